// What the kernels of the selective state-space scan share.
//
//   Delta = softplus(delta + bias),  h = exp(Delta A) h + (Delta u) B,  y = (C . h + D u) silu(z)
//
// for each channel with S states of its own; B and C are common to a group's channels.  Per state and step that is one
// exponential and four fp32 operations: with 16 exponentials and 128 fp32 operations a cycle and multiprocessor, the exponentials
// bind (the streams are 8 bytes a channel and step in bf16, read and written in less time than 16 states' exponentials take).  So a thread holds some
// states of one or two channels in registers and walks the time axis; LN neighbouring lanes share a channel.  What belongs to a channel and
// step (softplus, the gate) is formed once, by the thread that loads it into a tile of 16 (8) steps x 32, 64 or 128 channels.
#pragma once
#include <type_traits>

#include "common.cuh"
#include "scan.h"

namespace srwm {
namespace scan {

// C: neighbouring channels of a thread.  A step's B and C are then read once for C channels: with one, the shared-memory pipe (a 16-byte load
// is four of its cycles) is busier than the exponentials' one.
template <int S_, int C_, int TT_>
struct Shape {
  static constexpr int S = S_, C = C_, TT = TT_;              // TT: steps of a tile
  static constexpr int LN = S == 8 ? 2 : S == 64 ? 8 : 4;    // lanes of a channel
  static constexpr int ST = S / LN;                           // states of a thread and channel (4 or 8)
  static constexpr int NP = ST / 2;                           // pairs of them
  static constexpr int LC = 32 / LN;                          // channel groups of a warp
  static constexpr int WARPS = LN < 4 ? 4 : LN, WALK = 32 * WARPS;      // warps and threads that walk the time axis
  static constexpr int LOAD = 128, NT = WALK + LOAD;          // threads that load, prepare and write tiles beside them; all
  static constexpr int CH = WARPS * LC * C;                   // channels of a CTA
  static constexpr int PIECES = TT * CH / 4, NL = (PIECES + LOAD - 1) / LOAD;               // pieces of four channels of a tile; of a loading thread
  static constexpr int QUADS = TT * S / 4, NQ = (QUADS + LOAD - 1) / LOAD;     // pieces of four of B (and of C)
  // What a channel's lanes add up to goes through shared memory, a row a lane (one store a step; shuffles and selects are five times
  // the instructions), at a distance that keeps the rows' banks apart
  static constexpr int PAD = CH + (LN == 2 ? 16 : LN == 4 ? 8 : 4);
  // state j of lane q: whole pieces of four lie side by side over the lanes, so that a warp reads B and C without conflicts
  static __device__ __forceinline__ int first(int q, int piece) { return piece * 4 * LN + q * 4; }
};

__device__ __forceinline__ u64 mul2(u64 a, u64 b) {
  u64 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ u64 add2(u64 a, u64 b) {
  u64 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float sigmoid(float x) { return rcp(1.f + ex2(-LOG2E * x)); }
// max(x, 0) + log(1 + e), e = exp(-|x|): log(1 + e) / e as a polynomial (fitted for the least largest relative error on [0, 1]:
// 3e-8), so that small results (step sizes of 1e-3) keep fp32's relative precision, and without a reciprocal: the special-function pipe has enough
// to do.  Two at a time.
__device__ __forceinline__ u64 softplus2(u64 x) {
  float a, b;
  unpack2(x, a, b);
  const u64 e = pack2(ex2(-LOG2E * fabsf(a)), ex2(-LOG2E * fabsf(b)));
  u64 p = dup2(0.0052326880395412445f);
  p = fma2<true>(p, e, dup2(-0.029505213722586632f));
  p = fma2<true>(p, e, dup2(0.07822591066360474f));
  p = fma2<true>(p, e, dup2(-0.13663242757320404f));
  p = fma2<true>(p, e, dup2(0.19106005132198334f));
  p = fma2<true>(p, e, dup2(-0.2484298199415207f));
  p = fma2<true>(p, e, dup2(0.3331909775733948f));
  p = fma2<true>(p, e, dup2(-0.4999949336051941f));
  p = fma2<true>(p, e, dup2(0.9999999403953552f));
  // (fmaxf drops a NaN, which is in the other term)
  return fma2<true>(p, e, pack2(fmaxf(a, 0.f), fmaxf(b, 0.f)));
}
__device__ __forceinline__ float softplus(float x) {
  float r, other;
  unpack2(softplus2(pack2(x, x)), r, other);
  return r;
}

// Four neighbouring elements of a row, kept as they are loaded (a conversion would wait for the load)
template <typename T>
struct Raw;
template <>
struct Raw<float> { typedef float4 type; };
template <>
struct Raw<__nv_bfloat16> { typedef uint2 type; };
__device__ __forceinline__ float4 widen(float4 v) { return v; }
__device__ __forceinline__ float4 widen(uint2 v) {
  float4 r;
  bf16x2_to_f32(v.x, r.x, r.y);
  bf16x2_to_f32(v.y, r.z, r.w);
  return r;
}
__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void narrow(float v, float* p) { *p = v; }
__device__ __forceinline__ void narrow(float v, __nv_bfloat16* p) { *p = __float2bfloat16_rn(v); }

// VEC: every piece of four may be loaded and stored whole (otherwise by elements); a piece has four elements then, or none.
// Loads are predicated, not behind branches, so that many are on their way at a time.
template <typename T, bool VEC>
struct Quad {
  typename Raw<T>::type raw;
  __device__ __forceinline__ void fetch(const T* p, int valid) {
    raw = typename Raw<T>::type();
    if (valid > 0) raw = *reinterpret_cast<const typename Raw<T>::type*>(p);
  }
  __device__ __forceinline__ float4 get() const { return widen(raw); }
};
template <typename T>
struct Quad<T, false> {
  T e[4];
  __device__ __forceinline__ void fetch(const T* p, int valid) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      e[i] = T(0.f);
      if (valid > i) e[i] = p[i];
    }
  }
  __device__ __forceinline__ float4 get() const { return make_float4(to_float(e[0]), to_float(e[1]), to_float(e[2]), to_float(e[3])); }
};
template <bool VEC>
__device__ __forceinline__ void put4(float* p, int valid, float4 v) {
  if constexpr (VEC) {
    if (valid > 0) *reinterpret_cast<float4*>(p) = v;
  } else {
    const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (valid > i) p[i] = e[i];
  }
}
template <bool VEC>
__device__ __forceinline__ void put4(__nv_bfloat16* p, int valid, float4 v) {
  if constexpr (VEC) {
    if (valid > 0) *reinterpret_cast<uint2*>(p) = make_uint2(f32x2_to_bf16x2(v.x, v.y), f32x2_to_bf16x2(v.z, v.w));
  } else {
    const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (valid > i) p[i] = __float2bfloat16_rn(e[i]);
  }
}

// Four values as two pairs
struct Pairs {
  u64 lo, hi;
  __device__ __forceinline__ Pairs() : lo(0ull), hi(0ull) {}
  __device__ __forceinline__ Pairs(u64 a, u64 b) : lo(a), hi(b) {}
  __device__ __forceinline__ explicit Pairs(float4 v) : lo(pack2(v.x, v.y)), hi(pack2(v.z, v.w)) {}
  __device__ __forceinline__ explicit Pairs(const float* p) {
    const ulonglong2 t = *reinterpret_cast<const ulonglong2*>(p);
    lo = t.x;
    hi = t.y;
  }
  __device__ __forceinline__ float4 f4() const {
    float4 v;
    unpack2(lo, v.x, v.y);
    unpack2(hi, v.z, v.w);
    return v;
  }
};
__device__ __forceinline__ Pairs operator+(Pairs a, Pairs b) { return Pairs(add2(a.lo, b.lo), add2(a.hi, b.hi)); }
__device__ __forceinline__ Pairs operator*(Pairs a, Pairs b) { return Pairs(mul2(a.lo, b.lo), mul2(a.hi, b.hi)); }
__device__ __forceinline__ Pairs fma4(Pairs a, Pairs b, Pairs c) { return Pairs(fma2<true>(a.lo, b.lo, c.lo), fma2<true>(a.hi, b.hi, c.hi)); }
__device__ __forceinline__ Pairs softplus4(Pairs x) { return Pairs(softplus2(x.lo), softplus2(x.hi)); }
__device__ __forceinline__ Pairs sigmoid4(Pairs x) {
  const float4 v = x.f4();
  return Pairs(make_float4(sigmoid(v.x), sigmoid(v.y), sigmoid(v.z), sigmoid(v.w)));
}
// The same step's values of the LN lanes' rows, added up
template <typename Sh>
__device__ __forceinline__ Pairs sum_lanes(const float* p) {
  Pairs v(p);
#pragma unroll
  for (int q = 1; q < Sh::LN; ++q) v = v + Pairs(p + q * Sh::PAD);
  return v;
}
// Delta and Delta u of four channels side by side
__device__ __forceinline__ void store_staged(float2* p, Pairs a, Pairs b) {
  const float4 x = a.f4(), y = b.f4();
  reinterpret_cast<float4*>(p)[0] = make_float4(x.x, y.x, x.y, y.y);
  reinterpret_cast<float4*>(p)[1] = make_float4(x.z, y.z, x.w, y.w);
}
// Four of a vector over the channels
__device__ __forceinline__ Pairs four(const float* p, int valid) {
  float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
  if (p == nullptr) return Pairs(r);
  if (valid > 0) r.x = p[0];
  if (valid > 1) r.y = p[1];
  if (valid > 2) r.z = p[2];
  if (valid > 3) r.w = p[3];
  return Pairs(r);
}
template <int C>
__device__ __forceinline__ void store_channels(float* p, const float* v) {
  if constexpr (C == 2) *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]);
  else *p = v[0];
}

// A thread's states of a channel as pairs, from or to that channel's [S] floats
template <typename Sh>
__device__ __forceinline__ void load_states(const float* p, int q, u64* v) {
#pragma unroll
  for (int i = 0; i < Sh::ST / 4; ++i) {
    const ulonglong2 t = *reinterpret_cast<const ulonglong2*>(p + Sh::first(q, i));
    v[2 * i] = t.x; v[2 * i + 1] = t.y;
  }
}
template <typename Sh>
__device__ __forceinline__ void store_states(float* p, int q, const u64* v) {
#pragma unroll
  for (int i = 0; i < Sh::ST / 4; ++i)
    *reinterpret_cast<ulonglong2*>(p + Sh::first(q, i)) = make_ulonglong2(v[2 * i], v[2 * i + 1]);
}
// C neighbouring values of a staged row
template <int C>
__device__ __forceinline__ void load_channels(const float2* p, float2* v) {
  if constexpr (C == 2) {
    const float4 t = *reinterpret_cast<const float4*>(p);
    v[0] = make_float2(t.x, t.y);
    v[1] = make_float2(t.z, t.w);
  } else {
    v[0] = *p;
  }
}

// exp(Delta A) of a pair, with the factor log2(e) in A (or Delta) already.  ex2.approx is low on the average: by 1.8e-8 to 3.5e-8 of the
// value for arguments between -1 and -2^-8, 0.6e-8 nearer to zero.  A state's memory adds that up over its steps, so the product that
// makes the argument lifts it, at no cost (the same instruction with an addend): from -1/2 on the mean is within 1.1e-8 (in front, where
// a memory is two steps, the addend is less than half a step of the argument), and the
// errors of training passes against 64 bits fall to about half (58 outputs of lengths up to 1000: their sum 1.04 of a plain fp32
// form's before, 0.54 since; with 2^-25 0.52, but 1.5e-8 high for the longest memories; with 2^-26 0.66).
constexpr float EX2_LIFT = 1.5f / (1 << 26);
__device__ __forceinline__ u64 decay2(u64 delta, u64 A) {
  float a, b;
  unpack2(fma2<true>(delta, A, dup2(EX2_LIFT)), a, b);
  return pack2(ex2(a), ex2(b));
}

// The state (or its gradient) on the far side of a piece of the time axis, from the one on this side, what the piece adds and the square root of
// the product of its decays: steps as given may be negative, and a piece's growth (or decay) be beyond a float where what it makes of a small
// state is not.  A state of zero stays zero through any growth.  Where an episode begins inside the piece nothing goes through, not even a NaN
// or an infinity: such a piece leaves CUT, a zero that no exponential gives, and is told by it (a product of decays may well be +0).
constexpr u64 CUT = 0x8000000080000000ull;      // a pair of -0
__device__ __forceinline__ u64 piece_root(float sum_d, u64 A) { return decay2(dup2(0.5f * sum_d), A); }
template <int NP>
__device__ __forceinline__ void through_piece(u64 (&h)[NP], const u64 (&root)[NP], const u64 (&end)[NP]) {
  const bool cut = root[0] == CUT;
#pragma unroll
  for (int k = 0; k < NP; ++k) {
    float h0, h1, n0, n1, e0, e1;
    unpack2(h[k], h0, h1);
    unpack2(fma2<true>(root[k], mul2(root[k], h[k]), end[k]), n0, n1);
    unpack2(end[k], e0, e1);
    h[k] = pack2(cut || h0 == 0.f ? e0 : n0, cut || h1 == 0.f ? e1 : n1);
  }
}

// Where a CTA works: sequence, group, first channel, channels of the group from there on
template <int CH>
struct Place {
  int n, g, ch0, left, blk;
  __device__ __forceinline__ Place(const ScanParams& p, int index) {
    const int Dg = p.D / p.G, per = (Dg + CH - 1) / CH, blocks = per * p.G;
    n = index / blocks;
    const int b = index - n * blocks;
    g = b / per;
    blk = b - g * per;
    ch0 = blk * CH;
    left = Dg - ch0;
    ch0 += g * Dg;
  }
};

// Steps of the tile at t0 that begin an episode, as bits (the same for all threads)
__device__ __forceinline__ unsigned reset_bits(const ScanParams& p, int n, int t0, int steps) {
  if (p.done == nullptr) return 0u;
  const int lane = threadIdx.x % 32;
  const bool r = lane < steps && p.done[n * p.done_n + (long long)(t0 + lane) * p.done_l] != 0;
  return __ballot_sync(0xffffffffu, r);
}

inline long long blocks_of(const ScanParams& p, int channels) {
  const int Dg = p.D / p.G;
  return (long long)((Dg + channels - 1) / channels) * p.G * p.N;
}

// Raises a kernel's limit of dynamic shared memory, once a device
template <typename Kernel>
inline cudaError_t allow_smem(Kernel kern, int bytes, unsigned long long* raised) {
  if (bytes <= 48 * 1024) return cudaSuccess;
  int dev = 0;
  if (const cudaError_t e = cudaGetDevice(&dev); e != cudaSuccess) return e;
  const unsigned long long bit = 1ull << (dev & 63);
  if (__atomic_load_n(raised, __ATOMIC_ACQUIRE) & bit) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) __atomic_fetch_or(raised, bit, __ATOMIC_RELEASE);
  return e;
}

// f(element, states, vec) as types
template <typename T, bool VEC, typename F>
inline cudaError_t by_states(const ScanParams& p, F& f) {
  const std::bool_constant<VEC> vec;
  switch (p.S) {
    case 8: return f(T(), std::integral_constant<int, 8>(), vec);
    case 16: return f(T(), std::integral_constant<int, 16>(), vec);
    case 32: return f(T(), std::integral_constant<int, 32>(), vec);
    default: return f(T(), std::integral_constant<int, 64>(), vec);
  }
}
template <typename F>
inline cudaError_t by_shape(const ScanParams& p, F f) {
  if (p.bf16) return p.vec ? by_states<__nv_bfloat16, true>(p, f) : by_states<__nv_bfloat16, false>(p, f);
  return p.vec ? by_states<float, true>(p, f) : by_states<float, false>(p, f);
}

}  // namespace scan
}  // namespace srwm
