// What the kernels of the selective state-space scan share.
//
//   Delta = softplus(delta + bias),  h = exp(Delta A) h + (Delta u) B,  y = (C . h + D u) silu(z)
//
// for each channel with S states of its own; B and C are common to a group's channels.  Per state and step that is one
// exponential and four fp32 operations: with 16 exponentials and 128 fp32 operations a cycle and multiprocessor, the exponentials
// bind (the streams are 8 bytes a channel and step in bf16, read and written in less time than 16 states' exponentials take).  So a thread holds some
// states of one channel in registers and walks the time axis; LN neighbouring lanes share a channel.  What belongs to a channel and
// step (softplus, the gate) is formed once per tile of 16 steps x 32 channels, by the thread that loads it.
#pragma once
#include "common.cuh"
#include "scan.h"

namespace srwm {
namespace scan {

template <int S_>
struct Shape {
  static constexpr int S = S_;
  static constexpr int LN = S == 64 ? 8 : 4;    // lanes of a channel
  static constexpr int ST = S / LN;             // states of a thread (2, 4 or 8)
  static constexpr int LC = 32 / LN;            // channels of a warp
  static constexpr int NT = SCAN_CH * LN;       // threads
  static constexpr int QUADS = 2 * SCAN_TILE * S / 4;
  static constexpr int NQ = (QUADS + NT - 1) / NT;   // pieces of four of B and C that a thread loads
  // state j of lane q: whole pieces of four lie side by side over the lanes, so that a warp reads B and C without conflicts
  static __device__ __forceinline__ int first(int q, int piece) { return ST >= 4 ? piece * 4 * LN + q * 4 : q * ST; }
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

__device__ __forceinline__ float sigmoid(float x) { return rcp(1.f + ex2(-LOG2E * x)); }
// max(x, 0) + log(1 + e), e = exp(-|x|) <= 1, as 2 atanh(e / (2 + e)): its series in s^2 <= 1/9 keeps the relative error of small
// results (step sizes of 1e-3) near fp32's own, which a logarithm of 1 + e would not
__device__ __forceinline__ float softplus(float x) {
  const float e = ex2(-LOG2E * fabsf(x)), s = e * rcp(2.f + e), q = s * s;
  float p = fmaf(q, 1.f / 13.f, 1.f / 11.f);
  p = fmaf(q, p, 1.f / 9.f);
  p = fmaf(q, p, 1.f / 7.f);
  p = fmaf(q, p, 1.f / 5.f);
  p = fmaf(q, p, 1.f / 3.f);
  p = fmaf(q, p, 1.f);
  const float r = 2.f * s * p;
  return x > 0.f ? x + r : (x == x ? r : x);
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

template <typename T>
struct Quad {
  typename Raw<T>::type raw;
  // a row's piece ahead of time where it may be loaded whole; otherwise get() loads its elements
  __device__ __forceinline__ void fetch(const T* p, int vec, int valid) {
    if (vec && valid > 0) raw = *reinterpret_cast<const typename Raw<T>::type*>(p);
  }
  __device__ __forceinline__ float4 get(const T* p, int vec, int valid) const {
    if (valid <= 0) return make_float4(0.f, 0.f, 0.f, 0.f);
    if (vec) return widen(raw);
    float4 r = make_float4(to_float(p[0]), 0.f, 0.f, 0.f);
    if (valid > 1) r.y = to_float(p[1]);
    if (valid > 2) r.z = to_float(p[2]);
    if (valid > 3) r.w = to_float(p[3]);
    return r;
  }
};
__device__ __forceinline__ void put4(float* p, int vec, int valid, float4 v) {
  if (vec) { *reinterpret_cast<float4*>(p) = v; return; }
  p[0] = v.x;
  if (valid > 1) p[1] = v.y;
  if (valid > 2) p[2] = v.z;
  if (valid > 3) p[3] = v.w;
}
__device__ __forceinline__ void put4(__nv_bfloat16* p, int vec, int valid, float4 v) {
  if (vec) {
    *reinterpret_cast<uint2*>(p) = make_uint2(f32x2_to_bf16x2(v.x, v.y), f32x2_to_bf16x2(v.z, v.w));
    return;
  }
  p[0] = __float2bfloat16_rn(v.x);
  if (valid > 1) p[1] = __float2bfloat16_rn(v.y);
  if (valid > 2) p[2] = __float2bfloat16_rn(v.z);
  if (valid > 3) p[3] = __float2bfloat16_rn(v.w);
}

// Sums over a channel's LN lanes of LN steps' values: lane q gets step q's
template <int LN>
__device__ __forceinline__ float steps_to_lanes(float (&v)[LN], int q) {
#pragma unroll
  for (int w = 1; w < LN; w *= 2) {
    const bool up = q & w;
#pragma unroll
    for (int i = 0; i < LN; i += 2 * w) {
      const float keep = up ? v[i + w] : v[i], send = up ? v[i] : v[i + w];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, send, w);
    }
  }
  return v[0];
}

// A thread's states as pairs, from or to [S] floats of its channel
template <typename Sh>
__device__ __forceinline__ void load_states(const float* p, int q, u64 (&v)[Sh::ST / 2]) {
  if constexpr (Sh::ST >= 4) {
#pragma unroll
    for (int i = 0; i < Sh::ST / 4; ++i) {
      const ulonglong2 t = *reinterpret_cast<const ulonglong2*>(p + Sh::first(q, i));
      v[2 * i] = t.x; v[2 * i + 1] = t.y;
    }
  } else {
    v[0] = *reinterpret_cast<const u64*>(p + Sh::first(q, 0));
  }
}
template <typename Sh>
__device__ __forceinline__ void store_states(float* p, int q, const u64 (&v)[Sh::ST / 2]) {
  if constexpr (Sh::ST >= 4) {
#pragma unroll
    for (int i = 0; i < Sh::ST / 4; ++i)
      *reinterpret_cast<ulonglong2*>(p + Sh::first(q, i)) = make_ulonglong2(v[2 * i], v[2 * i + 1]);
  } else {
    *reinterpret_cast<u64*>(p + Sh::first(q, 0)) = v[0];
  }
}

// exp of a pair, with the factor log2(e) in x already
__device__ __forceinline__ u64 exp2_pair(u64 x) {
  float a, b;
  unpack2(x, a, b);
  return pack2(ex2(a), ex2(b));
}

// Where a CTA works: sequence, group, first channel in the group
struct Place {
  int n, g, ch0, left;      // left: channels of the group from ch0 on
  __device__ __forceinline__ Place(const ScanParams& p, int index) {
    const int Dg = p.D / p.G, per = (Dg + SCAN_CH - 1) / SCAN_CH, blocks = per * p.G;
    n = index / blocks;
    const int b = index - n * blocks;
    g = b / per;
    ch0 = (b - g * per) * SCAN_CH;
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

template <int S>
inline int blocks_of(const ScanParams& p) {
  const int Dg = p.D / p.G;
  return (Dg + SCAN_CH - 1) / SCAN_CH * p.G;
}

}  // namespace scan
}  // namespace srwm
