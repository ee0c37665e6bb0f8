// Selective state-space scan, backward.
//
// With g_t = dL/dh_t = C_t dy'_t + a_{t+1} g_{t+1} (dy' = dy silu(z), a = exp(Delta A)):
//   dC_t = sum_d dy'_t h_t        dB_t = sum_d g_t Delta_t u_t        dA = sum_t Delta_t g_t a_t h_{t-1}
//   du_t = D dy'_t + Delta_t (g_t . B_t)        dDelta_t = u_t (g_t . B_t) + sum_s A a_t h_{t-1} g_t
// A CTA takes its 64 (32) channels from the last step to the first.  The states in front of each eighth step are the forward's; within
// eight steps they are formed again, four at a time, a_t and a_t h_{t-1} staying in registers until the way back has used them.  Thirteen fp32
// operations per state and step bind.  Sums over states go through a channel's lanes, sums over channels (dB, dC) through the
// warp's other lanes and shared memory, and are added up over the CTAs by a second launch, in a fixed order.
#include <type_traits>

#include "device.h"
#include "scan.cuh"

namespace srwm {
namespace {
using namespace scan;

// The states of a thread are held in an order of its own: state j of piece i in register (i ^ pp, j ^ (2 x1 + x0)), where pp, x1, x0 are bits of its
// channel group.  The sums over the warp's groups then halve at each exchange without a select: a lane keeps its first
// half and sends the second, which is what the other lane keeps.
template <int ST, int LN>
struct Order {
  int pp, x1, x0;
  __device__ __forceinline__ explicit Order(int lane) {
    const int c = lane / LN;
    pp = ST == 8 ? c & 1 : 0;
    x1 = ST == 8 ? c >> 1 & 1 : c & 1;
    x0 = ST == 8 ? (LN == 8 ? 0 : c >> 2 & 1) : c >> 1 & 1;
  }
  __device__ __forceinline__ int copy() const { return x1 + 2 * x0; }      // of four in shared memory (side by side: no conflicts)
  __device__ __forceinline__ int state() const { return 2 * x1 + x0; }      // in register 0
  // into the order and out of it, a piece as two pairs
  __device__ __forceinline__ void turn(u64& lo, u64& hi) const {
    float a, b, c, d;
    unpack2(lo, a, b);
    unpack2(hi, c, d);
    const float a1 = x1 ? c : a, b1 = x1 ? d : b, c1 = x1 ? a : c, d1 = x1 ? b : d;
    lo = pack2(x0 ? b1 : a1, x0 ? a1 : b1);
    hi = pack2(x0 ? d1 : c1, x0 ? c1 : d1);
  }
};
template <typename Sh, typename O>
__device__ __forceinline__ void load_turned(const float* p, int q, const O& o, u64* v) {
#pragma unroll
  for (int i = 0; i < Sh::ST / 4; ++i) {
    const ulonglong2 t = *reinterpret_cast<const ulonglong2*>(p + Sh::first(q, i ^ o.pp));
    v[2 * i] = t.x; v[2 * i + 1] = t.y;
    o.turn(v[2 * i], v[2 * i + 1]);
  }
}
template <typename Sh, typename O>
__device__ __forceinline__ void store_turned(float* p, int q, const O& o, const u64* v) {
#pragma unroll
  for (int i = 0; i < Sh::ST / 4; ++i) {
    u64 lo = v[2 * i], hi = v[2 * i + 1];
    o.turn(lo, hi);
    *reinterpret_cast<ulonglong2*>(p + Sh::first(q, i ^ o.pp)) = make_ulonglong2(lo, hi);
  }
}
// Sums of eight values (8 / ST steps of a thread's states) over the warp's channel groups: v[0] (and v[1], with four groups) is what
// the lane keeps
template <int ST, int LN>
__device__ __forceinline__ void sum_groups(float* v, int lane) {
  auto other = [](float x, int w) { return __shfl_xor_sync(0xffffffffu, x, w); };
  if (ST == 8) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] += other(v[j + 4], LN);
#pragma unroll
    for (int j = 0; j < 2; ++j) v[j] += other(v[j + 2], 2 * LN);
    if (LN == 4) v[0] += other(v[1], 4 * LN);
  } else {
#pragma unroll
    for (int s = 0; s < 8; s += 4) {
      v[s] += other(v[s + 2], LN);
      v[s + 1] += other(v[s + 3], LN);
      v[s] += other(v[s + 1], 2 * LN);
    }
    const bool up = lane & (4 * LN);       // the second of the two steps
    const float keep = up ? v[4] : v[0], send = up ? v[0] : v[4];
    v[0] = keep + other(send, 4 * LN);
    if (LN == 2) v[0] += other(v[0], 16);
  }
}

// Two channels a thread with up to 16 states, one with more: eight states of a thread in all
template <int S>
using BwdShape = Shape<S, S <= 16 ? 2 : 1, SCAN_CKPT>;
template <int S>
using BwdCarryShape = Shape<S, S <= 16 ? 2 : 1, SCAN_TILE>;

// Two buffers: a tile is loaded and prepared, and the results of the one before it written, while the tile between is walked
template <int S>
struct BwdSmem {
  using Sh = BwdShape<S>;
  static constexpr int TT = Sh::TT, CH = Sh::CH, PAD = Sh::PAD;
  struct Tile {
    float2 dd[TT][CH];           // Delta, Delta u
    float gy[TT][CH];            // dy'
    float bc[2][TT][4][S];       // B and C, in the four orders of a piece's states
    float gb[TT][Sh::LN][PAD], sa[TT][Sh::LN][PAD], yp[TT][Sh::LN][PAD];      // g . B, A . (g a h), C . h: a row of each lane of a channel
    float part[Sh::WARPS][TT][2][S];
  } tile[2];
  float4 sums[2][Sh::PIECES];    // of dy' u and of the gradient of delta, a slot for each loading thread's piece
};

// Registers: the walking threads' share and the loading threads', which together are at most what the CTA is launched with (128 a thread, two
// CTAs a multiprocessor; S 64: 168 and one): a share beyond that would be waited for without end.
template <int S>
struct BwdRegs {
  using Sh = BwdShape<S>;
  static constexpr int CTAS = S == 64 ? 1 : 2, LOADERS = 104, WALKERS = S == 64 ? 200 : 152;
  static constexpr int ALL = Sh::WALK * WALKERS + Sh::LOAD * LOADERS;
  static_assert(ALL <= 65536 / CTAS / Sh::NT / 8 * 8 * Sh::NT, "more registers than the CTA is launched with");
};
template <int N>
__device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

template <typename T, int S, bool VEC>
__device__ __forceinline__ void scan_bwd_load(const ScanParams& p, BwdSmem<S>& sm) {
  using Sh = BwdShape<S>;
  constexpr int TT = Sh::TT, CH = Sh::CH, NL = Sh::NL, NQ = Sh::NQ;
  const int tid = threadIdx.x - Sh::WALK;
  const Place<CH> at(p, blockIdx.x);
  const int seg = blockIdx.y, t_first = seg * p.seglen, t_end = min(p.L, t_first + p.seglen);
  const int t_last = t_first + (t_end - t_first - 1) / TT * TT;
  const bool gate = p.z.p != nullptr;
  // piece k: row (tid + k LOAD) / (CH / 4), columns from (tid % (CH / 4)) * 4 on
  static_assert(Sh::LOAD % (CH / 4) == 0, "all pieces of a thread have the same columns");
  constexpr int RS = Sh::LOAD / (CH / 4);       // rows between a thread's pieces
  const bool loads = tid < Sh::PIECES;          // (32 channels: half of the threads have a piece)
  const int row = tid / (CH / 4), col = tid % (CH / 4) * 4, valid = loads ? max(0, min(4, at.left - col)) : 0;
  if (loads) {
#pragma unroll
    for (int k = 0; k < NL; ++k) sm.sums[0][tid + k * Sh::LOAD] = sm.sums[1][tid + k * Sh::LOAD] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  auto place = [&](const ScanRows& w, int t) { return reinterpret_cast<T*>(w.p) + at.n * w.sn + t * w.sl + at.ch0 + col; };
  float bias[4], skip[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    bias[i] = i < valid && p.bias ? p.bias[at.ch0 + col + i] : 0.f;
    skip[i] = i < valid && p.skip ? p.skip[at.ch0 + col + i] : 0.f;
  }
  Quad<T, VEC> fu[NL], fd[NL], fz[NL], fy[NL], fb[NQ], fc[NQ];
  auto fetch_rows = [&](int t0) {
#pragma unroll
    for (int k = 0; k < NL; ++k) {
      const int t = t0 + row + k * RS, v = t < t_end ? valid : 0;
      fu[k].fetch(place(p.u, t), v);
      fd[k].fetch(place(p.delta, t), v);
      fy[k].fetch(place(p.dy, t), v);
      if (gate) fz[k].fetch(place(p.z, t), v);
    }
  };
  auto fetch_bc = [&](int t0) {
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      const int id = tid + i * Sh::LOAD, c = id % (S / 4) * 4, t = t0 + id / (S / 4), v = id < Sh::QUADS && t < t_end ? 4 : 0;
      fb[i].fetch(reinterpret_cast<const T*>(p.B.p) + at.n * p.B.sn + at.g * p.B.sg + t * p.B.sl + c, v);
      fc[i].fetch(reinterpret_cast<const T*>(p.C.p) + at.n * p.C.sn + at.g * p.C.sg + t * p.C.sl + c, v);
    }
  };
  auto stage = [&](int buf) {
    auto& tl = sm.tile[buf];
#pragma unroll
    for (int k = 0; k < NL; ++k) {
      if (!loads) break;
      const float4 u4 = fu[k].get(), r4 = fd[k].get();
      u64 lo = add2(pack2(r4.x, r4.y), pack2(bias[0], bias[1])), hi = add2(pack2(r4.z, r4.w), pack2(bias[2], bias[3]));
      if (p.softplus) {
        lo = softplus2(lo);
        hi = softplus2(hi);
      }
      const u64 xlo = mul2(lo, pack2(u4.x, u4.y)), xhi = mul2(hi, pack2(u4.z, u4.w));
      float dl[4], du[4];
      float4 g = fy[k].get();
      unpack2(lo, dl[0], dl[1]); unpack2(hi, dl[2], dl[3]);
      unpack2(xlo, du[0], du[1]); unpack2(xhi, du[2], du[3]);
      if (gate) {
        const float4 z4 = fz[k].get();
        g.x *= z4.x * sigmoid(z4.x); g.y *= z4.y * sigmoid(z4.y); g.z *= z4.z * sigmoid(z4.z); g.w *= z4.w * sigmoid(z4.w);
      }
      float4* o = reinterpret_cast<float4*>(&tl.dd[row + k * RS][col]);
      o[0] = make_float4(dl[0], du[0], dl[1], du[1]);
      o[1] = make_float4(dl[2], du[2], dl[3], du[3]);
      *reinterpret_cast<float4*>(&tl.gy[row + k * RS][col]) = g;
    }
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      const int id = tid + i * Sh::LOAD, c = id % (S / 4) * 4, r = id / (S / 4);
      if (id >= Sh::QUADS) continue;
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const float4 v = w ? fc[i].get() : fb[i].get();
        float* o = &tl.bc[w][r][0][c];
        *reinterpret_cast<float4*>(o) = v;
        *reinterpret_cast<float4*>(o + S) = make_float4(v.z, v.w, v.x, v.y);
        *reinterpret_cast<float4*>(o + 2 * S) = make_float4(v.y, v.x, v.w, v.z);
        *reinterpret_cast<float4*>(o + 3 * S) = make_float4(v.w, v.z, v.y, v.x);
      }
    }
  };
  auto finish = [&](int t0, int buf) {
    const auto& tl = sm.tile[buf];
    const int steps = min(TT, t_end - t0);
    // this CTA's share of dB and dC
#pragma unroll 1
    for (int e = tid; e < steps * 2 * S / 4; e += Sh::LOAD) {
      const int s = e % (S / 4) * 4, arr = e / (S / 4) % 2, t = e / (S / 2);
      float4 v = *reinterpret_cast<const float4*>(&tl.part[0][t][arr][s]);
#pragma unroll
      for (int w = 1; w < Sh::WARPS; ++w) {
        const float4 o = *reinterpret_cast<const float4*>(&tl.part[w][t][arr][s]);
        v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w;
      }
      *reinterpret_cast<float4*>(p.part_bc + ((((long long)at.blk * 2 + arr) * p.N + at.n) * p.L + t0 + t) * p.G * S + at.g * S + s) = v;
    }
    // (the tile's rows again: they have left the registers)
#pragma unroll 1
    for (int k = 0; k < NL; ++k) {
      const int r = row + k * RS, t = t0 + r, v = r < steps ? valid : 0;
      if (v <= 0) break;
      Quad<T, VEC> q0, q1, q2, q3;
      q0.fetch(place(p.u, t), v);
      q1.fetch(place(p.delta, t), v);
      if (gate) {
        q2.fetch(place(p.z, t), v);
        q3.fetch(place(p.dy, t), v);
      }
      const float4 gb4 = sum_lanes<Sh>(&tl.gb[r][0][col]), sa4 = sum_lanes<Sh>(&tl.sa[r][0][col]);
      const float4 g4 = *reinterpret_cast<const float4*>(&tl.gy[r][col]);
      const float4* dk = reinterpret_cast<const float4*>(&tl.dd[r][col]);
      const float4 d01 = dk[0], d23 = dk[1], u4 = q0.get(), r4 = q1.get();
      const float dl[4] = {d01.x, d01.z, d23.x, d23.z}, us[4] = {u4.x, u4.y, u4.z, u4.w}, g[4] = {g4.x, g4.y, g4.z, g4.w};
      const float rs[4] = {r4.x, r4.y, r4.z, r4.w}, gb[4] = {gb4.x, gb4.y, gb4.z, gb4.w}, sa[4] = {sa4.x, sa4.y, sa4.z, sa4.w};
      float o1[4], o2[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        o1[i] = fmaf(g[i], skip[i], dl[i] * gb[i]);
        o2[i] = fmaf(us[i], gb[i], sa[i] * 0.6931471805599453f);      // (the walking threads' A has log2(e) in it)
        if (p.softplus) o2[i] *= sigmoid(rs[i] + bias[i]);
      }
      put4<VEC>(place(p.du, t), v, make_float4(o1[0], o1[1], o1[2], o1[3]));
      put4<VEC>(place(p.ddelta, t), v, make_float4(o2[0], o2[1], o2[2], o2[3]));
      const int id = tid + k * Sh::LOAD;
      float4 w = sm.sums[0][id];
      sm.sums[0][id] = make_float4(fmaf(g[0], us[0], w.x), fmaf(g[1], us[1], w.y), fmaf(g[2], us[2], w.z), fmaf(g[3], us[3], w.w));
      w = sm.sums[1][id];
      sm.sums[1][id] = make_float4(w.x + o2[0], w.y + o2[1], w.z + o2[2], w.w + o2[3]);
      if (gate) {
        const float4 yp4 = sum_lanes<Sh>(&tl.yp[r][0][col]), z4 = q2.get(), y4 = q3.get();
        const float yp[4] = {yp4.x, yp4.y, yp4.z, yp4.w}, zs[4] = {z4.x, z4.y, z4.z, z4.w}, os[4] = {y4.x, y4.y, y4.z, y4.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float sg = sigmoid(zs[i]);
          o1[i] = os[i] * fmaf(skip[i], us[i], yp[i]) * sg * fmaf(zs[i], 1.f - sg, 1.f);
        }
        put4<VEC>(place(p.dz, t), v, make_float4(o1[0], o1[1], o1[2], o1[3]));
      }
    }
  };
  fetch_rows(t_last);
  fetch_bc(t_last);
  stage(0);
  if (t_last - TT >= t_first) {
    fetch_rows(t_last - TT);
    fetch_bc(t_last - TT);
  }
  __syncthreads();
  int k0 = 0;
  for (int t0 = t_last; t0 >= t_first; t0 -= TT, k0 ^= 1) {
    if (t0 < t_last) finish(t0 + TT, k0 ^ 1);
    if (t0 - TT >= t_first) {
      stage(k0 ^ 1);
      if (t0 - 2 * TT >= t_first) {
        fetch_rows(t0 - 2 * TT);
        fetch_bc(t0 - 2 * TT);
      }
    }
    __syncthreads();
  }
  finish(t_first, k0 ^ 1);
  asm volatile("bar.sync 1, %0;" ::"n"(Sh::LOAD) : "memory");      // the loading threads alone
  const long long slot = (long long)at.n * p.nseg + seg;
  for (int e = tid; e < 2 * CH; e += Sh::LOAD) {
    const int c = e % CH, which = e / CH;
    const float* f = reinterpret_cast<const float*>(&sm.sums[which][0]) + c;
    float v = 0.f;
#pragma unroll
    for (int r = 0; r < TT; ++r) v += f[r * CH];
    if (c < at.left) p.part_v[(slot * 2 + which) * p.D + at.ch0 + c] = v;
  }
}

template <typename T, int S, bool VEC>
__device__ __forceinline__ void scan_bwd_walk(const ScanParams& p, BwdSmem<S>& sm) {
  using Sh = BwdShape<S>;
  constexpr int TT = Sh::TT, CH = Sh::CH, C = Sh::C, NP = Sh::NP, ST = Sh::ST, LN = Sh::LN;
  constexpr int SUB = 4, GS = 8 / ST;
  static_assert(TT == SCAN_CKPT && TT == 2 * SUB, "a tile's steps are those between two of the forward's states");
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, q = lane % LN, chl = (warp * Sh::LC + lane / LN) * C;
  const Place<CH> at(p, blockIdx.x);
  const int seg = blockIdx.y, t_first = seg * p.seglen, t_end = min(p.L, t_first + p.seglen);
  const int t_last = t_first + (t_end - t_first - 1) / TT * TT;
  const int d = at.ch0 + chl, mine = at.left - chl;
  const bool gate = p.z.p != nullptr;
  const Order<ST, LN> order(lane);

  u64 A2[C][NP], gc[C][NP], dA[C][NP];
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int i = 0; i < NP; ++i) A2[c][i] = gc[c][i] = dA[c][i] = 0ull;
  const long long states = (long long)p.N * p.D * S, own = ((long long)at.n * p.D + d) * S;
  const int nck = (p.L + TT - 1) / TT;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    if (c >= mine) continue;
    load_turned<Sh>(p.A + (long long)(d + c) * S, q, order, A2[c]);
#pragma unroll
    for (int i = 0; i < NP; ++i) A2[c][i] = mul2(A2[c][i], dup2(LOG2E));
    const long long o = own + c * S;
    if (p.dhT) load_turned<Sh>(p.dhT + o, q, order, gc[c]);
#pragma unroll 4
    for (int i = p.nseg - 1; i > seg; --i) {      // the pieces behind, the last first
      u64 decay[NP], end[NP];
      load_turned<Sh>(p.carry + (2 * i - 2) * states + o, q, order, end);
      load_turned<Sh>(p.carry + (2 * i - 1) * states + o, q, order, decay);
#pragma unroll
      for (int k = 0; k < NP; ++k) gc[c][k] = fma2<true>(decay[k], gc[c][k], end[k]);
    }
  }
  // in part[][][][]: of v[0] of sum_groups (ST 4: of the step that the lane keeps)
  const int kept_at = (warp * TT + (ST == 4 ? lane / LN >> 2 & 1 : 0)) * 2 * S + Sh::first(q, order.pp) + order.state();
  const bool keeps = LN > 2 || lane < 16;      // (sixteen groups: two lanes have the same sum)
  const int bc_at = order.copy() * S;
  u64 ck[C][NP];      // the states in front of the next tile
  auto checkpoint = [&](int t) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
#pragma unroll
      for (int i = 0; i < NP; ++i) ck[c][i] = 0ull;
      if (c >= mine || t < t_first) continue;
#pragma unroll
      for (int i = 0; i < ST / 4; ++i) {
        const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(p.ckpt + (((long long)at.n * nck + t / TT) * p.D + d + c) * S + Sh::first(q, i ^ order.pp));
        ck[c][2 * i] = v.x;
        ck[c][2 * i + 1] = v.y;
      }
    }
  };
  checkpoint(t_last);
  unsigned resets = reset_bits(p, at.n, t_last, t_end - t_last);
  __syncthreads();

  for (int t0 = t_last, k0 = 0; t0 >= t_first; t0 -= TT, k0 ^= 1) {
    auto& tl = sm.tile[k0];
    const int steps = min(TT, t_end - t0);
    const unsigned now = resets;
    if (t0 - TT >= t_first) resets = reset_bits(p, at.n, t0 - TT, TT);
    float* part_mine = &tl.part[0][0][0][0] + kept_at;
    u64 start[C][NP];
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int i = 0; i < NP; i += 2) {
        start[c][i] = ck[c][i];
        start[c][i + 1] = ck[c][i + 1];
        order.turn(start[c][i], start[c][i + 1]);
      }
    checkpoint(t0 - TT);
    auto load_bc = [&](int w, int t, u64* v) {
#pragma unroll
      for (int i = 0; i < ST / 4; ++i) {
        const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(&tl.bc[w][t][0][0] + bc_at + Sh::first(q, i ^ order.pp));
        v[2 * i] = x.x;
        v[2 * i + 1] = x.y;
      }
    };

    // Four steps at a time, the last first.  The second four have the first four walked on the way to them (without what they leave), so that a
    // and a h of no more than four stay in registers.
    auto tile = [&](auto whole) __attribute__((always_inline)) {
      constexpr bool WHOLE = decltype(whole)::value;
#pragma unroll 1
      for (int s0 = SUB; s0 >= 0; s0 -= SUB) {
        if (!WHOLE && s0 >= steps) continue;
        u64 h[C][NP];
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int i = 0; i < NP; ++i) h[c][i] = start[c][i];
        if (s0 > 0) {
          u64 a[SUB][C][NP], in[SUB][C][NP];      // (first what does not wait for the state)
#pragma unroll
          for (int k = 0; k < SUB; ++k) {
            float2 x[C];
            load_channels<C>(&tl.dd[k][chl], x);
            u64 b2[NP];
            load_bc(0, k, b2);
#pragma unroll
            for (int c = 0; c < C; ++c) {
              const u64 d2 = dup2(x[c].x), x2 = dup2(x[c].y);
#pragma unroll
              for (int i = 0; i < NP; ++i) {
                a[k][c][i] = exp2_pair(mul2(d2, A2[c][i]));
                in[k][c][i] = mul2(x2, b2[i]);
              }
            }
          }
#pragma unroll
          for (int k = 0; k < SUB; ++k) {
            const bool fresh = !WHOLE && (now >> k & 1u);
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
              for (int i = 0; i < NP; ++i) h[c][i] = fresh ? in[k][c][i] : fma2<true>(a[k][c][i], h[c][i], in[k][c][i]);
          }
        }
        u64 a[SUB][C][NP], ah[SUB][C][NP];      // ah: what is inserted first, then a h
#pragma unroll
        for (int k = 0; k < SUB; ++k) {
          float2 x[C];
          load_channels<C>(&tl.dd[s0 + k][chl], x);
          u64 b2[NP];
          load_bc(0, s0 + k, b2);
#pragma unroll
          for (int c = 0; c < C; ++c) {
            const u64 d2 = dup2(x[c].x), x2 = dup2(x[c].y);
#pragma unroll
            for (int i = 0; i < NP; ++i) {
              a[k][c][i] = exp2_pair(mul2(d2, A2[c][i]));
              ah[k][c][i] = mul2(x2, b2[i]);
            }
          }
        }
        float v8[8];
#pragma unroll
        for (int k = 0; k < SUB; ++k) {
          const int t = s0 + k;
          float* vk = v8 + k % GS * ST;
          if (WHOLE || t < steps) {
            const bool fresh = !WHOLE && (now >> t & 1u);
            u64 c2[NP], sum[NP];
            float y[C];
            load_bc(1, t, c2);
#pragma unroll
            for (int c = 0; c < C; ++c) {
              const u64 g2 = dup2(tl.gy[t][chl + c]);
              u64 acc = 0ull;
#pragma unroll
              for (int i = 0; i < NP; ++i) {
                const u64 in = ah[k][c][i];
                if (fresh) a[k][c][i] = h[c][i] = 0ull;
                ah[k][c][i] = mul2(a[k][c][i], h[c][i]);
                h[c][i] = add2(ah[k][c][i], in);
                acc = i == 0 ? mul2(h[c][i], c2[i]) : fma2<true>(h[c][i], c2[i], acc);
                sum[i] = c == 0 ? mul2(h[c][i], g2) : fma2<true>(h[c][i], g2, sum[i]);
              }
              y[c] = hsum2(acc);
            }
            if (gate) store_channels<C>(&tl.yp[t][q][chl], y);
#pragma unroll
            for (int i = 0; i < NP; ++i) unpack2(sum[i], vk[2 * i], vk[2 * i + 1]);
          } else {
#pragma unroll
            for (int i = 0; i < ST; ++i) vk[i] = 0.f;
          }
          if (k % GS == GS - 1) {
            sum_groups<ST, LN>(v8, lane);
            float* o = part_mine + (t - (GS - 1)) * 2 * S + S;
            if (LN == 8) *reinterpret_cast<float2*>(o) = make_float2(v8[0], v8[1]);
            else if (keeps) *o = v8[0];
          }
        }
#pragma unroll
        for (int k = SUB - 1; k >= 0; --k) {
          const int t = s0 + k;
          float* vk = v8 + k % GS * ST;
          if (WHOLE || t < steps) {
            float2 x[C];
            load_channels<C>(&tl.dd[t][chl], x);
            u64 b2[NP], c2[NP], sum[NP];
            float gbv[C], sav[C];
            load_bc(0, t, b2);
            load_bc(1, t, c2);
            const bool fresh = !WHOLE && (now >> t & 1u);
#pragma unroll
            for (int c = 0; c < C; ++c) {
              const u64 d2 = dup2(x[c].x), x2 = dup2(x[c].y), g2 = dup2(tl.gy[t][chl + c]);
              u64 gb = 0ull, sa = 0ull;
#pragma unroll
              for (int i = 0; i < NP; ++i) {
                const u64 g = fma2<true>(c2[i], g2, gc[c][i]), gah = mul2(g, ah[k][c][i]);
                gb = i == 0 ? mul2(g, b2[i]) : fma2<true>(g, b2[i], gb);
                sa = i == 0 ? mul2(gah, A2[c][i]) : fma2<true>(gah, A2[c][i], sa);
                dA[c][i] = fma2<true>(gah, d2, dA[c][i]);
                sum[i] = c == 0 ? mul2(g, x2) : fma2<true>(g, x2, sum[i]);
                gc[c][i] = fresh ? 0ull : mul2(a[k][c][i], g);
              }
              gbv[c] = hsum2(gb);
              sav[c] = hsum2(sa);
            }
            store_channels<C>(&tl.gb[t][q][chl], gbv);
            store_channels<C>(&tl.sa[t][q][chl], sav);
#pragma unroll
            for (int i = 0; i < NP; ++i) unpack2(sum[i], vk[2 * i], vk[2 * i + 1]);
          } else {
#pragma unroll
            for (int i = 0; i < ST; ++i) vk[i] = 0.f;
          }
          if (k % GS == 0) {
            sum_groups<ST, LN>(v8, lane);
            float* o = part_mine + t * 2 * S;
            if (LN == 8) *reinterpret_cast<float2*>(o) = make_float2(v8[0], v8[1]);
            else if (keeps) *o = v8[0];
          }
        }
      }
    };
    if (steps == TT && now == 0u) tile(std::true_type());
    else tile(std::false_type());
    __syncthreads();
  }
  const long long slot = (long long)at.n * p.nseg + seg;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    if (c >= mine) continue;
    store_turned<Sh>(p.part_a + (slot * p.D + d + c) * S, q, order, dA[c]);
    if (seg == 0 && p.dh0) store_turned<Sh>(p.dh0 + own + c * S, q, order, gc[c]);
  }
}

template <typename T, int S, bool VEC>
__global__ void __launch_bounds__(BwdShape<S>::NT, BwdRegs<S>::CTAS) scan_bwd_kernel(const ScanParams p) {
  extern __shared__ __align__(16) unsigned char raw_smem[];
  BwdSmem<S>& sm = *reinterpret_cast<BwdSmem<S>*>(raw_smem);
  if (threadIdx.x >= BwdShape<S>::WALK) {
    fewer_registers<BwdRegs<S>::LOADERS>();
    scan_bwd_load<T, S, VEC>(p, sm);
  } else {
    more_registers<BwdRegs<S>::WALKERS>();
    scan_bwd_walk<T, S, VEC>(p, sm);
  }
}

// What a piece of the time axis adds to the gradient of the state in front of it (from zero behind it), and the product of its
// decays, for pieces 1 .. nseg - 1.
template <typename T, int S, bool VEC>
__global__ void __launch_bounds__(BwdCarryShape<S>::NT) scan_bwd_carry_kernel(const ScanParams p) {
  using Sh = BwdCarryShape<S>;
  constexpr int TT = Sh::TT, CH = Sh::CH, C = Sh::C, NP = Sh::NP, NL = Sh::NL, NQ = Sh::NQ;
  __shared__ __align__(16) float2 dg[2][TT][CH];        // Delta, dy'
  __shared__ __align__(16) float cs[2][TT][S];
  const Place<CH> at(p, blockIdx.x);
  const int seg = blockIdx.y + 1, t_first = seg * p.seglen, t_end = min(p.L, t_first + p.seglen);
  const int t_last = t_first + (t_end - t_first - 1) / TT * TT;
  if (threadIdx.x >= Sh::WALK) {
  const int tid = threadIdx.x - Sh::WALK;
  const bool gate = p.z.p != nullptr;
  int row[NL], col[NL], valid[NL];
  float bias[NL][4];
#pragma unroll
  for (int k = 0; k < NL; ++k) {
    const int id = tid + k * Sh::LOAD;
    row[k] = id / (CH / 4);
    col[k] = id % (CH / 4) * 4;
    valid[k] = max(0, min(4, at.left - col[k]));
#pragma unroll
    for (int i = 0; i < 4; ++i) bias[k][i] = p.bias && i < valid[k] ? p.bias[at.ch0 + col[k] + i] : 0.f;
  }
  auto place = [&](const ScanRows& w, int t, int k) { return reinterpret_cast<const T*>(w.p) + at.n * w.sn + t * w.sl + at.ch0 + col[k]; };
  Quad<T, VEC> fd[NL], fz[NL], fy[NL], fc[NQ];
  auto fetch = [&](int t0) {
#pragma unroll
    for (int k = 0; k < NL; ++k) {
      const int t = t0 + row[k], v = t < t_end ? valid[k] : 0;
      fd[k].fetch(place(p.delta, t, k), v);
      fy[k].fetch(place(p.dy, t, k), v);
      if (gate) fz[k].fetch(place(p.z, t, k), v);
    }
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      const int id = tid + i * Sh::LOAD, t = t0 + id / (S / 4);
      fc[i].fetch(reinterpret_cast<const T*>(p.C.p) + at.n * p.C.sn + at.g * p.C.sg + t * p.C.sl + id % (S / 4) * 4, id < Sh::QUADS && t < t_end ? 4 : 0);
    }
  };
  auto stage = [&](int buf) {
#pragma unroll
    for (int k = 0; k < NL; ++k) {
      const float4 r4 = fd[k].get();
      float4 g = fy[k].get();
      u64 lo = add2(pack2(r4.x, r4.y), pack2(bias[k][0], bias[k][1])), hi = add2(pack2(r4.z, r4.w), pack2(bias[k][2], bias[k][3]));
      if (p.softplus) {
        lo = softplus2(lo);
        hi = softplus2(hi);
      }
      float dl[4];
      unpack2(lo, dl[0], dl[1]); unpack2(hi, dl[2], dl[3]);
      if (gate) {
        const float4 z4 = fz[k].get();
        g.x *= z4.x * sigmoid(z4.x); g.y *= z4.y * sigmoid(z4.y); g.z *= z4.z * sigmoid(z4.z); g.w *= z4.w * sigmoid(z4.w);
      }
      float4* o = reinterpret_cast<float4*>(&dg[buf][row[k]][col[k]]);
      o[0] = make_float4(dl[0], g.x, dl[1], g.y);
      o[1] = make_float4(dl[2], g.z, dl[3], g.w);
    }
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      const int id = tid + i * Sh::LOAD;
      if (id < Sh::QUADS) *reinterpret_cast<float4*>(&cs[buf][0][0] + id * 4) = fc[i].get();
    }
  };
  fetch(t_last);
  stage(0);
  if (t_last - TT >= t_first) fetch(t_last - TT);
  __syncthreads();
  for (int t0 = t_last, k0 = 0; t0 >= t_first; t0 -= TT, k0 ^= 1) {
    if (t0 - TT >= t_first) {
      stage(k0 ^ 1);
      if (t0 - 2 * TT >= t_first) fetch(t0 - 2 * TT);
    }
    __syncthreads();
  }
  return;
  }

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, q = lane % Sh::LN, chl = (warp * Sh::LC + lane / Sh::LN) * C;
  const int d = at.ch0 + chl, mine = at.left - chl;
  u64 A2[C][NP], gc[C][NP];
#pragma unroll
  for (int c = 0; c < C; ++c) {
#pragma unroll
    for (int i = 0; i < NP; ++i) A2[c][i] = gc[c][i] = 0ull;
    if (c < mine) load_states<Sh>(p.A + (long long)(d + c) * S, q, A2[c]);
#pragma unroll
    for (int i = 0; i < NP; ++i) A2[c][i] = mul2(A2[c][i], dup2(LOG2E));
  }
  float sum_d[C];
#pragma unroll
  for (int c = 0; c < C; ++c) sum_d[c] = 0.f;
  bool cut = false;
  unsigned resets = reset_bits(p, at.n, t_last, t_end - t_last);
  __syncthreads();
  for (int t0 = t_last, k0 = 0; t0 >= t_first; t0 -= TT, k0 ^= 1) {
    const int steps = min(TT, t_end - t0);
    const unsigned now = resets;
    if (t0 - TT >= t_first) resets = reset_bits(p, at.n, t0 - TT, TT);
    auto walk = [&](auto whole) {
      constexpr bool WHOLE = decltype(whole)::value;
#pragma unroll
      for (int t = TT - 1; t >= 0; --t) {
        if (!WHOLE && t >= steps) continue;
        float2 x[C];
        load_channels<C>(&dg[k0][t][chl], x);
        u64 c2[NP];
        load_states<Sh>(&cs[k0][t][0], q, c2);
        const bool fresh = !WHOLE && (now >> t & 1u);
        cut |= fresh;
#pragma unroll
        for (int c = 0; c < C; ++c) {
          const u64 d2 = dup2(x[c].x), g2 = dup2(x[c].y);
          sum_d[c] += x[c].x;
#pragma unroll
          for (int i = 0; i < NP; ++i) {
            const u64 g = fma2<true>(c2[i], g2, gc[c][i]), a = exp2_pair(mul2(d2, A2[c][i]));
            gc[c][i] = fresh ? 0ull : mul2(a, g);
          }
        }
      }
    };
    if (steps == TT && now == 0u) walk(std::true_type());
    else walk(std::false_type());
    __syncthreads();
  }
  const long long states = (long long)p.N * p.D * S, own = ((long long)at.n * p.D + d) * S;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    if (c >= mine) continue;
    u64 decay[NP];
#pragma unroll
    for (int i = 0; i < NP; ++i) decay[i] = cut ? 0ull : exp2_pair(mul2(dup2(sum_d[c]), A2[c][i]));
    store_states<Sh>(p.carry + (2 * seg - 2) * states + own + c * S, q, gc[c]);
    store_states<Sh>(p.carry + (2 * seg - 1) * states + own + c * S, q, decay);
  }
}

// The CTAs' shares added up: blocks below `bc_blocks` four values of dB or dC a thread, the others one of dA, dD or dbias
template <typename T>
__global__ void __launch_bounds__(256) scan_sums_kernel(const ScanParams p, int bc_blocks) {
  const int ch = scan_bwd_channels(p.S), per = (p.D / p.G + ch - 1) / ch, GS = p.G * p.S;
  if ((int)blockIdx.x < bc_blocks) {
    const long long rows = (long long)p.N * p.L, total = 2 * rows * GS;
    const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= total) return;
    float4 v = *reinterpret_cast<const float4*>(p.part_bc + i);
#pragma unroll 4
    for (int b = 1; b < per; ++b) {
      const float4 w = *reinterpret_cast<const float4*>(p.part_bc + b * total + i);
      v.x += w.x; v.y += w.y; v.z += w.z; v.w += w.w;
    }
    const bool second = i >= rows * GS;
    const long long k = i - (second ? rows * GS : 0), r = k / GS;
    const int e = (int)(k - r * GS), g = e / p.S, s = e - g * p.S;
    const ScanRows& o = second ? p.dC : p.dB;
    T* dst = reinterpret_cast<T*>(o.p) + r / p.L * o.sn + r % p.L * o.sl + g * o.sg + s;
    if (p.vec) put4<true>(dst, 4, v);
    else put4<false>(dst, 4, v);
    return;
  }
  const long long i = (long long)(blockIdx.x - bc_blocks) * 256 + threadIdx.x, na = (long long)p.D * p.S;
  if (i >= na + 2 * p.D) return;
  const bool vec = i >= na;
  const float* src = vec ? p.part_v + (i - na) : p.part_a + i;
  const long long step = vec ? 2 * p.D : na;
  float v = 0.f;
#pragma unroll 4
  for (int b = 0; b < p.N * p.nseg; ++b) v += src[b * step];
  if (!vec) p.dA[i] = v;
  else if (i - na < p.D) { if (p.dskip) p.dskip[i - na] = v; }
  else if (p.dbias) p.dbias[i - na - p.D] = v;
}

template <typename T, int S, bool VEC>
cudaError_t launch(const ScanParams& p, cudaStream_t s) {
  const unsigned grid = (unsigned)blocks_of(p, BwdShape<S>::CH);
  constexpr int smem = sizeof(BwdSmem<S>);
  static unsigned long long raised = 0;
  static int registers = 0;      // of a thread at launch: the kernel shares them out
  if (__atomic_load_n(&registers, __ATOMIC_RELAXED) == 0) {
    cudaFuncAttributes a;
    if (const cudaError_t e = cudaFuncGetAttributes(&a, scan_bwd_kernel<T, S, VEC>); e != cudaSuccess) return e;
    if (a.numRegs * BwdShape<S>::NT < BwdRegs<S>::ALL) return cudaErrorLaunchOutOfResources;
    __atomic_store_n(&registers, a.numRegs, __ATOMIC_RELAXED);
  }
  if (const cudaError_t e = allow_smem(scan_bwd_kernel<T, S, VEC>, smem, &raised); e != cudaSuccess) return e;
  if (p.nseg > 1) {
    scan_bwd_carry_kernel<T, S, VEC><<<dim3(grid, p.nseg - 1), BwdCarryShape<S>::NT, 0, s>>>(p);
    if (const cudaError_t e = cudaGetLastError(); e != cudaSuccess) return e;
  }
  scan_bwd_kernel<T, S, VEC><<<dim3(grid, p.nseg), BwdShape<S>::NT, smem, s>>>(p);
  if (const cudaError_t e = cudaGetLastError(); e != cudaSuccess) return e;
  const long long quads = 2ll * p.N * p.L * p.G * S / 4, bc_blocks = (quads + 255) / 256;
  const long long rest = ((long long)p.D * S + 2 * p.D + 255) / 256;
  scan_sums_kernel<T><<<(unsigned)(bc_blocks + rest), 256, 0, s>>>(p, (int)bc_blocks);
  return cudaGetLastError();
}
}  // namespace

long long scan_bwd_scratch(ScanParams& p, float* base) {
  const long long ch = scan_bwd_channels(p.S), per = (p.D / p.G + ch - 1) / ch, slots = (long long)p.N * p.nseg;
  const long long bc = per * 2 * p.N * p.L * p.G * p.S, a = slots * p.D * p.S, v = (slots * 2 * p.D + 3) / 4 * 4;
  const long long carry = p.nseg > 1 ? 2ll * (p.nseg - 1) * p.N * p.D * p.S : 0;
  if (base) {
    p.part_bc = base;
    p.part_a = base + bc;
    p.part_v = p.part_a + a;
    p.carry = p.part_v + v;
  }
  return bc + a + v + carry;
}
cudaError_t scan_backward(const ScanParams& p, cudaStream_t s) {
  return by_shape(p, [&](auto t, auto states, auto vec) { return launch<decltype(t), decltype(states)::value, decltype(vec)::value>(p, s); });
}

}  // namespace srwm
