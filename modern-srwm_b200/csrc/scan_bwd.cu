// Selective state-space scan, backward.
//
// With g_t = dL/dh_t = C_t dy'_t + a_{t+1} g_{t+1} (dy' = dy silu(z), a = exp(Delta A)):
//   dC_t = sum_d dy'_t h_t        dB_t = sum_d g_t Delta_t u_t        dA = sum_t Delta_t g_t a_t h_{t-1}
//   du_t = D dy'_t + Delta_t (g_t . B_t)        dDelta_t = u_t (g_t . B_t) + sum_s A a_t h_{t-1} g_t
// A CTA takes its 64 (32) channels from the last step to the first.  The states in front of each eighth step are the forward's; within
// eight steps they are formed again, four at a time, a_t and a_t h_{t-1} staying in registers until the way back has used them.  Thirteen fp32
// operations per state and step are its floor.  Sums over states go through shared memory, a row a lane; sums over channels (dB, dC) through
// the warp's lanes and shared memory, and are added up over the CTAs by a second launch, in a fixed order.
//
// 8 sequences x 2048 steps x 2048 channels, S 16, bf16: 738 us (1580 with every warp loading, walking and writing in turn and one channel
// a thread).  Four walking and four loading warps a CTA, two CTAs a multiprocessor by registers: issue is busy 53 % of the time, the
// fp32 pipe 43, shared memory 60; a scheduler has two walking warps, and each waits for its own chain.  Sums over lanes by shuffles, with
// selects, took 780; states of eight steps in registers spill at 168 a thread (2250).
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

// Registers: the walking threads' share and the loading threads' (88 for these spill: 1150 us against 970 forward and backward), which together are at most what the CTA is launched with (128 a thread, two
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
  // (each pointer walks with its tiles, the last first: the loads' two tiles in front of the results')
  auto place = [&](const ScanRows& w) { return reinterpret_cast<T*>(w.p) + at.n * w.sn + (t_last + row) * w.sl + at.ch0 + col; };
  const T *pu = place(p.u), *pd = place(p.delta), *pz = place(p.z), *py = place(p.dy);
  T *ou = place(p.du), *od = place(p.ddelta), *oz = place(p.dz);
  const int id0 = tid % Sh::QUADS, bc_row = tid < Sh::QUADS ? id0 / (S / 4) : p.L;      // (a row behind every piece's end)
  const T* pb = reinterpret_cast<const T*>(p.B.p) + at.n * p.B.sn + at.g * p.B.sg + (t_last + id0 / (S / 4)) * p.B.sl + id0 % (S / 4) * 4;
  const T* pc = reinterpret_cast<const T*>(p.C.p) + at.n * p.C.sn + at.g * p.C.sg + (t_last + id0 / (S / 4)) * p.C.sl + id0 % (S / 4) * 4;
  static_assert(NQ == 1, "a tile's B is a piece a thread");
  const Pairs bias = four(p.bias ? p.bias + at.ch0 + col : nullptr, valid), skip = four(p.skip ? p.skip + at.ch0 + col : nullptr, valid);
  // three tiles: being fetched, staged for the next walk, walked before (these two for the results; where they take more than 16
  // registers, the rows are loaded again instead)
  constexpr bool KEEP = VEC && NL * sizeof(T) == 2;
  struct Rows {
    Quad<T, VEC> u, d, z, y;
  } next[NL], staged[KEEP ? NL : 1], done[KEEP ? NL : 1];
  Quad<T, VEC> fb, fc;
  auto fetch = [&](int t0) {
#pragma unroll
    for (int k = 0; k < NL; ++k) {
      const int v = t0 + row + k * RS < t_end ? valid : 0;
      next[k].u.fetch(pu + k * RS * p.u.sl, v);
      next[k].d.fetch(pd + k * RS * p.delta.sl, v);
      next[k].y.fetch(py + k * RS * p.dy.sl, v);
      if (gate) next[k].z.fetch(pz + k * RS * p.z.sl, v);
    }
    pu -= TT * p.u.sl; pd -= TT * p.delta.sl; py -= TT * p.dy.sl; pz -= TT * p.z.sl;
    const int v = t0 + bc_row < t_end ? 4 : 0;
    fb.fetch(pb, v);
    fc.fetch(pc, v);
    pb -= TT * p.B.sl; pc -= TT * p.C.sl;
  };
  auto stage = [&](int buf) {
    auto& tl = sm.tile[buf];
#pragma unroll
    for (int k = 0; k < NL; ++k) {
      if (KEEP) {
        done[KEEP ? k : 0] = staged[KEEP ? k : 0];
        staged[KEEP ? k : 0] = next[k];
      }
      if (!loads) continue;
      Pairs dl = Pairs(next[k].d.get()) + bias, g(next[k].y.get());
      if (p.softplus) dl = softplus4(dl);
      if (gate) {
        const Pairs z(next[k].z.get());
        g = g * (z * sigmoid4(z));
      }
      store_staged(&tl.dd[row + k * RS][col], dl, dl * Pairs(next[k].u.get()));
      *reinterpret_cast<float4*>(&tl.gy[row + k * RS][col]) = g.f4();
    }
    if (tid < Sh::QUADS) {
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const float4 v = w ? fc.get() : fb.get();
        float* o = &tl.bc[w][id0 / (S / 4)][0][id0 % (S / 4) * 4];
        *reinterpret_cast<float4*>(o) = v;
        *reinterpret_cast<float4*>(o + S) = make_float4(v.z, v.w, v.x, v.y);
        *reinterpret_cast<float4*>(o + 2 * S) = make_float4(v.y, v.x, v.w, v.z);
        *reinterpret_cast<float4*>(o + 3 * S) = make_float4(v.w, v.z, v.y, v.x);
      }
    }
  };
  float* part = p.part_bc + ((long long)at.blk * 2 * p.N + at.n) * p.L * p.G * S + at.g * S;
  auto finish = [&](int t0, int buf) {
    const auto& tl = sm.tile[buf];
    const int steps = min(TT, t_end - t0);
    // this CTA's share of dB and dC
#pragma unroll
    for (int e0 = 0; e0 < 2 * Sh::QUADS; e0 += Sh::LOAD) {
      const int e = e0 + tid, s = e % (S / 4) * 4, arr = e / (S / 4) % 2, t = e / (S / 2);
      if (e >= 2 * Sh::QUADS || t >= steps) continue;
      Pairs v(&tl.part[0][t][arr][s]);
#pragma unroll
      for (int w = 1; w < Sh::WARPS; ++w) v = v + Pairs(&tl.part[w][t][arr][s]);
      *reinterpret_cast<float4*>(part + ((long long)arr * p.N * p.L + t0 + t) * p.G * S + s) = v.f4();
    }
#pragma unroll
    for (int k = 0; k < NL; ++k) {
      const int r = row + k * RS, v = r < steps ? valid : 0;
      if (v > 0) {
        Rows was = done[KEEP ? k : 0];
        if (!KEEP) {
          const int t = t0 - t_last + k * RS;      // (the pointers at the last tile, from the results')
          was.u.fetch(place(p.u) + t * p.u.sl, v);
          was.d.fetch(place(p.delta) + t * p.delta.sl, v);
          if (gate) {
            was.z.fetch(place(p.z) + t * p.z.sl, v);
            was.y.fetch(place(p.dy) + t * p.dy.sl, v);
          }
        }
        const Pairs g(&tl.gy[r][col]), u(was.u.get()), gb = sum_lanes<Sh>(&tl.gb[r][0][col]), sa = sum_lanes<Sh>(&tl.sa[r][0][col]);
        const float4* dk = reinterpret_cast<const float4*>(&tl.dd[r][col]);
        const float4 d01 = dk[0], d23 = dk[1];
        const Pairs dl(make_float4(d01.x, d01.z, d23.x, d23.z));
        put4<VEC>(ou + k * RS * p.du.sl, v, fma4(g, skip, dl * gb).f4());
        const u64 ln2 = dup2(0.6931471805599453f);      // (the walking threads' A has log2(e) in it)
        Pairs dr = fma4(u, gb, sa * Pairs(ln2, ln2));
        if (p.softplus) dr = dr * sigmoid4(Pairs(was.d.get()) + bias);
        put4<VEC>(od + k * RS * p.ddelta.sl, v, dr.f4());
        const int id = tid + k * Sh::LOAD;
        sm.sums[0][id] = fma4(g, u, Pairs(sm.sums[0][id])).f4();
        sm.sums[1][id] = (Pairs(sm.sums[1][id]) + dr).f4();
        if (gate) {      // silu'(z) = sigmoid (1 + z (1 - sigmoid))
          const u64 one = dup2(1.f), minus = dup2(-1.f);
          const Pairs y = fma4(skip, u, sum_lanes<Sh>(&tl.yp[r][0][col])), z(was.z.get()), sg = sigmoid4(z);
          const Pairs rest = fma4(sg, Pairs(minus, minus), Pairs(one, one));
          put4<VEC>(oz + k * RS * p.dz.sl, v, (Pairs(was.y.get()) * y * (sg * fma4(z, rest, Pairs(one, one)))).f4());
        }
      }
    }
    ou -= TT * p.du.sl; od -= TT * p.ddelta.sl; oz -= TT * p.dz.sl;
  };
  fetch(t_last);
  stage(0);
  if (t_last - TT >= t_first) fetch(t_last - TT);
  __syncthreads();
  int k0 = 0;
  for (int t0 = t_last; t0 >= t_first; t0 -= TT, k0 ^= 1) {
    if (t0 < t_last) finish(t0 + TT, k0 ^ 1);
    if (t0 - TT >= t_first) {
      stage(k0 ^ 1);
      if (t0 - 2 * TT >= t_first) fetch(t0 - 2 * TT);
    } else {
#pragma unroll
      for (int k = 0; k < (KEEP ? NL : 1); ++k) done[k] = staged[k];
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
  constexpr int SUB = 4, GS = 8 / ST, HOLD = ST == 4 ? SUB : 1;      // HOLD: steps whose sums over the groups are formed together
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
      u64 root[NP], end[NP];
      load_turned<Sh>(p.carry + (2 * i - 2) * states + o, q, order, end);
      load_turned<Sh>(p.carry + (2 * i - 1) * states + o, q, order, root);
      through_piece(gc[c], root, end);
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

    // HOLD steps' shares of dB or dC from t on
    auto leave = [&](float* v, int t, int arr) __attribute__((always_inline)) {
#pragma unroll
      for (int g = 0; g < HOLD / GS; ++g) sum_groups<ST, LN>(v + 8 * g, lane);
#pragma unroll
      for (int g = 0; g < HOLD / GS; ++g) {
        float* o = part_mine + ((t + g * GS) * 2 + arr) * S;
        if (LN == 8) *reinterpret_cast<float2*>(o) = make_float2(v[8 * g], v[8 * g + 1]);
        else if (keeps) *o = v[8 * g];
      }
    };
    // Four steps at a time, the last first.  The second four have the first four walked on the way to them (without what they leave), so that a
    // and a h of no more than four stay in registers.
    auto tile = [&](auto whole) __attribute__((always_inline)) {
      constexpr bool WHOLE = decltype(whole)::value;      // eight steps of one episode, all channels there
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
                a[k][c][i] = decay2(d2, A2[c][i]);
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
              a[k][c][i] = decay2(d2, A2[c][i]);
              ah[k][c][i] = mul2(x2, b2[i]);
            }
          }
        }
        float v[HOLD * ST];
#pragma unroll
        for (int k = 0; k < SUB; ++k) {
          const int t = s0 + k;
          float* vk = v + k % HOLD * ST;
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
                const u64 share = WHOLE || c < mine ? h[c][i] : 0ull;      // (no channel: B may be infinite, and 0 B not 0)
                sum[i] = c == 0 ? mul2(share, g2) : fma2<true>(share, g2, sum[i]);
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
          if (k % HOLD == HOLD - 1) leave(v, t - (HOLD - 1), 1);
        }
#pragma unroll
        for (int k = SUB - 1; k >= 0; --k) {
          const int t = s0 + k;
          float* vk = v + k % HOLD * ST;
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
                const u64 share = WHOLE || c < mine ? g : 0ull;
                sum[i] = c == 0 ? mul2(share, x2) : fma2<true>(share, x2, sum[i]);
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
          if (k % HOLD == 0) leave(v, t, 0);
        }
      }
    };
    if (steps == TT && now == 0u && at.left >= CH) tile(std::true_type());
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
            const u64 g = fma2<true>(c2[i], g2, gc[c][i]), a = decay2(d2, A2[c][i]);
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
    u64 root[NP];
#pragma unroll
    for (int i = 0; i < NP; ++i) root[i] = cut ? CUT : piece_root(sum_d[c], A2[c][i]);
    store_states<Sh>(p.carry + (2 * seg - 2) * states + own + c * S, q, gc[c]);
    store_states<Sh>(p.carry + (2 * seg - 1) * states + own + c * S, q, root);
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
