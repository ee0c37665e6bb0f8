// Selective state-space scan, backward.
//
// With g_t = dL/dh_t = C_t dy'_t + a_{t+1} g_{t+1} (dy' = dy silu(z), a = exp(Delta A)):
//   dC_t = sum_d dy'_t h_t        dB_t = sum_d g_t Delta_t u_t        dA = sum_t Delta_t g_t a_t h_{t-1}
//   du_t = D dy'_t + Delta_t (g_t . B_t)        dDelta_t = u_t (g_t . B_t) + sum_s A a_t h_{t-1} g_t
// A CTA takes its 32 channels from the last step to the first.  The states in front of each eighth step are the forward's; within
// eight steps they are formed again, a_t and a_t h_{t-1} staying in registers until the way back has used them (four steps of them
// where a thread has eight states: the first four are walked twice then).  Thirteen fp32
// operations per state and step bind.  Sums over states go through a channel's lanes, sums over channels (dB, dC) through the
// warp's other lanes and shared memory, and are added up over the CTAs by a second launch, in a fixed order.
#include <type_traits>

#include "device.h"
#include "scan.cuh"

namespace srwm {
namespace {
using namespace scan;

// Sums of eight values over a warp's LC channels: 8 / LC values stay with each lane, those from index `kept_of` on
template <int LN, int LC>
__device__ __forceinline__ void channels_to_lanes(float (&v)[8], int lane) {
#pragma unroll
  for (int w = LN, half = 4; w < 32; w *= 2, half /= 2) {
    const bool up = lane & w;
#pragma unroll
    for (int i = 0; i < half; ++i) {
      const float keep = up ? v[half + i] : v[i], send = up ? v[i] : v[half + i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, send, w);
    }
  }
}
template <int LN, int LC>
__device__ __forceinline__ int kept_of(int lane) {
  const int c = lane / LN;       // bits of the channel, the lowest first halves
  return LC == 8 ? (c & 1) * 4 + (c & 2) + (c >> 2) : (c & 1) * 4 + (c & 2);
}

template <int S>
struct BwdSmem {
  static constexpr int TT = SCAN_TILE, CH = SCAN_CH, PAD = CH + 8, WARPS = Shape<S>::NT / 32;
  float4 dd[TT][CH];           // Delta twice, Delta u twice
  float2 gy[TT][CH];           // dy' twice
  float bc[2][TT][S];
  float gb[TT][PAD], sa[TT][PAD], yp[TT][PAD];
  float part[WARPS][TT][2][S];
};

// Steps whose a and a h stay in registers, and CTAs that a multiprocessor is to hold (168 registers a thread, or 128)
template <int S>
struct BwdPlan {
  static constexpr int SUB = Shape<S>::ST == 8 ? 4 : 8, CTAS = S == 8 ? 4 : S == 64 ? 1 : 2;
};

template <typename T, int S, bool VEC>
__global__ void __launch_bounds__(Shape<S>::NT, BwdPlan<S>::CTAS) scan_bwd_kernel(const ScanParams p) {
  using Sh = Shape<S>;
  constexpr int TT = SCAN_TILE, CH = SCAN_CH, KT = SCAN_CKPT, NP = Sh::ST / 2, GS = 8 / Sh::ST, KEPT = 8 / Sh::LC, SUB = BwdPlan<S>::SUB;
  constexpr int WARPS = BwdSmem<S>::WARPS;
  extern __shared__ __align__(16) unsigned char raw_smem[];
  BwdSmem<S>& sm = *reinterpret_cast<BwdSmem<S>*>(raw_smem);
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, q = lane % Sh::LN, chl = warp * Sh::LC + lane / Sh::LN;
  const Place at(p, blockIdx.x);
  const int seg = blockIdx.y, t_first = seg * p.seglen, t_end = min(p.L, t_first + p.seglen);
  const int t_last = t_first + (t_end - t_first - 1) / TT * TT;
  const bool mine = chl < at.left;
  const int d = at.ch0 + chl, here = swizzled(chl);

  const bool loader = tid < TT * CH / 4;
  const int row = tid / (CH / 4), col = tid % (CH / 4) * 4, valid = loader ? max(0, min(4, at.left - col)) : 0;
  auto rows = [&](const ScanRows& w) { return reinterpret_cast<T*>(w.p) + at.n * w.sn + (t_last + row) * w.sl + at.ch0 + col; };
  const T *pu = rows(p.u), *pd = rows(p.delta), *pz = rows(p.z), *py = rows(p.dy);
  T *ou = rows(p.du), *od = rows(p.ddelta), *oz = rows(p.dz);
  const bool gate = p.z.p != nullptr;
  float bias[4], skip[4], sum_skip[4], sum_bias[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    bias[i] = i < valid && p.bias ? p.bias[at.ch0 + col + i] : 0.f;
    skip[i] = i < valid && p.skip ? p.skip[at.ch0 + col + i] : 0.f;
    sum_skip[i] = sum_bias[i] = 0.f;
  }
  const T* pbc[Sh::NQ];
  long long lbc[Sh::NQ];
  int rbc[Sh::NQ];
#pragma unroll
  for (int i = 0; i < Sh::NQ; ++i) {
    const int id = tid + i * Sh::NT, c = id % (S / 4) * 4, r = id / (S / 4) % TT;
    const bool second = id >= TT * S / 4;
    lbc[i] = (second ? p.C.sl : p.B.sl) * TT;
    pbc[i] = second ? reinterpret_cast<const T*>(p.C.p) + at.n * p.C.sn + at.g * p.C.sg + (t_last + r) * p.C.sl + c
                    : reinterpret_cast<const T*>(p.B.p) + at.n * p.B.sn + at.g * p.B.sg + (t_last + r) * p.B.sl + c;
    rbc[i] = id < Sh::QUADS ? r : p.L;
  }
  Quad<T, VEC> fu, fd, fz, fy, fbc[Sh::NQ];
  auto fetch = [&](int t0) {      // tiles are asked for in order, the last first
    const int v = t0 + row < t_end ? valid : 0;
    fu.fetch(pu, v);
    fd.fetch(pd, v);
    fy.fetch(py, v);
    if (gate) fz.fetch(pz, v);
    pu -= TT * p.u.sl; pd -= TT * p.delta.sl; py -= TT * p.dy.sl; pz -= TT * p.z.sl;
#pragma unroll
    for (int i = 0; i < Sh::NQ; ++i) {
      fbc[i].fetch(pbc[i], t0 + rbc[i] < t_end ? 4 : 0);
      pbc[i] -= lbc[i];
    }
  };

  u64 A2[NP], gc[NP], dA[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) A2[i] = gc[i] = dA[i] = 0ull;
  if (t_first < t_end) fetch(t_last);
  const long long states = (long long)p.N * p.D * S, own = ((long long)at.n * p.D + d) * S;
  const int nck = (p.L + KT - 1) / KT;
  if (mine) {
    load_states<Sh>(p.A + (long long)d * S, q, A2);
    const u64 l2 = dup2(LOG2E);
#pragma unroll
    for (int i = 0; i < NP; ++i) A2[i] = mul2(A2[i], l2);
    if (p.dhT) load_states<Sh>(p.dhT + own, q, gc);
#pragma unroll 4
    for (int i = p.nseg - 1; i > seg; --i) {      // the pieces behind, the last first
      u64 decay[NP], end[NP];
      load_states<Sh>(p.carry + (2 * i - 2) * states + own, q, end);
      load_states<Sh>(p.carry + (2 * i - 1) * states + own, q, decay);
#pragma unroll
      for (int k = 0; k < NP; ++k) gc[k] = fma2<true>(decay[k], gc[k], end[k]);
    }
  }
  const int kept = kept_of<Sh::LN, Sh::LC>(lane), kept_step = kept / Sh::ST, kept_j = kept % Sh::ST;
  const int kept_state = Sh::first(q, kept_j / 4) + (Sh::ST >= 4 ? kept_j % 4 : kept_j);
  float* part_mine = &sm.part[warp][kept_step][0][kept_state];

  for (int t0 = t_last; t0 >= t_first; t0 -= TT) {
    const int steps = min(TT, t_end - t0);
    // the states in front of the tile's two halves
    u64 ck[2][NP];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
      for (int i = 0; i < NP; ++i) ck[k][i] = 0ull;
      if (mine && k * KT < steps) load_states<Sh>(p.ckpt + (((long long)at.n * nck + t0 / KT + k) * p.D + d) * S, q, ck[k]);
    }
    const Quad<T, VEC> qu = fu, qd = fd, qz = fz, qy = fy;
    u64 dl2[2], g2v[2];      // Delta and dy' of this thread's piece
    dl2[0] = dl2[1] = g2v[0] = g2v[1] = 0ull;
    if (loader) {
      const float4 u4 = qu.get(), r4 = qd.get(), y4 = qy.get();
      dl2[0] = add2(pack2(r4.x, r4.y), pack2(bias[0], bias[1]));
      dl2[1] = add2(pack2(r4.z, r4.w), pack2(bias[2], bias[3]));
      if (p.softplus) {
        dl2[0] = softplus2(dl2[0]);
        dl2[1] = softplus2(dl2[1]);
      }
      const u64 xlo = mul2(dl2[0], pack2(u4.x, u4.y)), xhi = mul2(dl2[1], pack2(u4.z, u4.w));
      float dl[4], du[4], g[4] = {y4.x, y4.y, y4.z, y4.w};
      unpack2(dl2[0], dl[0], dl[1]); unpack2(dl2[1], dl[2], dl[3]);
      unpack2(xlo, du[0], du[1]); unpack2(xhi, du[2], du[3]);
      if (gate) {
        const float4 z4 = qz.get();
        g[0] *= z4.x * sigmoid(z4.x); g[1] *= z4.y * sigmoid(z4.y); g[2] *= z4.z * sigmoid(z4.z); g[3] *= z4.w * sigmoid(z4.w);
      }
      g2v[0] = pack2(g[0], g[1]); g2v[1] = pack2(g[2], g[3]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        sm.dd[row][swizzled(col + i)] = make_float4(dl[i], dl[i], du[i], du[i]);
        sm.gy[row][swizzled(col + i)] = make_float2(g[i], g[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < Sh::NQ; ++i) {
      const int id = tid + i * Sh::NT;
      if (id < Sh::QUADS) *reinterpret_cast<float4*>(&sm.bc[0][0][0] + id * 4) = fbc[i].get();
    }
    const unsigned resets = reset_bits(p, at.n, t0, steps);
    __syncthreads();
    if (t0 - TT >= t_first) fetch(t0 - TT);

    // SUB steps from s0 of the tile, h the state in front of them
    auto steps_of = [&](auto whole, int s0, u64* h) __attribute__((always_inline)) {
      constexpr bool WHOLE = decltype(whole)::value;
      u64 a[SUB][NP], ah[SUB][NP];
      float yv[Sh::LN], dc[8];
#pragma unroll
      for (int k = 0; k < SUB; ++k) {
        const int t = s0 + k;
        float* dck = dc + k % GS * Sh::ST;
        yv[k % Sh::LN] = 0.f;
#pragma unroll
        for (int i = 0; i < Sh::ST; ++i) dck[i] = 0.f;
        if (WHOLE || t < steps) {
          const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(&sm.dd[t][here]);
          const u64 g2 = *reinterpret_cast<const u64*>(&sm.gy[t][here]);
          const bool fresh = !WHOLE && (resets >> t & 1u);
          u64 b2[NP], c2[NP], acc = 0ull;
          load_states<Sh>(&sm.bc[0][t][0], q, b2);
          load_states<Sh>(&sm.bc[1][t][0], q, c2);
#pragma unroll
          for (int i = 0; i < NP; ++i) {
            a[k][i] = exp2_pair(mul2(x.x, A2[i]));
            if (fresh) a[k][i] = h[i] = 0ull;
            ah[k][i] = mul2(a[k][i], h[i]);
            h[i] = add2(ah[k][i], mul2(x.y, b2[i]));
            acc = i == 0 ? mul2(h[i], c2[i]) : fma2<true>(h[i], c2[i], acc);
            unpack2(mul2(h[i], g2), dck[2 * i], dck[2 * i + 1]);
          }
          yv[k % Sh::LN] = hsum2(acc);
        }
        if (k % GS == GS - 1) {
          channels_to_lanes<Sh::LN, Sh::LC>(dc, lane);
          float* o = part_mine + (s0 + k - (GS - 1)) * 2 * S + S;
#pragma unroll
          for (int i = 0; i < KEPT; ++i) o[i] = dc[i];
        }
        // (a piece's last steps may be fewer than the lanes: the values are zero then, and the row is not read)
        if (gate && (k % Sh::LN == Sh::LN - 1 || k == SUB - 1)) {
#pragma unroll
          for (int i = SUB; i < Sh::LN; ++i) yv[i] = 0.f;
          const float y = steps_to_lanes<Sh::LN>(yv, q);
          if (SUB >= Sh::LN || q < SUB) sm.yp[s0 + k - (SUB < Sh::LN ? SUB : Sh::LN) + 1 + q][chl] = y;
        }
      }
      float gbv[Sh::LN], sav[Sh::LN], db[8];
#pragma unroll
      for (int k = SUB - 1; k >= 0; --k) {
        const int t = s0 + k;
        float* dbk = db + k % GS * Sh::ST;
        gbv[k % Sh::LN] = sav[k % Sh::LN] = 0.f;
#pragma unroll
        for (int i = 0; i < Sh::ST; ++i) dbk[i] = 0.f;
        if (WHOLE || t < steps) {
          const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(&sm.dd[t][here]);
          const u64 g2 = *reinterpret_cast<const u64*>(&sm.gy[t][here]);
          u64 b2[NP], c2[NP], gb = 0ull, sa = 0ull;
          load_states<Sh>(&sm.bc[0][t][0], q, b2);
          load_states<Sh>(&sm.bc[1][t][0], q, c2);
          const bool fresh = !WHOLE && (resets >> t & 1u);
#pragma unroll
          for (int i = 0; i < NP; ++i) {
            const u64 g = fma2<true>(c2[i], g2, gc[i]), gah = mul2(g, ah[k][i]);
            gb = i == 0 ? mul2(g, b2[i]) : fma2<true>(g, b2[i], gb);
            sa = i == 0 ? mul2(gah, A2[i]) : fma2<true>(gah, A2[i], sa);
            dA[i] = fma2<true>(gah, x.x, dA[i]);
            unpack2(mul2(g, x.y), dbk[2 * i], dbk[2 * i + 1]);
            gc[i] = fresh ? 0ull : mul2(a[k][i], g);
          }
          gbv[k % Sh::LN] = hsum2(gb);
          sav[k % Sh::LN] = hsum2(sa);
        }
        if (k % GS == 0) {
          channels_to_lanes<Sh::LN, Sh::LC>(db, lane);
          float* o = part_mine + (s0 + k) * 2 * S;
#pragma unroll
          for (int i = 0; i < KEPT; ++i) o[i] = db[i];
        }
        if (k % Sh::LN == 0) {
#pragma unroll
          for (int i = SUB; i < Sh::LN; ++i) gbv[i] = sav[i] = 0.f;
          const float g = steps_to_lanes<Sh::LN>(gbv, q), s = steps_to_lanes<Sh::LN>(sav, q);
          if (SUB >= Sh::LN || q < SUB) {
            sm.gb[s0 + k + q][chl] = g;
            sm.sa[s0 + k + q][chl] = s * 0.6931471805599453f;      // (A2 has log2(e) in it)
          }
        }
      }
    };
    // eight steps at a time, the last first; where four stay in registers, the first four are walked on the way to the others
    auto halves = [&](auto whole) {
      constexpr bool WHOLE = decltype(whole)::value;
#pragma unroll 1
      for (int s0 = TT - SUB; s0 >= 0; s0 -= SUB) {
        if (!WHOLE && s0 >= steps) continue;
        u64 h[NP];
#pragma unroll
        for (int i = 0; i < NP; ++i) h[i] = s0 >= KT ? ck[1][i] : ck[0][i];
        if (SUB < KT && s0 % KT != 0) {
#pragma unroll
          for (int k = 0; k < SUB; ++k) {
            const int t = s0 - SUB + k;
            const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(&sm.dd[t][here]);
            u64 b2[NP];
            load_states<Sh>(&sm.bc[0][t][0], q, b2);
            const bool fresh = !WHOLE && (resets >> t & 1u);
#pragma unroll
            for (int i = 0; i < NP; ++i) {
              u64 a = exp2_pair(mul2(x.x, A2[i]));
              if (fresh) a = h[i] = 0ull;
              h[i] = add2(mul2(a, h[i]), mul2(x.y, b2[i]));
            }
          }
        }
        steps_of(whole, s0, h);
      }
    };
    if (steps == TT && resets == 0u) halves(std::true_type());
    else halves(std::false_type());
    __syncthreads();
    {   // this CTA's share of dB and dC
      const int per = ((p.D / p.G) + CH - 1) / CH, blk = (int)(blockIdx.x % (unsigned)per);
#pragma unroll
      for (int e = tid; e < TT * 2 * S / 4; e += Sh::NT) {
        const int s = e % (S / 4) * 4, arr = e / (S / 4) % 2, t = e / (S / 2);
        float4 v = *reinterpret_cast<const float4*>(&sm.part[0][t][arr][s]);
#pragma unroll
        for (int w = 1; w < WARPS; ++w) {
          const float4 o = *reinterpret_cast<const float4*>(&sm.part[w][t][arr][s]);
          v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w;
        }
        if (t < steps)
          *reinterpret_cast<float4*>(p.part_bc + ((((long long)blk * 2 + arr) * p.N + at.n) * p.L + t0 + t) * p.G * S + at.g * S + s) = v;
      }
    }
    const int v = row < steps ? valid : 0;
    if (v > 0) {
      const float4 gb4 = *reinterpret_cast<const float4*>(&sm.gb[row][col]), sa4 = *reinterpret_cast<const float4*>(&sm.sa[row][col]);
      const float4 u4 = qu.get(), r4 = qd.get();
      const float us[4] = {u4.x, u4.y, u4.z, u4.w}, rs[4] = {r4.x, r4.y, r4.z, r4.w};
      const float gb[4] = {gb4.x, gb4.y, gb4.z, gb4.w}, sa[4] = {sa4.x, sa4.y, sa4.z, sa4.w};
      float dl[4], g[4], o1[4], o2[4];
      unpack2(dl2[0], dl[0], dl[1]); unpack2(dl2[1], dl[2], dl[3]);
      unpack2(g2v[0], g[0], g[1]); unpack2(g2v[1], g[2], g[3]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        o1[i] = fmaf(g[i], skip[i], dl[i] * gb[i]);
        o2[i] = fmaf(us[i], gb[i], sa[i]);
        if (p.softplus) o2[i] *= sigmoid(rs[i] + bias[i]);
        if (i < v) {
          sum_skip[i] = fmaf(g[i], us[i], sum_skip[i]);
          sum_bias[i] += o2[i];
        }
      }
      put4<VEC>(ou, v, make_float4(o1[0], o1[1], o1[2], o1[3]));
      put4<VEC>(od, v, make_float4(o2[0], o2[1], o2[2], o2[3]));
      if (gate) {
        const float4 yp4 = *reinterpret_cast<const float4*>(&sm.yp[row][col]), z4 = qz.get(), y4 = qy.get();
        const float yp[4] = {yp4.x, yp4.y, yp4.z, yp4.w}, zs[4] = {z4.x, z4.y, z4.z, z4.w}, os[4] = {y4.x, y4.y, y4.z, y4.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float sg = sigmoid(zs[i]);
          o1[i] = os[i] * fmaf(skip[i], us[i], yp[i]) * sg * fmaf(zs[i], 1.f - sg, 1.f);
        }
        put4<VEC>(oz, v, make_float4(o1[0], o1[1], o1[2], o1[3]));
      }
    }
    ou -= TT * p.du.sl; od -= TT * p.ddelta.sl; oz -= TT * p.dz.sl;
  }
  const long long slot = (long long)at.n * p.nseg + seg;
  if (mine) {
    store_states<Sh>(p.part_a + (slot * p.D + d) * S, q, dA);
    if (seg == 0 && p.dh0) store_states<Sh>(p.dh0 + own, q, gc);
  }
  __syncthreads();
  if (loader) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      sm.gb[row][col + i] = sum_skip[i];
      sm.sa[row][col + i] = sum_bias[i];
    }
  }
  __syncthreads();
  if (tid < 2 * CH) {
    const int c = tid % CH, which = tid / CH;
    float v = 0.f;
#pragma unroll
    for (int r = 0; r < TT; ++r) v += which ? sm.sa[r][c] : sm.gb[r][c];
    if (c < at.left) p.part_v[(slot * 2 + which) * p.D + at.ch0 + c] = v;
  }
}

// What a piece of the time axis adds to the gradient of the state in front of it (from zero behind it), and the product of its
// decays, for pieces 1 .. nseg - 1.
template <typename T, int S, bool VEC>
__global__ void __launch_bounds__(Shape<S>::NT) scan_bwd_carry_kernel(const ScanParams p) {
  using Sh = Shape<S>;
  constexpr int TT = SCAN_TILE, CH = SCAN_CH, NP = Sh::ST / 2, NQ = (Sh::QUADS / 2 + Sh::NT - 1) / Sh::NT;
  __shared__ __align__(16) float4 dg[2][TT][CH];        // Delta twice, dy' twice
  __shared__ __align__(16) float cs[2][TT][S];
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, q = lane % Sh::LN, chl = warp * Sh::LC + lane / Sh::LN;
  const Place at(p, blockIdx.x);
  const int seg = blockIdx.y + 1, t_first = seg * p.seglen, t_end = min(p.L, t_first + p.seglen);
  const int t_last = t_first + (t_end - t_first - 1) / TT * TT;
  const bool mine = chl < at.left;
  const int d = at.ch0 + chl, here = swizzled(chl);
  const bool loader = tid < TT * CH / 4;
  const int row = tid / (CH / 4), col = tid % (CH / 4) * 4, valid = loader ? max(0, min(4, at.left - col)) : 0;
  auto rows = [&](const ScanRows& w) { return reinterpret_cast<const T*>(w.p) + at.n * w.sn + (t_last + row) * w.sl + at.ch0 + col; };
  const T *pd = rows(p.delta), *pz = rows(p.z), *py = rows(p.dy);
  const bool gate = p.z.p != nullptr;
  float bias[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) bias[i] = i < valid && p.bias ? p.bias[at.ch0 + col + i] : 0.f;
  const T* pc[NQ];
#pragma unroll
  for (int i = 0; i < NQ; ++i) {
    const int id = tid + i * Sh::NT;
    pc[i] = reinterpret_cast<const T*>(p.C.p) + at.n * p.C.sn + at.g * p.C.sg + (t_last + id / (S / 4)) * p.C.sl + id % (S / 4) * 4;
  }
  Quad<T, VEC> fd, fz, fy, fc[NQ];
  auto fetch = [&](int t0) {
    const int v = t0 + row < t_end ? valid : 0;
    fd.fetch(pd, v);
    fy.fetch(py, v);
    if (gate) fz.fetch(pz, v);
    pd -= TT * p.delta.sl; py -= TT * p.dy.sl; pz -= TT * p.z.sl;
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      const int r = (tid + i * Sh::NT) / (S / 4);
      fc[i].fetch(pc[i], r < TT && t0 + r < t_end ? 4 : 0);
      pc[i] -= TT * p.C.sl;
    }
  };
  auto stage = [&](int buf) {
    if (loader) {
      const float4 r4 = fd.get(), y4 = fy.get();
      u64 lo = add2(pack2(r4.x, r4.y), pack2(bias[0], bias[1])), hi = add2(pack2(r4.z, r4.w), pack2(bias[2], bias[3]));
      if (p.softplus) {
        lo = softplus2(lo);
        hi = softplus2(hi);
      }
      float dl[4], g[4] = {y4.x, y4.y, y4.z, y4.w};
      unpack2(lo, dl[0], dl[1]); unpack2(hi, dl[2], dl[3]);
      if (gate) {
        const float4 z4 = fz.get();
        g[0] *= z4.x * sigmoid(z4.x); g[1] *= z4.y * sigmoid(z4.y); g[2] *= z4.z * sigmoid(z4.z); g[3] *= z4.w * sigmoid(z4.w);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) dg[buf][row][swizzled(col + i)] = make_float4(dl[i], dl[i], g[i], g[i]);
    }
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      const int id = tid + i * Sh::NT;
      if (id < Sh::QUADS / 2) *reinterpret_cast<float4*>(&cs[buf][0][0] + id * 4) = fc[i].get();
    }
  };
  u64 A2[NP], gc[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) A2[i] = gc[i] = 0ull;
  if (t_first < t_end) fetch(t_last);
  if (mine) {
    load_states<Sh>(p.A + (long long)d * S, q, A2);
#pragma unroll
    for (int i = 0; i < NP; ++i) A2[i] = mul2(A2[i], dup2(LOG2E));
  }
  float sum_d = 0.f;
  bool cut = false;
  unsigned resets = 0u;
  if (t_first < t_end) {
    stage(0);
    resets = reset_bits(p, at.n, t_last, t_end - t_last);
    if (t_last - TT >= t_first) fetch(t_last - TT);
    __syncthreads();
  }
  for (int t0 = t_last, k0 = 0; t0 >= t_first; t0 -= TT, k0 ^= 1) {
    const int steps = min(TT, t_end - t0);
    const unsigned now = resets;
    if (t0 - TT >= t_first) {
      stage(k0 ^ 1);
      resets = reset_bits(p, at.n, t0 - TT, TT);
      if (t0 - 2 * TT >= t_first) fetch(t0 - 2 * TT);
    }
    auto walk = [&](auto whole) {
      constexpr bool WHOLE = decltype(whole)::value;
#pragma unroll
      for (int t = TT - 1; t >= 0; --t) {
        if (!WHOLE && t >= steps) continue;
        const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(&dg[k0][t][here]);
        u64 c2[NP];
        load_states<Sh>(&cs[k0][t][0], q, c2);
        const bool fresh = !WHOLE && (now >> t & 1u);
        cut |= fresh;
        sum_d += __uint_as_float((unsigned)x.x);
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const u64 g = fma2<true>(c2[i], x.y, gc[i]), a = exp2_pair(mul2(x.x, A2[i]));
          gc[i] = fresh ? 0ull : mul2(a, g);
        }
      }
    };
    if (steps == TT && now == 0u) walk(std::true_type());
    else walk(std::false_type());
    __syncthreads();
  }
  if (!mine) return;
  const long long states = (long long)p.N * p.D * S, own = ((long long)at.n * p.D + d) * S;
  u64 decay[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) decay[i] = cut ? 0ull : exp2_pair(mul2(dup2(sum_d), A2[i]));
  store_states<Sh>(p.carry + (2 * seg - 2) * states + own, q, gc);
  store_states<Sh>(p.carry + (2 * seg - 1) * states + own, q, decay);
}

// The CTAs' shares added up: blocks below `bc_blocks` four values of dB or dC a thread, the others one of dA, dD or dbias
template <typename T>
__global__ void __launch_bounds__(256) scan_sums_kernel(const ScanParams p, int bc_blocks) {
  const int per = (p.D / p.G + SCAN_CH - 1) / SCAN_CH, GS = p.G * p.S;
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
  const unsigned grid = (unsigned)(blocks_of(p) * p.N);
  constexpr int smem = sizeof(BwdSmem<S>);
  static unsigned long long raised = 0;      // devices whose limit is raised
  if (smem > 48 * 1024) {
    int dev = 0;
    if (const cudaError_t e = cudaGetDevice(&dev); e != cudaSuccess) return e;
    const unsigned long long bit = 1ull << (dev & 63);
    if (!(__atomic_load_n(&raised, __ATOMIC_ACQUIRE) & bit)) {
      const cudaError_t e = cudaFuncSetAttribute(scan_bwd_kernel<T, S, VEC>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
      if (e != cudaSuccess) return e;
      __atomic_fetch_or(&raised, bit, __ATOMIC_RELEASE);
    }
  }
  if (p.nseg > 1) {
    scan_bwd_carry_kernel<T, S, VEC><<<dim3(grid, p.nseg - 1), Shape<S>::NT, 0, s>>>(p);
    if (const cudaError_t e = cudaGetLastError(); e != cudaSuccess) return e;
  }
  scan_bwd_kernel<T, S, VEC><<<dim3(grid, p.nseg), Shape<S>::NT, smem, s>>>(p);
  if (const cudaError_t e = cudaGetLastError(); e != cudaSuccess) return e;
  const long long quads = 2ll * p.N * p.L * p.G * S / 4, bc_blocks = (quads + 255) / 256;
  const long long rest = ((long long)p.D * S + 2 * p.D + 255) / 256;
  scan_sums_kernel<T><<<(unsigned)(bc_blocks + rest), 256, 0, s>>>(p, (int)bc_blocks);
  return cudaGetLastError();
}
}  // namespace

int scan_bwd_segments(int N, int L, int D, int sms) { return scan_segments(N, L, D, sms); }

long long scan_bwd_scratch(ScanParams& p, float* base) {
  const long long per = (p.D / p.G + SCAN_CH - 1) / SCAN_CH, slots = (long long)p.N * p.nseg;
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
