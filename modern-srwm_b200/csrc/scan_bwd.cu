// Selective state-space scan, backward.
//
// With g_t = dL/dh_t = C_t dy'_t + a_{t+1} g_{t+1} (dy' = dy silu(z), a = exp(Delta A)):
//   dC_t = sum_d dy'_t h_t        dB_t = sum_d g_t Delta_t u_t        dA = sum_t Delta_t g_t a_t h_{t-1}
//   du_t = D dy'_t + Delta_t (g_t . B_t)        dDelta_t = u_t (g_t . B_t) + sum_s A a_t h_{t-1} g_t
// A CTA takes its 32 channels from the last step to the first.  The states in front of each eighth step are the forward's; within
// eight steps they are formed again, a_t and a_t h_{t-1} staying in registers until the way back has used them.  Thirteen fp32
// operations per state and step bind.  Sums over states go through a channel's lanes, sums over channels (dB, dC) through the
// warp's other lanes and shared memory, and are added up over the CTAs by a second launch, in a fixed order.
#include <type_traits>

#include "device.h"
#include "scan.cuh"

namespace srwm {
namespace {
using namespace scan;

__device__ __forceinline__ u64 add2(u64 a, u64 b) {
  u64 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

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
  float part[WARPS][SCAN_CKPT][2][S];
};

template <typename T, int S>
__global__ void __launch_bounds__(Shape<S>::NT) scan_bwd_kernel(const ScanParams p) {
  using Sh = Shape<S>;
  constexpr int TT = SCAN_TILE, CH = SCAN_CH, KT = SCAN_CKPT, NP = Sh::ST / 2, GS = 8 / Sh::ST, KEPT = 8 / Sh::LC;
  extern __shared__ __align__(16) unsigned char raw_smem[];
  BwdSmem<S>& sm = *reinterpret_cast<BwdSmem<S>*>(raw_smem);
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, q = lane % Sh::LN, chl = warp * Sh::LC + lane / Sh::LN;
  const Place at(p, blockIdx.x);
  const int seg = blockIdx.y, t_first = seg * p.seglen, t_end = min(p.L, t_first + p.seglen);
  const bool mine = chl < at.left;
  const int d = at.ch0 + chl;

  const bool loader = tid < TT * CH / 4;
  const int row = tid / (CH / 4), col = tid % (CH / 4) * 4, valid = loader ? min(4, at.left - col) : 0;
  auto rows = [&](const ScanRows& w) { return reinterpret_cast<T*>(w.p) + at.n * w.sn + at.ch0 + col; };
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
  Quad<T> ru, rd, rz, ry, rbc[Sh::NQ];
  const T* pbc[Sh::NQ];
  long long lbc[Sh::NQ];
  int rbc_row[Sh::NQ], vbc[Sh::NQ];
  float* sbc[Sh::NQ];
#pragma unroll
  for (int i = 0; i < Sh::NQ; ++i) {
    const int id = tid + i * Sh::NT, c = id % (S / 4) * 4, r = id / (S / 4) % TT;
    const bool second = id >= TT * S / 4;
    pbc[i] = second ? reinterpret_cast<const T*>(p.C.p) + at.n * p.C.sn + at.g * p.C.sg + c
                    : reinterpret_cast<const T*>(p.B.p) + at.n * p.B.sn + at.g * p.B.sg + c;
    lbc[i] = second ? p.C.sl : p.B.sl;
    vbc[i] = second ? p.C.vec : p.B.vec;
    rbc_row[i] = id < Sh::QUADS ? r : p.L;
    sbc[i] = &sm.bc[second][r][c];
  }
  auto fetch = [&](int t0) {
    const int t = t0 + row, v = t < t_end ? valid : 0;
    ru.fetch(pu + t * p.u.sl, p.u.vec, v);
    rd.fetch(pd + t * p.delta.sl, p.delta.vec, v);
    ry.fetch(py + t * p.dy.sl, p.dy.vec, v);
    if (gate) rz.fetch(pz + t * p.z.sl, p.z.vec, v);
#pragma unroll
    for (int i = 0; i < Sh::NQ; ++i)
      if (t0 + rbc_row[i] < t_end) rbc[i].fetch(pbc[i] + (t0 + rbc_row[i]) * lbc[i], vbc[i], 4);
  };

  u64 A2[NP], gc[NP], dA[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) A2[i] = gc[i] = dA[i] = 0ull;
  const long long states = (long long)p.N * p.D * S, own = ((long long)at.n * p.D + d) * S;
  const int nck = (p.L + KT - 1) / KT;
  if (mine) {
    load_states<Sh>(p.A + (long long)d * S, q, A2);
    const u64 l2 = dup2(LOG2E);
#pragma unroll
    for (int i = 0; i < NP; ++i) A2[i] = mul2(A2[i], l2);
    if (p.dhT) load_states<Sh>(p.dhT + own, q, gc);
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

  const int t_last = t_first + (t_end - t_first - 1) / TT * TT;
  if (t_first < t_end) fetch(t_last);
  for (int t0 = t_last; t0 >= t_first; t0 -= TT) {
    const int steps = min(TT, t_end - t0);
    float4 u4, z4, r4, y4;
    if (loader) {
      const int t = t0 + row, v = t < t_end ? valid : 0;
      u4 = ru.get(pu + t * p.u.sl, p.u.vec, v);
      r4 = rd.get(pd + t * p.delta.sl, p.delta.vec, v);
      y4 = ry.get(py + t * p.dy.sl, p.dy.vec, v);
      z4 = make_float4(0.f, 0.f, 0.f, 0.f);
      if (gate) z4 = rz.get(pz + t * p.z.sl, p.z.vec, v);
      const float us[4] = {u4.x, u4.y, u4.z, u4.w}, zs[4] = {z4.x, z4.y, z4.z, z4.w};
      float rs[4] = {r4.x, r4.y, r4.z, r4.w}, gs[4] = {y4.x, y4.y, y4.z, y4.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        rs[i] += bias[i];
        float dl = p.softplus ? softplus(rs[i]) : rs[i];
        dl = i < v ? dl : 0.f;
        const float du = dl * us[i], g = gate ? gs[i] * zs[i] * sigmoid(zs[i]) : gs[i];
        sm.dd[row][col + i] = make_float4(dl, dl, du, du);
        sm.gy[row][col + i] = make_float2(g, g);
      }
      r4 = make_float4(rs[0], rs[1], rs[2], rs[3]);
    }
#pragma unroll
    for (int i = 0; i < Sh::NQ; ++i)
      if (t0 + rbc_row[i] < t_end)
        *reinterpret_cast<float4*>(sbc[i]) = rbc[i].get(pbc[i] + (t0 + rbc_row[i]) * lbc[i], vbc[i], 4);
    const unsigned resets = reset_bits(p, at.n, t0, steps);
    __syncthreads();
    if (t0 - TT >= t_first) fetch(t0 - TT);

    auto half = [&](auto whole, int s0) {       // eight steps from s0 of the tile
      constexpr bool WHOLE = decltype(whole)::value;
      u64 a[KT][NP], ah[KT][NP], h[NP];
#pragma unroll
      for (int i = 0; i < NP; ++i) h[i] = 0ull;
      if (mine) load_states<Sh>(p.ckpt + (((long long)at.n * nck + (t0 + s0) / KT) * p.D + d) * S, q, h);
      float yv[Sh::LN], dc[8];
#pragma unroll
      for (int k = 0; k < KT; ++k) {
        const int t = s0 + k;
        float* dck = dc + k % GS * Sh::ST;
        yv[k % Sh::LN] = 0.f;
#pragma unroll
        for (int i = 0; i < Sh::ST; ++i) dck[i] = 0.f;
        if (WHOLE || t < steps) {
          const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(&sm.dd[t][chl]);
          const u64 g2 = *reinterpret_cast<const u64*>(&sm.gy[t][chl]);
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
#pragma unroll
          for (int i = 0; i < KEPT; ++i) sm.part[warp][k - (GS - 1) + kept_step][1][kept_state + i] = dc[i];
        }
        if (gate && k % Sh::LN == Sh::LN - 1) {
          const float y = steps_to_lanes<Sh::LN>(yv, q);
          sm.yp[s0 + k - (Sh::LN - 1) + q][chl] = y;
        }
      }
      float gbv[Sh::LN], sav[Sh::LN], db[8];
#pragma unroll
      for (int k = KT - 1; k >= 0; --k) {
        const int t = s0 + k;
        float* dbk = db + k % GS * Sh::ST;
        gbv[k % Sh::LN] = sav[k % Sh::LN] = 0.f;
#pragma unroll
        for (int i = 0; i < Sh::ST; ++i) dbk[i] = 0.f;
        if (WHOLE || t < steps) {
          const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(&sm.dd[t][chl]);
          const u64 g2 = *reinterpret_cast<const u64*>(&sm.gy[t][chl]);
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
#pragma unroll
          for (int i = 0; i < KEPT; ++i) sm.part[warp][k + kept_step][0][kept_state + i] = db[i];
        }
        if (k % Sh::LN == 0) {
          const float g = steps_to_lanes<Sh::LN>(gbv, q), s = steps_to_lanes<Sh::LN>(sav, q);
          sm.gb[s0 + k + q][chl] = g;
          sm.sa[s0 + k + q][chl] = s * 0.6931471805599453f;      // (A2 has log2(e) in it)
        }
      }
    };
    for (int s0 = TT - KT; s0 >= 0; s0 -= KT) {
      if (s0 >= steps) continue;
      if (steps == TT && resets == 0u) half(std::true_type(), s0);
      else half(std::false_type(), s0);
      __syncthreads();
      // this CTA's share of dB and dC of the eight steps
      for (int e = tid; e < KT * 2 * S; e += Sh::NT) {
        const int s = e % S, arr = e / S % 2, k = e / (2 * S), t = t0 + s0 + k;
        float v = sm.part[0][k][arr][s];
#pragma unroll
        for (int w = 1; w < BwdSmem<S>::WARPS; ++w) v += sm.part[w][k][arr][s];
        const int per = ((p.D / p.G) + CH - 1) / CH, blk = (int)(blockIdx.x % (unsigned)per);
        if (t < t_end) p.part_bc[((((long long)blk * 2 + arr) * p.N + at.n) * p.L + t) * p.G * S + at.g * S + s] = v;
      }
      __syncthreads();
    }
    if (loader && t0 + row < t_end && valid > 0) {
      const int t = t0 + row;
      const float4 gb4 = *reinterpret_cast<const float4*>(&sm.gb[row][col]), sa4 = *reinterpret_cast<const float4*>(&sm.sa[row][col]);
      float4 yp4 = make_float4(0.f, 0.f, 0.f, 0.f);
      if (gate) yp4 = *reinterpret_cast<const float4*>(&sm.yp[row][col]);
      const float us[4] = {u4.x, u4.y, u4.z, u4.w}, rs[4] = {r4.x, r4.y, r4.z, r4.w}, zs[4] = {z4.x, z4.y, z4.z, z4.w};
      const float os[4] = {y4.x, y4.y, y4.z, y4.w}, gb[4] = {gb4.x, gb4.y, gb4.z, gb4.w}, sa[4] = {sa4.x, sa4.y, sa4.z, sa4.w};
      const float yp[4] = {yp4.x, yp4.y, yp4.z, yp4.w};
      float ru4[4], rd4[4], rz4[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float g = sm.gy[row][col + i].x, dl = sm.dd[row][col + i].x;
        ru4[i] = fmaf(g, skip[i], dl * gb[i]);
        float dr = fmaf(us[i], gb[i], sa[i]);
        if (p.softplus) dr *= sigmoid(rs[i]);
        rd4[i] = dr;
        const float sg = sigmoid(zs[i]);
        rz4[i] = os[i] * fmaf(skip[i], us[i], yp[i]) * sg * fmaf(zs[i], 1.f - sg, 1.f);
        if (i < valid) {
          sum_skip[i] = fmaf(g, us[i], sum_skip[i]);
          sum_bias[i] += dr;
        }
      }
      put4(ou + t * p.du.sl, p.du.vec, valid, make_float4(ru4[0], ru4[1], ru4[2], ru4[3]));
      put4(od + t * p.ddelta.sl, p.ddelta.vec, valid, make_float4(rd4[0], rd4[1], rd4[2], rd4[3]));
      if (gate) put4(oz + t * p.dz.sl, p.dz.vec, valid, make_float4(rz4[0], rz4[1], rz4[2], rz4[3]));
    }
    __syncthreads();
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
    for (int r = 0; r < TT; ++r) v += which ? sm.sa[r][c] : sm.gb[r][c];
    if (c < at.left) p.part_v[(slot * 2 + which) * p.D + at.ch0 + c] = v;
  }
}

// What a piece of the time axis adds to the gradient of the state in front of it (from zero behind it), and the product of its
// decays, for pieces 1 .. nseg - 1.
template <typename T, int S>
__global__ void __launch_bounds__(Shape<S>::NT) scan_bwd_carry_kernel(const ScanParams p) {
  using Sh = Shape<S>;
  constexpr int TT = SCAN_TILE, CH = SCAN_CH, NP = Sh::ST / 2, NQ = (Sh::QUADS / 2 + Sh::NT - 1) / Sh::NT;
  __shared__ __align__(16) float4 dg[TT][CH];        // Delta twice, dy' twice
  __shared__ __align__(16) float cs[TT][S];
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, q = lane % Sh::LN, chl = warp * Sh::LC + lane / Sh::LN;
  const Place at(p, blockIdx.x);
  const int seg = blockIdx.y + 1, t_first = seg * p.seglen, t_end = min(p.L, t_first + p.seglen);
  const bool mine = chl < at.left;
  const int d = at.ch0 + chl;
  const bool loader = tid < TT * CH / 4;
  const int row = tid / (CH / 4), col = tid % (CH / 4) * 4, valid = loader ? min(4, at.left - col) : 0;
  auto rows = [&](const ScanRows& w) { return reinterpret_cast<const T*>(w.p) + at.n * w.sn + at.ch0 + col; };
  const T *pd = rows(p.delta), *pz = rows(p.z), *py = rows(p.dy);
  const bool gate = p.z.p != nullptr;
  float bias[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) bias[i] = i < valid && p.bias ? p.bias[at.ch0 + col + i] : 0.f;
  const T* pc = reinterpret_cast<const T*>(p.C.p) + at.n * p.C.sn + at.g * p.C.sg;
  Quad<T> rd, rz, ry, rc[NQ];
  auto fetch = [&](int t0) {
    const int t = t0 + row, v = t < t_end ? valid : 0;
    rd.fetch(pd + t * p.delta.sl, p.delta.vec, v);
    ry.fetch(py + t * p.dy.sl, p.dy.vec, v);
    if (gate) rz.fetch(pz + t * p.z.sl, p.z.vec, v);
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      const int id = tid + i * Sh::NT, r = id / (S / 4);
      if (r < TT && t0 + r < t_end) rc[i].fetch(pc + (t0 + r) * p.C.sl + id % (S / 4) * 4, p.C.vec, 4);
    }
  };
  u64 A2[NP], gc[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) A2[i] = gc[i] = 0ull;
  if (mine) {
    load_states<Sh>(p.A + (long long)d * S, q, A2);
#pragma unroll
    for (int i = 0; i < NP; ++i) A2[i] = mul2(A2[i], dup2(LOG2E));
  }
  float sum_d = 0.f;
  bool cut = false;
  const int t_last = t_first + (t_end - t_first - 1) / TT * TT;
  if (t_first < t_end) fetch(t_last);
  for (int t0 = t_last; t0 >= t_first; t0 -= TT) {
    const int steps = min(TT, t_end - t0);
    if (loader) {
      const int t = t0 + row, v = t < t_end ? valid : 0;
      const float4 r4 = rd.get(pd + t * p.delta.sl, p.delta.vec, v), y4 = ry.get(py + t * p.dy.sl, p.dy.vec, v);
      float4 z4 = make_float4(0.f, 0.f, 0.f, 0.f);
      if (gate) z4 = rz.get(pz + t * p.z.sl, p.z.vec, v);
      const float rs[4] = {r4.x, r4.y, r4.z, r4.w}, gs[4] = {y4.x, y4.y, y4.z, y4.w}, zs[4] = {z4.x, z4.y, z4.z, z4.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = rs[i] + bias[i], g = gate ? gs[i] * zs[i] * sigmoid(zs[i]) : gs[i];
        float dl = p.softplus ? softplus(x) : x;
        dl = i < v ? dl : 0.f;
        dg[row][col + i] = make_float4(dl, dl, g, g);
      }
    }
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      const int id = tid + i * Sh::NT, r = id / (S / 4), c = id % (S / 4) * 4;
      if (r < TT && t0 + r < t_end) *reinterpret_cast<float4*>(&cs[r][c]) = rc[i].get(pc + (t0 + r) * p.C.sl + c, p.C.vec, 4);
    }
    const unsigned resets = reset_bits(p, at.n, t0, steps);
    __syncthreads();
    if (t0 - TT >= t_first) fetch(t0 - TT);
#pragma unroll 4
    for (int t = steps - 1; t >= 0; --t) {
      const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(&dg[t][chl]);
      u64 c2[NP];
      load_states<Sh>(&cs[t][0], q, c2);
      const bool fresh = resets >> t & 1u;
      cut |= fresh;
      sum_d += dg[t][chl].x;
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const u64 g = fma2<true>(c2[i], x.y, gc[i]), a = exp2_pair(mul2(x.x, A2[i]));
        gc[i] = fresh ? 0ull : mul2(a, g);
      }
    }
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
    put4(dst, o.vec, 4, v);
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

template <typename T, int S>
cudaError_t launch(const ScanParams& p, cudaStream_t s) {
  const unsigned grid = (unsigned)(blocks_of<S>(p) * p.N);
  constexpr int smem = sizeof(BwdSmem<S>);
  static unsigned long long raised = 0;      // devices whose limit is raised
  if (smem > 48 * 1024) {
    int dev = 0;
    if (const cudaError_t e = cudaGetDevice(&dev); e != cudaSuccess) return e;
    const unsigned long long bit = 1ull << (dev & 63);
    if (!(__atomic_load_n(&raised, __ATOMIC_ACQUIRE) & bit)) {
      const cudaError_t e = cudaFuncSetAttribute(scan_bwd_kernel<T, S>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
      if (e != cudaSuccess) return e;
      __atomic_fetch_or(&raised, bit, __ATOMIC_RELEASE);
    }
  }
  if (p.nseg > 1) {
    scan_bwd_carry_kernel<T, S><<<dim3(grid, p.nseg - 1), Shape<S>::NT, 0, s>>>(p);
    if (const cudaError_t e = cudaGetLastError(); e != cudaSuccess) return e;
  }
  scan_bwd_kernel<T, S><<<dim3(grid, p.nseg), Shape<S>::NT, smem, s>>>(p);
  if (const cudaError_t e = cudaGetLastError(); e != cudaSuccess) return e;
  const long long quads = 2ll * p.N * p.L * p.G * S / 4, bc_blocks = (quads + 255) / 256;
  const long long rest = ((long long)p.D * S + 2 * p.D + 255) / 256;
  scan_sums_kernel<T><<<(unsigned)(bc_blocks + rest), 256, 0, s>>>(p, (int)bc_blocks);
  return cudaGetLastError();
}
template <typename T>
cudaError_t by_states(const ScanParams& p, cudaStream_t s) {
  switch (p.S) {
    case 8: return launch<T, 8>(p, s);
    case 16: return launch<T, 16>(p, s);
    case 32: return launch<T, 32>(p, s);
    default: return launch<T, 64>(p, s);
  }
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
  return p.bf16 ? by_states<__nv_bfloat16>(p, s) : by_states<float>(p, s);
}

}  // namespace srwm
