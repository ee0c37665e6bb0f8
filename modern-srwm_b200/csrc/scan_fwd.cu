// Selective state-space scan, forward: sequences (scan_fwd_kernel) and single tokens (scan_step_kernel).
#include <type_traits>

#include "chain.h"
#include "device.h"
#include "scan.cuh"

namespace srwm {
namespace {
using namespace scan;

// CARRY: only what a piece of the time axis makes of the state (its end from zero, and the product of its decays), for the
// pieces behind it; one CTA per 32 channels and piece.
template <typename T, int S, bool CARRY>
__global__ void __launch_bounds__(Shape<S>::NT) scan_fwd_kernel(const ScanParams p) {
  using Sh = Shape<S>;
  constexpr int TT = SCAN_TILE, CH = SCAN_CH, PAD = CH + 8;
  __shared__ __align__(16) float4 dd[TT][CH];        // Delta twice, Delta u twice
  __shared__ __align__(16) float bc[2][TT][S];
  __shared__ __align__(16) float ys[TT][PAD];
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, q = lane % Sh::LN, chl = warp * Sh::LC + lane / Sh::LN;
  const Place at(p, blockIdx.x);
  const int seg = blockIdx.y, t_first = seg * p.seglen, t_end = min(p.L, t_first + p.seglen);
  const bool mine = chl < at.left;
  const int d = at.ch0 + chl;

  // the piece of the tile that this thread loads, and stores again
  const bool loader = tid < TT * CH / 4;
  const int row = tid / (CH / 4), col = tid % (CH / 4) * 4, valid = loader ? min(4, at.left - col) : 0;
  const T* pu = reinterpret_cast<const T*>(p.u.p) + at.n * p.u.sn + at.ch0 + col;
  const T* pd = reinterpret_cast<const T*>(p.delta.p) + at.n * p.delta.sn + at.ch0 + col;
  const T* pz = reinterpret_cast<const T*>(p.z.p) + at.n * p.z.sn + at.ch0 + col;
  T* py = reinterpret_cast<T*>(p.y.p) + at.n * p.y.sn + at.ch0 + col;
  const bool gate = !CARRY && p.z.p != nullptr;
  float bias[4], skip[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    bias[i] = i < valid && p.bias ? p.bias[at.ch0 + col + i] : 0.f;
    skip[i] = !CARRY && i < valid && p.skip ? p.skip[at.ch0 + col + i] : 0.f;
  }
  Quad<T> ru, rd, rz, rbc[Sh::NQ];

  // the pieces of B and C that it loads
  const T* pbc[Sh::NQ];
  long long lbc[Sh::NQ];
  int rbc_row[Sh::NQ], vbc[Sh::NQ];
  float* sbc[Sh::NQ];
#pragma unroll
  for (int i = 0; i < Sh::NQ; ++i) {
    const int id = tid + i * Sh::NT, c = id % (S / 4) * 4, r = id / (S / 4) % TT;
    const bool second = !CARRY && id >= TT * S / 4;
    pbc[i] = second ? reinterpret_cast<const T*>(p.C.p) + at.n * p.C.sn + at.g * p.C.sg + c
                    : reinterpret_cast<const T*>(p.B.p) + at.n * p.B.sn + at.g * p.B.sg + c;
    lbc[i] = second ? p.C.sl : p.B.sl;
    vbc[i] = second ? p.C.vec : p.B.vec;
    rbc_row[i] = id < (CARRY ? Sh::QUADS / 2 : Sh::QUADS) ? r : p.L;      // (a row behind every piece's end)
    sbc[i] = &bc[second][r][c];
  }
  auto fetch = [&](int t0) {
    const int t = t0 + row, v = t < t_end ? valid : 0;
    ru.fetch(pu + t * p.u.sl, p.u.vec, v);
    rd.fetch(pd + t * p.delta.sl, p.delta.vec, v);
    if (gate) rz.fetch(pz + t * p.z.sl, p.z.vec, v);
#pragma unroll
    for (int i = 0; i < Sh::NQ; ++i) {
      if (t0 + rbc_row[i] < t_end) rbc[i].fetch(pbc[i] + (t0 + rbc_row[i]) * lbc[i], vbc[i], 4);
    }
  };

  u64 h[Sh::ST / 2], A2[Sh::ST / 2];
#pragma unroll
  for (int i = 0; i < Sh::ST / 2; ++i) h[i] = A2[i] = 0ull;
  if (t_first < t_end) fetch(t_first);
  const long long states = (long long)p.N * p.D * S, own = ((long long)at.n * p.D + d) * S;
  if (mine) {
    load_states<Sh>(p.A + (long long)d * S, q, A2);
    if (CARRY || p.nseg == 1) {
      if (seg == 0 && p.h0) load_states<Sh>(p.h0 + own, q, h);
      if (CARRY && seg == 0) store_states<Sh>(p.carry + own, q, h);    // (hT may be h0's memory)
    } else {
      load_states<Sh>(p.carry + own, q, h);
      for (int i = 0; i < seg; ++i) {     // the pieces in front, in order
        u64 decay[Sh::ST / 2], end[Sh::ST / 2];
        load_states<Sh>(p.carry + (2 * i + 1) * states + own, q, end);
        load_states<Sh>(p.carry + (2 * i + 2) * states + own, q, decay);
#pragma unroll
        for (int k = 0; k < Sh::ST / 2; ++k) h[k] = fma2<true>(decay[k], h[k], end[k]);
      }
    }
    const u64 l2 = dup2(LOG2E);
#pragma unroll
    for (int i = 0; i < Sh::ST / 2; ++i) A2[i] = mul2(A2[i], l2);
  }
  if (CARRY) {
#pragma unroll
    for (int i = 0; i < Sh::ST / 2; ++i) h[i] = 0ull;
  }
  float sum_d = 0.f;
  bool cut = false;      // CARRY: an episode begins inside the piece
  const int nck = (p.L + SCAN_CKPT - 1) / SCAN_CKPT;

  for (int t0 = t_first; t0 < t_end; t0 += TT) {
    const int steps = min(TT, t_end - t0);
    float4 u4, z4;
    if (loader) {
      const int t = t0 + row, v = t < t_end ? valid : 0;
      u4 = ru.get(pu + t * p.u.sl, p.u.vec, v);
      const float4 r4 = rd.get(pd + t * p.delta.sl, p.delta.vec, v);
      if (gate) z4 = rz.get(pz + t * p.z.sl, p.z.vec, v);
      const float us[4] = {u4.x, u4.y, u4.z, u4.w}, rs[4] = {r4.x, r4.y, r4.z, r4.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = rs[i] + bias[i];
        float dl = p.softplus ? softplus(x) : x;
        dl = i < v ? dl : 0.f;
        const float du = dl * us[i];
        dd[row][col + i] = make_float4(dl, dl, du, du);
      }
    }
#pragma unroll
    for (int i = 0; i < Sh::NQ; ++i) {
      if (t0 + rbc_row[i] < t_end)
        *reinterpret_cast<float4*>(sbc[i]) = rbc[i].get(pbc[i] + (t0 + rbc_row[i]) * lbc[i], vbc[i], 4);
    }
    const unsigned resets = reset_bits(p, at.n, t0, steps);
    __syncthreads();
    if (t0 + TT < t_end) fetch(t0 + TT);

    auto walk = [&](auto whole) {       // whole: sixteen steps of one episode
      constexpr bool WHOLE = decltype(whole)::value;
#pragma unroll
      for (int g4 = 0; g4 < TT; g4 += Sh::LN) {
        if (!WHOLE && g4 >= steps) break;
        float yv[Sh::LN];
#pragma unroll
        for (int k = 0; k < Sh::LN; ++k) {
          const int t = g4 + k;
          yv[k] = 0.f;
          if (!WHOLE && t >= steps) continue;
          if (!CARRY && t % SCAN_CKPT == 0 && p.ckpt && mine)
            store_states<Sh>(p.ckpt + (((long long)at.n * nck + (t0 + t) / SCAN_CKPT) * p.D + d) * S, q, h);
          const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(&dd[t][chl]);
          const bool fresh = !WHOLE && (resets >> t & 1u);
          if (fresh) {
#pragma unroll
            for (int i = 0; i < Sh::ST / 2; ++i) h[i] = 0ull;
            if (CARRY) cut = true;
          }
          if (CARRY) sum_d += dd[t][chl].x;
          u64 b2[Sh::ST / 2], c2[Sh::ST / 2];
          load_states<Sh>(&bc[0][t][0], q, b2);
          if (!CARRY) load_states<Sh>(&bc[1][t][0], q, c2);
          u64 acc = 0ull;
#pragma unroll
          for (int i = 0; i < Sh::ST / 2; ++i) {
            u64 a = exp2_pair(mul2(x.x, A2[i]));
            if (fresh) a = 0ull;
            h[i] = fma2<true>(a, h[i], mul2(x.y, b2[i]));
            if (!CARRY) acc = i == 0 ? mul2(h[i], c2[i]) : fma2<true>(h[i], c2[i], acc);
          }
          yv[k] = hsum2(acc);
        }
        if (!CARRY) {
          const float s = steps_to_lanes<Sh::LN>(yv, q);
          ys[g4 + q][chl] = s;
        }
      }
    };
    if (steps == TT && resets == 0u) walk(std::true_type());
    else walk(std::false_type());
    __syncthreads();
    if (!CARRY && loader && t0 + row < t_end && valid > 0) {
      float4 y4 = *reinterpret_cast<const float4*>(&ys[row][col]);
      y4.x = fmaf(skip[0], u4.x, y4.x); y4.y = fmaf(skip[1], u4.y, y4.y);
      y4.z = fmaf(skip[2], u4.z, y4.z); y4.w = fmaf(skip[3], u4.w, y4.w);
      if (gate) {
        y4.x *= z4.x * sigmoid(z4.x); y4.y *= z4.y * sigmoid(z4.y);
        y4.z *= z4.z * sigmoid(z4.z); y4.w *= z4.w * sigmoid(z4.w);
      }
      put4(py + (t0 + row) * p.y.sl, p.y.vec, valid, y4);
    }
  }
  if (!mine) return;
  if (CARRY) {
    u64 decay[Sh::ST / 2];
#pragma unroll
    for (int i = 0; i < Sh::ST / 2; ++i) decay[i] = cut ? 0ull : exp2_pair(mul2(dup2(sum_d), A2[i]));
    store_states<Sh>(p.carry + (2 * seg + 1) * states + own, q, h);
    store_states<Sh>(p.carry + (2 * seg + 2) * states + own, q, decay);
  } else if (seg == p.nseg - 1 && p.hT) {
    store_states<Sh>(p.hT + own, q, h);
  }
}

// A few steps, states in registers, everything else straight from memory: what an actor or a server does for each token.  Bound by the state's
// bytes, and by its launch where these are few.
template <typename T, int S>
__global__ void __launch_bounds__(Shape<S>::NT) scan_step_kernel(const ScanParams p) {
  using Sh = Shape<S>;
  chained();
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, q = lane % Sh::LN, chl = warp * Sh::LC + lane / Sh::LN;
  const Place at(p, blockIdx.x);
  const bool mine = chl < at.left;
  const int d = mine ? at.ch0 + chl : at.ch0;
  const long long own = ((long long)at.n * p.D + d) * S;
  u64 h[Sh::ST / 2], A2[Sh::ST / 2], b2[Sh::ST / 2], c2[Sh::ST / 2];
#pragma unroll
  for (int i = 0; i < Sh::ST / 2; ++i) h[i] = 0ull;
  if (p.h0) load_states<Sh>(p.h0 + own, q, h);
  load_states<Sh>(p.A + (long long)d * S, q, A2);
  const u64 l2 = dup2(LOG2E);
#pragma unroll
  for (int i = 0; i < Sh::ST / 2; ++i) A2[i] = mul2(A2[i], l2);
  const float bias = p.bias ? p.bias[d] : 0.f, skip = p.skip ? p.skip[d] : 0.f;
  for (int t = 0; t < p.L; ++t) {
    const float u = to_float(reinterpret_cast<const T*>(p.u.p)[at.n * p.u.sn + t * p.u.sl + d]);
    const float x = to_float(reinterpret_cast<const T*>(p.delta.p)[at.n * p.delta.sn + t * p.delta.sl + d]) + bias;
    const float z = p.z.p ? to_float(reinterpret_cast<const T*>(p.z.p)[at.n * p.z.sn + t * p.z.sl + d]) : 0.f;
    const bool fresh = p.done && p.done[at.n * p.done_n + t * p.done_l] != 0;
    auto row = [&](const ScanRows& w, u64 (&v)[Sh::ST / 2]) {
      const T* r = reinterpret_cast<const T*>(w.p) + at.n * w.sn + at.g * w.sg + t * w.sl;
#pragma unroll
      for (int i = 0; i < (Sh::ST + 3) / 4; ++i) {
        const T* f = r + Sh::first(q, i);
        if (Sh::ST >= 4 && w.vec) {
          const float4 t4 = widen(*reinterpret_cast<const typename Raw<T>::type*>(f));
          v[2 * i] = pack2(t4.x, t4.y);
          if constexpr (Sh::ST >= 4) v[2 * i + 1] = pack2(t4.z, t4.w);
        } else {
          v[2 * i] = pack2(to_float(f[0]), to_float(f[1]));
          if constexpr (Sh::ST >= 4) v[2 * i + 1] = pack2(to_float(f[2]), to_float(f[3]));
        }
      }
    };
    row(p.B, b2);
    row(p.C, c2);
    const float dl = p.softplus ? softplus(x) : x;
    const u64 d2 = dup2(dl), x2 = dup2(dl * u);
    u64 acc = 0ull;
#pragma unroll
    for (int i = 0; i < Sh::ST / 2; ++i) {
      u64 a = exp2_pair(mul2(d2, A2[i]));
      if (fresh) a = h[i] = 0ull;
      h[i] = fma2<true>(a, h[i], mul2(x2, b2[i]));
      acc = fma2<true>(h[i], c2[i], acc);
    }
    float y = hsum2(acc);
#pragma unroll
    for (int w = 1; w < Sh::LN; w *= 2) y += __shfl_xor_sync(0xffffffffu, y, w);
    y = fmaf(skip, u, y);
    if (p.z.p) y *= z * sigmoid(z);
    if (mine && q == 0) narrow(y, reinterpret_cast<T*>(p.y.p) + at.n * p.y.sn + t * p.y.sl + d);
  }
  if (mine && p.hT) store_states<Sh>(p.hT + own, q, h);
}

template <typename T, int S>
cudaError_t launch(const ScanParams& p, cudaStream_t s) {
  const unsigned grid = (unsigned)(blocks_of<S>(p) * p.N);
  if (p.L <= SCAN_STEPS_DIRECT && !p.ckpt) return launch_behind(scan_step_kernel<T, S>, p, dim3(grid), Shape<S>::NT, 0, s);
  if (p.nseg > 1) {
    scan_fwd_kernel<T, S, true><<<dim3(grid, p.nseg - 1), Shape<S>::NT, 0, s>>>(p);
    if (const cudaError_t e = cudaGetLastError(); e != cudaSuccess) return e;
  }
  scan_fwd_kernel<T, S, false><<<dim3(grid, p.nseg), Shape<S>::NT, 0, s>>>(p);
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

// One piece where the channels alone give every scheduler a warp; otherwise enough pieces for two, of 64 steps at least (a piece's
// exponentials are formed twice).
int scan_segments(int N, int L, int D, int sms) {
  const long long ctas = (long long)N * ((D + SCAN_CH - 1) / SCAN_CH);
  if (ctas >= sms || L < 128) return 1;
  long long n = (2 * sms + ctas - 1) / ctas;
  if (n > L / 64) n = L / 64;
  if (n > 64) n = 64;
  return n < 3 ? 1 : (int)n;
}
long long scan_fwd_scratch(const ScanParams& p) {
  return p.nseg > 1 ? (2ll * p.nseg - 1) * p.N * p.D * p.S : 0;
}
cudaError_t scan_forward(const ScanParams& p, cudaStream_t s) {
  return p.bf16 ? by_states<__nv_bfloat16>(p, s) : by_states<float>(p, s);
}

}  // namespace srwm
