// Selective state-space scan, forward: sequences (scan_fwd_kernel) and single tokens (scan_step_kernel).
#include <type_traits>

#include "chain.h"
#include "device.h"
#include "scan.cuh"

namespace srwm {
namespace {
using namespace scan;

// CARRY: only what a piece of the time axis makes of the state (its end from zero, and the product of its decays), for the
// pieces behind it; one CTA per 32 channels and piece.  A tile is staged, and the one before it written, while the tile between is walked: one
// barrier a tile.
template <typename T, int S, bool VEC, bool CARRY>
__global__ void __launch_bounds__(Shape<S>::NT) scan_fwd_kernel(const ScanParams p) {
  using Sh = Shape<S>;
  constexpr int TT = SCAN_TILE, CH = SCAN_CH, PAD = CH + 8, NP = Sh::ST / 2;
  constexpr int NQ = CARRY ? (Sh::QUADS / 2 + Sh::NT - 1) / Sh::NT : Sh::NQ;
  __shared__ __align__(16) float4 dd[2][TT][CH];     // Delta twice, Delta u twice
  __shared__ __align__(16) float bc[2][CARRY ? 1 : 2][TT][S];
  __shared__ __align__(16) float ys[CARRY ? 1 : 2][TT][PAD];
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, q = lane % Sh::LN, chl = warp * Sh::LC + lane / Sh::LN;
  const Place at(p, blockIdx.x);
  const int seg = blockIdx.y, t_first = seg * p.seglen, t_end = min(p.L, t_first + p.seglen);
  const bool mine = chl < at.left;
  const int d = at.ch0 + chl, here = swizzled(chl);

  // the piece of a tile that this thread loads, and stores again
  const bool loader = tid < TT * CH / 4;
  const int row = tid / (CH / 4), col = tid % (CH / 4) * 4, valid = loader ? max(0, min(4, at.left - col)) : 0;
  const T* pu = reinterpret_cast<const T*>(p.u.p) + at.n * p.u.sn + (t_first + row) * p.u.sl + at.ch0 + col;
  const T* pd = reinterpret_cast<const T*>(p.delta.p) + at.n * p.delta.sn + (t_first + row) * p.delta.sl + at.ch0 + col;
  const T* pz = reinterpret_cast<const T*>(p.z.p) + at.n * p.z.sn + (t_first + row) * p.z.sl + at.ch0 + col;
  T* py = reinterpret_cast<T*>(p.y.p) + at.n * p.y.sn + (t_first + row) * p.y.sl + at.ch0 + col;
  const bool gate = !CARRY && p.z.p != nullptr;
  float bias[4], skip[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    bias[i] = i < valid && p.bias ? p.bias[at.ch0 + col + i] : 0.f;
    skip[i] = !CARRY && i < valid && p.skip ? p.skip[at.ch0 + col + i] : 0.f;
  }
  // the pieces of B and C that it loads
  const T* pbc[NQ];
  long long lbc[NQ];
  int rbc[NQ];
#pragma unroll
  for (int i = 0; i < NQ; ++i) {
    const int id = tid + i * Sh::NT, c = id % (S / 4) * 4, r = id / (S / 4) % TT;
    const bool second = !CARRY && id >= TT * S / 4;
    lbc[i] = (second ? p.C.sl : p.B.sl) * TT;
    pbc[i] = second ? reinterpret_cast<const T*>(p.C.p) + at.n * p.C.sn + at.g * p.C.sg + (t_first + r) * p.C.sl + c
                    : reinterpret_cast<const T*>(p.B.p) + at.n * p.B.sn + at.g * p.B.sg + (t_first + r) * p.B.sl + c;
    rbc[i] = id < (CARRY ? Sh::QUADS / 2 : Sh::QUADS) ? r : p.L;      // (a row behind every piece's end)
  }
  // three tiles: being fetched, staged for the next walk (u and z stay for its result), walked before
  Quad<T, VEC> fu, fd, fz, fbc[NQ], u1, z1, u0, z0;
  auto fetch = [&](int t0) {      // tiles are asked for in order
    const int v = t0 + row < t_end ? valid : 0;
    fu.fetch(pu, v);
    fd.fetch(pd, v);
    if (gate) fz.fetch(pz, v);
    pu += TT * p.u.sl; pd += TT * p.delta.sl; pz += TT * p.z.sl;
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      fbc[i].fetch(pbc[i], t0 + rbc[i] < t_end ? 4 : 0);
      pbc[i] += lbc[i];
    }
  };
  auto stage = [&](int buf) {
    u0 = u1; z0 = z1;
    u1 = fu; z1 = fz;
    if (loader) {
      const float4 u4 = fu.get(), r4 = fd.get();
      u64 lo = add2(pack2(r4.x, r4.y), pack2(bias[0], bias[1])), hi = add2(pack2(r4.z, r4.w), pack2(bias[2], bias[3]));
      if (p.softplus) {
        lo = softplus2(lo);
        hi = softplus2(hi);
      }
      const u64 xlo = mul2(lo, pack2(u4.x, u4.y)), xhi = mul2(hi, pack2(u4.z, u4.w));
      float dl[4], du[4];
      unpack2(lo, dl[0], dl[1]); unpack2(hi, dl[2], dl[3]);
      unpack2(xlo, du[0], du[1]); unpack2(xhi, du[2], du[3]);
#pragma unroll
      for (int i = 0; i < 4; ++i) dd[buf][row][swizzled(col + i)] = make_float4(dl[i], dl[i], du[i], du[i]);
    }
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      const int id = tid + i * Sh::NT;
      if (id < (CARRY ? Sh::QUADS / 2 : Sh::QUADS)) *reinterpret_cast<float4*>(&bc[buf][0][0][0] + id * 4) = fbc[i].get();
    }
  };
  auto finish = [&](int t0, int buf) {      // y of the tile walked before
    const int v = t0 + row < t_end ? valid : 0;
    if (v > 0) {
      const float4 s4 = *reinterpret_cast<const float4*>(&ys[buf][row][col]), u4 = u0.get();
      float4 y4 = make_float4(fmaf(skip[0], u4.x, s4.x), fmaf(skip[1], u4.y, s4.y), fmaf(skip[2], u4.z, s4.z), fmaf(skip[3], u4.w, s4.w));
      if (gate) {
        const float4 z4 = z0.get();
        y4.x *= z4.x * sigmoid(z4.x); y4.y *= z4.y * sigmoid(z4.y);
        y4.z *= z4.z * sigmoid(z4.z); y4.w *= z4.w * sigmoid(z4.w);
      }
      put4<VEC>(py, v, y4);
    }
    py += TT * p.y.sl;
  };

  u64 h[NP], A2[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) h[i] = A2[i] = 0ull;
  if (t_first < t_end) fetch(t_first);
  const long long states = (long long)p.N * p.D * S, own = ((long long)at.n * p.D + d) * S;
  if (mine) {
    load_states<Sh>(p.A + (long long)d * S, q, A2);
    if (CARRY || p.nseg == 1) {
      if (seg == 0 && p.h0) load_states<Sh>(p.h0 + own, q, h);
      if (CARRY && seg == 0) store_states<Sh>(p.carry + own, q, h);    // (hT may be h0's memory)
    } else {
      load_states<Sh>(p.carry + own, q, h);
#pragma unroll 4
      for (int i = 0; i < seg; ++i) {     // the pieces in front, in order
        u64 decay[NP], end[NP];
        load_states<Sh>(p.carry + (2 * i + 1) * states + own, q, end);
        load_states<Sh>(p.carry + (2 * i + 2) * states + own, q, decay);
#pragma unroll
        for (int k = 0; k < NP; ++k) h[k] = fma2<true>(decay[k], h[k], end[k]);
      }
    }
    const u64 l2 = dup2(LOG2E);
#pragma unroll
    for (int i = 0; i < NP; ++i) A2[i] = mul2(A2[i], l2);
  }
  if (CARRY) {
#pragma unroll
    for (int i = 0; i < NP; ++i) h[i] = 0ull;
  }
  float sum_d = 0.f;
  bool cut = false;      // CARRY: an episode begins inside the piece
  const int nck = (p.L + SCAN_CKPT - 1) / SCAN_CKPT;
  float* ck = p.ckpt + (((long long)at.n * nck + t_first / SCAN_CKPT) * p.D + d) * S;

  unsigned resets = 0u;
  if (t_first < t_end) {
    stage(0);
    resets = reset_bits(p, at.n, t_first, min(TT, t_end - t_first));
    if (t_first + TT < t_end) fetch(t_first + TT);
    __syncthreads();
  }
  for (int t0 = t_first, k0 = 0; t0 < t_end; t0 += TT, k0 ^= 1) {
    const int steps = min(TT, t_end - t0);
    const unsigned now = resets;
    if (t0 + TT < t_end) {
      stage(k0 ^ 1);
      resets = reset_bits(p, at.n, t0 + TT, min(TT, t_end - t0 - TT));
      if (t0 + 2 * TT < t_end) fetch(t0 + 2 * TT);
    } else {
      u0 = u1; z0 = z1;
    }
    const float4(*dk)[CH] = dd[k0];
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
          if (!CARRY && t % SCAN_CKPT == 0 && p.ckpt) {
            if (mine) store_states<Sh>(ck, q, h);
            ck += (long long)p.D * S;
          }
          const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(&dk[t][here]);
          const bool fresh = !WHOLE && (now >> t & 1u);
          if (fresh) {
#pragma unroll
            for (int i = 0; i < NP; ++i) h[i] = 0ull;
            if (CARRY) cut = true;
          }
          if (CARRY) sum_d += __uint_as_float((unsigned)x.x);
          u64 b2[NP], c2[NP];
          load_states<Sh>(&bc[k0][0][t][0], q, b2);
          if (!CARRY) load_states<Sh>(&bc[k0][CARRY ? 0 : 1][t][0], q, c2);
          u64 acc = 0ull;
#pragma unroll
          for (int i = 0; i < NP; ++i) {
            u64 a = exp2_pair(mul2(x.x, A2[i]));
            if (fresh) a = 0ull;
            h[i] = fma2<true>(a, h[i], mul2(x.y, b2[i]));
            if (!CARRY) acc = i == 0 ? mul2(h[i], c2[i]) : fma2<true>(h[i], c2[i], acc);
          }
          yv[k] = hsum2(acc);
        }
        if (!CARRY) {
          const float s = steps_to_lanes<Sh::LN>(yv, q);
          ys[CARRY ? 0 : k0][g4 + q][chl] = s;
        }
      }
    };
    if (steps == TT && now == 0u) walk(std::true_type());
    else walk(std::false_type());
    __syncthreads();
    if (!CARRY) finish(t0, k0);
  }
  if (!mine) return;
  if (CARRY) {
    u64 decay[NP];
#pragma unroll
    for (int i = 0; i < NP; ++i) decay[i] = cut ? 0ull : exp2_pair(mul2(dup2(sum_d), A2[i]));
    store_states<Sh>(p.carry + (2 * seg + 1) * states + own, q, h);
    store_states<Sh>(p.carry + (2 * seg + 2) * states + own, q, decay);
  } else if (seg == p.nseg - 1 && p.hT) {
    store_states<Sh>(p.hT + own, q, h);
  }
}

// A few steps, states in registers, everything else straight from memory: what an actor or a server does for each token.  Bound by the state's
// bytes, and by its launch where these are few.  NB: sequences of a thread, whose loads are all on their way before the first is used; more
// than one where there are enough of them (256 sequences x 2048 channels, S 16, bf16: 34 us with one, see the rule).
template <typename T, int S, bool VEC, int NB>
__global__ void __launch_bounds__(Shape<S>::NT) scan_step_kernel(const ScanParams p) {
  using Sh = Shape<S>;
  constexpr int NP = Sh::ST / 2;
  chained();
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, q = lane % Sh::LN, chl = warp * Sh::LC + lane / Sh::LN;
  const Place at(p, blockIdx.x);       // (its n: of the first of NB sequences, counted in such groups)
  const int n0 = at.n * NB;
  const bool mine = chl < at.left;
  const int d = mine ? at.ch0 + chl : at.ch0;
  u64 h[NB][NP], A2[NP];
#pragma unroll
  for (int b = 0; b < NB; ++b) {
#pragma unroll
    for (int i = 0; i < NP; ++i) h[b][i] = 0ull;
    if (p.h0 && n0 + b < p.N) load_states<Sh>(p.h0 + ((long long)(n0 + b) * p.D + d) * S, q, h[b]);
  }
  load_states<Sh>(p.A + (long long)d * S, q, A2);
  const float bias = p.bias ? p.bias[d] : 0.f, skip = p.skip ? p.skip[d] : 0.f;
  for (int t = 0; t < p.L; ++t) {
    float u[NB], x[NB], z[NB];
    bool fresh[NB];
    u64 b2[NB][NP], c2[NB][NP];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const int n = min(n0 + b, p.N - 1);
      u[b] = to_float(reinterpret_cast<const T*>(p.u.p)[n * p.u.sn + t * p.u.sl + d]);
      x[b] = to_float(reinterpret_cast<const T*>(p.delta.p)[n * p.delta.sn + t * p.delta.sl + d]);
      z[b] = p.z.p ? to_float(reinterpret_cast<const T*>(p.z.p)[n * p.z.sn + t * p.z.sl + d]) : 0.f;
      fresh[b] = p.done && p.done[n * p.done_n + t * p.done_l] != 0;
      auto row = [&](const ScanRows& w, u64 (&v)[NP]) {
        const T* r = reinterpret_cast<const T*>(w.p) + n * w.sn + at.g * w.sg + t * w.sl;
        if constexpr (Sh::ST >= 4) {
#pragma unroll
          for (int i = 0; i < Sh::ST / 4; ++i) {
            Quad<T, VEC> f;
            f.fetch(r + Sh::first(q, i), 4);
            const float4 t4 = f.get();
            v[2 * i] = pack2(t4.x, t4.y);
            v[2 * i + 1] = pack2(t4.z, t4.w);
          }
        } else {
          v[0] = pack2(to_float(r[Sh::first(q, 0)]), to_float(r[Sh::first(q, 0) + 1]));
        }
      };
      row(p.B, b2[b]);
      row(p.C, c2[b]);
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const float dl = p.softplus ? softplus(x[b] + bias) : x[b] + bias;
      const u64 d2 = dup2(dl * LOG2E), x2 = dup2(dl * u[b]);
      u64 acc = 0ull;
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        u64 a = exp2_pair(mul2(d2, A2[i]));
        if (fresh[b]) a = h[b][i] = 0ull;
        h[b][i] = fma2<true>(a, h[b][i], mul2(x2, b2[b][i]));
        acc = fma2<true>(h[b][i], c2[b][i], acc);
      }
      float y = hsum2(acc);
#pragma unroll
      for (int w = 1; w < Sh::LN; w *= 2) y += __shfl_xor_sync(0xffffffffu, y, w);
      y = fmaf(skip, u[b], y);
      if (p.z.p) y *= z[b] * sigmoid(z[b]);
      if (mine && q == 0 && n0 + b < p.N) narrow(y, reinterpret_cast<T*>(p.y.p) + (n0 + b) * p.y.sn + t * p.y.sl + d);
    }
  }
  if (!mine || !p.hT) return;
#pragma unroll
  for (int b = 0; b < NB; ++b)
    if (n0 + b < p.N) store_states<Sh>(p.hT + ((long long)(n0 + b) * p.D + d) * S, q, h[b]);
}

template <typename T, int S, bool VEC>
cudaError_t launch(const ScanParams& p, cudaStream_t s) {
  const unsigned grid = (unsigned)(blocks_of(p) * p.N);
  if (p.L <= SCAN_STEPS_DIRECT && !p.ckpt) {
    constexpr int NB = S <= 16 ? 4 : 2;
    if (grid < 32u * common_sms()) return launch_behind(scan_step_kernel<T, S, VEC, 1>, p, dim3(grid), Shape<S>::NT, 0, s);
    return launch_behind(scan_step_kernel<T, S, VEC, NB>, p, dim3((unsigned)(blocks_of(p) * ((p.N + NB - 1) / NB))), Shape<S>::NT, 0, s);
  }
  if (p.nseg > 1) {
    scan_fwd_kernel<T, S, VEC, true><<<dim3(grid, p.nseg - 1), Shape<S>::NT, 0, s>>>(p);
    if (const cudaError_t e = cudaGetLastError(); e != cudaSuccess) return e;
  }
  scan_fwd_kernel<T, S, VEC, false><<<dim3(grid, p.nseg), Shape<S>::NT, 0, s>>>(p);
  return cudaGetLastError();
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
  return by_shape(p, [&](auto t, auto states, auto vec) { return launch<decltype(t), decltype(states)::value, decltype(vec)::value>(p, s); });
}

}  // namespace srwm
