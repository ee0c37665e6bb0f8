// Selective state-space scan, forward: sequences (scan_fwd_kernel) and single tokens (scan_step_kernel).
#include <type_traits>

#include "chain.h"
#include "device.h"
#include "scan.cuh"

namespace srwm {
namespace {
using namespace scan;

template <typename Sh, bool CARRY>
struct FwdSmem {
  float2 dd[2][Sh::TT][Sh::CH];                                            // Delta, Delta u
  float bc[2][CARRY ? 1 : 2][Sh::TT][Sh::S];
  float ys[CARRY ? 1 : 2][CARRY ? 1 : Sh::TT][CARRY ? 1 : Sh::LN][Sh::PAD];   // C . h, a row of each lane of a channel
};

// CARRY: only what a piece of the time axis makes of the state (its end from zero, and the product of its decays), for the
// pieces behind it; one CTA per 32 or 64 channels and piece.
//
// Four warps load and prepare a tile, and write the one before it, while the others walk the tile between: one barrier a tile.  8 sequences x
// 2048 steps x 2048 channels, S 16, bf16: 229 us, of which the exponentials alone are 119 (their pipe is busy 60 % of the time, issue 52 %);
// with the loading in the same warps 264, with one channel a thread 288, without the exponentials formed ahead of the chain 341.
// 256 CTAs are two on some multiprocessors and one on others, 14 % of it.
template <typename T, int S, bool VEC, int C, bool CARRY>
__global__ void __launch_bounds__(Shape<S, C, SCAN_TILE>::NT, S == 64 && C == 2 ? 1 : 2) scan_fwd_kernel(const ScanParams p) {
  using Sh = Shape<S, C, SCAN_TILE>;
  constexpr int TT = SCAN_TILE, CH = Sh::CH, NP = Sh::NP, NL = Sh::NL, NQ = Sh::NQ, BUFS = CARRY ? 1 : 2;
  extern __shared__ __align__(16) unsigned char raw_smem[];
  FwdSmem<Sh, CARRY>& sm = *reinterpret_cast<FwdSmem<Sh, CARRY>*>(raw_smem);
  auto& dd = sm.dd;
  auto& bc = sm.bc;
  auto& ys = sm.ys;
  const Place<CH> at(p, blockIdx.x);
  const int seg = blockIdx.y, t_first = seg * p.seglen, t_end = min(p.L, t_first + p.seglen);
  if (threadIdx.x >= Sh::WALK) {
    const int tid = threadIdx.x - Sh::WALK;
    // the pieces of a tile that this thread loads, and stores again: the same four channels, RS rows apart
    constexpr int RS = Sh::LOAD / (CH / 4);
    static_assert(Sh::LOAD % (CH / 4) == 0 && Sh::PIECES % Sh::LOAD == 0, "a thread's pieces have the same columns");
    const bool gate = !CARRY && p.z.p != nullptr;
    const int row = tid / (CH / 4), col = tid % (CH / 4) * 4, valid = max(0, min(4, at.left - col));
    auto place = [&](const ScanRows& w) { return reinterpret_cast<T*>(w.p) + at.n * w.sn + (t_first + row) * w.sl + at.ch0 + col; };
    const T *pu = place(p.u), *pd = place(p.delta), *pz = place(p.z);
    T* py = place(p.y);
    const int id0 = tid % Sh::QUADS, bc_row = tid < Sh::QUADS ? id0 / (S / 4) : p.L;      // (a row behind every piece's end)
    constexpr int RBC = Sh::LOAD / (S / 4);
    const T* pb = reinterpret_cast<const T*>(p.B.p) + at.n * p.B.sn + at.g * p.B.sg + (t_first + id0 / (S / 4)) * p.B.sl + id0 % (S / 4) * 4;
    const T* pc = reinterpret_cast<const T*>(p.C.p) + at.n * p.C.sn + at.g * p.C.sg + (t_first + id0 / (S / 4)) * p.C.sl + id0 % (S / 4) * 4;
    const Pairs bias = four(p.bias ? p.bias + at.ch0 + col : nullptr, valid), skip = four(!CARRY && p.skip ? p.skip + at.ch0 + col : nullptr, valid);
    // three tiles: being fetched, staged for the next walk (u and z stay for its result), walked before
    Quad<T, VEC> fu[NL], fd[NL], fz[NL], fb[NQ], fc[NQ], u1[NL], z1[NL], u0[NL], z0[NL];
    auto fetch = [&](int t0) {      // tiles are asked for in order
#pragma unroll
      for (int k = 0; k < NL; ++k) {
        const int v = t0 + row + k * RS < t_end ? valid : 0;
        fu[k].fetch(pu + k * RS * p.u.sl, v);
        fd[k].fetch(pd + k * RS * p.delta.sl, v);
        if (gate) fz[k].fetch(pz + k * RS * p.z.sl, v);
      }
      pu += TT * p.u.sl; pd += TT * p.delta.sl; pz += TT * p.z.sl;
#pragma unroll
      for (int i = 0; i < NQ; ++i) {
        const int v = t0 + bc_row + i * RBC < t_end ? 4 : 0;
        fb[i].fetch(pb + i * RBC * p.B.sl, v);
        if (!CARRY) fc[i].fetch(pc + i * RBC * p.C.sl, v);
      }
      pb += TT * p.B.sl; pc += TT * p.C.sl;
    };
    auto stage = [&](int buf) {
#pragma unroll
      for (int k = 0; k < NL; ++k) {
        u0[k] = u1[k]; z0[k] = z1[k];
        u1[k] = fu[k]; z1[k] = fz[k];
        Pairs dl = Pairs(fd[k].get()) + bias;
        if (p.softplus) dl = softplus4(dl);
        store_staged(&dd[buf][row + k * RS][col], dl, dl * Pairs(fu[k].get()));
      }
#pragma unroll
      for (int i = 0; i < NQ; ++i) {
        if (tid >= Sh::QUADS) continue;
        *reinterpret_cast<float4*>(&bc[buf][0][0][0] + (tid + i * Sh::LOAD) * 4) = fb[i].get();
        if (!CARRY) *reinterpret_cast<float4*>(&bc[buf][BUFS - 1][0][0] + (tid + i * Sh::LOAD) * 4) = fc[i].get();
      }
    };
    auto finish = [&](int t0, int buf) {      // y of the tile walked before
#pragma unroll
      for (int k = 0; k < NL; ++k) {
        const int v = t0 + row + k * RS < t_end ? valid : 0;
        if (v > 0) {
          Pairs y = fma4(skip, Pairs(u0[k].get()), sum_lanes<Sh>(&ys[buf][row + k * RS][0][col]));
          if (gate) {
            const Pairs z(z0[k].get());
            y = y * (z * sigmoid4(z));
          }
          put4<VEC>(py + k * RS * p.y.sl, v, y.f4());
        }
      }
      py += TT * p.y.sl;
    };
    if (t_first < t_end) {
      fetch(t_first);
      stage(0);
      if (t_first + TT < t_end) fetch(t_first + TT);
    }
    __syncthreads();
    int k0 = 0;
    for (int t0 = t_first; t0 < t_end; t0 += TT, k0 ^= 1) {
      if (!CARRY && t0 > t_first) finish(t0 - TT, k0 ^ 1);
      if (t0 + TT < t_end) {
        stage(k0 ^ 1);
        if (t0 + 2 * TT < t_end) fetch(t0 + 2 * TT);
      } else {
#pragma unroll
        for (int k = 0; k < NL; ++k) {
          u0[k] = u1[k];
          z0[k] = z1[k];
        }
      }
      __syncthreads();
    }
    if (!CARRY && t_first < t_end) finish(t_first + (t_end - t_first - 1) / TT * TT, k0 ^ 1);
    return;
  }

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, q = lane % Sh::LN, chl = (warp * Sh::LC + lane / Sh::LN) * C;
  const int d = at.ch0 + chl, mine = at.left - chl;      // channels of this thread that there are: mine > 0, mine > 1
  u64 h[C][NP], A2[C][NP];
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int i = 0; i < NP; ++i) h[c][i] = A2[c][i] = 0ull;
  const long long states = (long long)p.N * p.D * S, own = ((long long)at.n * p.D + d) * S;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    if (c >= mine) continue;
    load_states<Sh>(p.A + (long long)(d + c) * S, q, A2[c]);
    const long long o = own + c * S;
    if (CARRY || p.nseg == 1) {
      if (seg == 0 && p.h0) load_states<Sh>(p.h0 + o, q, h[c]);
      if (CARRY && seg == 0) store_states<Sh>(p.carry + o, q, h[c]);    // (hT may be h0's memory)
    } else {
      load_states<Sh>(p.carry + o, q, h[c]);
#pragma unroll 4
      for (int i = 0; i < seg; ++i) {     // the pieces in front, in order
        u64 root[NP], end[NP];
        load_states<Sh>(p.carry + (2 * i + 1) * states + o, q, end);
        load_states<Sh>(p.carry + (2 * i + 2) * states + o, q, root);
        through_piece(h[c], root, end);
      }
    }
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      A2[c][i] = mul2(A2[c][i], dup2(LOG2E));
      if (CARRY) h[c][i] = 0ull;
    }
  }
  float sum_d[C];
#pragma unroll
  for (int c = 0; c < C; ++c) sum_d[c] = 0.f;
  bool cut = false;      // CARRY: an episode begins inside the piece
  const int nck = (p.L + SCAN_CKPT - 1) / SCAN_CKPT;
  float* ck = p.ckpt + (((long long)at.n * nck + t_first / SCAN_CKPT) * p.D + d) * S;

  unsigned resets = t_first < t_end ? reset_bits(p, at.n, t_first, min(TT, t_end - t_first)) : 0u;
  __syncthreads();
  for (int t0 = t_first, k0 = 0; t0 < t_end; t0 += TT, k0 ^= 1) {
    const int steps = min(TT, t_end - t0);
    const unsigned now = resets;
    if (t0 + TT < t_end) resets = reset_bits(p, at.n, t0 + TT, min(TT, t_end - t0 - TT));
    // whole: sixteen steps of one episode.  What does not wait for the state (the decays and what is inserted) is formed PU steps
    // ahead of the chain through it, so that the exponentials' pipe does not wait for it either.
    auto walk = [&](auto whole) {
      constexpr bool WHOLE = decltype(whole)::value;
      constexpr int PU = Sh::ST == 8 ? 1 : 4 / C;      // (eight states a thread: 438 us with two, 411 with one; S 64, 8 x 2048 x 1024, bf16)
      u64 a[2][PU][C][NP], in[2][PU][C][NP], c2[2][PU][NP];
      auto ahead = [&](int t1, int b) __attribute__((always_inline)) {      // steps t1 .. t1 + PU - 1
#pragma unroll
        for (int k = 0; k < PU; ++k) {
          const int t = t1 + k;
          float2 x[C];
          u64 b2[NP];
          load_channels<C>(&dd[k0][t][chl], x);
          load_states<Sh>(&bc[k0][0][t][0], q, b2);
          if (!CARRY) load_states<Sh>(&bc[k0][BUFS - 1][t][0], q, c2[b][k]);
#pragma unroll
          for (int c = 0; c < C; ++c) {
            const u64 d2 = dup2(x[c].x), x2 = dup2(x[c].y);
            if (CARRY && (WHOLE || t < steps)) sum_d[c] += x[c].x;
#pragma unroll
            for (int i = 0; i < NP; ++i) {
              a[b][k][c][i] = decay2(d2, A2[c][i]);
              in[b][k][c][i] = mul2(x2, b2[i]);
            }
          }
        }
      };
      ahead(0, 0);
#pragma unroll
      for (int t1 = 0; t1 < TT; t1 += PU) {
        const int b = t1 / PU % 2;
        if (!WHOLE && t1 >= steps) break;
        if (t1 + PU < TT) ahead(t1 + PU, b ^ 1);
#pragma unroll
        for (int k = 0; k < PU; ++k) {
          const int t = t1 + k;
          if (!CARRY && t % SCAN_CKPT == 0 && p.ckpt && (WHOLE || t < steps)) {
#pragma unroll
            for (int c = 0; c < C; ++c)
              if (c < mine) store_states<Sh>(ck + c * S, q, h[c]);
            ck += (long long)p.D * S;
          }
          const bool fresh = !WHOLE && (now >> t & 1u);
          if (CARRY && fresh) cut = true;
          float y[C];
#pragma unroll
          for (int c = 0; c < C; ++c) {
            u64 acc = 0ull;
#pragma unroll
            for (int i = 0; i < NP; ++i) {
              const u64 next = fresh ? in[b][k][c][i] : fma2<true>(a[b][k][c][i], h[c][i], in[b][k][c][i]);
              h[c][i] = WHOLE || t < steps ? next : h[c][i];
              if (!CARRY) acc = i == 0 ? mul2(h[c][i], c2[b][k][i]) : fma2<true>(h[c][i], c2[b][k][i], acc);
            }
            y[c] = hsum2(acc);
          }
          if (!CARRY) store_channels<C>(&ys[CARRY ? 0 : k0][CARRY ? 0 : t][CARRY ? 0 : q][chl], y);
        }
      }
    };
    if (steps == TT && now == 0u) walk(std::true_type());
    else walk(std::false_type());
    __syncthreads();
  }
#pragma unroll
  for (int c = 0; c < C; ++c) {
    if (c >= mine) continue;
    const long long o = own + c * S;
    if (CARRY) {
      u64 root[NP];
#pragma unroll
      for (int i = 0; i < NP; ++i) root[i] = cut ? CUT : piece_root(sum_d[c], A2[c][i]);
      store_states<Sh>(p.carry + (2 * seg + 1) * states + o, q, h[c]);
      store_states<Sh>(p.carry + (2 * seg + 2) * states + o, q, root);
    } else if (seg == p.nseg - 1 && p.hT) {
      store_states<Sh>(p.hT + o, q, h[c]);
    }
  }
}

// A few steps, states in registers, everything else straight from memory: what an actor or a server does for each token.  Bound by the state's
// bytes, and by its launch where these are few.  NB: sequences of a thread.  With four, what belongs to a channel and sequence (softplus,
// gate) is formed by one of the channel's lanes each and passed around; with one, by all of them (256 sequences x 2048 channels, S 16,
// bf16: 17.5 us; 33 with one, 25 with four and no passing around).
template <typename T, int S, bool VEC, int NB>
__global__ void __launch_bounds__(Shape<S, 1, SCAN_TILE>::WALK) scan_step_kernel(const ScanParams p) {
  using Sh = Shape<S, 1, SCAN_TILE>;
  constexpr int NP = Sh::NP, LN = Sh::LN, OWN = NB > LN ? NB / LN : 1;      // OWN: sequences whose values a lane forms
  chained();
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, q = lane % LN, chl = warp * Sh::LC + lane / LN;
  const Place<Sh::CH> at(p, blockIdx.x);       // (its n: of the first of NB sequences, counted in such groups)
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
    float u[OWN], x[OWN], z[OWN];
#pragma unroll
    for (int o = 0; o < OWN; ++o) {
      const long long n = min(n0 + (NB == 1 ? 0 : (q + o * LN) % NB), p.N - 1);
      u[o] = to_float(reinterpret_cast<const T*>(p.u.p)[n * p.u.sn + t * p.u.sl + d]);
      x[o] = to_float(reinterpret_cast<const T*>(p.delta.p)[n * p.delta.sn + t * p.delta.sl + d]) + bias;
      z[o] = p.z.p ? to_float(reinterpret_cast<const T*>(p.z.p)[n * p.z.sn + t * p.z.sl + d]) : 0.f;
    }
    bool fresh[NB];
    u64 b2[NB][NP], c2[NB][NP];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const long long n = min(n0 + b, p.N - 1);
      fresh[b] = p.done && p.done[n * p.done_n + t * p.done_l] != 0;
      auto row = [&](const ScanRows& w, u64* v) {
        const T* r = reinterpret_cast<const T*>(w.p) + n * w.sn + at.g * w.sg + t * w.sl;
#pragma unroll
        for (int i = 0; i < Sh::ST / 4; ++i) {
          Quad<T, VEC> f;
          f.fetch(r + Sh::first(q, i), 4);
          const float4 t4 = f.get();
          v[2 * i] = pack2(t4.x, t4.y);
          v[2 * i + 1] = pack2(t4.z, t4.w);
        }
      };
      row(p.B, b2[b]);
      row(p.C, c2[b]);
    }
    float dl[OWN], du[OWN], y[NB];
#pragma unroll
    for (int o = 0; o < OWN; ++o) {
      dl[o] = p.softplus ? softplus(x[o]) : x[o];
      du[o] = dl[o] * u[o];
      dl[o] *= LOG2E;
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const float db = NB == 1 ? dl[0] : __shfl_sync(0xffffffffu, dl[b / LN], b % LN, LN);
      const float xb = NB == 1 ? du[0] : __shfl_sync(0xffffffffu, du[b / LN], b % LN, LN);
      u64 acc = 0ull;
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        u64 a = decay2(dup2(db), A2[i]);
        if (fresh[b]) a = h[b][i] = 0ull;
        h[b][i] = fma2<true>(a, h[b][i], mul2(dup2(xb), b2[b][i]));
        acc = i == 0 ? mul2(h[b][i], c2[b][i]) : fma2<true>(h[b][i], c2[b][i], acc);
      }
      y[b] = hsum2(acc);
    }
    // the sums over the lanes; with four sequences lane q ends with those of its own
    constexpr int W = NB < LN ? NB : LN;
#pragma unroll
    for (int w = W; w < LN; w *= 2) {
#pragma unroll
      for (int b = 0; b < NB; ++b) y[b] += __shfl_xor_sync(0xffffffffu, y[b], w);
    }
#pragma unroll
    for (int w = 1; w < W; w *= 2) {
      const bool up = q & w;
#pragma unroll
      for (int b = 0; b < NB; b += 2 * w) {
        const float keep = up ? y[b + w] : y[b], send = up ? y[b] : y[b + w];
        y[b] = keep + __shfl_xor_sync(0xffffffffu, send, w);
      }
    }
#pragma unroll
    for (int o = 0; o < OWN; ++o) {
      const int b = q + o * LN;
      float r = fmaf(skip, u[o], y[o * LN < NB ? o * LN : 0]);
      if (p.z.p) r *= z[o] * sigmoid(z[o]);
      if (mine && b < NB && n0 + b < p.N) narrow(r, reinterpret_cast<T*>(p.y.p) + (long long)(n0 + b) * p.y.sn + t * p.y.sl + d);
    }
  }
  if (!mine || !p.hT) return;
#pragma unroll
  for (int b = 0; b < NB; ++b)
    if (n0 + b < p.N) store_states<Sh>(p.hT + ((long long)(n0 + b) * p.D + d) * S, q, h[b]);
}

template <typename T, int S, bool VEC, int C>
cudaError_t sequences(const ScanParams& p, cudaStream_t s) {
  using Sh = Shape<S, C, SCAN_TILE>;
  const unsigned grid = (unsigned)blocks_of(p, Sh::CH);
  static unsigned long long raised[2] = {0, 0};
  if (p.nseg > 1) {
    constexpr int smem = sizeof(FwdSmem<Sh, true>);
    if (const cudaError_t e = allow_smem(scan_fwd_kernel<T, S, VEC, C, true>, smem, &raised[0]); e != cudaSuccess) return e;
    scan_fwd_kernel<T, S, VEC, C, true><<<dim3(grid, p.nseg - 1), Sh::NT, smem, s>>>(p);
    if (const cudaError_t e = cudaGetLastError(); e != cudaSuccess) return e;
  }
  constexpr int smem = sizeof(FwdSmem<Sh, false>);
  if (const cudaError_t e = allow_smem(scan_fwd_kernel<T, S, VEC, C, false>, smem, &raised[1]); e != cudaSuccess) return e;
  scan_fwd_kernel<T, S, VEC, C, false><<<dim3(grid, p.nseg), Sh::NT, smem, s>>>(p);
  return cudaGetLastError();
}
template <typename T, int S, bool VEC>
cudaError_t launch(const ScanParams& p, cudaStream_t s) {
  if (p.L <= SCAN_STEPS_DIRECT && !p.ckpt) {
    constexpr int NB = 4;      // (48 sequences x 512 channels leave most of the GPU idle either way: the launch is what counts there)
    const long long grid = blocks_of(p, Shape<S, 1, SCAN_TILE>::CH);
    if (grid < 32 * common_sms()) return launch_behind(scan_step_kernel<T, S, VEC, 1>, p, dim3((unsigned)grid), Shape<S, 1, SCAN_TILE>::WALK, 0, s);
    return launch_behind(scan_step_kernel<T, S, VEC, NB>, p, dim3((unsigned)(grid / p.N * ((p.N + NB - 1) / NB))), Shape<S, 1, SCAN_TILE>::WALK, 0, s);
  }
  // two channels a thread where these CTAs still fill the multiprocessors: 8 x 1024 x 2048, S 32, 184 us against 208 (S 64: 346 against
  // 373); 8 x 2048 x 1024, S 64 (128 CTAs), 376 with one against 411
  if constexpr (S > 8)
    if (blocks_of(p, Shape<S, 2, SCAN_TILE>::CH) * p.nseg >= 1 * common_sms()) return sequences<T, S, VEC, 2>(p, s);
  return sequences<T, S, VEC, 1>(p, s);
}

}  // namespace

// The pieces of the time axis.  One where the channels alone come near to filling the GPU; otherwise as many as fill it once, of 64 steps at
// least.  A piece's exponentials are formed twice, so two pieces gain nothing.
int scan_segments(const ScanParams& p, int channels, int sms) {
  const long long ctas = blocks_of(p, channels), room = (long long)sms * (p.S == 64 ? 1 : 2);
  if (ctas == 0 || p.L < 192) return 1;
  long long n = room / ctas;
  if (n > p.L / 64) n = p.L / 64;
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
