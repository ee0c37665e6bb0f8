// Causal convolution along time in front of the selective scan, K = 2, 3 or 4 taps of a channel's own, forward and backward:
//   y_t = act(bias + sum_i w_{K-1-i} x_{t-i}),   act = silu or the identity,
// with the K - 1 inputs before the call carried as a state, and none read across an episode's start.
//
// Bound by HBM: one read and one write of [N, L, D].  A thread takes four channels and a chunk of steps in time order, its window in
// registers, the next steps' rows on their way; the K - 1 steps in front of its own come from L2.  8 x 2048 x 2048, K 4, bf16: forward 32 us
// (21 at the copy bandwidth), backward 57 (31: x is read again).  Chunks as long as fill the GPU once, and steps inside a chunk without
// conditions, took them there from 39 and 75 with chunks of 16.  Both wait for memory: issue is busy 41 % of the time, the loads are the first
// stall, and the backward's three blocks of 144 registers a thread have 24 KB of rows on their way a multiprocessor, where the copy
// bandwidth times its latency is some 35.  (Some variants keep a value or two of a thread on the stack, 4 to 48 bytes.)
#include <type_traits>

#include "chain.h"
#include "conv.h"
#include "device.h"
#include "scan.cuh"

namespace srwm {
namespace {
using namespace scan;

// w[j]: tap j of four channels
template <int K>
__device__ __forceinline__ void load_taps(const ConvParams& p, int d, int valid, Pairs (&w)[K], Pairs& b) {
  b = four(p.bias ? p.bias + d : nullptr, valid);
#pragma unroll
  for (int j = 0; j < K; ++j) {
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < valid ? p.w[(long long)(d + i) * K + j] : 0.f;
    w[j] = Pairs(make_float4(v[0], v[1], v[2], v[3]));
  }
}
__device__ __forceinline__ bool starts(const ConvParams& p, int n, int t) {
  return p.done && p.done[n * p.done_n + (long long)t * p.done_l] != 0;
}
// x_t of the call, or of the state in front of it
template <typename T, int K, bool VEC>
__device__ __forceinline__ Quad<T, VEC> input(const ConvParams& p, int n, int t, int d, int valid) {
  const bool before = t < 0;
  const char* base = before ? p.s0.p : p.x.p;
  const long long at = before ? n * p.s0.sn + (t + K - 1) * p.s0.sl : n * p.x.sn + t * p.x.sl;
  Quad<T, VEC> q;
  q.fetch(reinterpret_cast<const T*>(base) + at + d, base ? valid : 0);
  return q;
}

// AH: steps whose rows are on their way.  A thread takes p.chunk steps.
template <typename T, bool VEC, int K, int AH, bool DONE>
__global__ void __launch_bounds__(128) conv_fwd_kernel(const ConvParams p) {
  chained();
  const int quads = (p.D + 3) / 4, chunks = p.L == 0 ? 1 : (p.L + p.chunk - 1) / p.chunk;
  const long long id = (long long)blockIdx.x * 128 + threadIdx.x;
  const int d = (int)(id % quads) * 4, chunk = (int)(id / quads % chunks), valid = min(4, p.D - d);
  const long long n_ = id / quads / chunks;
  if (n_ >= p.N) return;
  const int n = (int)n_, t0 = chunk * p.chunk, t_end = min(p.L, t0 + p.chunk);
  const T* px = reinterpret_cast<const T*>(p.x.p) + n * p.x.sn + t0 * p.x.sl + d;
  T* py = reinterpret_cast<T*>(p.y.p) + n * p.y.sn + t0 * p.y.sl + d;
  Quad<T, VEC> row[AH], past[K];
  bool cut[AH];
#pragma unroll
  for (int k = 0; k < AH; ++k) {
    row[k].fetch(px, t0 + k < t_end ? valid : 0);
    px += p.x.sl;
    if (DONE) cut[k] = t0 + k < t_end && starts(p, n, t0 + k);
  }
#pragma unroll
  for (int j = 1; j < K; ++j) past[j] = input<T, K, VEC>(p, n, t0 - K + j, d, valid);
  Pairs w[K], b, win[K];       // win: x_{t-K+1} .. x_t
  load_taps<K>(p, d, valid, w, b);
#pragma unroll
  for (int j = 1; j < K; ++j) {
    const int t = t0 - K + j;
    win[j] = Pairs(past[j].get());
    if (DONE && t >= 0 && starts(p, n, t)) {
#pragma unroll
      for (int k = 1; k < j; ++k) win[k] = Pairs();
    }
  }
  auto steps = [&](auto inner, int t1) __attribute__((always_inline)) {      // AH of them; inner: none behind the chunk's end
    constexpr bool INNER = decltype(inner)::value;
#pragma unroll
    for (int k = 0; k < AH; ++k) {
      const int t = t1 + k;
      if (!INNER && t >= t_end) break;
#pragma unroll
      for (int j = 0; j + 1 < K; ++j) win[j] = DONE && cut[k] ? Pairs() : win[j + 1];
      win[K - 1] = Pairs(row[k].get());
      if (AH > 1) {
        row[k].fetch(px, t + AH < t_end ? valid : 0);
        px += p.x.sl;
        if (DONE) cut[k] = t + AH < t_end && starts(p, n, t + AH);
      }
      Pairs y = b;
#pragma unroll
      for (int j = 0; j < K; ++j) y = fma4(w[j], win[j], y);
      const Pairs f = y * sigmoid4(y);
      put4<VEC>(py, valid, (p.silu ? f : y).f4());
      py += p.y.sl;
    }
  };
  int t1 = t0;
  for (; t1 + AH <= t_end; t1 += AH) steps(std::true_type(), t1);
  if (t1 < t_end) steps(std::false_type(), t1);
  if (t_end == p.L && p.sT.p) {
    T* ps = reinterpret_cast<T*>(p.sT.p) + n * p.sT.sn + d;
#pragma unroll
    for (int j = 1; j < K; ++j) put4<VEC>(ps + (j - 1) * p.sT.sl, valid, win[j].f4());
  }
}

// A warp takes 32 quads of channels and p.chunk steps at a time, the block's four warps one chunk after another's; the sums of dw
// and dbias stay with the threads.  What the outputs behind the chunk give to its inputs comes from K - 1 more steps of dy.
// An episode's start is read with the rows, AH steps ahead: forward and backward at N 8, L 2048, D 2048 in 16 bits with starts 125 us
// (132 when each step read its own); without starts 97.
template <typename T, bool VEC, int K, bool DONE>
__global__ void __launch_bounds__(128) conv_bwd_kernel(const ConvParams p) {
  __shared__ float4 red[4][32];
  constexpr int AH = 4;      // steps whose rows are on their way
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int d = ((int)blockIdx.x * 32 + lane) * 4, valid = max(0, min(4, p.D - d));
  const int chunks = (p.L + p.chunk - 1) / p.chunk;
  const long long units = (long long)p.N * chunks;
  Pairs w[K], b, dw[K], db;
  load_taps<K>(p, d, valid, w, b);
  const u64 one = dup2(1.f), minus = dup2(-1.f);
  const Pairs ones(one, one), minuses(minus, minus);
  for (long long u = (long long)blockIdx.y * 4 + warp; u < units; u += (long long)gridDim.y * 4) {
    if (valid == 0) break;
    const int n = (int)(u / chunks), t0 = (int)(u % chunks) * p.chunk, t_end = min(p.L, t0 + p.chunk), t_all = t_end + K - 1;
    const T* px = reinterpret_cast<const T*>(p.x.p) + n * p.x.sn + t0 * p.x.sl + d;
    const T* py = reinterpret_cast<const T*>(p.dy.p) + n * p.dy.sn + t0 * p.dy.sl + d;
    T* ox = reinterpret_cast<T*>(p.dx.p) + n * p.dx.sn + t0 * p.dx.sl + d;
    Quad<T, VEC> rx[AH], ry[AH], past[K];
    bool cut[AH];
#pragma unroll
    for (int j = 1; j < K; ++j) past[j] = input<T, K, VEC>(p, n, t0 - K + j, d, valid);
#pragma unroll
    for (int k = 0; k < AH; ++k) {
      const int v = t0 + k < p.L && t0 + k < t_all ? valid : 0;
      if (DONE) cut[k] = v > 0 && starts(p, n, t0 + k);
      rx[k].fetch(px, v);
      ry[k].fetch(py, v);
      px += p.x.sl;
      py += p.dy.sl;
    }
    // From the chunk's first step on, K - 1 steps beyond its last: dx[s] (of the state's rows too, in the first chunk) is whole
    // once the step K - 1 behind it is done.  Steps beyond the call's end have no gradient.
    const bool last = t_all > p.L - (K - 1) && p.dsT.p != nullptr;      // some of the inputs are in the state behind the call
    Pairs win[K], acc[K];       // acc[j]: of the input at t - K + 1 + j
    int age = K - 1;            // steps since the episode's start, as far as they matter
#pragma unroll
    for (int j = 1; j < K; ++j) {
      const int t = t0 - K + j;
      win[j] = Pairs(past[j].get());
      if (DONE && t >= 0) {
        const bool cut = starts(p, n, t);
        if (cut) {
#pragma unroll
          for (int k = 1; k < j; ++k) win[k] = Pairs();
        }
        age = cut ? 0 : min(K - 1, age + 1);
      }
    }
    // what the state behind the call gives to the input at s
    auto carried = [&](int s) {
      Quad<T, VEC> q;
      bool kept = s >= p.L - (K - 1) && s < p.L;
      if (DONE && kept)
        for (int r = max(s + 1, 0); r < p.L; ++r) kept = kept && !starts(p, n, r);
      q.fetch(reinterpret_cast<const T*>(p.dsT.p) + n * p.dsT.sn + (long long)(s - (p.L - (K - 1))) * p.dsT.sl + d, kept ? valid : 0);
      return Pairs(q.get());
    };
    if (last) {
#pragma unroll
      for (int j = 1; j < K; ++j) acc[j] = carried(t0 - K + j);
    }
    // AH steps; inner: all of the chunk's own, their inputs' gradients too, and none of them in the state behind the call
    auto steps = [&](auto inner, int t1) __attribute__((always_inline)) {
      constexpr bool INNER = decltype(inner)::value;
#pragma unroll
      for (int k = 0; k < AH; ++k) {
        const int t = t1 + k, s = t - (K - 1);
        if (!INNER && t >= t_all) break;
#pragma unroll
        for (int j = 0; j + 1 < K; ++j) acc[j] = acc[j + 1];
        acc[K - 1] = Pairs();
        if (!INNER && last) acc[K - 1] = carried(t);
        const bool fresh = DONE && cut[k];
        if (DONE) age = fresh ? 0 : min(K - 1, age + 1);
#pragma unroll
        for (int j = 0; j + 1 < K; ++j) win[j] = DONE && fresh ? Pairs() : win[j + 1];
        win[K - 1] = Pairs(rx[k].get());
        Pairs gp(ry[k].get()), a = b;
        const int v = t + AH < p.L && t + AH < t_all ? valid : 0;
        if (DONE) cut[k] = v > 0 && starts(p, n, t + AH);
        rx[k].fetch(px, v);
        ry[k].fetch(py, v);
        px += p.x.sl;
        py += p.dy.sl;
#pragma unroll
        for (int j = 0; j < K; ++j) a = fma4(w[j], win[j], a);
        const Pairs sg = sigmoid4(a), f = gp * (sg * fma4(a, fma4(sg, minuses, ones), ones));      // silu'(a) = sigmoid (1 + a (1 - sigmoid))
        gp = p.silu ? f : gp;
        if (!INNER && t >= p.L) gp = Pairs();      // (whatever the window holds)
#pragma unroll
        for (int j = 0; j < K; ++j)
          if (!DONE || K - 1 - j <= age) acc[j] = fma4(w[j], gp, acc[j]);
        if (INNER || t < t_end) {
          db = db + gp;
#pragma unroll
          for (int j = 0; j < K; ++j)
            if (!DONE || K - 1 - j <= age) dw[j] = fma4(gp, win[j], dw[j]);
        }
        if (INNER || s >= t0) {
          put4<VEC>(ox, valid, acc[0].f4());
          ox += p.dx.sl;
        } else if (t0 == 0 && p.ds0.p) {
          put4<VEC>(reinterpret_cast<T*>(p.ds0.p) + n * p.ds0.sn + (s + K - 1) * p.ds0.sl + d, valid, acc[0].f4());
        }
      }
    };
    for (int t1 = t0; t1 < t_all; t1 += AH) {
      if (t1 >= t0 + K - 1 && t1 + AH <= t_end && t1 + AH <= p.L - (K - 1)) steps(std::true_type(), t1);
      else steps(std::false_type(), t1);
    }
  }
  float* out = p.part + (long long)blockIdx.y * p.D * (K + 1);
#pragma unroll
  for (int j = 0; j <= K; ++j) {
    __syncthreads();
    red[warp][lane] = (j < K ? dw[j < K ? j : 0] : db).f4();
    __syncthreads();
    if (warp == 0) {
      float4 s = red[0][lane];
#pragma unroll
      for (int k = 1; k < 4; ++k) {
        const float4 o = red[k][lane];
        s.x += o.x; s.y += o.y; s.z += o.z; s.w += o.w;
      }
      const float r[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < valid) out[(long long)(d + i) * (K + 1) + j] = r[i];
    }
  }
}

struct ConvSums {
  const float* part;
  float *dw, *dbias;
  int parts, D, K;
};
// [parts][D][K + 1] -> dw [D][K], dbias [D]: 32 values a block, 32 slices of the parts
__global__ void __launch_bounds__(1024) conv_sums_kernel(const ConvSums a) {
  chained();
  __shared__ float s[32][33];
  const int c = threadIdx.x % 32, slice = threadIdx.x / 32;
  const long long total = (long long)a.D * (a.K + 1);
  long long i = blockIdx.x * 32ll + c;
  float t = 0.f;
  if (i < total) {
#pragma unroll 8
    for (int b = slice; b < a.parts; b += 32) t += a.part[b * total + i];
  }
  s[slice][c] = t;
  __syncthreads();
  t = allreduce_warp(s[c][slice]);
  i = blockIdx.x * 32ll + slice;
  if (c != 0 || i >= total) return;
  const long long d = i / (a.K + 1);
  const int j = (int)(i - d * (a.K + 1));
  if (j < a.K) a.dw[d * a.K + j] = t;
  else if (a.dbias) a.dbias[d] = t;
}

constexpr int CONV_FWD_THREADS = 768;      // of a multiprocessor at once (bf16: six blocks at 80 registers a thread; 640 and 1280 take as long)

// Steps of a chunk, so that the N sequences' chunks are as many as are taken at once; 16 at least (each reads K - 1 steps in front of its own)
int chunk_of(const ConvParams& p, long long at_once) {
  const long long each = p.N > 0 && at_once > p.N ? at_once / p.N : 1, steps = (p.L + each - 1) / each;
  return (int)(steps < CONV_CHUNK ? CONV_CHUNK : steps);
}
// Blocks of a strip of 128 channels in the backward: three of a multiprocessor in all, as many as are there at once
long long conv_blocks(const ConvParams& p) {
  const long long n = 3ll * common_sms() / ((p.D + 127) / 128);
  return n < 1 ? 1 : n;
}

template <typename T, bool VEC, int K>
cudaError_t fwd(ConvParams p, cudaStream_t s) {
  const long long quads = (p.D + 3) / 4;
  auto run = [&](auto ah) {
    constexpr int AH = decltype(ah)::value;
    const long long chunks = p.L == 0 ? 1 : (p.L + p.chunk - 1) / p.chunk, blocks = (quads * chunks * p.N + 127) / 128;
    return p.done ? launch_behind(conv_fwd_kernel<T, VEC, K, AH, true>, p, dim3((unsigned)blocks), 128, 0, s)
                  : launch_behind(conv_fwd_kernel<T, VEC, K, AH, false>, p, dim3((unsigned)blocks), 128, 0, s);
  };
  // as many threads as are there at once
  p.chunk = chunk_of(p, CONV_FWD_THREADS * common_sms() / quads);
  if (p.L <= 1) return run(std::integral_constant<int, 1>());
  return run(std::integral_constant<int, 8>());
}
template <typename T, bool VEC, int K>
cudaError_t bwd(ConvParams p, cudaStream_t s) {
  const int parts = conv_parts(p);
  const dim3 grid((unsigned)((p.D + 127) / 128), (unsigned)parts);
  p.chunk = chunk_of(p, 4 * conv_blocks(p));
  if (p.done) conv_bwd_kernel<T, VEC, K, true><<<grid, 128, 0, s>>>(p);
  else conv_bwd_kernel<T, VEC, K, false><<<grid, 128, 0, s>>>(p);
  if (const cudaError_t e = cudaGetLastError(); e != cudaSuccess) return e;
  return launch_behind(conv_sums_kernel, ConvSums{p.part, p.dw, p.dbias, parts, p.D, K}, dim3((unsigned)((p.D * (K + 1ll) + 31) / 32)), 1024, 0, s);
}
// f(element, VEC, K)
template <typename F>
cudaError_t by_type(const ConvParams& p, F f) {
  auto taps = [&](auto t, auto vec) {
    switch (p.K) {
      case 2: return f(t, vec, std::integral_constant<int, 2>());
      case 3: return f(t, vec, std::integral_constant<int, 3>());
      default: return f(t, vec, std::integral_constant<int, 4>());
    }
  };
  if (p.bf16) return p.vec ? taps(__nv_bfloat16(), std::true_type()) : taps(__nv_bfloat16(), std::false_type());
  return p.vec ? taps(float(), std::true_type()) : taps(float(), std::false_type());
}

}  // namespace

int conv_parts(const ConvParams& p) {
  const long long most = conv_blocks(p), chunk = chunk_of(p, 4 * most), want = (p.N * ((p.L + chunk - 1) / chunk) + 3) / 4;
  return (int)(want < 1 ? 1 : want < most ? want : most);
}
cudaError_t conv_forward(const ConvParams& p, cudaStream_t s) {
  return by_type(p, [&](auto t, auto v, auto k) { return fwd<decltype(t), decltype(v)::value, decltype(k)::value>(p, s); });
}
cudaError_t conv_backward(const ConvParams& p, cudaStream_t s) {
  return by_type(p, [&](auto t, auto v, auto k) { return bwd<decltype(t), decltype(v)::value, decltype(k)::value>(p, s); });
}

}  // namespace srwm
