// Causal convolution along time in front of the selective scan, K = 2, 3 or 4 taps of a channel's own, forward and backward:
//   y_t = act(bias + sum_i w_{K-1-i} x_{t-i}),   act = silu or the identity,
// with the K - 1 inputs before the call carried as a state, and none read across an episode's start.
//
// Bound by HBM: one read and one write of [N, L, D].  A thread takes four channels and up to 16 steps in time order, its window in
// registers; the K - 1 steps in front of its own come from L2.
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

// TS: steps of a thread, whose loads are all on their way before the first is used
template <typename T, bool VEC, int K, int TS, bool DONE>
__global__ void __launch_bounds__(128) conv_fwd_kernel(const ConvParams p) {
  chained();
  const int quads = (p.D + 3) / 4, chunks = p.L == 0 ? 1 : (p.L + TS - 1) / TS;
  const long long id = (long long)blockIdx.x * 128 + threadIdx.x;
  const int d = (int)(id % quads) * 4, chunk = (int)(id / quads % chunks), valid = min(4, p.D - d);
  const long long n_ = id / quads / chunks;
  if (n_ >= p.N) return;
  const int n = (int)n_, t0 = chunk * TS, t_end = min(p.L, t0 + TS);
  const T* px = reinterpret_cast<const T*>(p.x.p) + n * p.x.sn + t0 * p.x.sl + d;
  T* py = reinterpret_cast<T*>(p.y.p) + n * p.y.sn + t0 * p.y.sl + d;
  Quad<T, VEC> row[TS], past[K];
  bool cut[TS];
#pragma unroll
  for (int k = 0; k < TS; ++k) {
    row[k].fetch(px + k * p.x.sl, t0 + k < t_end ? valid : 0);
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
#pragma unroll
  for (int k = 0; k < TS; ++k) {
    if (t0 + k >= t_end) break;
#pragma unroll
    for (int j = 0; j + 1 < K; ++j) win[j] = DONE && cut[k] ? Pairs() : win[j + 1];
    win[K - 1] = Pairs(row[k].get());
    Pairs y = b;
#pragma unroll
    for (int j = 0; j < K; ++j) y = fma4(w[j], win[j], y);
    if (p.silu) y = y * sigmoid4(y);
    put4<VEC>(py + k * p.y.sl, valid, y.f4());
  }
  if (t_end == p.L && p.sT.p) {
    T* ps = reinterpret_cast<T*>(p.sT.p) + n * p.sT.sn + d;
#pragma unroll
    for (int j = 1; j < K; ++j) put4<VEC>(ps + (j - 1) * p.sT.sl, valid, win[j].f4());
  }
}

// A warp takes 32 quads of channels and a chunk of TS steps at a time, the block's four warps one chunk after another's; the sums of dw
// and dbias stay with the threads.  What the outputs behind the chunk give to its inputs comes from TS + K - 1 steps of dy.
template <typename T, bool VEC, int K, int TS, bool DONE>
__global__ void __launch_bounds__(128) conv_bwd_kernel(const ConvParams p) {
  __shared__ float4 red[4][32];
  constexpr int ALL = TS + K - 1, AHEAD = 4;      // steps of a chunk, and how many of them are on their way
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int d = ((int)blockIdx.x * 32 + lane) * 4, valid = max(0, min(4, p.D - d));
  const int chunks = (p.L + TS - 1) / TS;
  const long long units = (long long)p.N * chunks;
  Pairs w[K], b, dw[K], db;
  load_taps<K>(p, d, valid, w, b);
  const u64 one = dup2(1.f), minus = dup2(-1.f);
  const Pairs ones(one, one), minuses(minus, minus);
  for (long long u = (long long)blockIdx.y * 4 + warp; u < units; u += (long long)gridDim.y * 4) {
    if (valid == 0) break;
    const int n = (int)(u / chunks), t0 = (int)(u % chunks) * TS;
    const T* px = reinterpret_cast<const T*>(p.x.p) + n * p.x.sn + t0 * p.x.sl + d;
    const T* py = reinterpret_cast<const T*>(p.dy.p) + n * p.dy.sn + t0 * p.dy.sl + d;
    T* ox = reinterpret_cast<T*>(p.dx.p) + n * p.dx.sn + t0 * p.dx.sl + d;
    Quad<T, VEC> rx[AHEAD], ry[AHEAD], past[K];
#pragma unroll
    for (int j = 1; j < K; ++j) past[j] = input<T, K, VEC>(p, n, t0 - K + j, d, valid);
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int v = t0 + k < p.L ? valid : 0;
      rx[k].fetch(px, v);
      ry[k].fetch(py, v);
      px += p.x.sl;
      py += p.dy.sl;
    }
    // From the chunk's first step on, K - 1 steps beyond its last: dx[s] (of the state's rows too, in the first chunk) is whole
    // once the step K - 1 behind it is done.  Steps beyond the call's end have no gradient.
    const bool last = t0 + TS > p.L - (K - 1) && p.dsT.p != nullptr;      // some of the inputs are in the state behind the call
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
      bool kept = last && s >= p.L - (K - 1) && s < p.L;
      if (DONE && kept)
        for (int r = max(s + 1, 0); r < p.L; ++r) kept = kept && !starts(p, n, r);
      q.fetch(reinterpret_cast<const T*>(p.dsT.p) + n * p.dsT.sn + (long long)(s - (p.L - (K - 1))) * p.dsT.sl + d, kept ? valid : 0);
      return Pairs(q.get());
    };
    if (last) {
#pragma unroll
      for (int j = 1; j < K; ++j) acc[j] = carried(t0 - K + j);
    }
#pragma unroll
    for (int k = 0; k < ALL; ++k) {
      const int t = t0 + k;
      if (t >= p.L + K - 1) break;
#pragma unroll
      for (int j = 0; j + 1 < K; ++j) acc[j] = acc[j + 1];
      acc[K - 1] = last ? carried(t) : Pairs();
      const bool fresh = DONE && t < p.L && starts(p, n, t);
      if (DONE) age = fresh ? 0 : min(K - 1, age + 1);
#pragma unroll
      for (int j = 0; j + 1 < K; ++j) win[j] = DONE && fresh ? Pairs() : win[j + 1];
      win[K - 1] = Pairs(rx[k % AHEAD].get());
      Pairs gp(ry[k % AHEAD].get());
      if (k + AHEAD < ALL) {
        const int v = t + AHEAD < p.L ? valid : 0;
        rx[k % AHEAD].fetch(px, v);
        ry[k % AHEAD].fetch(py, v);
        px += p.x.sl;
        py += p.dy.sl;
      }
      if (p.silu) {      // silu'(a) = sigmoid (1 + a (1 - sigmoid))
        Pairs a = b;
#pragma unroll
        for (int j = 0; j < K; ++j) a = fma4(w[j], win[j], a);
        const Pairs sg = sigmoid4(a);
        gp = gp * (sg * fma4(a, fma4(sg, minuses, ones), ones));
        if (t >= p.L) gp = Pairs();      // (whatever the window holds)
      }
#pragma unroll
      for (int j = 0; j < K; ++j)
        if (!DONE || K - 1 - j <= age) acc[j] = fma4(w[j], gp, acc[j]);
      if (k < TS) {
        db = db + gp;
#pragma unroll
        for (int j = 0; j < K; ++j)
          if (!DONE || K - 1 - j <= age) dw[j] = fma4(gp, win[j], dw[j]);
      }
      if (k >= K - 1) {
        put4<VEC>(ox, t - (K - 1) < p.L ? valid : 0, acc[0].f4());
        ox += p.dx.sl;
      } else if (t0 == 0 && p.ds0.p) {
        put4<VEC>(reinterpret_cast<T*>(p.ds0.p) + n * p.ds0.sn + k * p.ds0.sl + d, valid, acc[0].f4());
      }
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
  const int c = threadIdx.x % 32, slice = threadIdx.x / 32, total = a.D * (a.K + 1);
  int i = blockIdx.x * 32 + c;
  float t = 0.f;
  if (i < total) {
#pragma unroll 8
    for (int b = slice; b < a.parts; b += 32) t += a.part[(long long)b * total + i];
  }
  s[slice][c] = t;
  __syncthreads();
  t = allreduce_warp(s[c][slice]);
  i = blockIdx.x * 32 + slice;
  if (c != 0 || i >= total) return;
  const int d = i / (a.K + 1), j = i % (a.K + 1);
  if (j < a.K) a.dw[(long long)d * a.K + j] = t;
  else if (a.dbias) a.dbias[d] = t;
}

template <typename T, bool VEC, int K>
cudaError_t fwd(const ConvParams& p, cudaStream_t s) {
  const long long quads = (p.D + 3) / 4;
  auto run = [&](auto ts) {
    constexpr int TS = decltype(ts)::value;
    const long long chunks = p.L == 0 ? 1 : (p.L + TS - 1) / TS, blocks = (quads * chunks * p.N + 127) / 128;
    return p.done ? launch_behind(conv_fwd_kernel<T, VEC, K, TS, true>, p, dim3((unsigned)blocks), 128, 0, s)
                  : launch_behind(conv_fwd_kernel<T, VEC, K, TS, false>, p, dim3((unsigned)blocks), 128, 0, s);
  };
  if (p.L <= 1) return run(std::integral_constant<int, 1>());
  return run(std::integral_constant<int, CONV_CHUNK>());
}
template <typename T, bool VEC, int K>
cudaError_t bwd(const ConvParams& p, cudaStream_t s) {
  const int parts = conv_parts(p);
  const dim3 grid((unsigned)((p.D + 127) / 128), (unsigned)parts);
  if (p.done) conv_bwd_kernel<T, VEC, K, CONV_CHUNK, true><<<grid, 128, 0, s>>>(p);
  else conv_bwd_kernel<T, VEC, K, CONV_CHUNK, false><<<grid, 128, 0, s>>>(p);
  if (const cudaError_t e = cudaGetLastError(); e != cudaSuccess) return e;
  return launch_behind(conv_sums_kernel, ConvSums{p.part, p.dw, p.dbias, parts, p.D, K}, dim3((unsigned)((p.D * (K + 1) + 31) / 32)), 1024, 0, s);
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

// Four chunks a block and turn; blocks for eight of a multiprocessor at most, each of which leaves a part to be added up
int conv_parts(const ConvParams& p) {
  const long long units = (long long)p.N * ((p.L + CONV_CHUNK - 1) / CONV_CHUNK), want = (units + 3) / 4;
  const long long most = 8ll * common_sms() / ((p.D + 127) / 128);
  const long long n = want < most ? want : most;
  return n < 1 ? 1 : (int)n;
}
cudaError_t conv_forward(const ConvParams& p, cudaStream_t s) {
  return by_type(p, [&](auto t, auto v, auto k) { return fwd<decltype(t), decltype(v)::value, decltype(k)::value>(p, s); });
}
cudaError_t conv_backward(const ConvParams& p, cudaStream_t s) {
  return by_type(p, [&](auto t, auto v, auto k) { return bwd<decltype(t), decltype(v)::value, decltype(k)::value>(p, s); });
}

}  // namespace srwm
