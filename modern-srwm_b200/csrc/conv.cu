// Causal convolution along time in front of the selective scan, K = 2, 3 or 4 taps of a channel's own, forward and backward:
//   y_t = act(bias + sum_i w_{K-1-i} x_{t-i}),   act = silu or the identity,
// with the K - 1 inputs before the call carried as a state, and none read across an episode's start.
//
// Bound by HBM: one read and one write of [N, L, D].  A thread takes four channels and up to 16 steps in time order, its window in
// registers, loads four steps ahead; the K - 1 steps in front of its own come from L2.
#include <type_traits>

#include "chain.h"
#include "conv.h"
#include "device.h"
#include "scan.cuh"

namespace srwm {
namespace {
using namespace scan;

struct Chan4 {
  float v[4];
  __device__ __forceinline__ Chan4() { v[0] = v[1] = v[2] = v[3] = 0.f; }
  __device__ __forceinline__ explicit Chan4(float4 f) { v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w; }
  __device__ __forceinline__ float4 f4() const { return make_float4(v[0], v[1], v[2], v[3]); }
};

// w[j][i]: tap j of channel i
template <int K>
__device__ __forceinline__ void load_taps(const ConvParams& p, int d, int valid, float (&w)[K][4], float (&b)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    b[i] = i < valid && p.bias ? p.bias[d + i] : 0.f;
#pragma unroll
    for (int j = 0; j < K; ++j) w[j][i] = i < valid ? p.w[(long long)(d + i) * K + j] : 0.f;
  }
}
__device__ __forceinline__ bool starts(const ConvParams& p, int n, int t) {
  return p.done && p.done[n * p.done_n + (long long)t * p.done_l] != 0;
}
// x_t of the call, or of the state in front of it
template <typename T, int K>
__device__ __forceinline__ Chan4 input(const ConvParams& p, int n, int t, int d, int valid) {
  const ScanRows& r = t >= 0 ? p.x : p.s0;
  if (r.p == nullptr) return Chan4();
  const T* ptr = reinterpret_cast<const T*>(r.p) + n * r.sn + (long long)(t >= 0 ? t : t + K - 1) * r.sl + d;
  Quad<T> qd;
  qd.fetch(ptr, r.vec, valid);
  return Chan4(qd.get(ptr, r.vec, valid));
}

// TS: steps of a thread
template <typename T, int K, int TS>
__global__ void __launch_bounds__(128) conv_fwd_kernel(const ConvParams p) {
  chained();
  const int quads = (p.D + 3) / 4, chunks = p.L == 0 ? 1 : (p.L + TS - 1) / TS;
  const long long id = (long long)blockIdx.x * 128 + threadIdx.x;
  const int d = (int)(id % quads) * 4, chunk = (int)(id / quads % chunks), valid = min(4, p.D - d);
  const long long n_ = id / quads / chunks;
  if (n_ >= p.N) return;
  const int n = (int)n_, t0 = chunk * TS, t_end = min(p.L, t0 + TS);
  float w[K][4], b[4];
  load_taps<K>(p, d, valid, w, b);
  Chan4 win[K];       // x_{t-K+1} .. x_t
#pragma unroll
  for (int j = 1; j < K; ++j) {
    const int t = t0 - K + j;
    win[j] = input<T, K>(p, n, t, d, valid);
    if (t >= 0 && starts(p, n, t)) {
#pragma unroll
      for (int k = 1; k < j; ++k) win[k] = Chan4();
    }
  }
  constexpr int AH = TS < 4 ? TS : 4;       // steps loaded at a time
  const T* px = reinterpret_cast<const T*>(p.x.p) + n * p.x.sn + d;
  T* py = reinterpret_cast<T*>(p.y.p) + n * p.y.sn + d;
  Quad<T> next[AH];
  bool cut[AH];
#pragma unroll
  for (int k = 0; k < AH; ++k) {
    const int t = t0 + k;
    next[k].fetch(px + t * p.x.sl, p.x.vec, t < t_end ? valid : 0);
    cut[k] = t < t_end && starts(p, n, t);
  }
#pragma unroll
  for (int g = 0; g < TS; g += AH) {
    Quad<T> cur[AH];
    bool fresh[AH];
#pragma unroll
    for (int k = 0; k < AH; ++k) {
      cur[k] = next[k];
      fresh[k] = cut[k];
      const int t = t0 + g + AH + k;
      if (g + AH < TS) {
        next[k].fetch(px + t * p.x.sl, p.x.vec, t < t_end ? valid : 0);
        cut[k] = t < t_end && starts(p, n, t);
      }
    }
#pragma unroll
    for (int k = 0; k < AH; ++k) {
      const int t = t0 + g + k;
      if (t >= t_end) break;
#pragma unroll
      for (int j = 0; j + 1 < K; ++j) win[j] = fresh[k] ? Chan4() : win[j + 1];
      win[K - 1] = Chan4(cur[k].get(px + t * p.x.sl, p.x.vec, valid));
      Chan4 y;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float a = b[i];
#pragma unroll
        for (int j = 0; j < K; ++j) a = fmaf(w[j][i], win[j].v[i], a);
        y.v[i] = p.silu ? a * sigmoid(a) : a;
      }
      put4(py + t * p.y.sl, p.y.vec, valid, y.f4());
    }
  }
  if (t_end == p.L && p.sT.p) {
    T* ps = reinterpret_cast<T*>(p.sT.p) + n * p.sT.sn + d;
#pragma unroll
    for (int j = 1; j < K; ++j) put4(ps + (j - 1) * p.sT.sl, p.sT.vec, valid, win[j].f4());
  }
}

// A warp takes 32 quads of channels and a chunk of TS steps at a time, the block's four warps one chunk after another's; the sums of dw
// and dbias stay with the threads.  What the outputs behind the chunk give to its inputs comes from TS + K - 1 steps of dy.
template <typename T, int K, int TS>
__global__ void __launch_bounds__(128) conv_bwd_kernel(const ConvParams p) {
  __shared__ float4 red[4][32];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int d = ((int)blockIdx.x * 32 + lane) * 4, valid = max(0, min(4, p.D - d));
  const int chunks = (p.L + TS - 1) / TS;
  const long long units = (long long)p.N * chunks;
  float w[K][4], b[4], dw[K][4], db[4];
  load_taps<K>(p, d, valid, w, b);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    db[i] = 0.f;
#pragma unroll
    for (int j = 0; j < K; ++j) dw[j][i] = 0.f;
  }
  for (long long u = (long long)blockIdx.y * 4 + warp; u < units; u += (long long)gridDim.y * 4) {
    if (valid == 0) break;
    const int n = (int)(u / chunks), t0 = (int)(u % chunks) * TS, t_end = min(p.L, t0 + TS);
    // from the chunk's first step (the state's first row in front of the first chunk) on: dx[s] is whole once the step K - 1 behind it is done
    Chan4 win[K], acc[K];       // acc[j]: of the input at t - K + 1 + j
    int age = K - 1;            // steps since the episode's start, as far as they matter
#pragma unroll
    for (int j = 1; j < K; ++j) {
      const int t = t0 - K + j;
      win[j] = input<T, K>(p, n, t, d, valid);
      if (t >= 0) {
        const bool cut = starts(p, n, t);
        if (cut) {
#pragma unroll
          for (int k = 1; k < j; ++k) win[k] = Chan4();
        }
        age = cut ? 0 : min(K - 1, age + 1);
      }
    }
    const T* px = reinterpret_cast<const T*>(p.x.p) + n * p.x.sn + d;
    const T* py = reinterpret_cast<const T*>(p.dy.p) + n * p.dy.sn + d;
    T* ox = reinterpret_cast<T*>(p.dx.p) + n * p.dx.sn + d;
    constexpr int AH = 4;
    Quad<T> nx[AH], ny[AH];
    const int t_all = min(p.L, t_end + K - 1);     // steps whose outputs read the chunk's inputs
#pragma unroll
    for (int k = 0; k < AH; ++k) {
      const int t = t0 + k, v = t < t_all ? valid : 0;
      nx[k].fetch(px + t * p.x.sl, p.x.vec, v);
      ny[k].fetch(py + t * p.dy.sl, p.dy.vec, v);
    }
    for (int g = t0; g < t_end + K - 1; g += AH) {
      Quad<T> cx[AH], cy[AH];
#pragma unroll
      for (int k = 0; k < AH; ++k) {
        cx[k] = nx[k];
        cy[k] = ny[k];
        const int t = g + AH + k, v = t < t_all ? valid : 0;
        nx[k].fetch(px + t * p.x.sl, p.x.vec, v);
        ny[k].fetch(py + t * p.dy.sl, p.dy.vec, v);
      }
#pragma unroll
      for (int k = 0; k < AH; ++k) {
        const int t = g + k;
        if (t >= t_end + K - 1) break;
#pragma unroll
        for (int j = 0; j + 1 < K; ++j) acc[j] = acc[j + 1];
        acc[K - 1] = Chan4();
        if (t < p.L) {
          const bool fresh = starts(p, n, t);
          age = fresh ? 0 : min(K - 1, age + 1);
#pragma unroll
          for (int j = 0; j + 1 < K; ++j) win[j] = fresh ? Chan4() : win[j + 1];
          win[K - 1] = Chan4(cx[k].get(px + t * p.x.sl, p.x.vec, valid));
          const Chan4 go(cy[k].get(py + t * p.dy.sl, p.dy.vec, valid));
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float a = b[i];
#pragma unroll
            for (int j = 0; j < K; ++j) a = fmaf(w[j][i], win[j].v[i], a);
            float gp = go.v[i];
            if (p.silu) {
              const float sg = sigmoid(a);
              gp *= sg * fmaf(a, 1.f - sg, 1.f);
            }
#pragma unroll
            for (int j = 0; j < K; ++j)
              if (K - 1 - j <= age) acc[j].v[i] = fmaf(w[j][i], gp, acc[j].v[i]);
            if (t < t_end) {
              db[i] += gp;
#pragma unroll
              for (int j = 0; j < K; ++j) dw[j][i] = fmaf(gp, win[j].v[i], dw[j][i]);
            }
          }
        }
        const int s = t - (K - 1);      // the input whose gradient is whole now
        if (s >= t0 || t0 == 0) {
          Chan4 o = acc[0];
          if (s >= p.L - (K - 1) && p.dsT.p) {      // it is in the state behind the call, unless an episode began after it
            bool kept = true;
            for (int r = max(s + 1, 0); r < p.L; ++r) kept = kept && !starts(p, n, r);
            if (kept) {
              const T* pg = reinterpret_cast<const T*>(p.dsT.p) + n * p.dsT.sn + (long long)(s - (p.L - (K - 1))) * p.dsT.sl + d;
              Quad<T> qd;
              qd.fetch(pg, p.dsT.vec, valid);
              const Chan4 gs(qd.get(pg, p.dsT.vec, valid));
#pragma unroll
              for (int i = 0; i < 4; ++i) o.v[i] += gs.v[i];
            }
          }
          if (s >= t0) put4(ox + s * p.dx.sl, p.dx.vec, valid, o.f4());
          else if (p.ds0.p) put4(reinterpret_cast<T*>(p.ds0.p) + n * p.ds0.sn + (long long)(s + K - 1) * p.ds0.sl + d, p.ds0.vec, valid, o.f4());
        }
      }
    }
  }
  float* out = p.part + (long long)blockIdx.y * p.D * (K + 1);
#pragma unroll
  for (int j = 0; j <= K; ++j) {
    const float* v = j < K ? dw[j < K ? j : 0] : db;
    __syncthreads();
    red[warp][lane] = make_float4(v[0], v[1], v[2], v[3]);
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

// [parts][D][K + 1] -> dw [D][K], dbias [D]: 32 values a block, eight slices of the parts
__global__ void __launch_bounds__(256) conv_sums_kernel(const float* part, int parts, int D, int K, float* dw, float* dbias) {
  __shared__ float s[8][33];
  const int c = threadIdx.x % 32, slice = threadIdx.x / 32, total = D * (K + 1), i = blockIdx.x * 32 + c;
  float t = 0.f;
  if (i < total) {
#pragma unroll 4
    for (int b = slice; b < parts; b += 8) t += part[(long long)b * total + i];
  }
  s[slice][c] = t;
  __syncthreads();
  if (slice != 0 || i >= total) return;
#pragma unroll
  for (int k = 1; k < 8; ++k) t += s[k][c];
  const int d = i / (K + 1), j = i % (K + 1);
  if (j < K) dw[(long long)d * K + j] = t;
  else if (dbias) dbias[d] = t;
}

template <typename T, int K>
cudaError_t fwd(const ConvParams& p, cudaStream_t s) {
  const long long quads = (p.D + 3) / 4;
  auto run = [&](auto ts) {
    constexpr int TS = decltype(ts)::value;
    const long long chunks = p.L == 0 ? 1 : (p.L + TS - 1) / TS, blocks = (quads * chunks * p.N + 127) / 128;
    return launch_behind(conv_fwd_kernel<T, K, TS>, p, dim3((unsigned)blocks), 128, 0, s);
  };
  if (p.L <= 1) return run(std::integral_constant<int, 1>());
  return run(std::integral_constant<int, CONV_CHUNK>());
}
template <typename T, int K>
cudaError_t bwd(const ConvParams& p, cudaStream_t s) {
  const int parts = conv_parts(p);
  conv_bwd_kernel<T, K, CONV_CHUNK><<<dim3((unsigned)((p.D + 127) / 128), (unsigned)parts), 128, 0, s>>>(p);
  if (const cudaError_t e = cudaGetLastError(); e != cudaSuccess) return e;
  conv_sums_kernel<<<(unsigned)((p.D * (K + 1) + 31) / 32), 256, 0, s>>>(p.part, parts, p.D, K, p.dw, p.dbias);
  return cudaGetLastError();
}
template <typename F>
cudaError_t by_type(const ConvParams& p, F f) {
  auto taps = [&](auto t) {
    switch (p.K) {
      case 2: return f(t, std::integral_constant<int, 2>());
      case 3: return f(t, std::integral_constant<int, 3>());
      default: return f(t, std::integral_constant<int, 4>());
    }
  };
  return p.bf16 ? taps(__nv_bfloat16()) : taps(float());
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
  return by_type(p, [&](auto t, auto k) { return fwd<decltype(t), decltype(k)::value>(p, s); });
}
cudaError_t conv_backward(const ConvParams& p, cudaStream_t s) {
  return by_type(p, [&](auto t, auto k) { return bwd<decltype(t), decltype(k)::value>(p, s); });
}

}  // namespace srwm
