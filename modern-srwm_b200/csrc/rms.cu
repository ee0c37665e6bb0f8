// Root-mean-square norm with the residual's addition:
//   s = x + res (rounded to their type: the stream that the next block reads),  y = s rstd w,  rstd = (mean s^2 + eps)^-1/2
// y in the type of x, or in e4m3 with one scale a row: scale = max |y| / 448 (at least 2^-126), y / scale rounded to nearest.
//
// Bound by HBM: x and res in, s and y out, once each.  A row stays in registers between its sum and its result: up to 1024 columns with a
// warp, above with a block of eight warps.  The weight's gradient is kept per thread over all rows of a block and added up over
// the blocks by a second launch, in a fixed order.
#include "rms.h"

#include <cuda_fp8.h>

#include <type_traits>

#include "chain.h"
#include "device.h"
#include "scan.cuh"

namespace srwm {
namespace {
using namespace scan;

// A row's threads: a warp (eight rows a block) or the whole block
template <bool BLOCK>
struct Team {
  static constexpr int SIZE = BLOCK ? 256 : 32, ROWS = 256 / SIZE;
  static __device__ __forceinline__ float sum(float v, float* red) {
    v = allreduce_warp(v);
    if constexpr (BLOCK) {
      __syncthreads();       // (red is used again)
      if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = v;
      __syncthreads();
      v = ((red[0] + red[1]) + (red[2] + red[3])) + ((red[4] + red[5]) + (red[6] + red[7]));
    }
    return v;
  }
  // the largest, NaN where one is among them (bits of values that are not negative order as they do, with NaN on top)
  static __device__ __forceinline__ float top(float v, float* red) {
    v = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v)));
    if constexpr (BLOCK) {
      __syncthreads();
      if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = v;
      __syncthreads();
      unsigned m = __float_as_uint(red[0]);
#pragma unroll
      for (int i = 1; i < 8; ++i) m = max(m, __float_as_uint(red[i]));
      v = __uint_as_float(m);
    }
    return v;
  }
};

template <typename T>
__device__ __forceinline__ float4 row4(const T* p, bool vec, int valid) {
  Quad<T> q;
  q.fetch(p, vec, valid);
  return q.get(p, vec, valid);
}
template <typename T>
__device__ __forceinline__ float4 rounded(float4 v) {
  if constexpr (sizeof(T) == 2) {
    const uint2 r = make_uint2(f32x2_to_bf16x2(v.x, v.y), f32x2_to_bf16x2(v.z, v.w));
    return widen(r);
  }
  return v;
}
template <typename T>
inline bool quads_ok(const void* p, long long row, int D) {
  return (uintptr_t)p % (4 * sizeof(T)) == 0 && row % 4 == 0 && D % 4 == 0;
}

struct RmsLaunch {
  RmsParams p;
  int vx, vr, vy, vs, vw, vg;     // rows of x, res, y, sum, w, dsum in pieces of four
};

// NV: pieces of four columns of a thread
template <typename T, bool BLOCK, int NV, bool FP8>
__global__ void __launch_bounds__(256) rms_fwd_kernel(const RmsLaunch a) {
  chained();
  using G = Team<BLOCK>;
  __shared__ float red[8];
  const RmsParams& p = a.p;
  const int lane = threadIdx.x % G::SIZE, sub = threadIdx.x / G::SIZE;
  const float inv_d = 1.f / (float)p.D;
  for (long long row = (long long)blockIdx.x * G::ROWS + sub; row < p.rows; row += (long long)gridDim.x * G::ROWS) {
    const T* px = reinterpret_cast<const T*>(p.x) + row * p.x_row;
    const T* pr = reinterpret_cast<const T*>(p.res) + row * p.res_row;
    float4 v[NV];
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * G::SIZE + lane) * 4, valid = min(4, p.D - c);
      v[i] = row4(px + c, a.vx, valid);
      if (p.res != nullptr) {
        const float4 r = row4(pr + c, a.vr, valid);
        v[i] = rounded<T>(make_float4(v[i].x + r.x, v[i].y + r.y, v[i].z + r.z, v[i].w + r.w));
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * G::SIZE + lane) * 4, valid = min(4, p.D - c);
      if (p.sum != nullptr && valid > 0) put4(reinterpret_cast<T*>(p.sum) + row * p.D + c, a.vs, valid, v[i]);
      q += (v[i].x * v[i].x + v[i].y * v[i].y) + (v[i].z * v[i].z + v[i].w * v[i].w);
    }
    const float rstd = rsqrtf(G::sum(q, red) * inv_d + p.eps);
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * G::SIZE + lane) * 4, valid = min(4, p.D - c);
      const float4 w = row4(p.w + c, a.vw, valid);
      v[i] = make_float4(v[i].x * rstd * w.x, v[i].y * rstd * w.y, v[i].z * rstd * w.z, v[i].w * rstd * w.w);
      if constexpr (FP8) {
        // (as bits, so that NaN stays on top)
        const unsigned m = max(max(__float_as_uint(fabsf(v[i].x)), __float_as_uint(fabsf(v[i].y))),
                               max(__float_as_uint(fabsf(v[i].z)), __float_as_uint(fabsf(v[i].w))));
        top = __uint_as_float(max(__float_as_uint(top), m));
      } else if (valid > 0) {
        put4(reinterpret_cast<T*>(p.y) + row * p.D + c, a.vy, valid, v[i]);
      }
    }
    if constexpr (FP8) {
      top = G::top(top, red);
      float scale = __fdiv_rn(top, 448.f);
      if (scale < 1.17549435e-38f) scale = 1.17549435e-38f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * G::SIZE + lane) * 4, valid = min(4, p.D - c);
        const unsigned lo = __nv_cvt_float2_to_fp8x2(make_float2(__fdiv_rn(v[i].x, scale), __fdiv_rn(v[i].y, scale)), __NV_SATFINITE, __NV_E4M3);
        const unsigned hi = __nv_cvt_float2_to_fp8x2(make_float2(__fdiv_rn(v[i].z, scale), __fdiv_rn(v[i].w, scale)), __NV_SATFINITE, __NV_E4M3);
        const unsigned b = lo | hi << 16;
        uint8_t* o = reinterpret_cast<uint8_t*>(p.y) + row * p.D + c;
        if (a.vy && valid > 0) *reinterpret_cast<unsigned*>(o) = b;
        else {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (k < valid) o[k] = (uint8_t)(b >> 8 * k);
        }
      }
      if (lane == 0) p.scale[row] = scale;
    }
    if (lane == 0 && p.rstd != nullptr) p.rstd[row] = rstd;
  }
}

template <typename T, bool BLOCK, int NV>
__global__ void __launch_bounds__(256) rms_bwd_kernel(const RmsLaunch a) {
  using G = Team<BLOCK>;
  __shared__ float red[8];
  __shared__ float4 add[BLOCK ? 1 : 8][32];
  const RmsParams& p = a.p;
  const int lane = threadIdx.x % G::SIZE, sub = threadIdx.x / G::SIZE;
  const float inv_d = 1.f / (float)p.D;
  float4 gw[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) gw[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (long long row = (long long)blockIdx.x * G::ROWS + sub; row < p.rows; row += (long long)gridDim.x * G::ROWS) {
    const float rstd = p.rstd[row];
    float4 xh[NV], g[NV], o[NV];
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * G::SIZE + lane) * 4, valid = min(4, p.D - c);
      const float4 x = row4(reinterpret_cast<const T*>(p.sum) + row * p.sum_row + c, a.vs, valid);
      const float4 d = row4(reinterpret_cast<const T*>(p.dy) + row * p.dy_row + c, a.vx, valid);
      o[i] = p.dsum ? row4(reinterpret_cast<const T*>(p.dsum) + row * p.dsum_row + c, a.vg, valid) : make_float4(0.f, 0.f, 0.f, 0.f);
      const float4 w = row4(p.w + c, a.vw, valid);
      xh[i] = make_float4(x.x * rstd, x.y * rstd, x.z * rstd, x.w * rstd);
      gw[i].x = fmaf(d.x, xh[i].x, gw[i].x); gw[i].y = fmaf(d.y, xh[i].y, gw[i].y);
      gw[i].z = fmaf(d.z, xh[i].z, gw[i].z); gw[i].w = fmaf(d.w, xh[i].w, gw[i].w);
      g[i] = make_float4(d.x * w.x, d.y * w.y, d.z * w.z, d.w * w.w);
      s += (g[i].x * xh[i].x + g[i].y * xh[i].y) + (g[i].z * xh[i].z + g[i].w * xh[i].w);
    }
    const float m = G::sum(s, red) * inv_d;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * G::SIZE + lane) * 4, valid = min(4, p.D - c);
      if (valid <= 0) continue;
      put4(reinterpret_cast<T*>(p.y) + row * p.D + c, a.vy, valid,
           make_float4(fmaf(rstd, g[i].x - xh[i].x * m, o[i].x), fmaf(rstd, g[i].y - xh[i].y * m, o[i].y),
                       fmaf(rstd, g[i].z - xh[i].z * m, o[i].z), fmaf(rstd, g[i].w - xh[i].w * m, o[i].w)));
    }
  }
  float* out = p.part + (long long)blockIdx.x * p.D;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * G::SIZE + lane) * 4;
    float4 t = gw[i];
    if constexpr (!BLOCK) {
      __syncthreads();
      add[sub][lane] = t;
      __syncthreads();
      if (sub != 0) continue;
#pragma unroll
      for (int k = 1; k < 8; ++k) {
        const float4 v = add[k][lane];
        t.x += v.x; t.y += v.y; t.z += v.z; t.w += v.w;
      }
    }
    if (c < p.D) put4(out + c, 0, min(4, p.D - c), t);
  }
}

// [blocks][D] -> dw: 32 columns a block, eight slices
__global__ void __launch_bounds__(256) rms_sums_kernel(const float* part, int blocks, int D, float* dw) {
  __shared__ float s[8][33];
  const int col = threadIdx.x % 32, slice = threadIdx.x / 32, c = blockIdx.x * 32 + col;
  float t = 0.f;
  if (c < D) {
#pragma unroll 4
    for (int b = slice; b < blocks; b += 8) t += part[(long long)b * D + c];
  }
  s[slice][col] = t;
  __syncthreads();
  if (slice != 0 || c >= D) return;
#pragma unroll
  for (int k = 1; k < 8; ++k) t += s[k][col];
  dw[c] = t;
}

template <typename F>
cudaError_t by_width(int D, F f) {
  using std::integral_constant;
  if (D <= 128) return f(std::false_type(), integral_constant<int, 1>());
  if (D <= 256) return f(std::false_type(), integral_constant<int, 2>());
  if (D <= 512) return f(std::false_type(), integral_constant<int, 4>());
  if (D <= 1024) return f(std::false_type(), integral_constant<int, 8>());
  if (D <= 2048) return f(std::true_type(), integral_constant<int, 2>());
  if (D <= 4096) return f(std::true_type(), integral_constant<int, 4>());
  return f(std::true_type(), integral_constant<int, 8>());
}

template <typename T>
cudaError_t forward(const RmsParams& p, cudaStream_t s) {
  RmsLaunch a = {p};
  a.vx = quads_ok<T>(p.x, p.x_row, p.D);
  a.vr = quads_ok<T>(p.res, p.res_row, p.D);
  a.vy = p.fp8 ? (uintptr_t)p.y % 4 == 0 && p.D % 4 == 0 : quads_ok<T>(p.y, p.D, p.D);
  a.vs = quads_ok<T>(p.sum, p.D, p.D);
  a.vw = quads_ok<float>(p.w, 0, p.D);
  return by_width(p.D, [&](auto block, auto nv) {
    constexpr bool B = decltype(block)::value;
    constexpr int NV = decltype(nv)::value;
    const long long blocks = (p.rows + Team<B>::ROWS - 1) / Team<B>::ROWS, most = 16ll * common_sms();
    const dim3 grid((unsigned)(blocks < most ? blocks : most));
    return p.fp8 ? launch_behind(rms_fwd_kernel<T, B, NV, true>, a, grid, 256, 0, s)
                 : launch_behind(rms_fwd_kernel<T, B, NV, false>, a, grid, 256, 0, s);
  });
}
template <typename T>
cudaError_t backward(const RmsParams& p, cudaStream_t s) {
  RmsLaunch a = {p};
  a.vx = quads_ok<T>(p.dy, p.dy_row, p.D);
  a.vg = quads_ok<T>(p.dsum, p.dsum_row, p.D);
  a.vy = quads_ok<T>(p.y, p.D, p.D);
  a.vs = quads_ok<T>(p.sum, p.sum_row, p.D);
  a.vw = quads_ok<float>(p.w, 0, p.D);
  const int blocks = rms_blocks(p.rows, p.D);
  const cudaError_t e = by_width(p.D, [&](auto block, auto nv) {
    rms_bwd_kernel<T, decltype(block)::value, decltype(nv)::value><<<blocks, 256, 0, s>>>(a);
    return cudaGetLastError();
  });
  if (e != cudaSuccess) return e;
  rms_sums_kernel<<<(p.D + 31) / 32, 256, 0, s>>>(p.part, blocks, p.D, p.dw);
  return cudaGetLastError();
}

}  // namespace

// Four blocks of a multiprocessor, each with a part of dw to be added up; fewer rows, fewer blocks
int rms_blocks(long long rows, int D) {
  const long long per = D <= 1024 ? 8 : 1, b = (rows + per - 1) / per, most = 4ll * common_sms();
  return (int)(b < most ? b : most);
}
cudaError_t rms_forward(const RmsParams& p, cudaStream_t s) {
  return p.bf16 ? forward<__nv_bfloat16>(p, s) : forward<float>(p, s);
}
cudaError_t rms_backward(const RmsParams& p, cudaStream_t s) {
  return p.bf16 ? backward<__nv_bfloat16>(p, s) : backward<float>(p, s);
}

}  // namespace srwm
