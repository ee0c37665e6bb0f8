// Root-mean-square norm with the residual's addition:
//   s = x + res (rounded to their type: the stream that the next block reads),  y = s rstd w,  rstd = (mean s^2 + eps)^-1/2
// y in the type of x, or in e4m3 with one scale a row: scale = max |y| / 448 (at least 2^-126), y / scale rounded to nearest.
//
// Bound by HBM: x and res in, s and y out, once each (16384 x 512 fp32 with the residual: forward 19 us, backward 20 + 4, 20.5 each
// at the copy bandwidth, which L2 has part of in passes one after another; loads behind branches instead of predicates took 29 and 55).  A row stays in registers between its sum and its result: up to 1024 columns with a
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

// A row's threads: a warp (some rows a block) or the whole block
template <bool BLOCK, int THREADS = 256>
struct Team {
  static constexpr int SIZE = BLOCK ? 256 : 32, ROWS = THREADS / SIZE;
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

template <bool VEC, typename T>
__device__ __forceinline__ float4 row4(const T* p, int valid) {
  Quad<T, VEC> q;
  q.fetch(p, valid);
  return q.get();
}
template <typename T>
__device__ __forceinline__ float4 rounded(float4 v) {
  if constexpr (sizeof(T) == 2) {
    const uint2 r = make_uint2(f32x2_to_bf16x2(v.x, v.y), f32x2_to_bf16x2(v.z, v.w));
    return widen(r);
  }
  return v;
}
inline bool quads_ok(const void* p, long long row, int D, int es) { return (uintptr_t)p % (4 * es) == 0 && row % 4 == 0 && D % 4 == 0; }

// NV: pieces of four columns of a thread
template <typename T, bool VEC, bool BLOCK, int NV, bool FP8>
__global__ void __launch_bounds__(BLOCK ? 256 : 128) rms_fwd_kernel(const RmsParams p) {
  chained();
  using G = Team<BLOCK, BLOCK ? 256 : 128>;
  __shared__ float red[8];
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
      v[i] = row4<VEC>(px + c, valid);
      if (p.res != nullptr) {
        const float4 r = row4<VEC>(pr + c, valid);
        v[i] = rounded<T>(make_float4(v[i].x + r.x, v[i].y + r.y, v[i].z + r.z, v[i].w + r.w));
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * G::SIZE + lane) * 4, valid = min(4, p.D - c);
      if (p.sum != nullptr) put4<VEC>(reinterpret_cast<T*>(p.sum) + row * p.D + c, valid, v[i]);
      q += (v[i].x * v[i].x + v[i].y * v[i].y) + (v[i].z * v[i].z + v[i].w * v[i].w);
    }
    const float rstd = rsqrtf(G::sum(q, red) * inv_d + p.eps);
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * G::SIZE + lane) * 4, valid = min(4, p.D - c);
      const float4 w = row4<VEC>(p.w + c, valid);
      v[i] = make_float4(v[i].x * rstd * w.x, v[i].y * rstd * w.y, v[i].z * rstd * w.z, v[i].w * rstd * w.w);
      if constexpr (FP8) {
        // (as bits, so that NaN stays on top)
        const unsigned m = max(max(__float_as_uint(fabsf(v[i].x)), __float_as_uint(fabsf(v[i].y))),
                               max(__float_as_uint(fabsf(v[i].z)), __float_as_uint(fabsf(v[i].w))));
        top = __uint_as_float(max(__float_as_uint(top), m));
      } else {
        put4<VEC>(reinterpret_cast<T*>(p.y) + row * p.D + c, valid, v[i]);
      }
    }
    if constexpr (FP8) {
      top = G::top(top, red);
      float scale = __fdiv_rn(top, 448.f);
      if (scale < 1.17549435e-38f) scale = 1.17549435e-38f;
      const float inv = __frcp_rn(scale);      // (2^126 at most; its rounding moves a value by 2^-24 in front of one to 2^-4)
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * G::SIZE + lane) * 4, valid = min(4, p.D - c);
        const unsigned lo = __nv_cvt_float2_to_fp8x2(make_float2(v[i].x * inv, v[i].y * inv), __NV_SATFINITE, __NV_E4M3);
        const unsigned hi = __nv_cvt_float2_to_fp8x2(make_float2(v[i].z * inv, v[i].w * inv), __NV_SATFINITE, __NV_E4M3);
        const unsigned b = lo | hi << 16;
        uint8_t* o = reinterpret_cast<uint8_t*>(p.y) + row * p.D + c;
        if (VEC) {
          if (valid > 0) *reinterpret_cast<unsigned*>(o) = b;
        } else {
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

template <typename T, bool VEC, bool BLOCK, int NV>
__global__ void __launch_bounds__(256) rms_bwd_kernel(const RmsParams p) {
  using G = Team<BLOCK>;
  __shared__ float red[8];
  __shared__ float4 add[BLOCK ? 1 : 8][32];
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
      const float4 x = row4<VEC>(reinterpret_cast<const T*>(p.sum) + row * p.sum_row + c, valid);
      const float4 d = row4<VEC>(reinterpret_cast<const T*>(p.dy) + row * p.dy_row + c, valid);
      o[i] = p.dsum ? row4<VEC>(reinterpret_cast<const T*>(p.dsum) + row * p.dsum_row + c, valid) : make_float4(0.f, 0.f, 0.f, 0.f);
      const float4 w = row4<VEC>(p.w + c, valid);
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
      put4<VEC>(reinterpret_cast<T*>(p.y) + row * p.D + c, valid,
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
    put4<VEC>(out + c, min(4, p.D - c), t);
  }
}

struct RmsSums {
  const float* part;
  float* dw;
  int blocks, D;
};
// [blocks][D] -> dw: 32 columns a block, 32 slices
__global__ void __launch_bounds__(1024) rms_sums_kernel(const RmsSums a) {
  chained();
  __shared__ float s[32][33];
  const int col = threadIdx.x % 32, slice = threadIdx.x / 32;
  int c = blockIdx.x * 32 + col;
  float t = 0.f;
  if (c < a.D) {
#pragma unroll 8
    for (int b = slice; b < a.blocks; b += 32) t += a.part[(long long)b * a.D + c];
  }
  s[slice][col] = t;
  __syncthreads();
  t = allreduce_warp(s[col][slice]);
  if (col == 0 && (c = blockIdx.x * 32 + slice) < a.D) a.dw[c] = t;
}

// f(element, VEC, BLOCK, NV)
template <typename T, bool VEC, typename F>
cudaError_t by_width(int D, F& f) {
  using std::integral_constant;
  const std::bool_constant<VEC> vec;
  const std::false_type warp;
  const std::true_type block;
  if (D <= 128) return f(T(), vec, warp, integral_constant<int, 1>());
  if (D <= 256) return f(T(), vec, warp, integral_constant<int, 2>());
  if (D <= 512) return f(T(), vec, warp, integral_constant<int, 4>());
  if (D <= 1024) return f(T(), vec, warp, integral_constant<int, 8>());
  if (D <= 2048) return f(T(), vec, block, integral_constant<int, 2>());
  if (D <= 4096) return f(T(), vec, block, integral_constant<int, 4>());
  return f(T(), vec, block, integral_constant<int, 8>());
}
template <typename F>
cudaError_t by_rows(const RmsParams& p, bool vec, F f) {
  if (p.bf16) return vec ? by_width<__nv_bfloat16, true>(p.D, f) : by_width<__nv_bfloat16, false>(p.D, f);
  return vec ? by_width<float, true>(p.D, f) : by_width<float, false>(p.D, f);
}

}  // namespace

// Two blocks of a multiprocessor, all resident, each with a part of dw to be added up; fewer rows, fewer blocks
int rms_blocks(long long rows, int D) {
  const long long per = D <= 1024 ? 8 : 1, b = (rows + per - 1) / per, most = 2ll * common_sms();
  return (int)(b < most ? b : most);
}
cudaError_t rms_forward(const RmsParams& p, cudaStream_t s) {
  const int es = p.bf16 ? 2 : 4;
  const bool vec = quads_ok(p.x, p.x_row, p.D, es) && quads_ok(p.res, p.res_row, p.D, es) && quads_ok(p.y, 0, p.D, p.fp8 ? 1 : es) &&
                   quads_ok(p.sum, 0, p.D, es) && quads_ok(p.w, 0, p.D, 4);
  return by_rows(p, vec, [&](auto t, auto v, auto block, auto nv) {
    using T = decltype(t);
    constexpr bool V = decltype(v)::value, B = decltype(block)::value;
    constexpr int NV = decltype(nv)::value;
    constexpr int THREADS = B ? 256 : 128, ROWS = Team<B, THREADS>::ROWS;
    const long long blocks = (p.rows + ROWS - 1) / ROWS, most = 32ll * common_sms();
    const dim3 grid((unsigned)(blocks < most ? blocks : most));
    return p.fp8 ? launch_behind(rms_fwd_kernel<T, V, B, NV, true>, p, grid, THREADS, 0, s)
                 : launch_behind(rms_fwd_kernel<T, V, B, NV, false>, p, grid, THREADS, 0, s);
  });
}
cudaError_t rms_backward(const RmsParams& p, cudaStream_t s) {
  const int es = p.bf16 ? 2 : 4, blocks = rms_blocks(p.rows, p.D);
  const bool vec = quads_ok(p.dy, p.dy_row, p.D, es) && quads_ok(p.dsum, p.dsum_row, p.D, es) && quads_ok(p.y, 0, p.D, es) &&
                   quads_ok(p.sum, p.sum_row, p.D, es) && quads_ok(p.w, 0, p.D, 4) && quads_ok(p.part, 0, p.D, 4);
  const cudaError_t e = by_rows(p, vec, [&](auto t, auto v, auto block, auto nv) {
    rms_bwd_kernel<decltype(t), decltype(v)::value, decltype(block)::value, decltype(nv)::value><<<blocks, 256, 0, s>>>(p);
    return cudaGetLastError();
  });
  if (e != cudaSuccess) return e;
  return launch_behind(rms_sums_kernel, RmsSums{p.part, p.dw, blocks, p.D}, dim3((p.D + 31) / 32), 1024, 0, s);
}

}  // namespace srwm
