// The 2-norm over all values of many tensors, and their scaling by min(1, max_norm / (norm + 1e-6)).
//
// Bound by HBM: the tensors are read for the norm, and read and written for the scaling.  A launch takes up to 64 (or 1024) tensors: their
// addresses are its arguments, cut into chunks of 8192 values that the blocks take in turn.  Squares are added in fp32 over
// 32 values of a thread, in fp64 from there on, in a fixed order; each block leaves one sum, and every block of the
// scaling adds all of those again (a few KB).  The scaling goes through the chunks backwards: the last ones read are still in L2.
// 160 M fp32 values: norm 104 us (6.15 TB/s), scaling 208 (6.15 TB/s).
#include "grads.h"

#include "chain.h"
#include "common.cuh"
#include "device.h"

namespace srwm {
namespace {

constexpr int THREADS = 256;

template <int MOST>
struct Table {
  void* ptr[MOST];
  long long n[MOST];
  int first[MOST + 1];          // of each tensor's chunks
  unsigned half[MOST / 32];     // bits: bf16
  int count, parts, all_parts, write;
  double* part;                 // this launch's sums
  const double* all;            // every launch's
  float max_norm;
  float* norm;
};

// Tensor of a chunk, by halves
template <int MOST>
__device__ __forceinline__ int tensor_of(const Table<MOST>& t, int chunk) {
  int lo = 0, hi = t.count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (t.first[mid] <= chunk) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ double sum_block(double v, double* red) {
#pragma unroll
  for (int w = 16; w > 0; w /= 2) v += __shfl_xor_sync(0xffffffffu, v, w);
  if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int i = 1; i < THREADS / 32; ++i) v += red[i];
  return v;
}

template <int MOST>
__global__ void __launch_bounds__(THREADS) grads_norm_kernel(const __grid_constant__ Table<MOST> t) {
  __shared__ double red[THREADS / 32];
  double sum = 0.;
  for (int c = blockIdx.x; c < t.first[t.count]; c += gridDim.x) {
    const int k = tensor_of(t, c);
    const long long at = (long long)(c - t.first[k]) * GRADS_CHUNK;
    const int n = (int)min((long long)GRADS_CHUNK, t.n[k] - at), tid = threadIdx.x;
    float s = 0.f;
    if (t.half[k / 32] >> k % 32 & 1u) {
      const __nv_bfloat16* p = reinterpret_cast<const __nv_bfloat16*>(t.ptr[k]) + at;
      int done = 0;
      if ((uintptr_t)p % 16 == 0) {
        done = n / 8 * 8;
#pragma unroll 4
        for (int i = tid * 8; i < done; i += THREADS * 8) {
          float v[8];
          ld_vec<8>(p + i, v);
#pragma unroll
          for (int j = 0; j < 8; ++j) s = fmaf(v[j], v[j], s);
        }
      }
      for (int i = done + tid; i < n; i += THREADS) {
        const float v = __bfloat162float(p[i]);
        s = fmaf(v, v, s);
      }
    } else {
      const float* p = reinterpret_cast<const float*>(t.ptr[k]) + at;
      int done = 0;
      if ((uintptr_t)p % 16 == 0) {
        done = n / 4 * 4;
#pragma unroll 8
        for (int i = tid * 4; i < done; i += THREADS * 4) {
          const float4 v = *reinterpret_cast<const float4*>(p + i);
          s = fmaf(v.x, v.x, s); s = fmaf(v.y, v.y, s); s = fmaf(v.z, v.z, s); s = fmaf(v.w, v.w, s);
        }
      }
      for (int i = done + tid; i < n; i += THREADS) s = fmaf(p[i], p[i], s);
    }
    sum += (double)s;
  }
  sum = sum_block(sum, red);
  if (threadIdx.x == 0) t.part[blockIdx.x] = sum;
}

template <int MOST>
__global__ void __launch_bounds__(THREADS) grads_scale_kernel(const __grid_constant__ Table<MOST> t) {
  chained();
  __shared__ double red[THREADS / 32];
  double sum = 0.;
  for (int i = threadIdx.x; i < t.all_parts; i += THREADS) sum += t.all[i];
  const float norm = (float)sqrt(sum_block(sum, red));
  if (blockIdx.x == 0 && threadIdx.x == 0 && t.norm) *t.norm = norm;
  const float coef = __fdiv_rn(t.max_norm, norm + 1e-6f);
  if (!t.write || coef >= 1.f) return;      // (a NaN goes into every value)
  const int chunks = t.first[t.count];
  for (int b = blockIdx.x; b < chunks; b += gridDim.x) {
    const int c = chunks - 1 - b, k = tensor_of(t, c);
    const long long at = (long long)(c - t.first[k]) * GRADS_CHUNK;
    const int n = (int)min((long long)GRADS_CHUNK, t.n[k] - at), tid = threadIdx.x;
    if (t.half[k / 32] >> k % 32 & 1u) {
      __nv_bfloat16* p = reinterpret_cast<__nv_bfloat16*>(t.ptr[k]) + at;
      int done = 0;
      if ((uintptr_t)p % 16 == 0) {
        done = n / 8 * 8;
#pragma unroll 4
        for (int i = tid * 8; i < done; i += THREADS * 8) {
          float v[8];
          ld_vec<8>(p + i, v);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] *= coef;
          st_vec<8>(p + i, v);
        }
      }
      for (int i = done + tid; i < n; i += THREADS) p[i] = __float2bfloat16_rn(__bfloat162float(p[i]) * coef);
    } else {
      float* p = reinterpret_cast<float*>(t.ptr[k]) + at;
      int done = 0;
      if ((uintptr_t)p % 16 == 0) {
        done = n / 4 * 4;
#pragma unroll 8
        for (int i = tid * 4; i < done; i += THREADS * 4) {
          float4 v = *reinterpret_cast<const float4*>(p + i);
          v.x *= coef; v.y *= coef; v.z *= coef; v.w *= coef;
          *reinterpret_cast<float4*>(p + i) = v;
        }
      }
      for (int i = done + tid; i < n; i += THREADS) p[i] *= coef;
    }
  }
}

constexpr int FEW = 64, MANY = 1024;

int blocks_for(long long chunks) {
  const long long most = 8ll * common_sms();
  return (int)(chunks < 1 ? 1 : chunks < most ? chunks : most);
}
long long chunks_of(const GradTensor* t, int count) {
  long long c = 0;
  for (int i = 0; i < count; ++i) c += (t[i].n + GRADS_CHUNK - 1) / GRADS_CHUNK;
  return c;
}
template <int MOST>
void fill(Table<MOST>& a, const GradTensor* t, int count) {
  a = {};
  a.count = count;
  for (int i = 0; i < count; ++i) {
    a.ptr[i] = t[i].p;
    a.n[i] = t[i].n;
    a.first[i + 1] = a.first[i] + (int)((t[i].n + GRADS_CHUNK - 1) / GRADS_CHUNK);
    if (t[i].bf16) a.half[i / 32] |= 1u << i % 32;
  }
}
// f(table with `count` tensors from t on, blocks) for each launch
template <typename F>
cudaError_t each(const GradTensor* t, int count, F f) {
  if (count <= FEW) {
    Table<FEW> a;
    fill(a, t, count);
    return f(a, blocks_for(a.first[count]));
  }
  for (int i = 0; i < count; i += MANY) {
    Table<MANY> a;
    const int n = count - i < MANY ? count - i : MANY;
    fill(a, t + i, n);
    if (const cudaError_t e = f(a, blocks_for(a.first[n])); e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace

int grads_parts(const GradTensor* t, int count) {
  if (count <= FEW) return blocks_for(chunks_of(t, count));
  int parts = 0;
  for (int i = 0; i < count; i += MANY) parts += blocks_for(chunks_of(t + i, count - i < MANY ? count - i : MANY));
  return parts;
}
cudaError_t grads_norm(const GradTensor* t, int count, double* part, float* norm, cudaStream_t s) {
  int at = 0;
  const cudaError_t e = each(t, count, [&](auto& a, int blocks) {
    a.part = part + at;
    at += blocks;
    constexpr int MOST = sizeof(a.half) / 4 * 32;
    grads_norm_kernel<MOST><<<blocks, THREADS, 0, s>>>(a);
    return cudaGetLastError();
  });
  if (e != cudaSuccess || !norm) return e;
  Table<FEW> a = {};
  a.all = part;
  a.all_parts = at;
  a.norm = norm;
  return launch_behind(grads_scale_kernel<FEW>, a, dim3(1), THREADS, 0, s);
}
cudaError_t grads_clip(const GradTensor* t, int count, const double* part, float max_norm, float* norm, cudaStream_t s) {
  const int parts = grads_parts(t, count);
  bool first = true;
  return each(t, count, [&](auto& a, int blocks) {
    a.all = part;
    a.all_parts = parts;
    a.write = 1;
    a.max_norm = max_norm;
    a.norm = first ? norm : nullptr;
    constexpr int MOST = sizeof(a.half) / 4 * 32;
    const cudaError_t e = launch_behind(grads_scale_kernel<MOST>, a, dim3(blocks), THREADS, 0, s);
    first = false;
    return e;
  });
}

}  // namespace srwm
