// Norm over many tensors and clipping by it (grads.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace srwm {

constexpr int GRADS_CHUNK = 8192;        // values of a tensor that a block takes at a time

struct GradTensor {
  void* p;
  long long n;
  int bf16;
};
int grads_parts(const GradTensor* t, int count);       // doubles of working memory
cudaError_t grads_norm(const GradTensor* t, int count, double* part, float* norm, cudaStream_t s);
cudaError_t grads_clip(const GradTensor* t, int count, const double* part, float max_norm, float* norm, cudaStream_t s);

}  // namespace srwm
