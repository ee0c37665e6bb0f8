// Root-mean-square norm over the last dimension with the residual's addition (rms.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace srwm {

constexpr int RMS_MAX_D = 8192;

struct RmsParams {
  const void *x, *res;             // [rows, D] with row strides in elements; res NULL: none
  long long x_row, res_row;
  const float* w;                  // [D]
  void* y;                         // dense, x's type or e4m3
  void* sum;                       // x + res rounded to x's type, dense; NULL: not wanted
  float *rstd, *scale;             // [rows]; rstd NULL: not wanted; scale: with e4m3
  long long rows;
  int D, bf16, fp8;
  float eps;
  // backward: sum is read, y is the gradient of x and res
  const void *dy, *dsum;           // dsum NULL: none
  long long dy_row, dsum_row, sum_row;
  float *dw, *part;
};
int rms_blocks(long long rows, int D);
cudaError_t rms_forward(const RmsParams& p, cudaStream_t s);
cudaError_t rms_backward(const RmsParams& p, cudaStream_t s);

}  // namespace srwm
