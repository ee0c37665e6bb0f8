// Causal convolution of a few steps along time (conv.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "scan.h"

namespace srwm {

constexpr int CONV_CHUNK = 16;     // steps of a thread at least (a shorter call is one chunk)

struct ConvParams {
  int N, L, D, K;
  int chunk;                       // steps of a thread (set by the launch)
  int bf16, silu, vec;             // vec: all rows' pieces of four channels are aligned to their size
  ScanRows x, y, s0, sT;           // [N, L, D]; the states [N, K-1, D], NULL: zeros / not wanted
  const float *w, *bias;           // [D, K], [D] or NULL
  const uint8_t* done;
  long long done_n, done_l;
  // backward
  ScanRows dy, dx, dsT, ds0;
  float *dw, *dbias, *part;
};
int conv_parts(const ConvParams& p);          // the backward's partial sums [conv_parts][D][K + 1]
cudaError_t conv_forward(const ConvParams& p, cudaStream_t s);
cudaError_t conv_backward(const ConvParams& p, cudaStream_t s);

}  // namespace srwm
