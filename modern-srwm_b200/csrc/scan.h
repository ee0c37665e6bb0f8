// Selective state-space scan (scan_fwd.cu, scan_bwd.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace srwm {

constexpr int SCAN_CKPT = 8;    // steps between the states that a training forward keeps
constexpr int SCAN_TILE = 16;   // steps that a CTA stages at a time
constexpr int SCAN_STEPS_DIRECT = 4;   // up to so many steps without gradients take the kernel of single tokens

struct ScanRows {               // [N, L, D] (or [N, L, G, S]), innermost dense; strides in elements
  char* p;
  long long sn, sl, sg;
};

struct ScanParams {
  int N, L, D, G, S;
  int bf16, softplus;
  int vec;                      // all rows' pieces of four elements are aligned to their size
  int nseg, seglen;             // pieces of the time axis (seglen a multiple of SCAN_TILE)
  ScanRows u, delta, z, y, B, C;
  const float *A, *skip, *bias, *h0;
  float* hT;
  const uint8_t* done;
  long long done_n, done_l;
  float* ckpt;                  // [N][ceil(L / SCAN_CKPT)][D][S], the state in front of each eighth step
  float* carry;                 // nseg > 1: each piece's end from zero and the product of its decays (its root), [N][D][S] each (forward: the first state in front)
  // backward
  ScanRows dy, du, ddelta, dz, dB, dC;
  const float* dhT;
  float *dh0, *dA, *dskip, *dbias;
  float *part_bc, *part_a, *part_v;
};

__host__ __device__ constexpr int scan_bwd_channels(int S) { return S == 8 ? 128 : S == 16 ? 64 : 32; }      // of a CTA of the backward
constexpr int SCAN_FWD_CHANNELS = 64;                     // of a CTA of the forward (32 where these would not fill the GPU; S 8: 64)
int scan_segments(const ScanParams& p, int channels, int sms);      // pieces that a call's time axis is cut into
long long scan_fwd_scratch(const ScanParams& p);           // floats
long long scan_bwd_scratch(ScanParams& p, float* base);    // floats; base not NULL: sets the pointers into it
cudaError_t scan_forward(const ScanParams& p, cudaStream_t s);
cudaError_t scan_backward(const ScanParams& p, cudaStream_t s);

}  // namespace srwm
