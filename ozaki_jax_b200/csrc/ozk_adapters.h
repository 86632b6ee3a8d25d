// The adapters' own gradients (ozk_adapters_grad.cu), as ozk_adapters_grad calls them.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace ozk {

struct OuterProduct {
  bool bf16;
  int64_t M, N, K;
  int r, E;
  const int32_t* ids;
  const void* X;        // 16-bit [M][K], or int8 codes when exps is set; X and dY on 16 bytes,
                        // row strides too
  int64_t ldx;
  const int8_t* exps;
  const void* dY;       // [M][N]
  int64_t ldy;
  const uint16_t* U;    // [M][2 split_half(r)]: high parts, low parts times low_up
  const float* T;       // [M][r]
  void *dA, *dB;        // [E][r][K], [E][N][r]
  int32_t* status;
};

size_t outer_scratch_bytes(int64_t M, int64_t N, int64_t K, int r, int E, int dev);
// First the row lists and T's split (the kernel that follows may start early and
// must wait for them before it ends), then, after the kernel that makes U, the
// sums.
int launch_outer_rows(const OuterProduct& p, void* scratch, int dev, cudaStream_t stream);
int launch_outer(const OuterProduct& p, void* scratch, int dev, cudaStream_t stream);

}  // namespace ozk
