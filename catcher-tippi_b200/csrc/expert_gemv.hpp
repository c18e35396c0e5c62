// The fp8 linear for few rows: see expert_gemv.cu.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "expert_ops.hpp"

namespace cq {

// What the rows of x are: T, brought to e4m3 on the way where the weights are, or
// e4m3 codes with their scales.
enum ExpertSource : int { kSourceT = 0, kSourceCodes = 1 };

constexpr int kGemvMaxRows = 24;

struct ExpertGemvArgs {
  const void* x;  // codes: 16-byte aligned rows
  int64_t ldx;
  const float* x_scales;  // codes: [k blocks][rows]
  int rows;
  const void* w;  // codes [N][ldw], rows padded with zeros to 128 bytes
  int64_t ldw;
  const float* w_scales;
  const void* bias;
  int N, K, act;
  void* y;
  int64_t ldy;
};

// Whether the kernel takes the call: few rows, by measured times, that fit shared memory.
bool expert_gemv_fits(int rows, int N, int K);
cudaError_t launch_expert_gemv(int dtype, int source, const ExpertGemvArgs& a, int num_sms, cudaStream_t stream, bool pdl);

}  // namespace cq
