// The grouped product for few rows: see expert_gemv.cu.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "expert_ops.hpp"

namespace cq {

// What the rows of x are: T or f32 (brought to e4m3 by the kernel where the
// weights are), or e4m3 codes with their scales.
enum ExpertSource : int { kSourceT = 0, kSourceF32 = 1, kSourceCodes = 2 };

struct ExpertGemvArgs {
  const void* x;
  int64_t ldx;
  const int32_t* row_index;  // row r is x row row_index[r]; outside [0, x_rows) it is zero; null: x row r
  int x_rows;
  const float* x_scales;  // codes: [k blocks][rows]
  int rows;
  const void* w;  // [experts][N][ldw], rows padded with zeros to 128 bytes
  int64_t ldw;
  const float* w_scales;
  const void* bias;
  const int32_t* offsets;
  int experts, N, K, act;
  int y_f32;
  void* y;
  int64_t ldy;
};

// Whether the kernel can take the call (its rows fit shared memory).
bool expert_gemv_fits(bool e4m3, int rows, int K);
cudaError_t launch_expert_gemv(int dtype, bool e4m3, int source, const ExpertGemvArgs& a, int num_sms,
                               cudaStream_t stream, bool pdl);

}  // namespace cq
