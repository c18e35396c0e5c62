// Kernels of the fp8 linear and of the linears of experts: bringing rows and
// weights to e4m3, the grouped product, the router and the combine.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace cq {

constexpr int kMaxExperts = 1024;
constexpr int kMaxTop = 32;

// x rows -> e4m3 codes [rows][ld] (ld a multiple of 16; zero from cols to the
// next multiple of 128 or ld) and scales [ceil(cols / 128)][rows].  With
// row_index, row r is x row row_index[r]; where that is outside [0, x_rows) the
// codes are left as they are and the scales are 1.
struct QuantizeRowsArgs {
  const void* x;
  int64_t ldx;
  const int32_t* row_index;
  int x_rows, rows, cols;
  uint8_t* codes;
  int64_t ld;
  float* scales;
};
cudaError_t launch_quantize_rows(int dtype, const QuantizeRowsArgs& a, cudaStream_t stream, bool pdl);

// Weight f32 [rows, cols] -> codes and the scales of 128 x 128 blocks.
cudaError_t launch_quantize_weight(const float* w, int rows, int cols, uint8_t* codes, float* scales,
                                   cudaStream_t stream);

// f32 -> T (kF16 or kBF16), to nearest.
cudaError_t launch_round(int dtype, const float* v, int64_t n, void* out, cudaStream_t stream);

// 16-bit rows x[row_index[r]] (or x[r]) -> out rows of stride ld, a multiple
// of 8 at least cols; rows whose index is outside [0, x_rows) are left as they are.
struct GatherRowsArgs {
  const void* x;
  int64_t ldx;
  const int32_t* row_index;
  int x_rows, rows, cols;
  void* out;
  int64_t ld;
};
cudaError_t launch_gather_rows(const GatherRowsArgs& a, cudaStream_t stream, bool pdl);

struct RouteArgs {
  const void* logits;
  int64_t ld;
  int tokens, experts, top, renormalize;
  int32_t* expert;
  float* weight;
  int32_t* offsets;
  int32_t* token;
  int32_t* position;
  int32_t* counts;  // workspace: route_workspace bytes
};
size_t route_workspace(int tokens, int experts);
cudaError_t launch_route(int dtype, const RouteArgs& a, cudaStream_t stream, bool pdl);

struct CombineArgs {
  const void* z;
  int64_t ldz;
  const int32_t* position;
  const float* weight;
  int rows, tokens, top, dims;
  void* y;
  int64_t ldy;
  int z_f32;  // z is f32 instead of T
};
cudaError_t launch_combine(int dtype, const CombineArgs& a, cudaStream_t stream, bool pdl);

}  // namespace cq
