// The grouped product on the 5th-generation tensor cores: see expert_gemm.cu.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "expert_ops.hpp"

namespace cq {

constexpr int kGemmRows = 128;  // rows of x per CTA
constexpr int kGemmBoxRows = 32;  // rows of one copy where a tile is not full

// What a value of y becomes: T, f32, e4m3 codes with their scales, or two of T
// whose sum it is (16-bit weights): the high parts of all rows, and after them
// what those leave.
enum ExpertOut : int { kOutT = 0, kOutF32 = 1, kOutCodes = 2, kOutParts = 3 };

struct ExpertGemmArgs {
  const float* x_scales;  // e4m3: [k blocks][rows]
  const float* w_scales;  // e4m3: [experts][n blocks][k blocks]
  const void* bias;       // T [experts][N] or null
  int x_parts;            // 16-bit: 2 where x comes as kOutParts, else 1
  const int32_t* offsets; // null: all rows meet expert 0
  int offsets_ready;      // the kernel launched before this one began after what wrote the offsets was done
  int rows, experts, N, K, act;
  int out;
  void* y;  // T, f32 or codes, row stride ldy
  int64_t ldy;
  float* y_scales;  // kOutCodes: [ceil(N / 128)][rows]
  int* status;
  int tile_store;
};

// The box of a tile store: 64 bytes of 32 rows.
constexpr int kStoreRows = 32, kStoreBytes = 64;

// Tensor maps of one call.  x, x_part: [rows, K], box 128 bytes x 128 and x 32
// rows; w: [experts * N, K], box 128 bytes x bn rows; all with the
// 128-byte swizzle.  y: [rows, N] in its own type, box 64 bytes x 32 rows, 64-byte
// swizzle, used where tile_store says that y's rows allow it (16-byte aligned).
// With 16-bit weights x, x_part and y have a third dimension, the parts.
struct ExpertGemmMaps {
  CUtensorMap x, x_part, w, y;
};

// `bn`: weight rows of a tile, 64, 128 or 256 (codes: 128 or 256); what
// plan_expert_gemm returns.
cudaError_t launch_expert_gemm(int dtype, bool e4m3, int bn, const ExpertGemmMaps& maps, const ExpertGemmArgs& a,
                               int num_sms, cudaStream_t stream, bool pdl);
int plan_expert_gemm(bool e4m3, int rows, int experts, int N, int K, int x_parts, int act, int out, int num_sms);

}  // namespace cq
