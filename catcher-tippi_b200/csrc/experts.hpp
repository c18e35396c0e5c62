// Host layer of the fp8 linear (include/cqfp8.h) and the linears of experts
// (include/cqexperts.h): weight layout, checks of arguments, workspaces and
// dispatch.  An fp8 linear is an expert linear with one expert.
#pragma once

#include <cuda_runtime.h>

#include <memory>

#include "cqexperts.h"
#include "cqfp8.h"
#include "device_buffer.hpp"

namespace nemotron_cuda {

class ExpertLinear {
 public:
  // Arrays in host or device memory; the layer owns copies whose rows are
  // padded with zeros to a multiple of 128 bytes.
  ExpertLinear(const void* weight, const float* scales, const void* bias, int experts, int output_dims,
               int input_dims, cq_weight_format format, cq_dtype dtype, int device);
  // An f32 weight (host or device) brought to e4m3; one expert.
  static std::unique_ptr<ExpertLinear> from_f32(const float* weight, const float* bias, int output_dims,
                                                int input_dims, cq_dtype dtype, int device);

  // bytes of forward's workspace; `grouped`: with offsets
  size_t workspace(int rows, bool grouped) const;
  // offsets null: all rows meet the only expert.
  void forward(const void* x, int64_t ldx, int rows, const int32_t* offsets, void* y, int64_t ldy, int act,
               void* workspace, size_t workspace_bytes, cudaStream_t stream) const;
  void forward_codes(const uint8_t* codes, int64_t ld, const float* scales, int rows, void* y, int64_t ldy, int act,
                     cudaStream_t stream) const;

  int experts() const { return experts_; }
  int input_dims() const { return K_; }
  int output_dims() const { return N_; }
  bool e4m3() const { return format_ == CQ_WEIGHT_E4M3; }
  cq_dtype dtype() const { return dtype_; }
  int device() const { return device_; }

  // Rows of a product: T, or e4m3 codes with their
  // scales [k blocks][rows], as cq::ExpertSource says; row r is x row
  // row_index[r] where that is given (T only).
  struct Rows {
    int source;
    const void* x;
    int64_t ld;
    const float* scales;
    const int32_t* row_index;
    int x_rows;
    int parts = 1;  // 2: T as cq::kOutParts made it
    // the kernel that the product follows on the stream began after what wrote
    // the offsets was done (and says so to its dependents only then)
    bool offsets_ready = false;
  };
  // Bytes in which product() brings rows to the form that the tensor cores'
  // tile copies take.
  size_t staging_bytes(int64_t rows) const;
  // What a product makes: a cq::ExpertOut; codes need y_scales [n blocks][rows]
  // and rows padded to whole blocks, and rows that few_rows() does not take; parts
  // need 2 x rows rows.
  struct Out {
    int kind;
    void* y;
    int64_t ld;
    float* scales;
  };
  // The product alone, arguments checked.
  void product(const Rows& x, int rows, const int32_t* offsets, const Out& out, int act, void* staging,
               cudaStream_t stream) const;
  // True when calls on `rows` rows stream the weights (expert_gemv.cu) instead
  // of running tiles on the tensor cores (expert_gemm.cu).
  bool few_rows(int rows, bool grouped) const;

 private:
  ExpertLinear(int experts, int output_dims, int input_dims, cq_weight_format format, cq_dtype dtype, int device);
  void check_rows(const void* x, int64_t ldx, int rows, const void* y, int64_t ldy, int act) const;

  int experts_, N_, K_;
  cq_weight_format format_;
  cq_dtype dtype_;
  int device_;
  int64_t ldw_;  // elements per padded weight row
  DeviceBuffer weight_, scales_, bias_;
};

// x rows -> e4m3 (cq_fp8_quantize_rows).
void quantize_rows(const void* x, int64_t ldx, int rows, int cols, cq_dtype dtype, uint8_t* codes, int64_t ld,
                   float* scales, cudaStream_t stream);

// f32 weight -> e4m3 by blocks of 128 x 128 (cq_fp8_quantize_weight).
void quantize_weight(const float* w, int rows, int cols, uint8_t* codes, float* scales, cudaStream_t stream);

size_t route_workspace_bytes(int tokens, int experts, int top);
void route(const void* logits, int64_t ld, cq_dtype dtype, int tokens, int experts, int top, bool renormalize,
           int32_t* expert, float* weight, int32_t* offsets, int32_t* token, int32_t* position, void* workspace,
           size_t workspace_bytes, cudaStream_t stream);
void combine(const void* z, int64_t ldz, int rows, const int32_t* position, const float* weight, int tokens, int top,
             int dims, cq_dtype dtype, void* y, int64_t ldy, cudaStream_t stream);

size_t expert_ffn_workspace(const ExpertLinear& up, const ExpertLinear& down, int tokens, int top);
void expert_ffn(const ExpertLinear& up, const ExpertLinear& down, const void* x, int64_t ldx, int tokens,
                const void* logits, int64_t ld_logits, cq_dtype logits_dtype, int top, bool renormalize, int act,
                void* y, int64_t ldy, void* workspace, size_t workspace_bytes, cudaStream_t stream);

}  // namespace nemotron_cuda
