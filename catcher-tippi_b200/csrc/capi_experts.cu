// extern "C" entry points of include/cqfp8.h and include/cqexperts.h over
// ExpertLinear and the functions of experts.hpp.
#include <memory>

#include "capi_guard.hpp"
#include "expert_ops.hpp"
#include "experts.hpp"

using namespace nemotron_cuda;

struct cq_fp8_linear {
  std::unique_ptr<ExpertLinear> impl;
};

struct cq_expert_linear {
  std::unique_ptr<ExpertLinear> impl;
};

namespace {

cudaStream_t as_stream(void* s) { return static_cast<cudaStream_t>(s); }

// A size, or SIZE_MAX (with the message kept) where `f` refuses.
template <class F>
size_t size_or_refuse(F&& f) {
  size_t n = 0;
  return guarded([&] { n = f(); }) == CQ_OK ? n : SIZE_MAX;
}

size_t rows_workspace(const ExpertLinear& layer, int32_t rows, bool grouped) {
  if (rows < 0) throw_invalid("negative row count");
  return layer.workspace(rows, grouped);
}

}  // namespace

extern "C" {

cq_status cq_fp8_linear_create(const uint8_t* codes, const float* scales, const void* bias_or_null,
                               int32_t output_dims, int32_t input_dims, cq_dtype dtype, int32_t device,
                               cq_fp8_linear** out) {
  return guarded([&] {
    need_handle(out, "out");
    *out = nullptr;
    auto h = std::make_unique<cq_fp8_linear>();
    h->impl = std::make_unique<ExpertLinear>(codes, scales, bias_or_null, 1, output_dims, input_dims, CQ_WEIGHT_E4M3,
                                             dtype, device);
    *out = h.release();
  });
}

cq_status cq_fp8_linear_create_from_f32(const float* weight, const float* bias_or_null, int32_t output_dims,
                                        int32_t input_dims, cq_dtype dtype, int32_t device, cq_fp8_linear** out) {
  return guarded([&] {
    need_handle(out, "out");
    *out = nullptr;
    auto h = std::make_unique<cq_fp8_linear>();
    h->impl = ExpertLinear::from_f32(weight, bias_or_null, output_dims, input_dims, dtype, device);
    *out = h.release();
  });
}

size_t cq_fp8_linear_workspace(const cq_fp8_linear* layer, int32_t rows) {
  return size_or_refuse([&] {
    need_handle(layer, "layer");
    return rows_workspace(*layer->impl, rows, false);
  });
}

cq_status cq_fp8_linear_forward(cq_fp8_linear* layer, const void* x, int64_t ldx, int32_t rows, void* y, int64_t ldy,
                                cq_act act, void* workspace, size_t workspace_bytes, void* stream) {
  return guarded([&] {
    need_handle(layer, "layer");
    layer->impl->forward(x, ldx, rows, nullptr, y, ldy, act, workspace, workspace_bytes, as_stream(stream));
  });
}

cq_status cq_fp8_linear_forward_codes(cq_fp8_linear* layer, const uint8_t* codes, int64_t ld, const float* scales,
                                      int32_t rows, void* y, int64_t ldy, cq_act act, void* stream) {
  return guarded([&] {
    need_handle(layer, "layer");
    layer->impl->forward_codes(codes, ld, scales, rows, y, ldy, act, as_stream(stream));
  });
}

int32_t cq_fp8_linear_input_dims(const cq_fp8_linear* layer) { return layer ? layer->impl->input_dims() : -1; }
int32_t cq_fp8_linear_output_dims(const cq_fp8_linear* layer) { return layer ? layer->impl->output_dims() : -1; }
void cq_fp8_linear_destroy(cq_fp8_linear* layer) { delete layer; }

cq_status cq_fp8_quantize_rows(const void* x, int64_t ldx, int32_t rows, int32_t cols, cq_dtype dtype, uint8_t* codes,
                               int64_t ld, float* scales, void* stream) {
  return guarded([&] {
    quantize_rows(x, ldx, rows, cols, dtype, codes, ld, scales, as_stream(stream));
  });
}

cq_status cq_fp8_quantize_weight(const float* w, int32_t rows, int32_t cols, uint8_t* codes, float* scales,
                                 void* stream) {
  return guarded([&] { quantize_weight(w, rows, cols, codes, scales, as_stream(stream)); });
}

cq_status cq_expert_linear_create(const void* weight, const float* scales, const void* bias_or_null, int32_t experts,
                                  int32_t output_dims, int32_t input_dims, cq_weight_format format, cq_dtype dtype,
                                  int32_t device, cq_expert_linear** out) {
  return guarded([&] {
    need_handle(out, "out");
    *out = nullptr;
    auto h = std::make_unique<cq_expert_linear>();
    h->impl = std::make_unique<ExpertLinear>(weight, scales, bias_or_null, experts, output_dims, input_dims, format,
                                             dtype, device);
    *out = h.release();
  });
}

size_t cq_expert_linear_workspace(const cq_expert_linear* layer, int32_t rows) {
  return size_or_refuse([&] {
    need_handle(layer, "layer");
    return rows_workspace(*layer->impl, rows, true);
  });
}

cq_status cq_expert_linear_forward(cq_expert_linear* layer, const void* x, int64_t ldx, int32_t rows,
                                   const int32_t* offsets, void* y, int64_t ldy, cq_act act, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  return guarded([&] {
    need_handle(layer, "layer");
    need_handle(offsets, "offsets");
    layer->impl->forward(x, ldx, rows, offsets, y, ldy, act, workspace, workspace_bytes, as_stream(stream));
  });
}

int32_t cq_expert_linear_experts(const cq_expert_linear* layer) { return layer ? layer->impl->experts() : -1; }
int32_t cq_expert_linear_input_dims(const cq_expert_linear* layer) { return layer ? layer->impl->input_dims() : -1; }
int32_t cq_expert_linear_output_dims(const cq_expert_linear* layer) { return layer ? layer->impl->output_dims() : -1; }
void cq_expert_linear_destroy(cq_expert_linear* layer) { delete layer; }

size_t cq_route_workspace(int32_t tokens, int32_t experts, int32_t top) {
  return size_or_refuse([&] { return route_workspace_bytes(tokens, experts, top); });
}

cq_status cq_route(const void* logits, int64_t ld, cq_dtype dtype, int32_t tokens, int32_t experts, int32_t top,
                   int32_t renormalize, int32_t* expert, float* weight, int32_t* offsets, int32_t* token,
                   int32_t* position, void* workspace, size_t workspace_bytes, void* stream) {
  return guarded([&] {
    route(logits, ld, dtype, tokens, experts, top, renormalize != 0, expert, weight, offsets, token, position,
          workspace, workspace_bytes, as_stream(stream));
  });
}

cq_status cq_expert_combine(const void* z, int64_t ldz, int32_t rows, const int32_t* position, const float* weight,
                            int32_t tokens, int32_t top, int32_t dims, cq_dtype dtype, void* y, int64_t ldy,
                            void* stream) {
  return guarded([&] { combine(z, ldz, rows, position, weight, tokens, top, dims, dtype, y, ldy, as_stream(stream)); });
}

size_t cq_expert_ffn_workspace(const cq_expert_linear* up, const cq_expert_linear* down, int32_t tokens, int32_t top) {
  return size_or_refuse([&] {
    need_handle(up, "up");
    need_handle(down, "down");
    return expert_ffn_workspace(*up->impl, *down->impl, tokens, top);
  });
}

cq_status cq_expert_ffn_forward(cq_expert_linear* up, cq_expert_linear* down, const void* x, int64_t ldx,
                                int32_t tokens, const void* logits, int64_t ld_logits, cq_dtype logits_dtype,
                                int32_t top, int32_t renormalize, cq_act act, void* y, int64_t ldy, void* workspace,
                                size_t workspace_bytes, void* stream) {
  return guarded([&] {
    need_handle(up, "up");
    need_handle(down, "down");
    expert_ffn(*up->impl, *down->impl, x, ldx, tokens, logits, ld_logits, logits_dtype, top, renormalize != 0, act, y,
               ldy, workspace, workspace_bytes, as_stream(stream));
  });
}

}  // extern "C"
