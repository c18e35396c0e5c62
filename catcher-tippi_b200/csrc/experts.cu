// Host layer of the fp8 linear and the linears of experts; see experts.hpp.
#include "experts.hpp"

#include <algorithm>
#include <string>

#include "expert_gemm.hpp"
#include "expert_gemv.hpp"
#include "expert_ops.hpp"
#include "qlinear.hpp"

namespace nemotron_cuda {

namespace {

constexpr int kBlock = 128;  // values that share an e4m3 scale
constexpr int kMaxDims = 1 << 20;

int64_t round_up(int64_t v, int64_t a) { return (v + a - 1) / a * a; }

// Hands out pieces of a workspace; with a null base it only adds up sizes, so
// that sizing and use are one piece of code.
class Arena {
 public:
  explicit Arena(void* base) : base_(static_cast<char*>(base)) {}
  template <class T>
  T* take(size_t count) {
    char* p = base_ == nullptr ? nullptr : base_ + used_;
    used_ += round_up(count * sizeof(T), 256);
    return reinterpret_cast<T*>(p);
  }
  size_t used() const { return used_; }

 private:
  char* base_;
  size_t used_ = 0;
};

void check_workspace(const void* workspace, size_t bytes, size_t need) {
  if (need == 0) return;
  if (workspace == nullptr || bytes < need)
    throw_invalid("workspace has " + std::to_string(workspace == nullptr ? 0 : bytes) + " bytes, expected " +
                  std::to_string(need));
  if ((reinterpret_cast<uintptr_t>(workspace) & 255) != 0) throw_invalid("workspace must be 256-byte aligned");
}

void check_act(int act) {
  if (act != CQ_ACT_NONE && act != CQ_ACT_SILU && act != CQ_ACT_RELU)
    throw_invalid("unknown activation " + std::to_string(act));
}

void check_aligned(const void* p, int bytes, const char* what) {
  if ((reinterpret_cast<uintptr_t>(p) & (bytes - 1)) != 0)
    throw_invalid(std::string(what) + " must be aligned to " + std::to_string(bytes) + " bytes");
}

void check_dtype16(cq_dtype dtype) {
  if (dtype != CQ_F16 && dtype != CQ_BF16) throw_invalid("dtype must be f16 or bf16, got " + std::to_string(dtype));
}

void check_dtype(cq_dtype dtype) {
  if (dtype != CQ_F16 && dtype != CQ_BF16 && dtype != CQ_F32)
    throw_invalid("unknown dtype " + std::to_string(dtype));
}

// The device that holds p, for entries without a handle.
int device_of(const void* p, const char* what) {
  cudaPointerAttributes attr{};
  check_cuda(cudaPointerGetAttributes(&attr, p), what);
  if (attr.type != cudaMemoryTypeDevice && attr.type != cudaMemoryTypeManaged)
    throw_invalid(std::string(what) + " must be device memory");
  return attr.device;
}

}  // namespace

ExpertLinear::ExpertLinear(int experts, int output_dims, int input_dims, cq_weight_format format, cq_dtype dtype,
                           int device)
    : experts_(experts), N_(output_dims), K_(input_dims), format_(format), dtype_(dtype), device_(device) {
  check_dtype16(dtype);
  if (format != CQ_WEIGHT_T && format != CQ_WEIGHT_E4M3)
    throw_invalid("unknown weight format " + std::to_string(format));
  if (experts < 1 || experts > cq::kMaxExperts)
    throw_invalid("experts must be 1 to " + std::to_string(cq::kMaxExperts) + ", got " + std::to_string(experts));
  if (output_dims < 1 || input_dims < 1 || output_dims > kMaxDims || input_dims > kMaxDims ||
      static_cast<int64_t>(experts) * output_dims > INT32_MAX)
    throw_invalid("invalid linear shape " + std::to_string(experts) + "x" + std::to_string(output_dims) + "x" +
                  std::to_string(input_dims));
  ldw_ = round_up(input_dims, e4m3() ? 128 : 64);
}

ExpertLinear::ExpertLinear(const void* weight, const float* scales, const void* bias, int experts, int output_dims,
                           int input_dims, cq_weight_format format, cq_dtype dtype, int device)
    : ExpertLinear(experts, output_dims, input_dims, format, dtype, device) {
  if (weight == nullptr) throw_invalid("weight must not be null");
  if (e4m3() && scales == nullptr) throw_invalid("scales must not be null");
  device_context(device);
  DeviceGuard guard(device);
  // the arrays may come from work on any stream
  check_cuda(cudaDeviceSynchronize(), "wait for the weight");
  const size_t size = e4m3() ? 1 : 2;
  const size_t rows = static_cast<size_t>(experts_) * N_;
  weight_ = DeviceBuffer(rows * ldw_ * size);
  if (ldw_ != K_) check_cuda(cudaMemset(weight_.get(), 0, rows * ldw_ * size), "clear weight");
  check_cuda(cudaMemcpy2D(weight_.get(), ldw_ * size, weight, K_ * size, K_ * size, rows, cudaMemcpyDefault),
             "copy weight");
  if (e4m3()) {
    const size_t count = static_cast<size_t>(experts_) * (round_up(N_, kBlock) / kBlock) * (ldw_ / kBlock);
    scales_ = DeviceBuffer(count * sizeof(float));
    check_cuda(cudaMemcpy(scales_.get(), scales, count * sizeof(float), cudaMemcpyDefault), "copy scales");
  }
  if (bias != nullptr) {
    bias_ = DeviceBuffer(rows * 2);
    check_cuda(cudaMemcpy(bias_.get(), bias, rows * 2, cudaMemcpyDefault), "copy bias");
  }
  check_cuda(cudaDeviceSynchronize(), "bind weight");
}

std::unique_ptr<ExpertLinear> ExpertLinear::from_f32(const float* weight, const float* bias, int output_dims,
                                                     int input_dims, cq_dtype dtype, int device) {
  if (weight == nullptr) throw_invalid("weight must not be null");
  std::unique_ptr<ExpertLinear> checked(
      new ExpertLinear(1, output_dims, input_dims, CQ_WEIGHT_E4M3, dtype, device));  // the shape's checks
  device_context(device);
  DeviceGuard guard(device);
  check_cuda(cudaDeviceSynchronize(), "wait for the weight");
  const size_t n = output_dims, k = input_dims;
  DeviceBuffer w(n * k * sizeof(float)), codes(n * k), bias_f32, bias_t;
  DeviceBuffer scales((round_up(n, kBlock) / kBlock) * (round_up(k, kBlock) / kBlock) * sizeof(float));
  check_cuda(cudaMemcpy(w.get(), weight, n * k * sizeof(float), cudaMemcpyDefault), "copy weight");
  check_cuda(cq::launch_quantize_weight(w.as<float>(), output_dims, input_dims, codes.as<uint8_t>(),
                                        scales.as<float>(), nullptr),
             "quantize weight");
  if (bias != nullptr) {
    bias_f32 = DeviceBuffer(n * sizeof(float));
    bias_t = DeviceBuffer(n * 2);
    check_cuda(cudaMemcpy(bias_f32.get(), bias, n * sizeof(float), cudaMemcpyDefault), "copy bias");
    check_cuda(cq::launch_round(dtype, bias_f32.as<float>(), static_cast<int64_t>(n), bias_t.get(), nullptr),
               "round bias");
  }
  return std::make_unique<ExpertLinear>(codes.get(), scales.as<float>(), bias_t.get(), 1, output_dims, input_dims,
                                        CQ_WEIGHT_E4M3, dtype, device);
}

size_t ExpertLinear::staging_bytes(int64_t rows) const {
  if (!e4m3()) return rows * round_up(K_, 8) * 2;
  const int64_t ld = round_up(K_, kBlock);
  return round_up(rows * ld, 256) + rows * (ld / kBlock) * sizeof(float);
}

size_t ExpertLinear::workspace(int rows, bool grouped) const {
  // the streaming kernel needs none
  return few_rows(rows, grouped) ? 0 : round_up(staging_bytes(rows), 256);
}

bool ExpertLinear::few_rows(int rows, bool grouped) const {
  return !grouped && e4m3() && cq::expert_gemv_fits(rows, N_, K_);
}

void ExpertLinear::check_rows(const void* x, int64_t ldx, int rows, const void* y, int64_t ldy, int act) const {
  if (rows < 0) throw_invalid("negative row count");
  if (rows > 0 && (x == nullptr || y == nullptr)) throw_invalid("input and output must not be null");
  if (ldx < K_) throw_invalid("input row stride " + std::to_string(ldx) + " is smaller than " + std::to_string(K_));
  if (ldy < N_) throw_invalid("output row stride " + std::to_string(ldy) + " is smaller than " + std::to_string(N_));
  check_aligned(y, 2, "output");
  check_act(act);
}

void ExpertLinear::product(const Rows& x, int rows, const int32_t* offsets, const Out& out, int act, void* staging,
                           cudaStream_t stream) const {
  DeviceContext& ctx = device_context(device_);
  const bool pdl = pdl_enabled();
  if (few_rows(rows, offsets != nullptr)) {
    const cq::ExpertGemvArgs a{x.x, x.ld, x.scales, rows, weight_.get(), ldw_, scales_.as<float>(), bias_.get(),
                               N_,  K_,   act,      out.y, out.ld};
    check_cuda(cq::launch_expert_gemv(dtype_, x.source, a, ctx.num_sms, stream, pdl), "expert product");
    return;
  }
  // rows as the tile copies take them: codes, or 16-byte aligned rows of T
  const void* from = x.x;
  int64_t ld = x.ld;
  const float* x_scales = x.scales;
  bool staged = false;
  if (e4m3() && x.source != cq::kSourceCodes) {
    ld = round_up(K_, kBlock);
    float* s = reinterpret_cast<float*>(static_cast<char*>(staging) + round_up(rows * ld, 256));
    const cq::QuantizeRowsArgs q{x.x, x.ld, x.row_index, x.x_rows, rows, K_, static_cast<uint8_t*>(staging), ld, s};
    check_cuda(cq::launch_quantize_rows(dtype_, q, stream, pdl), "quantize rows");
    from = staging;
    x_scales = s;
    staged = true;
  } else if (!e4m3() && (x.row_index != nullptr || x.ld % 8 != 0 || (reinterpret_cast<uintptr_t>(x.x) & 15) != 0)) {
    ld = round_up(K_, 8);
    const cq::GatherRowsArgs g{x.x, x.ld, x.row_index, x.x_rows, rows, K_, staging, ld};
    check_cuda(cq::launch_gather_rows(g, stream, pdl), "gather rows");
    from = staging;
    staged = true;
  }
  cq::ExpertGemmArgs a{};
  a.x_scales = x_scales;
  a.w_scales = scales_.as<float>();
  a.bias = bias_.get();
  a.offsets = offsets;
  a.offsets_ready = staged || x.offsets_ready;
  a.rows = rows;
  a.experts = experts_;
  a.N = N_;
  a.K = K_;
  a.x_parts = x.parts;
  a.act = act;
  a.out = out.kind;
  a.y = out.y;
  a.ldy = out.ld;
  a.y_scales = out.scales;
  a.status = ctx.status;
  const bool codes = out.kind == cq::kOutCodes;
  const int bn = cq::plan_expert_gemm(e4m3(), rows, experts_, N_, K_, x.parts, act, out.kind, ctx.num_sms);
  const int size = e4m3() ? 1 : 2, k = 128 / size;
  const int ysize = codes ? 1 : out.kind == cq::kOutF32 ? 4 : 2;
  a.tile_store = out.ld * ysize % 16 == 0 && (reinterpret_cast<uintptr_t>(out.y) & 15) == 0;
  cq::ExpertGemmMaps maps;
  // (16-bit: with the parts as a third dimension)
  const auto rows_map = [&](const void* base, int elem, int parts, int cols, int64_t stride, int box_rows, int box_cols,
                            CUtensorMapSwizzle swizzle) {
    return e4m3() ? make_map_2d(base, elem, rows, cols, stride, box_rows, box_cols, swizzle)
                  : make_map_3d(base, elem, parts, rows, cols, stride, box_rows, box_cols, swizzle);
  };
  maps.x = rows_map(from, size, x.parts, K_, ld, cq::kGemmRows, k, CU_TENSOR_MAP_SWIZZLE_128B);
  maps.x_part = rows_map(from, size, x.parts, K_, ld, cq::kGemmBoxRows, k, CU_TENSOR_MAP_SWIZZLE_128B);
  maps.w = make_map_2d(weight_.get(), size, experts_ * N_, K_, ldw_, bn, k, CU_TENSOR_MAP_SWIZZLE_128B);
  maps.y = !a.tile_store ? maps.x
                         : rows_map(out.y, ysize, out.kind == cq::kOutParts ? 2 : 1,
                                    codes ? static_cast<int>(out.ld) : N_, out.ld, cq::kStoreRows,
                                    cq::kStoreBytes / ysize, CU_TENSOR_MAP_SWIZZLE_64B);
  check_cuda(cq::launch_expert_gemm(dtype_, e4m3(), bn, maps, a, ctx.num_sms, stream, pdl), "expert product");
}

void ExpertLinear::forward(const void* x, int64_t ldx, int rows, const int32_t* offsets, void* y, int64_t ldy, int act,
                           void* workspace, size_t workspace_bytes, cudaStream_t stream) const {
  check_rows(x, ldx, rows, y, ldy, act);
  check_aligned(x, 2, "input");
  if (rows == 0) return;
  check_workspace(workspace, workspace_bytes, this->workspace(rows, offsets != nullptr));
  DeviceGuard guard(device_);
  product({cq::kSourceT, x, ldx, nullptr, nullptr, rows}, rows, offsets, {cq::kOutT, y, ldy, nullptr}, act,
          workspace, stream);
}

void ExpertLinear::forward_codes(const uint8_t* codes, int64_t ld, const float* scales, int rows, void* y, int64_t ldy,
                                 int act, cudaStream_t stream) const {
  check_rows(codes, ld, rows, y, ldy, act);
  if (ld % 16 != 0) throw_invalid("the row stride of codes must be a multiple of 16");
  check_aligned(codes, 16, "codes");
  if (rows == 0) return;
  if (scales == nullptr) throw_invalid("scales must not be null");
  check_aligned(scales, 4, "scales");
  DeviceGuard guard(device_);
  product({cq::kSourceCodes, codes, ld, scales, nullptr, rows}, rows, nullptr, {cq::kOutT, y, ldy, nullptr}, act,
          nullptr, stream);
}

void quantize_rows(const void* x, int64_t ldx, int rows, int cols, cq_dtype dtype, uint8_t* codes, int64_t ld,
                   float* scales, cudaStream_t stream) {
  check_dtype(dtype);
  if (rows < 0 || cols < 1 || cols > kMaxDims) throw_invalid("invalid shape " + std::to_string(rows) + "x" + std::to_string(cols));
  if (ldx < cols) throw_invalid("input row stride " + std::to_string(ldx) + " is smaller than " + std::to_string(cols));
  if (ld < cols || ld % 16 != 0)
    throw_invalid("the row stride of codes must be a multiple of 16 and at least " + std::to_string(cols));
  if (rows == 0) return;
  if (x == nullptr || codes == nullptr || scales == nullptr) throw_invalid("input, codes and scales must not be null");
  check_aligned(x, dtype == CQ_F32 ? 4 : 2, "input");
  check_aligned(codes, 16, "codes");
  check_aligned(scales, 4, "scales");
  DeviceGuard guard(device_of(codes, "codes"));
  const cq::QuantizeRowsArgs q{x, ldx, nullptr, rows, rows, cols, codes, ld, scales};
  check_cuda(cq::launch_quantize_rows(dtype, q, stream, pdl_enabled()), "quantize rows");
}

void quantize_weight(const float* w, int rows, int cols, uint8_t* codes, float* scales, cudaStream_t stream) {
  if (rows < 0 || cols < 1 || rows > kMaxDims || cols > kMaxDims)
    throw_invalid("invalid shape " + std::to_string(rows) + "x" + std::to_string(cols));
  if (rows == 0) return;
  if (w == nullptr || codes == nullptr || scales == nullptr) throw_invalid("weight, codes and scales must not be null");
  check_aligned(w, 4, "weight");
  check_aligned(scales, 4, "scales");
  DeviceGuard guard(device_of(codes, "codes"));
  check_cuda(cq::launch_quantize_weight(w, rows, cols, codes, scales, stream), "quantize weight");
}

namespace {

void check_route(int tokens, int experts, int top) {
  if (tokens < 0) throw_invalid("negative token count");
  if (experts < 1 || experts > cq::kMaxExperts)
    throw_invalid("experts must be 1 to " + std::to_string(cq::kMaxExperts) + ", got " + std::to_string(experts));
  if (top < 1 || top > experts || top > cq::kMaxTop)
    throw_invalid("top must be 1 to the smaller of experts and " + std::to_string(cq::kMaxTop) + ", got " +
                  std::to_string(top));
  if (static_cast<int64_t>(tokens) * top > INT32_MAX) throw_invalid("tokens * top does not fit 32 bits");
}

}  // namespace

size_t route_workspace_bytes(int tokens, int experts, int top) {
  check_route(tokens, experts, top);
  return round_up(cq::route_workspace(tokens, experts), 256);
}

void route(const void* logits, int64_t ld, cq_dtype dtype, int tokens, int experts, int top, bool renormalize,
           int32_t* expert, float* weight, int32_t* offsets, int32_t* token, int32_t* position, void* workspace,
           size_t workspace_bytes, cudaStream_t stream) {
  check_dtype(dtype);
  const size_t need = route_workspace_bytes(tokens, experts, top);
  if (ld < experts) throw_invalid("logits row stride " + std::to_string(ld) + " is smaller than " + std::to_string(experts));
  if (offsets == nullptr) throw_invalid("offsets must not be null");
  if (tokens > 0 &&
      (logits == nullptr || expert == nullptr || weight == nullptr || token == nullptr || position == nullptr))
    throw_invalid("logits and outputs must not be null");
  check_aligned(logits, dtype == CQ_F32 ? 4 : 2, "logits");
  for (const void* p : {static_cast<const void*>(expert), static_cast<const void*>(weight),
                        static_cast<const void*>(offsets), static_cast<const void*>(token),
                        static_cast<const void*>(position)})
    check_aligned(p, 4, "outputs");
  check_workspace(workspace, workspace_bytes, need);
  DeviceGuard guard(device_of(offsets, "offsets"));
  const cq::RouteArgs a{logits, ld, tokens, experts, top, renormalize ? 1 : 0, expert, weight, offsets, token, position,
                        static_cast<int32_t*>(workspace)};
  check_cuda(cq::launch_route(dtype, a, stream, pdl_enabled()), "route");
}

void combine(const void* z, int64_t ldz, int rows, const int32_t* position, const float* weight, int tokens, int top,
             int dims, cq_dtype dtype, void* y, int64_t ldy, cudaStream_t stream) {
  check_dtype16(dtype);
  if (rows < 0 || tokens < 0) throw_invalid("negative row count");
  if (top < 1) throw_invalid("top must be positive, got " + std::to_string(top));
  if (dims < 1 || dims > kMaxDims) throw_invalid("invalid dims " + std::to_string(dims));
  if (ldz < dims || ldy < dims) throw_invalid("row strides must be at least " + std::to_string(dims));
  if (tokens == 0) return;
  if ((z == nullptr && rows > 0) || position == nullptr || weight == nullptr || y == nullptr)
    throw_invalid("rows, positions, weights and output must not be null");
  check_aligned(z, 2, "rows");
  check_aligned(y, 2, "output");
  check_aligned(position, 4, "positions");
  check_aligned(weight, 4, "weights");
  DeviceGuard guard(device_of(y, "output"));
  const cq::CombineArgs a{z, ldz, position, weight, rows, tokens, top, dims, y, ldy, 0};
  check_cuda(cq::launch_combine(dtype, a, stream, pdl_enabled()), "combine");
}

// ------------------------------------------------------------------ feed-forward module

namespace {

struct FfnScratch {
  int32_t *expert, *offsets, *token, *position;
  float* weight;
  void* route;
  size_t route_bytes;
  void* x;  // the first product's staging
  void* h;  // up's result: two parts of T, or codes and scales
  int64_t ld_h;
  float* z;  // f32: the sum over a token's experts is rounded once
};

FfnScratch take_ffn(Arena& arena, const ExpertLinear& up, const ExpertLinear& down, int tokens, int top) {
  FfnScratch s{};
  const int64_t pairs = static_cast<int64_t>(tokens) * top;
  s.expert = arena.take<int32_t>(pairs);
  s.weight = arena.take<float>(pairs);
  s.offsets = arena.take<int32_t>(up.experts() + 1);
  s.token = arena.take<int32_t>(pairs);
  s.position = arena.take<int32_t>(pairs);
  s.route_bytes = route_workspace_bytes(tokens, up.experts(), top);
  s.route = arena.take<uint8_t>(s.route_bytes);
  s.x = arena.take<uint8_t>(up.staging_bytes(pairs));
  s.ld_h = round_up(up.output_dims(), 8);
  s.h = arena.take<uint8_t>(up.e4m3() ? down.staging_bytes(pairs) : 2 * pairs * s.ld_h * 2);
  s.z = arena.take<float>(pairs * down.output_dims());
  return s;
}

void check_ffn(const ExpertLinear& up, const ExpertLinear& down, int tokens, int top) {
  if (up.experts() != down.experts() || up.e4m3() != down.e4m3() || up.dtype() != down.dtype() ||
      up.device() != down.device())
    throw_invalid("the two linears of a feed-forward module must agree in experts, format, dtype and device");
  if (down.input_dims() != up.output_dims())
    throw_invalid("the second linear takes " + std::to_string(down.input_dims()) + " values, the first makes " +
                  std::to_string(up.output_dims()));
  check_route(tokens, up.experts(), top);
}

}  // namespace

size_t expert_ffn_workspace(const ExpertLinear& up, const ExpertLinear& down, int tokens, int top) {
  check_ffn(up, down, tokens, top);
  Arena arena(nullptr);
  take_ffn(arena, up, down, tokens, top);
  return arena.used();
}

void expert_ffn(const ExpertLinear& up, const ExpertLinear& down, const void* x, int64_t ldx, int tokens,
                const void* logits, int64_t ld_logits, cq_dtype logits_dtype, int top, bool renormalize, int act,
                void* y, int64_t ldy, void* workspace, size_t workspace_bytes, cudaStream_t stream) {
  const size_t need = expert_ffn_workspace(up, down, tokens, top);
  check_act(act);
  check_dtype(logits_dtype);
  const int d = up.input_dims(), out = down.output_dims();
  if (ldx < d) throw_invalid("input row stride " + std::to_string(ldx) + " is smaller than " + std::to_string(d));
  if (ldy < out) throw_invalid("output row stride " + std::to_string(ldy) + " is smaller than " + std::to_string(out));
  if (tokens == 0) return;
  if (x == nullptr || logits == nullptr || y == nullptr) throw_invalid("input, logits and output must not be null");
  check_aligned(x, 2, "input");
  check_aligned(y, 2, "output");
  check_workspace(workspace, workspace_bytes, need);
  Arena arena(workspace);
  const FfnScratch s = take_ffn(arena, up, down, tokens, top);
  const int pairs = tokens * top;
  DeviceGuard guard(up.device());
  route(logits, ld_logits, logits_dtype, tokens, up.experts(), top, renormalize, s.expert, s.weight, s.offsets,
        s.token, s.position, s.route, s.route_bytes, stream);
  const ExpertLinear::Rows rows{cq::kSourceT, x, ldx, nullptr, s.token, tokens};
  ExpertLinear::Rows h{cq::kSourceT, s.h, s.ld_h, nullptr, nullptr, pairs};
  if (!up.e4m3()) {
    // h as the sum of two values of T, so that it keeps twice T's fraction: one
    // rounding of h to T alone was as large as that of y
    up.product(rows, pairs, s.offsets, {cq::kOutParts, s.h, s.ld_h, nullptr}, act, s.x, stream);
    h.parts = 2;
    h.offsets_ready = true;  // a gather and the first product ran since the route
  } else {
    // from f32 sums to codes inside the first product
    const int64_t ld = round_up(up.output_dims(), kBlock);
    float* scales = reinterpret_cast<float*>(static_cast<char*>(s.h) + round_up(pairs * ld, 256));
    up.product(rows, pairs, s.offsets, {cq::kOutCodes, s.h, ld, scales}, act, s.x, stream);
    h = {cq::kSourceCodes, s.h, ld, scales, nullptr, pairs};
    h.offsets_ready = true;  // the first product ran between the route and the second
  }
  down.product(h, pairs, s.offsets, {cq::kOutF32, s.z, out, nullptr}, CQ_ACT_NONE, nullptr, stream);
  const cq::CombineArgs c{s.z, out, s.position, s.weight, pairs, tokens, top, out, y, ldy, 1};
  check_cuda(cq::launch_combine(up.dtype(), c, stream, pdl_enabled()), "combine");
}

}  // namespace nemotron_cuda
