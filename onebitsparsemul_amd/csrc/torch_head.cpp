// Torch side of onebit_head.h: checks of the operands, results, workspaces and the current stream. Activations, codes of tokens and logits that the
// kernels do not read where they lie are copied first, a weight is refused.
#include "torch_operands.h"

#include <ATen/MemoryOverlap.h>

#include <limits>
#include <variant>

namespace {

std::tuple<torch::Tensor, torch::Tensor> quantize_rows(const torch::Tensor& x) {
  at::AutoDispatchBelowADInplaceOrView guard_dispatch;
  const c10::Device device = x.device();
  TORCH_CHECK_VALUE(x.is_cuda() && x.dim() >= 1, "x must live on the GPU with shape (..., columns)");
  TORCH_CHECK_TYPE(dtype_code(x.scalar_type()) >= 0, "x must be float16, bfloat16 or float32, got ", x.scalar_type());
  const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(device);
  auto [codes, scales] = empty_codes(x.sizes(), device);
  if (x.numel() == 0) return {codes, scales};
  const torch::Tensor rows = rows_of(x, x.size(-1));
  TORCH_CHECK_VALUE(rows.size(0) < (1ll << 31) && rows.size(1) <= (1ll << 30), "x exceeds the int range");
  const onebit_codes out = codes_of(codes, scales);
  check_status(onebit_quantize_rows(rows.data_ptr(), dtype_code(rows.scalar_type()), rows.size(0) > 1 ? rows.stride(0) : 0, (int)rows.size(0),
                                    (int)rows.size(1), &out, current_stream(device)));
  return {codes, scales};
}

void check_codes(const torch::Tensor& t, const char* name, const c10::Device& device) {
  check_gpu(t, name, device);
  TORCH_CHECK_TYPE(t.scalar_type() == torch::kFloat8_e4m3fn, name, " must be float8_e4m3fn, got ", t.scalar_type());
  TORCH_CHECK_VALUE(!t.is_neg(), name, " must not be a negated view");
}
void check_scales(const torch::Tensor& t, const char* name, const c10::Device& device) {
  check_gpu(t, name, device);
  TORCH_CHECK_TYPE(t.scalar_type() == torch::kFloat32, name, " must be float32, got ", t.scalar_type());
}
bool readable(const torch::Tensor& codes, const torch::Tensor& scales) {
  return codes.stride(1) == 1 && (codes.size(0) == 1 || codes.stride(0) % 16 == 0) && reinterpret_cast<uintptr_t>(codes.data_ptr()) % 16 == 0 &&
         (scales.stride(1) == 1 || scales.size(1) == 1) && !scales.is_neg();
}

torch::Tensor block_linear(const torch::Tensor& codes, const torch::Tensor& scales, const torch::Tensor& weight_codes, const torch::Tensor& weight_scales,
                           const OptionalTensor& bias, c10::ScalarType out_dtype, const OptionalTensor& out) {
  at::AutoDispatchBelowADInplaceOrView guard_dispatch;
  const c10::Device device = codes.device();
  TORCH_CHECK_VALUE(codes.is_cuda() && codes.dim() >= 1, "codes must live on the GPU with shape (..., columns)");
  check_codes(codes, "codes", device);
  check_scales(scales, "scales", device);
  check_codes(weight_codes, "weight_codes", device);
  check_scales(weight_scales, "weight_scales", device);
  const int64_t columns = codes.size(-1), groups = columns / ONEBIT_CODE_GROUP;
  TORCH_CHECK_VALUE(columns % ONEBIT_CODE_GROUP == 0 && columns > 0, "rows of codes have a positive multiple of 128 columns, got ", codes.sizes());
  TORCH_CHECK_VALUE(scales.dim() == codes.dim() && scales.sizes().slice(0, codes.dim() - 1) == codes.sizes().slice(0, codes.dim() - 1) && scales.size(-1) == groups,
                    "scales must have one entry for each 128 columns of codes, got ", scales.sizes(), " for ", codes.sizes());
  TORCH_CHECK_VALUE(weight_codes.dim() == 2 && weight_codes.size(1) == columns, "weight_codes must have shape (rows, ", columns, "), got ", weight_codes.sizes());
  const int64_t rows = weight_codes.size(0);
  TORCH_CHECK_VALUE(weight_scales.dim() == 2 && weight_scales.size(0) == (rows + ONEBIT_CODE_GROUP - 1) / ONEBIT_CODE_GROUP && weight_scales.size(1) == groups,
                    "weight_scales must have one entry for each 128 x 128 codes, got ", weight_scales.sizes(), " for ", weight_codes.sizes());
  std::vector<int64_t> shape = codes.sizes().vec();
  shape.back() = rows;
  const c10::ScalarType type = out.has_value() ? out->scalar_type() : out_dtype;
  TORCH_CHECK_TYPE(dtype_code(type) >= 0, "the result must be float16, bfloat16 or float32, got ", type);
  if (bias.has_value()) {
    check_gpu(*bias, "bias", device);
    TORCH_CHECK_TYPE(dtype_code(bias->scalar_type()) >= 0, "bias must be float16, bfloat16 or float32, got ", bias->scalar_type());
    TORCH_CHECK_VALUE(bias->dim() == 1 && bias->size(0) == rows && bias->is_contiguous() && !bias->is_neg(), "bias must be contiguous with shape (", rows, ",), got ", bias->sizes());
  }
  if (out.has_value()) {
    check_gpu(*out, "out", device);
    at::assert_no_internal_overlap(*out);
    TORCH_CHECK_VALUE(out->sizes() == at::IntArrayRef(shape) && !out->is_neg() && (out->is_contiguous() || (out->dim() == 2 && (out->stride(1) == 1 || rows == 1))),
                      "out must have shape ", at::IntArrayRef(shape), " with whole rows, got ", out->sizes());
    for (const torch::Tensor* t : {&codes, &scales, &weight_codes, &weight_scales})
      TORCH_CHECK_VALUE(!may_meet(*t, *out), "out must lie apart from the operands");
    TORCH_CHECK_VALUE(!bias.has_value() || !may_meet(*bias, *out), "out must lie apart from the operands");
    TORCH_CHECK_VALUE(out->is_contiguous() || out->size(0) < 2 || out->stride(0) >= rows, "out's rows must not overlap");
  }
  const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(device);
  torch::Tensor y = out.has_value() ? *out : empty_result(shape, type, device);
  if (y.numel() == 0) return y;
  TORCH_CHECK_VALUE(readable(weight_codes, weight_scales), "weight_codes must be 16-byte aligned with whole rows a multiple of 16 apart, weight_scales of whole rows");
  torch::Tensor x = codes.dim() == 2 ? codes : codes.reshape({-1, columns}), x_scales = scales.dim() == 2 ? scales : scales.reshape({-1, groups});
  if (!readable(x, x_scales)) {
    x = x.clone(at::MemoryFormat::Contiguous);
    x_scales = x_scales.resolve_neg().clone(at::MemoryFormat::Contiguous);
  }
  const int64_t tokens = x.size(0);
  TORCH_CHECK_VALUE(tokens < (1ll << 31) && rows < (1ll << 31) && columns < (1ll << 31), "the product exceeds the int range");
  onebit_block_product p = {};
  p.x = codes_of(x, x_scales);
  p.weight = codes_of(weight_codes, weight_scales);
  p.bias = bias.has_value() ? bias->data_ptr() : nullptr;
  p.y = y.data_ptr();
  p.y_stride = y.dim() == 2 ? tokens > 1 ? y.stride(0) : 0 : rows;
  p.tokens = (int)tokens, p.rows = (int)rows, p.columns = (int)columns;
  p.y_dtype = dtype_code(type), p.bias_dtype = bias.has_value() ? dtype_code(bias->scalar_type()) : 0;
  const size_t bytes = onebit_block_linear_workspace(&p);
  torch::Tensor workspace;  // of the current stream, as the kernels that use it: free again with this call
  if (bytes) workspace = empty_result({(int64_t)bytes}, torch::kUInt8, device);
  check_status(onebit_block_linear(&p, bytes ? workspace.data_ptr() : nullptr, current_stream(device)));
  return y;
}

// A sampling parameter: one for each row, or a number for all
template <class Number, class Value>
void parameter(const std::optional<std::variant<torch::Tensor, Number>>& given, const char* name, c10::ScalarType type, at::IntArrayRef shape, const c10::Device& device,
               const Value*& each, Value& all) {
  if (!given.has_value()) return;
  if (const Number* number = std::get_if<Number>(&*given)) {
    all = std::is_integral<Value>::value ? (Value)std::min<Number>(std::max<Number>(*number, 0), std::numeric_limits<int>::max()) : (Value)*number;
    return;
  }
  const torch::Tensor& t = std::get<torch::Tensor>(*given);
  check_gpu(t, name, device);
  TORCH_CHECK_TYPE(t.scalar_type() == type, name, " must be a number or ", type, ", got ", t.scalar_type());
  TORCH_CHECK_VALUE(t.sizes() == shape && t.is_contiguous() && !t.is_neg(), name, " must be a number or contiguous with one entry for each row, got shape ", t.sizes());
  each = (const Value*)t.data_ptr();
}

torch::Tensor sample(const torch::Tensor& logits, const torch::Tensor& uniform, const std::optional<std::variant<torch::Tensor, double>>& temperature,
                     const std::optional<std::variant<torch::Tensor, int64_t>>& top_k, const std::optional<std::variant<torch::Tensor, double>>& top_p,
                     const std::optional<std::variant<torch::Tensor, double>>& min_p) {
  at::AutoDispatchBelowADInplaceOrView guard_dispatch;
  const c10::Device device = logits.device();
  TORCH_CHECK_VALUE(logits.is_cuda() && logits.dim() >= 1, "logits must live on the GPU with shape (..., vocabulary)");
  TORCH_CHECK_TYPE(dtype_code(logits.scalar_type()) >= 0, "logits must be float16, bfloat16 or float32, got ", logits.scalar_type());
  const at::IntArrayRef shape = logits.sizes().slice(0, logits.dim() - 1);
  check_gpu(uniform, "uniform", device);
  TORCH_CHECK_TYPE(uniform.scalar_type() == torch::kFloat32, "uniform must be float32, got ", uniform.scalar_type());
  TORCH_CHECK_VALUE(uniform.sizes() == shape && uniform.is_contiguous() && !uniform.is_neg(), "uniform must be contiguous with one number for each row, got shape ",
                    uniform.sizes(), " for logits ", logits.sizes());
  onebit_sampling a = {};
  a.temperature = 1.f, a.top_p = 1.f;
  parameter(temperature, "temperature", torch::kFloat32, shape, device, a.temperatures, a.temperature);
  parameter(top_k, "top_k", torch::kInt32, shape, device, a.top_ks, a.top_k);
  parameter(top_p, "top_p", torch::kFloat32, shape, device, a.top_ps, a.top_p);
  parameter(min_p, "min_p", torch::kFloat32, shape, device, a.min_ps, a.min_p);
  const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(device);
  torch::Tensor tokens = empty_result(shape, torch::kInt64, device);
  if (tokens.numel() == 0) return tokens;
  TORCH_CHECK_VALUE(logits.size(-1) > 0, "logits must have a vocabulary, got shape ", logits.sizes());
  const torch::Tensor rows = rows_of(logits, logits.size(-1));
  TORCH_CHECK_VALUE(rows.size(0) < (1ll << 31) && rows.size(1) < (1ll << 31), "logits exceed the int range");
  a.logits = rows.data_ptr();
  a.logits_stride = rows.size(0) > 1 ? rows.stride(0) : 0;
  a.logits_dtype = dtype_code(rows.scalar_type());
  a.rows = (int)rows.size(0), a.vocabulary = (int)rows.size(1);
  a.uniform = (const float*)uniform.data_ptr();
  a.tokens = (long long*)tokens.data_ptr();
  const size_t bytes = onebit_sample_workspace(&a);
  torch::Tensor workspace;
  if (bytes) workspace = empty_result({(int64_t)bytes}, torch::kUInt8, device);
  check_status(onebit_sample(&a, bytes ? workspace.data_ptr() : nullptr, current_stream(device)));
  return tokens;
}

}  // namespace

void bind_head(pybind11::module_& m) {
  using NoGil = pybind11::call_guard<pybind11::gil_scoped_release>;
  m.def("quantize_rows", &quantize_rows, NoGil());
  m.def("block_linear", &block_linear, NoGil());
  m.def("sample", &sample, NoGil());
}
