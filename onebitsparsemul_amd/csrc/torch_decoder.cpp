// Torch side of onebit_decoder.h: checks of the operands, results, workspace and the current stream. Operands that the kernels
// do not read where they lie (rows inside a head that are no whole 16-byte units, a negated view, elements on which a result given by the caller is
// written in another order) are copied first.
#include "torch_operands.h"

#include "onebit_head.h"

#include <ATen/MemoryOverlap.h>

#include <algorithm>
#include <cmath>
#include <vector>

namespace {

// Whether two tensors are the same element by element
bool are_same(const torch::Tensor& a, const torch::Tensor& b) {
  if (a.data_ptr() != b.data_ptr() || a.scalar_type() != b.scalar_type() || a.sizes() != b.sizes()) return false;
  for (int64_t i = 0; i < a.dim(); ++i)
    if (a.size(i) > 1 && a.stride(i) != b.stride(i)) return false;
  return true;
}
// An operand that is read while `out` is written: as it is where the two are apart or the same element by element, else a copy.
torch::Tensor beside(const torch::Tensor& in, const torch::Tensor& out) {
  return are_same(in, out) || !may_meet(in, out) ? in : in.clone(at::MemoryFormat::Contiguous);
}

bool in_vectors(const torch::Tensor& t) {
  if (t.stride(-1) != 1 || t.is_neg() || reinterpret_cast<uintptr_t>(t.data_ptr()) % 16) return false;
  for (int64_t i = 0; i + 1 < t.dim(); ++i)
    if (t.size(i) > 1 && t.stride(i) % 8) return false;
  return true;
}
// (tokens, heads, head_dim) as the kernels read it
torch::Tensor readable_heads(const torch::Tensor& t) {
  return in_vectors(t) ? t : t.resolve_neg().clone(at::MemoryFormat::Contiguous);
}
onebit_heads heads_of(const torch::Tensor& t) {
  // (the stride of a dimension of one is anything)
  return {t.data_ptr(), t.size(0) > 1 ? t.stride(0) : 0, t.size(1) > 1 ? t.stride(1) : 0};
}
void check_heads(const torch::Tensor& t, const char* name, const c10::Device& device) {
  check_gpu(t, name, device);
  TORCH_CHECK_VALUE(t.dim() == 3, name, " must have shape (tokens, heads, head_dim), got ", t.sizes());
  TORCH_CHECK_TYPE(dtype_code(t.scalar_type()) >= 0, name, " must be float16, bfloat16 or float32, got ", t.scalar_type());
}

onebit_cache cache_of(const torch::Tensor& k, const torch::Tensor& v, const torch::Tensor& k_scale, const torch::Tensor& v_scale,
                      const c10::Device& device) {
  TORCH_CHECK_TYPE(k.scalar_type() == torch::kFloat8_e4m3fn || k.scalar_type() == torch::kInt8, "k_cache must be float8_e4m3fn or int8, got ", k.scalar_type());
  check_table(k, "k_cache", k.scalar_type(), 4, device);
  check_table(v, "v_cache", k.scalar_type(), 4, device);
  TORCH_CHECK_VALUE(v.sizes() == k.sizes(), "k_cache and v_cache must have one shape (pages, kv_heads, block, head_dim), got ", k.sizes(), " and ", v.sizes());
  check_table(k_scale, "k_scale", torch::kFloat32, 2, device);
  check_table(v_scale, "v_scale", torch::kFloat32, 2, device);
  TORCH_CHECK_VALUE(k_scale.sizes() == k.sizes().slice(0, 2) && v_scale.sizes() == k.sizes().slice(0, 2), "k_scale and v_scale must have shape (pages, kv_heads)");
  for (int64_t size : k.sizes()) TORCH_CHECK_VALUE(size < (1ll << 31), "the cache's dimensions exceed the int range");
  return {k.data_ptr(), v.data_ptr(), (float*)k_scale.data_ptr(), (float*)v_scale.data_ptr(), (int)k.size(0), (int)k.size(1), (int)k.size(2),
          (int)k.size(3), k.scalar_type() == torch::kInt8 ? ONEBIT_CODE_INT8 : ONEBIT_CODE_E4M3};
}

onebit_sequences sequences_of(const torch::Tensor& pages, const torch::Tensor& lengths, const OptionalTensor& starts, int64_t tokens,
                              std::optional<int64_t> max_new, std::optional<int64_t> max_length, const c10::Device& device) {
  check_table(pages, "pages", torch::kInt32, 2, device);
  check_table(lengths, "lengths", torch::kInt32, 1, device);
  const int64_t count = pages.size(0);
  TORCH_CHECK_VALUE(lengths.size(0) == count, "lengths must have one entry for each of the ", count, " sequences");
  if (starts.has_value()) {
    check_table(*starts, "starts", torch::kInt32, 1, device);
    TORCH_CHECK_VALUE(starts->size(0) == count + 1, "starts must have ", count + 1, " entries");
  }
  TORCH_CHECK_VALUE(tokens < (1ll << 31) && pages.numel() < (1ll << 31), "too many tokens or pages");
  TORCH_CHECK_VALUE(!max_new.has_value() || *max_new > 0, "max_new must be positive");
  TORCH_CHECK_VALUE(!max_length.has_value() || *max_length > 0, "max_length must be positive");
  return {(const int*)pages.data_ptr(), (const int*)lengths.data_ptr(), starts.has_value() ? (const int*)starts->data_ptr() : nullptr, (int)count,
          (int)pages.size(1), (int)tokens, (int)std::min(max_new.value_or(tokens), tokens),
          (int)std::min<int64_t>(max_length.value_or(0), INT_MAX)};
}

struct Turning {
  const float* table = nullptr;
  int rows = 0, rotary_dim = 0;
};
Turning turning_of(const torch::Tensor& table, const c10::Device& device) {
  check_table(table, "the rotary table", torch::kFloat32, 2, device);
  TORCH_CHECK_VALUE(table.size(0) < (1ll << 31) && table.size(1) < (1ll << 31), "the rotary table exceeds the int range");
  return {(const float*)table.data_ptr(), (int)table.size(0), (int)table.size(1)};
}

torch::Tensor rotary(const torch::Tensor& x, const torch::Tensor& positions, const torch::Tensor& table, bool interleaved, const OptionalTensor& out) {
  at::AutoDispatchBelowADInplaceOrView guard_dispatch;
  const c10::Device device = x.device();
  TORCH_CHECK_VALUE(x.is_cuda(), "x must live on the GPU");
  check_heads(x, "x", device);
  const int64_t tokens = x.size(0), heads = x.size(1), dim = x.size(2);
  TORCH_CHECK_TYPE(positions.scalar_type() == torch::kInt32 || positions.scalar_type() == torch::kInt64, "positions must be int32 or int64, got ", positions.scalar_type());
  check_table(positions, "positions", positions.scalar_type(), 1, device);
  TORCH_CHECK_VALUE(positions.size(0) == tokens, "positions must have one entry for each of the ", tokens, " tokens");
  const Turning turning = turning_of(table, device);
  if (out.has_value()) {
    check_heads(*out, "out", device);
    at::assert_no_internal_overlap(*out);
    TORCH_CHECK_VALUE(out->sizes() == x.sizes() && out->scalar_type() == x.scalar_type() && out->stride(2) == 1 && !out->is_neg(),
                      "out must have x's shape and type and whole heads");
  }
  const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(device);
  torch::Tensor y = out.has_value() ? *out : empty_result(x.sizes(), x.scalar_type(), device);
  if (x.numel() == 0) return y;
  TORCH_CHECK_VALUE(tokens < (1ll << 31) && heads < (1ll << 31) && dim < (1ll << 31), "x exceeds the int range");
  auto read = [&](const torch::Tensor& t) { return out.has_value() ? beside(t, y) : t; };
  const torch::Tensor in = read(x.stride(2) == 1 && !x.is_neg() ? x : x.resolve_neg().clone(at::MemoryFormat::Contiguous));
  const torch::Tensor places = read(positions), angles = read(table);
  const onebit_heads from = heads_of(in), to = heads_of(y);
  check_status(onebit_rotary(&from, &to, dtype_code(x.scalar_type()), (int)tokens, (int)heads, (int)dim, places.data_ptr(),
                             places.scalar_type() == torch::kInt64, (const float*)angles.data_ptr(), turning.rows, turning.rotary_dim, interleaved, current_stream(device)));
  return y;
}

OptionalTensor cache_append(const torch::Tensor& k, const torch::Tensor& v, const torch::Tensor& k_cache, const torch::Tensor& v_cache,
                            const torch::Tensor& k_scale, const torch::Tensor& v_scale, const torch::Tensor& pages, const torch::Tensor& lengths,
                            const OptionalTensor& starts, const OptionalTensor& q, const OptionalTensor& table, bool interleaved,
                            std::optional<int64_t> max_new) {
  at::AutoDispatchBelowADInplaceOrView guard_dispatch;
  const c10::Device device = k.device();
  TORCH_CHECK_VALUE(k.is_cuda(), "k must live on the GPU");
  check_heads(k, "k", device);
  check_heads(v, "v", device);
  const onebit_cache cache = cache_of(k_cache, v_cache, k_scale, v_scale, device);
  TORCH_CHECK_VALUE(!may_meet(k_cache, v_cache) && !may_meet(k_scale, v_scale), "an append writes keys and values: their codes and scales must not share memory");
  TORCH_CHECK_VALUE(v.sizes() == k.sizes() && v.scalar_type() == k.scalar_type(), "k and v must have one shape and type");
  TORCH_CHECK_VALUE(k.size(1) == cache.kv_heads && k.size(2) == cache.head_dim, "k and v must have shape (tokens, ", cache.kv_heads, ", ", cache.head_dim,
                    ") for this cache, got ", k.sizes());
  const int64_t tokens = k.size(0);
  const onebit_sequences sequences = sequences_of(pages, lengths, starts, tokens, max_new, std::nullopt, device);
  Turning turning;
  if (table.has_value()) turning = turning_of(*table, device);
  if (q.has_value()) {
    check_heads(*q, "q", device);
    TORCH_CHECK_VALUE(q->size(0) == tokens && q->size(2) == cache.head_dim && q->scalar_type() == k.scalar_type(), "q must have k's tokens, head_dim and type");
    TORCH_CHECK_VALUE(table.has_value(), "queries are only turned: q needs a rotary table");
  }
  const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(device);
  OptionalTensor turned;
  if (q.has_value()) turned = empty_result(q->sizes(), q->scalar_type(), device);
  if (tokens == 0) return turned;
  const torch::Tensor k_in = readable_heads(k), v_in = readable_heads(v);
  const bool with_q = q.has_value() && q->numel() > 0;
  const torch::Tensor q_in = with_q ? readable_heads(*q) : k_in;
  const onebit_heads k_heads = heads_of(k_in), v_heads = heads_of(v_in), q_heads = heads_of(q_in);
  const onebit_heads out = with_q ? heads_of(*turned) : onebit_heads{};
  check_status(onebit_cache_append(&cache, &sequences, &k_heads, &v_heads, with_q ? &q_heads : nullptr, with_q ? &out : nullptr,
                                   with_q ? (int)q->size(1) : 0, dtype_code(k.scalar_type()), turning.table, turning.rows, turning.rotary_dim,
                                   interleaved, current_stream(device)));
  return turned;
}

torch::Tensor cache_attention(const torch::Tensor& q, const torch::Tensor& k_cache, const torch::Tensor& v_cache, const torch::Tensor& k_scale,
                              const torch::Tensor& v_scale, const torch::Tensor& pages, const torch::Tensor& lengths, const OptionalTensor& starts,
                              std::optional<double> scale, std::optional<int64_t> max_new, std::optional<int64_t> max_length, const OptionalTensor& out) {
  at::AutoDispatchBelowADInplaceOrView guard_dispatch;
  const c10::Device device = q.device();
  TORCH_CHECK_VALUE(q.is_cuda(), "q must live on the GPU");
  check_heads(q, "q", device);
  TORCH_CHECK_TYPE(q.scalar_type() != torch::kFloat32, "q must be float16 or bfloat16, got ", q.scalar_type());
  const onebit_cache cache = cache_of(k_cache, v_cache, k_scale, v_scale, device);
  const int64_t tokens = q.size(0), heads = q.size(1);
  TORCH_CHECK_VALUE(q.size(2) == cache.head_dim && heads < (1ll << 31), "q must have shape (tokens, heads, ", cache.head_dim, ") for this cache, got ", q.sizes());
  const onebit_sequences sequences = sequences_of(pages, lengths, starts, tokens, max_new, max_length, device);
  if (out.has_value()) {
    check_heads(*out, "out", device);
    at::assert_no_internal_overlap(*out);
    TORCH_CHECK_VALUE(out->sizes() == q.sizes() && out->scalar_type() == q.scalar_type() && in_vectors(*out),
                      "out must have q's shape and type and be 16-byte aligned, with strides that are multiples of eight");
  }
  const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(device);
  torch::Tensor y = out.has_value() ? *out : empty_result(q.sizes(), q.scalar_type(), device);
  if (q.numel() == 0) return y;
  const torch::Tensor in = out.has_value() ? beside(readable_heads(q), y) : readable_heads(q);
  const onebit_heads from = heads_of(in), to = heads_of(y);
  const size_t bytes = onebit_cache_attention_workspace(&cache, &sequences, (int)heads);
  torch::Tensor workspace;  // of the current stream, as the kernels that use it: free again with this call
  if (bytes) workspace = empty_result({(int64_t)bytes}, torch::kUInt8, device);
  check_status(onebit_cache_attention(&cache, &sequences, &from, &to, (int)heads, dtype_code(q.scalar_type()),
                                      (float)scale.value_or(1.0 / std::sqrt((double)cache.head_dim)), bytes ? workspace.data_ptr() : nullptr,
                                      current_stream(device)));
  return y;
}

// (h, y, scales): y as codes, or in its type and no scales
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> normed(const OptionalTensor& x, const torch::Tensor& residual, const torch::Tensor& weight,
                                                               const OptionalTensor& bias, const OptionalTensor& post_weight, const OptionalTensor& post_bias,
                                                               const OptionalTensor& gate, double residual_scale, double block_scale, double eps,
                                                               const std::string& kind, std::optional<c10::ScalarType> out_dtype,
                                                               const OptionalTensor& residual_out, bool as_codes) {
  at::AutoDispatchBelowADInplaceOrView guard_dispatch;
  const c10::Device device = residual.device();
  TORCH_CHECK_VALUE(residual.is_cuda() && residual.dim() >= 1, "residual must live on the GPU with shape (..., hidden)");
  TORCH_CHECK_VALUE(kind == "rms" || kind == "layer", "kind must be 'rms' or 'layer', got '", kind, "'");
  const int64_t hidden = residual.size(-1);
  auto check_type = [&](const torch::Tensor& t, const char* name) {
    check_gpu(t, name, device);
    TORCH_CHECK_TYPE(dtype_code(t.scalar_type()) >= 0, name, " must be float16, bfloat16 or float32, got ", t.scalar_type());
  };
  check_type(residual, "residual");
  if (x.has_value()) {
    check_type(*x, "x");
    TORCH_CHECK_VALUE(x->sizes() == residual.sizes(), "x must have the residual's shape ", residual.sizes(), ", got ", x->sizes());
  }
  auto check_vector = [&](const torch::Tensor& t, const char* name) {
    check_type(t, name);
    TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == hidden && t.is_contiguous() && !t.is_neg(), name, " must be contiguous with shape (", hidden, ",), got ", t.sizes());
    TORCH_CHECK_TYPE(t.scalar_type() == weight.scalar_type(), name, " must have the weight's type");
  };
  check_vector(weight, "weight");
  if (bias.has_value()) check_vector(*bias, "bias");
  if (post_weight.has_value()) check_vector(*post_weight, "post_weight");
  if (post_bias.has_value()) check_vector(*post_bias, "post_bias");
  const c10::ScalarType y_type = out_dtype.value_or(x.has_value() ? x->scalar_type() : residual.scalar_type());
  TORCH_CHECK_TYPE(dtype_code(y_type) >= 0, "out_dtype must be float16, bfloat16 or float32, got ", y_type);
  if (residual_out.has_value())
    TORCH_CHECK_VALUE(residual_out->device() == device && residual_out->sizes() == residual.sizes() && residual_out->scalar_type() == residual.scalar_type() &&
                          residual_out->is_contiguous() && !residual_out->is_neg(),
                      "residual_out must be contiguous with the residual's shape and type");
  const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(device);
  torch::Tensor y, scales;
  if (as_codes) std::tie(y, scales) = empty_codes(residual.sizes(), device);
  else y = empty_result(residual.sizes(), y_type, device);
  // without a block the residual is only normed, unless it is scaled or wanted elsewhere
  const bool writes = x.has_value() || residual_scale != 1.0 || (residual_out.has_value() && (!are_same(residual, *residual_out) || residual.is_neg()));
  torch::Tensor h = residual_out.has_value() ? *residual_out : writes ? empty_result(residual.sizes(), residual.scalar_type(), device) : residual;
  if (residual.numel() == 0) return {h, y, scales};
  const bool given = residual_out.has_value();
  auto read = [&](const torch::Tensor& t) { return given ? beside(t, h) : t; };
  const torch::Tensor residual_rows = rows_of(read(residual), hidden), x_rows = x.has_value() ? rows_of(read(*x), hidden) : residual_rows;
  TORCH_CHECK_VALUE(residual_rows.size(0) < (1ll << 31) && hidden < (1ll << 31), "too many rows");
  onebit_norm n = {};
  torch::Tensor gate_rows;
  if (gate.has_value()) {
    check_type(*gate, "gate");
    const int64_t last = gate->dim() > 0 ? gate->size(-1) : 1;
    TORCH_CHECK_VALUE(gate->numel() == 1 || (gate->dim() == 1 && last == hidden) || (gate->dim() == residual.dim() && (last == hidden || last == 1) &&
                      gate->sizes().slice(0, gate->dim() - 1) == residual.sizes().slice(0, residual.dim() - 1)),
                      "gate must have shape (hidden,), (..., 1) or (..., hidden), or one value, got ", gate->sizes());
    gate_rows = gate->numel() == 1 ? gate->reshape({1, 1}) : gate->dim() == 1 ? gate->reshape({1, hidden}) : gate->reshape({-1, last});
    if (gate_rows.is_neg() || (gate_rows.size(1) > 1 && gate_rows.stride(1) != 1 && gate_rows.stride(1) != 0)) gate_rows = gate_rows.resolve_neg().clone(at::MemoryFormat::Contiguous);
    gate_rows = read(gate_rows);
    n.gate = gate_rows.data_ptr();
    n.gate_row_stride = gate_rows.size(0) > 1 ? gate_rows.stride(0) : 0;
    n.gate_column_stride = gate_rows.size(1) > 1 ? (int)gate_rows.stride(1) : 0;
    n.gate_dtype = dtype_code(gate_rows.scalar_type());
  }
  n.x = x.has_value() ? x_rows.data_ptr() : nullptr;
  n.residual = residual_rows.data_ptr();
  n.h_out = writes ? h.data_ptr() : nullptr;
  n.y = y.data_ptr();
  const torch::Tensor vectors[] = {read(weight), bias.has_value() ? read(*bias) : torch::Tensor(), post_weight.has_value() ? read(*post_weight) : torch::Tensor(),
                                   post_bias.has_value() ? read(*post_bias) : torch::Tensor()};
  auto address = [](const torch::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
  n.weight = address(vectors[0]);
  n.bias = address(vectors[1]);
  n.post_weight = address(vectors[2]);
  n.post_bias = address(vectors[3]);
  n.x_stride = x_rows.size(0) > 1 ? x_rows.stride(0) : 0;
  n.residual_stride = residual_rows.size(0) > 1 ? residual_rows.stride(0) : 0;
  n.h_stride = n.y_stride = residual_rows.size(0) > 1 ? hidden : 0;
  n.x_dtype = dtype_code(x_rows.scalar_type());
  n.residual_dtype = dtype_code(residual.scalar_type());
  n.y_dtype = dtype_code(y_type);
  n.weight_dtype = dtype_code(weight.scalar_type());
  n.rows = (int)residual_rows.size(0);
  n.hidden = (int)hidden;
  n.kind = kind == "layer";
  n.residual_scale = (float)residual_scale;
  n.block_scale = (float)block_scale;
  n.eps = (float)eps;
  if (as_codes) {
    const onebit_codes codes = codes_of(y, scales);
    check_status(onebit_block_norm_codes(&n, &codes, current_stream(device)));
  } else {
    check_status(onebit_block_norm(&n, current_stream(device)));
  }
  return {h, y, scales};
}

std::tuple<torch::Tensor, torch::Tensor> block_norm(const OptionalTensor& x, const torch::Tensor& residual, const torch::Tensor& weight,
                                                    const OptionalTensor& bias, const OptionalTensor& post_weight, const OptionalTensor& post_bias,
                                                    const OptionalTensor& gate, double residual_scale, double block_scale, double eps,
                                                    const std::string& kind, std::optional<c10::ScalarType> out_dtype, const OptionalTensor& residual_out) {
  auto [h, y, scales] = normed(x, residual, weight, bias, post_weight, post_bias, gate, residual_scale, block_scale, eps, kind, out_dtype, residual_out, false);
  return {h, y};
}

std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> block_norm_codes(const OptionalTensor& x, const torch::Tensor& residual, const torch::Tensor& weight,
                                                                         const OptionalTensor& bias, const OptionalTensor& post_weight,
                                                                         const OptionalTensor& post_bias, const OptionalTensor& gate, double residual_scale,
                                                                         double block_scale, double eps, const std::string& kind,
                                                                         const OptionalTensor& residual_out) {
  return normed(x, residual, weight, bias, post_weight, post_bias, gate, residual_scale, block_scale, eps, kind, std::nullopt, residual_out, true);
}

}  // namespace

void bind_decoder(pybind11::module_& m) {
  using NoGil = pybind11::call_guard<pybind11::gil_scoped_release>;
  m.def("rotary", &rotary, NoGil());
  m.def("cache_append", &cache_append, NoGil());
  m.def("cache_attention", &cache_attention, NoGil());
  m.def("block_norm", &block_norm, NoGil());
  m.def("block_norm_codes", &block_norm_codes, NoGil());
}
