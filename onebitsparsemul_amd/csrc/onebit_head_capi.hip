// C ABI of onebit_head.h (but for the norm, whose checks are onebit_block_norm's): argument validation and launches. Host code only.
#include "onebit_decoder_checks.h"
#include "onebit_head_launch.h"

using onebit::aligned;
using onebit::is_type;
using onebit::launched;
using onebit::refuse;

namespace {

int check_product(const onebit_block_product* p) {
  if (!p || !p->y) return refuse("y must not be null");
  CHECKED(onebit::check_codes(&p->x, "x"));
  CHECKED(onebit::check_codes(&p->weight, "the weight"));
  constexpr int kMost = 1 << 30;
  if (p->tokens < 1 || p->rows < 1 || p->tokens > kMost || p->rows > kMost) return refuse("tokens and rows must be positive and at most 2^30 (got %d, %d)", p->tokens, p->rows);
  if (p->columns < ONEBIT_CODE_GROUP || p->columns % ONEBIT_CODE_GROUP || p->columns > kMost) return refuse("columns = %d: rows of codes have a positive multiple of 128, at most 2^30", p->columns);
  if (p->tokens > 1 && p->y_stride < p->rows) return refuse("rows of y must not overlap (stride %lld)", p->y_stride);
  if (!is_type(p->y_dtype) || (p->bias && !is_type(p->bias_dtype))) return refuse("dtype codes must be 0 (fp32), 1 (fp16) or 2 (bf16)");
  return ONEBIT_OK;
}

int check_sampling(const onebit_sampling* a) {
  if (!a || !a->logits || !a->uniform || !a->tokens) return refuse("logits, uniform and tokens must not be null");
  if (!is_type(a->logits_dtype)) return refuse("dtype code must be 0 (fp32), 1 (fp16) or 2 (bf16), got %d", a->logits_dtype);
  if (a->rows < 1 || a->vocabulary < 1 || a->vocabulary > 1 << 20) return refuse("rows must be positive and the vocabulary 1 to 2^20 (got %d, %d)", a->rows, a->vocabulary);
  return ONEBIT_OK;
}

}  // namespace

extern "C" {

int onebit_quantize_rows(const void* x, int dtype, long long x_stride, int rows, int columns, const onebit_codes* out, void* stream) {
  onebit::report(ONEBIT_OK, "");
  if (!x) return refuse("x must not be null");
  if (!is_type(dtype)) return refuse("dtype code must be 0 (fp32), 1 (fp16) or 2 (bf16), got %d", dtype);
  if (rows < 1 || columns < 1 || columns > 1 << 30) return refuse("rows must be positive and columns 1 to 2^30 (got %d, %d)", rows, columns);
  CHECKED(onebit::check_codes(out, "the result"));
  CHECKED(onebit::check_apart(*out, rows, columns));
  return launched(onebit::launch_quantize_rows(x, dtype, x_stride, rows, columns, *out, (hipStream_t)stream), "onebit_quantize_rows");
}

size_t onebit_block_linear_workspace(const onebit_block_product* product) {
  onebit::report(ONEBIT_OK, "");
  if (check_product(product)) return 0;
  return onebit::block_workspace(*product, onebit::plan_block(*product, onebit::device_compute_units()));
}

int onebit_block_linear(const onebit_block_product* product, void* workspace, void* stream) {
  onebit::report(ONEBIT_OK, "");
  CHECKED(check_product(product));
  onebit::BlockGrid grid = onebit::plan_block(*product, onebit::device_compute_units());
  if (const size_t bytes = onebit::block_workspace(*product, grid)) {
    if (!workspace || !aligned(workspace, 16)) return refuse("this call needs a workspace of %zu bytes, 16-byte aligned", bytes);
    grid.partial = (float*)workspace;
  }
  return launched(onebit::launch_block_linear(*product, grid, (hipStream_t)stream), "onebit_block_linear");
}

size_t onebit_sample_workspace(const onebit_sampling* sampling) {
  onebit::report(ONEBIT_OK, "");
  return check_sampling(sampling) ? 0 : onebit::sample_workspace(*sampling);
}

int onebit_sample(const onebit_sampling* sampling, void* workspace, void* stream) {
  onebit::report(ONEBIT_OK, "");
  CHECKED(check_sampling(sampling));
  const size_t bytes = onebit::sample_workspace(*sampling);
  if (bytes && (!workspace || !aligned(workspace, 16))) return refuse("this call needs a workspace of %zu bytes, 16-byte aligned", bytes);
  return launched(onebit::launch_sample(*sampling, workspace, (hipStream_t)stream), "onebit_sample");
}

}  // extern "C"
