/*
 * C ABI of libonebitmul for the way from a decoder's last layer to its next tokens on MI355X (gfx950): 8-bit codes with a scale for each
 * 128 values, behind a norm (onebit_decoder.h) or by themselves, the matrix product of such codes, and the choice of tokens
 * from logits. No counterpart in the reference, whose layers stop at the projection (onebit_sparse_mul/__init__.py:101-145).
 *
 * All data pointers are DEVICE pointers, the structs themselves are HOST memory, read before the call returns. Work is
 * enqueued on `stream` (hipStream_t as void*, NULL = default stream) and the calls return without synchronising. They allocate
 * nothing, keep nothing between calls, and can be captured in a HIP graph. Status codes, dtype codes and
 * onebit_sparse_last_error() are those of onebit_sparse_tensor.h; a call of more than 2^32 threads is refused as HIP refuses it.
 * Results lie apart from the operands, their rows from each other, and the workspace from all.
 */
#ifndef ONEBIT_HEAD_H_
#define ONEBIT_HEAD_H_

#include "onebit_decoder.h"

#ifdef __cplusplus
extern "C" {
#endif

#define ONEBIT_CODE_GROUP 128 /* values that share a scale */

/*
 * Rows of OCP e4m3 codes (448 the largest, no infinities) with a scale for each 128 columns. The columns are a multiple of 128: rows of
 * other lengths end in codes 0. codes: 16-byte aligned; row_stride in codes, a multiple of 16; scale_stride in floats.
 */
typedef struct onebit_codes {
  void *codes;
  float *scales;
  long long row_stride, scale_stride;
} onebit_codes;

/*
 * rows x columns values (x_stride between rows) as codes: scale = largest magnitude of the group / 448, code = value / scale rounded to
 * nearest even, 0 where the scale is 0, all in fp32. A NaN or an infinity makes its group's scale NaN or infinite and the codes 0, so that a
 * product with them is NaN. Columns beyond `columns`, up to the next multiple of 128, become 0.
 */
int onebit_quantize_rows(const void *x, int dtype, long long x_stride, int rows, int columns, const onebit_codes *out, void *stream);

/* onebit_block_norm whose y leaves as codes, from the unrounded values; norm->y and its dtype and stride are not looked at. */
int onebit_block_norm_codes(const onebit_norm *norm, const onebit_codes *out, void *stream);

/*
 * y[t][m] = sum over groups g of (x.scales[t][g] * weight.scales[m / 128][g]) * (sum over the group's columns k of x[t][k] * weight[m][k])
 * + bias[m]: tokens x rows values, fp32, fp16 or bf16 (y_dtype), y_stride between tokens. Products of codes are exact, their sums and everything behind
 * them fp32, y is rounded once; but for fp16 and bf16 results of more than 16 tokens the products of eight neighbouring columns are cut off
 * at 2^-13 of the largest of them, as the 8-bit matrix instruction does: y is then off by less than 7 2^-13 of the sum of the largest magnitudes of all eights, beside
 * its rounding, whatever is left of y where large products cancel. (Measured over 4096 columns, of y's norm: normal values 1.5e-5, of one sign 3e-6, one column of
 * eight hundreds of times the others 6.3e-5.) fp32 results are never cut: who needs such sums in 16 bits rounds those. weight: `rows` rows of codes, scales for each 128 rows and
 * columns (ceil(rows / 128) rows of them). columns: a multiple of 128. tokens, rows, columns: at most 2^30. bias: `rows` values (bias_dtype), or NULL. workspace:
 * onebit_block_linear_workspace() bytes, 16-byte aligned (NULL where that is 0). A NaN among a token's codes or scales reaches that token's results alone.
 */
typedef struct onebit_block_product {
  onebit_codes x, weight;
  const void *bias;
  void *y;
  long long y_stride;
  int tokens, rows, columns;
  int y_dtype, bias_dtype;
} onebit_block_product;
size_t onebit_block_linear_workspace(const onebit_block_product *product);
int onebit_block_linear(const onebit_block_product *product, void *workspace, void *stream);

/*
 * A token for each row of logits. With w_i = exp((logit_i - the row's largest) / temperature) and the tokens in the order of falling logits, equal ones by
 * rising index: the first top_k stay; of these those in front of which less than top_p of their mass lies; of these those with
 * w >= min_p; of all filters the first token always stays. The result is the first of them, by index, at which the running sum of w exceeds
 * uniform times its total. temperature 0 (or less, or NaN): the largest logit, the lowest index among equals. top_k 0 or less, top_p 1 or more,
 * min_p 0 or less: no such filter. A uniform number below 0 or NaN counts as 0, of 1 and above it takes the last token with a weight.
 * A row with a NaN, and one with nothing above -inf, gives -1. +inf: tokens that have it share the mass. Weights are multiples of 2^-42 of the largest,
 * rounded to nearest: integers, so that results do not depend on the order in which they are added; smaller weights are 0. Of more than 8192 logits the whole row's mass is that of each
 * 4096 in 2^-42 of their own largest, added in 64-bit floats in one order.
 * Parameters: a value for all rows, or with its pointer set one for each row. vocabulary: at most 2^20. workspace: onebit_sample_workspace() bytes,
 * 16-byte aligned (NULL where that is 0).
 */
typedef struct onebit_sampling {
  const void *logits; /* rows x vocabulary, logits_stride between rows */
  long long logits_stride;
  int logits_dtype, rows, vocabulary;
  const float *uniform;                        /* rows */
  const float *temperatures, *top_ps, *min_ps; /* rows each, or NULL */
  const int *top_ks;
  float temperature, top_p, min_p;
  int top_k;
  long long *tokens; /* rows */
} onebit_sampling;
size_t onebit_sample_workspace(const onebit_sampling *sampling);
int onebit_sample(const onebit_sampling *sampling, void *workspace, void *stream);

#ifdef __cplusplus
}
#endif
#endif
