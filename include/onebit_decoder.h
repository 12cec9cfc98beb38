/*
 * C ABI of libonebitmul for what a decoder layer runs around its one-bit projections (onebit_sparse_tensor.h) on MI355X
 * (gfx950): rotary positions, a paged cache of 8-bit keys and values with the attention that reads it, and the norms around
 * a block with its residual sum. No counterpart in the reference, whose layers stop at the projection
 * (onebit_sparse_mul/__init__.py:101-145).
 *
 * All data pointers are DEVICE pointers, the structs themselves are HOST memory, read before the call returns. Work is
 * enqueued on `stream` (hipStream_t as void*, NULL = default stream) and the calls return without synchronising. They allocate
 * nothing, keep nothing between calls, and can be captured in a HIP graph. Status codes, dtype codes and
 * onebit_sparse_last_error() are those of onebit_sparse_tensor.h; a call of more than 2^32 threads is refused as HIP refuses it.
 * Results lie apart from the operands unless a function says that the two may be the same memory.
 */
#ifndef ONEBIT_DECODER_H_
#define ONEBIT_DECODER_H_

#include "onebit_sparse_tensor.h"

#ifdef __cplusplus
extern "C" {
#endif

/* 8-bit codes of a cache */
#define ONEBIT_CODE_E4M3 0 /* OCP e4m3 (448 the largest, no infinities) */
#define ONEBIT_CODE_INT8 1 /* -127 ... 127 */

/* (tokens x heads x head_dim) values: consecutive within a head; strides in elements */
typedef struct onebit_heads {
  void *data;
  long long token_stride, head_stride;
} onebit_heads;

/*
 * Keys and values of one layer. Codes: pages x kv_heads x block x head_dim, 16-byte aligned; a token's value is its code
 * times the scale of its page and head (pages x kv_heads, fp32, not negative). block: 16, 32, 64 or 128 tokens; head_dim: 64 or 128.
 * Codes of a sequence's tokens are not NaN (an append writes none): attention would carry one to rows that do not see its token.
 * Attention takes a v_scale below 2^-99 as good as 0; a row that sees no values but some 2^-100 of those that rows beside it see may take them as 0 too. The
 * largest v_scale is 2^122, and sums of values over a sequence's keys are fp32: what exceeds it is infinite.
 */
typedef struct onebit_cache {
  void *k, *v;
  float *k_scale, *v_scale;
  int pages, kv_heads, block, head_dim;
  int code; /* ONEBIT_CODE_* */
} onebit_cache;

/*
 * The sequences of a call. Tokens [j * block, (j + 1) * block) of sequence s lie in page page_table[s * width + j]; an entry
 * outside of [0, pages) holds none (it is neither written nor attended to). lengths[s] counts the tokens of the sequence WITH
 * the call's new ones, which are its last: rows starts[s] ... starts[s + 1] - 1 of the call's token-major operands, or, with
 * starts NULL, tokens / count rows each. Lengths beyond width * block (at most 2^30) and starts outside of [0, tokens] are clamped.
 * Rows of no sequence are not read; what results hold there is not defined.
 */
typedef struct onebit_sequences {
  const int *page_table; /* count x width */
  const int *lengths;    /* count */
  const int *starts;     /* count + 1, or NULL */
  int count, width;
  int tokens;     /* rows of the token-major operands */
  int max_new;    /* no sequence has more new tokens (an append writes no keys and values of those beyond; attention does all, slower) */
  int max_length; /* what the launch is planned for; longer sequences are right and slower. 0: width * block */
} onebit_sequences;

/*
 * Rotary positions: of the first rotary_dim elements of each head, the pair (a, b) = (x[i], x[i + rotary_dim / 2]), or
 * (x[2 i], x[2 i + 1]) with interleaved != 0, becomes (a c - b s, b c + a s) in fp32, rounded once to the type of x; the other elements
 * are copied. table: fp32, positions x rotary_dim, a row's cosines c first, then its sines s. positions: tokens values, int32, or int64
 * with wide_positions != 0; a position outside of the table gives NaN. x and out may be the same memory (with equal strides).
 */
int onebit_rotary(const onebit_heads *x, const onebit_heads *out, int dtype, int tokens, int heads, int head_dim, const void *positions,
                  int wide_positions, const float *table, int table_rows, int rotary_dim, int interleaved, void *stream);

/*
 * Writes the new tokens' keys and values into the cache. With a table (else NULL) keys are turned as by onebit_rotary, by their
 * positions in their sequences, and so are the queries q into q_out (q NULL: none; q needs a table). scale' of a page and head is the
 * larger of the scale that its older tokens have and the new tokens' largest magnitude / 448 or 127; codes are value / scale' rounded
 * to nearest even, and where scale' grew, the older codes become (code * scale) / scale'. All in fp32. A page that starts with a
 * new token forgets its old scale. A NaN or an infinity among the new values makes the scale NaN or infinite and the codes 0, so that
 * what attends to the page is NaN. No two sequences may write into one page, and keys and values (with their scales) share no memory.
 */
int onebit_cache_append(const onebit_cache *cache, const onebit_sequences *sequences, const onebit_heads *k, const onebit_heads *v,
                        const onebit_heads *q, const onebit_heads *q_out, int heads, int dtype, const float *table, int table_rows,
                        int rotary_dim, int interleaved, void *stream);

/*
 * out = softmax(scale q k^T) v: the i-th of a sequence's n new tokens attends to its first length - n + i + 1 tokens, head h through
 * key/value head h / (heads / kv_heads). A row that attends to nothing is 0. scale may be negative. q and out: fp16 or bf16 (dtype), 16-byte aligned rows.
 * q and out may be the same memory (with equal strides). workspace: onebit_cache_attention_workspace() bytes, 16-byte aligned (NULL where that is 0).
 */
size_t onebit_cache_attention_workspace(const onebit_cache *cache, const onebit_sequences *sequences, int heads);
int onebit_cache_attention(const onebit_cache *cache, const onebit_sequences *sequences, const onebit_heads *q, const onebit_heads *out,
                           int heads, int dtype, float scale, void *workspace, void *stream);

/*
 * The norms around a block: h = residual_scale * residual + block_scale * gate * post(x), y = pre(h), with one pass over the rows.
 * post is left out where post_weight is NULL, the gate where it is NULL, and with x NULL h is residual_scale * residual. kind 0:
 * h / sqrt(mean(h^2) + eps) * weight + bias, kind 1: (h - mean(h)) / sqrt(var(h) + eps) * weight + bias (a bias NULL: none). All in fp32 from
 * the unrounded h; h and y are rounded once. h_out may be residual or x (with equal strides and types), or NULL (h is not wanted). Rows are hidden consecutive
 * values; strides in elements. gate: gate_row_stride between rows, gate_column_stride 0 or 1. hidden: at most 32768.
 */
typedef struct onebit_norm {
  const void *x, *residual;                         /* rows x hidden */
  void *h_out, *y;                                  /* rows x hidden */
  const void *weight, *bias, *post_weight, *post_bias; /* hidden values each */
  const void *gate;
  long long x_stride, residual_stride, h_stride, y_stride, gate_row_stride;
  int gate_column_stride;
  int x_dtype, residual_dtype /* and h_out's */, y_dtype, weight_dtype /* of the four */, gate_dtype;
  int rows, hidden, kind;
  float residual_scale, block_scale, eps;
} onebit_norm;
int onebit_block_norm(const onebit_norm *norm, void *stream);

#ifdef __cplusplus
}
#endif
#endif
