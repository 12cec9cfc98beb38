// C ABI of onebit_decoder.h: argument validation and launches. Host code only.
#include "onebit_decoder_launch.h"

#include <algorithm>
#include <cstdarg>
#include <cstdio>

namespace {

int fail(int code, const char* fmt, ...) {
  char text[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(text, sizeof text, fmt, ap);
  va_end(ap);
  return onebit::report(code, text);
}
template <class... Values>
int refuse(const char* fmt, Values... values) { return fail(ONEBIT_ERR_ARGUMENT, fmt, values...); }
int launched(hipError_t status, const char* what) {
  return status == hipSuccess ? ONEBIT_OK : fail(ONEBIT_ERR_HIP, "HIP error '%s' from %s", hipGetErrorString(status), what);
}

bool aligned(const void* p, int to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }
bool is_type(int dtype) { return dtype == ONEBIT_DTYPE_F32 || dtype == ONEBIT_DTYPE_F16 || dtype == ONEBIT_DTYPE_BF16; }

int check_cache(const onebit_cache* c) {
  if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale) return refuse("null pointer in the cache");
  if (!aligned(c->k, 16) || !aligned(c->v, 16)) return refuse("the cache's codes must be 16-byte aligned");
  if (c->pages < 1 || c->kv_heads < 1 || c->kv_heads > 65535) return refuse("a cache has pages and 1 to 65535 heads (got %d, %d)", c->pages, c->kv_heads);
  if (c->block != 16 && c->block != 32 && c->block != 64 && c->block != 128) return refuse("block = %d: pages hold 16, 32, 64 or 128 tokens", c->block);
  if (c->head_dim != 64 && c->head_dim != 128) return refuse("head_dim = %d: the cache takes heads of 64 and 128", c->head_dim);
  if (c->code != ONEBIT_CODE_E4M3 && c->code != ONEBIT_CODE_INT8) return refuse("code must be 0 (e4m3) or 1 (int8), got %d", c->code);
  return ONEBIT_OK;
}
int check_sequences(const onebit_sequences* q, int block) {
  if (!q || !q->page_table || !q->lengths) return refuse("null pointer in the sequences");
  if (q->count < 1 || q->count > 65535 || q->width < 1) return refuse("1 to 65535 sequences and a page table of some width (got %d, %d)", q->count, q->width);
  if ((long long)q->width * block > 1ll << 30) return refuse("%d pages of %d tokens to a sequence exceed the int range that positions have: 2^30 tokens", q->width, block);
  if (q->tokens < 1 || q->max_new < 1 || q->max_length < 0) return refuse("tokens and max_new must be positive (got %d, %d)", q->tokens, q->max_new);
  if (!q->starts && q->tokens % q->count) return refuse("%d tokens do not divide into %d sequences: pass starts", q->tokens, q->count);
  return ONEBIT_OK;
}
// rows of heads in 16-byte vectors
int check_vectors(const onebit_heads* x, const char* name) {
  if (!x || !x->data) return refuse("%s must not be null", name);
  if (!aligned(x->data, 16) || x->token_stride % 8 || x->head_stride % 8)
    return refuse("%s must be 16-byte aligned, with strides that are multiples of eight", name);
  return ONEBIT_OK;
}
int check_table(const float* table, int rows, int rotary_dim, int head_dim) {
  if (!table || rows < 1) return refuse("the rotary table must have rows");
  if (rotary_dim < 2 || rotary_dim % 2 || rotary_dim > head_dim) return refuse("rotary_dim = %d must be even, from 2 to head_dim = %d", rotary_dim, head_dim);
  return ONEBIT_OK;
}
#define CHECKED(call) \
  if (const int code_ = (call)) return code_

onebit_sequences planned(const onebit_sequences& q) {
  onebit_sequences r = q;
  r.max_new = q.starts ? std::min(q.max_new, q.tokens) : q.tokens / q.count;
  return r;
}

int attention_args(const onebit_cache* cache, const onebit_sequences* sequences, int heads, onebit::AttentionArgs& args) {
  CHECKED(check_cache(cache));
  CHECKED(check_sequences(sequences, cache->block));
  if (heads < 1 || heads % cache->kv_heads) return refuse("heads = %d must be a multiple of kv_heads = %d", heads, cache->kv_heads);
  if ((long long)sequences->tokens * heads >= 1ll << 31) return refuse("tokens * heads exceeds the int range");
  args.cache = *cache;
  args.sequences = planned(*sequences);
  args.heads = heads;
  args.group = heads / cache->kv_heads;
  if (args.group > 32768) return refuse("%d heads to a key/value head: at most 32768", args.group);
  args.group_inverse = (uint32_t)(((1ull << 32) + args.group - 1) / args.group);
  onebit::plan_attention(args, onebit::device_compute_units());
  return ONEBIT_OK;
}

}  // namespace

extern "C" {

int onebit_rotary(const onebit_heads* x, const onebit_heads* out, int dtype, int tokens, int heads, int head_dim, const void* positions,
                  int wide_positions, const float* table, int table_rows, int rotary_dim, int interleaved, void* stream) {
  onebit::report(ONEBIT_OK, "");
  if (!x || !x->data || !out || !out->data || !positions) return refuse("null operand pointer");
  if (!is_type(dtype)) return refuse("dtype code must be 0 (fp32), 1 (fp16) or 2 (bf16), got %d", dtype);
  if (tokens < 1 || heads < 1 || head_dim < 2 || head_dim % 2 || head_dim > 65536)
    return refuse("tokens and heads must be positive and head_dim even (got %d, %d, %d)", tokens, heads, head_dim);
  if ((long long)heads * head_dim >= 1 << 24) return refuse("heads * head_dim exceeds 2^24");
  CHECKED(check_table(table, table_rows, rotary_dim, head_dim));
  const onebit::RotaryArgs args = {*x, *out, tokens, heads, head_dim, positions, wide_positions, table, table_rows, rotary_dim, interleaved};
  return launched(onebit::launch_rotary(args, dtype, (hipStream_t)stream), "onebit_rotary");
}

int onebit_cache_append(const onebit_cache* cache, const onebit_sequences* sequences, const onebit_heads* k, const onebit_heads* v,
                        const onebit_heads* q, const onebit_heads* q_out, int heads, int dtype, const float* table, int table_rows,
                        int rotary_dim, int interleaved, void* stream) {
  onebit::report(ONEBIT_OK, "");
  CHECKED(check_cache(cache));
  CHECKED(check_sequences(sequences, cache->block));
  CHECKED(check_vectors(k, "k"));
  CHECKED(check_vectors(v, "v"));
  if (!is_type(dtype)) return refuse("dtype code must be 0 (fp32), 1 (fp16) or 2 (bf16), got %d", dtype);
  if (table) {
    CHECKED(check_table(table, table_rows, rotary_dim, cache->head_dim));
    if (rotary_dim % 16 || !aligned(table, 16)) return refuse("an append turns multiples of 16 elements (got %d), by a table that is 16-byte aligned", rotary_dim);
  }
  if (q) {
    if (!table) return refuse("queries are only turned: q needs a rotary table");
    CHECKED(check_vectors(q, "q"));
    CHECKED(check_vectors(q_out, "q_out"));
    if (heads < 1 || heads > 65535) return refuse("heads must be 1 to 65535 (got %d)", heads);
  }
  onebit::AppendArgs args = {*cache, planned(*sequences), *k, *v, {}, {}, 0, table, table_rows, rotary_dim, interleaved, 0};
  if (q) args.q = *q, args.q_out = *q_out, args.heads = heads;
  return launched(onebit::launch_append(args, dtype, (hipStream_t)stream), "onebit_cache_append");
}

size_t onebit_cache_attention_workspace(const onebit_cache* cache, const onebit_sequences* sequences, int heads) {
  onebit::report(ONEBIT_OK, "");
  onebit::AttentionArgs args = {};
  return attention_args(cache, sequences, heads, args) ? 0 : onebit::attention_workspace(args);
}

int onebit_cache_attention(const onebit_cache* cache, const onebit_sequences* sequences, const onebit_heads* q, const onebit_heads* out,
                           int heads, int dtype, float scale, void* workspace, void* stream) {
  onebit::report(ONEBIT_OK, "");
  onebit::AttentionArgs args = {};
  CHECKED(attention_args(cache, sequences, heads, args));
  CHECKED(check_vectors(q, "q"));
  CHECKED(check_vectors(out, "out"));
  if (dtype != ONEBIT_DTYPE_F16 && dtype != ONEBIT_DTYPE_BF16) return refuse("q's dtype code must be 1 (fp16) or 2 (bf16), got %d", dtype);
  if (args.splits > 1 && (!workspace || !aligned(workspace, 16))) return refuse("this call needs a workspace of %zu bytes, 16-byte aligned", onebit::attention_workspace(args));
  args.q = *q;
  args.out = *out;
  args.dtype = dtype;
  args.scale = scale;
  args.workspace = (float*)workspace;
  return launched(onebit::launch_attention(args, (hipStream_t)stream), "onebit_cache_attention");
}

int onebit_block_norm(const onebit_norm* n, void* stream) {
  onebit::report(ONEBIT_OK, "");
  if (!n || !n->residual || !n->y || !n->weight) return refuse("residual, y and weight must not be null");
  if (n->rows < 1 || n->hidden < 1 || n->hidden > 32768) return refuse("rows must be positive and hidden 1 to 32768 (got %d, %d)", n->rows, n->hidden);
  if (n->kind != 0 && n->kind != 1) return refuse("kind must be 0 (rms) or 1 (layer), got %d", n->kind);
  if ((n->x && !is_type(n->x_dtype)) || !is_type(n->residual_dtype) || !is_type(n->y_dtype) || !is_type(n->weight_dtype) || (n->gate && !is_type(n->gate_dtype)))
    return refuse("dtype codes must be 0 (fp32), 1 (fp16) or 2 (bf16)");
  if (!n->x && (n->post_weight || n->gate)) return refuse("a norm behind the block and a gate need the block's output x");
  if (n->post_bias && !n->post_weight) return refuse("post_bias needs post_weight");
  if (n->gate && n->gate_column_stride != 0 && n->gate_column_stride != 1) return refuse("gate_column_stride must be 0 or 1 (got %d)", n->gate_column_stride);
  return launched(onebit::launch_norm(*n, (hipStream_t)stream), "onebit_block_norm");
}

}  // extern "C"
