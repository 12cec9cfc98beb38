// Host-visible launch interface of the kernels around the one-bit projections (internal to libonebitmul). Arguments are those of
// onebit_decoder.h, checked.
#pragma once
#include "onebit_decoder.h"
#include "onebit_launch.h"

namespace onebit {

struct RotaryArgs {
  onebit_heads x, out;
  int tokens, heads, head_dim;
  const void* positions;
  int wide_positions;
  const float* table;
  int table_rows, rotary_dim, interleaved;
};
hipError_t launch_rotary(const RotaryArgs& args, int dtype, hipStream_t stream);

struct AppendArgs {
  onebit_cache cache;
  onebit_sequences sequences;
  onebit_heads k, v, q, q_out;
  int heads;  // of q; 0: no q
  const float* table;
  int table_rows, rotary_dim, interleaved;
  int slots;  // pages a sequence's new tokens may touch, filled by the launcher
};
hipError_t launch_append(AppendArgs args, int dtype, hipStream_t stream);

struct AttentionArgs {
  onebit_cache cache;
  onebit_sequences sequences;
  onebit_heads q, out;
  int heads, group;  // group: heads of a key/value head
  uint32_t group_inverse;  // 2^32 / group, rounded up
  int dtype;
  float scale;
  int wide;  // few_rows_kernel with twice as many wavefronts
  int rows;  // of q to a workgroup: 16 (few_rows_kernel) or many_rows() (many_rows_kernel)
  // keys split over workgroups: split i takes keys [i * keys_per_split, ...) of its sequence; workspace: splits x tokens x heads rows of
  // head_dim fp32 sums, then as many pairs (running maximum, sum); splits == 1: none
  int splits, keys_per_split;
  float* workspace;
};
// Rows of q to a workgroup of many_rows_kernel
constexpr int many_rows(int head_dim) { return head_dim == 64 ? 128 : 256; }
// Fills rows and the split of `args`.
void plan_attention(AttentionArgs& args, int compute_units);
size_t attention_workspace(const AttentionArgs& args);
hipError_t launch_attention(const AttentionArgs& args, hipStream_t stream);
hipError_t launch_many_rows(const AttentionArgs& args, hipStream_t stream);  // without the pass that joins splits

hipError_t launch_norm(const onebit_norm& args, hipStream_t stream);

}  // namespace onebit
