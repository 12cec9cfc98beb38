// Host-visible launch interface of the kernels behind onebit_head.h (internal to libonebitmul). Arguments are checked.
#pragma once
#include "onebit_head.h"
#include "onebit_launch.h"

namespace onebit {

hipError_t launch_quantize_rows(const void* x, int dtype, long long x_stride, int rows, int columns, const onebit_codes& out, hipStream_t stream);

// A product's launch. Groups of 128 columns split over workgroups: split s takes groups [s * groups_per_split, ...) of all, and writes fp32 sums to
// partial + s * tokens * rows; a second kernel adds them in order. splits == 1: straight into y.
enum BlockKernel { kBlock16, kBlock16Wide, kBlock64, kBlock128x32, kBlock64x64, kBlock128x64, kBlock256x128, kBlock256x256, kBlockMixed };
// (rows of the weight, wide: on eight wavefronts; rows x tokens; mixed: the last two)
constexpr int kLeastTileGroups = 4;  // of a tile's split
// Tiles for 16-bit results of many tokens take the 8-bit matrix instruction, twice as fast. It cuts the products of eight neighbouring columns off at 2^-13 of the largest: over 4096
// columns 1.5e-5 of the result's norm for normal values, 6.3e-5 with one column of eight hundreds of times the others, where an fp16 result's own rounding is 2.1e-4. (At most 7 2^-13
// of the sum of those largest: more than the rounding where they cancel.) The others take the products in fp16.
inline bool narrow_products(const onebit_block_product& p) { return p.y_dtype != ONEBIT_DTYPE_F32 && p.tokens > 16; }
struct BlockGrid {
  int tiles_n;  // of tokens, filled by the launcher
  int kernel;
  int large;    // kBlockMixed: how many tiles of 256 x 256, whole rows of them
  int splits, groups_per_split;
  int xcds;  // workgroup b runs on XCD b % xcds
  float* partial;
};
BlockGrid plan_block(const onebit_block_product& args, int compute_units);
size_t block_workspace(const onebit_block_product& args, const BlockGrid& grid);
hipError_t launch_block_linear(const onebit_block_product& args, const BlockGrid& grid, hipStream_t stream);
hipError_t launch_block_tiles(const onebit_block_product& args, const BlockGrid& grid, hipStream_t stream);  // without the pass that adds splits

size_t sample_workspace(const onebit_sampling& args);
hipError_t launch_sample(const onebit_sampling& args, void* workspace, hipStream_t stream);

}  // namespace onebit
