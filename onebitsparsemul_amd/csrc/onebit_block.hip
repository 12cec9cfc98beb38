// The product of 8-bit codes with a scale for each 128 (onebit_head.h): few tokens, and which kernel takes a call.
//
// Codes go into the matrix instructions as fp16, exactly, whose products are exact and whose sums are fp32 (v_mfma_f32_16x16x32_f16: 9e-9 off over a group of 128
// normal values; those of the 8-bit instructions cut the products of eight neighbours off at 2^-13 of the largest, 1.5e-5 over normal values: they serve 16-bit results of many tokens). The sum of a group, from 0 on, times the
// product of the two scales is added to the sums in fp32. The weight is the matrix operand A, the tokens are B's columns: a lane then holds four neighbouring rows of y of
// one token, so that its scale is one register, the weight's is the same for all lanes, and y is written in vectors.
#include "onebit_block.h"

#include <algorithm>

namespace onebit {
namespace {

// Few tokens: the weight goes by once, which bounds it: 16 tokens x 4096 -> 131072 109 us for 541 MB = 4.95 TB/s, as a large copy; small ones are a chain of a few loads (512 -> 4096 2.8 us). Loads of the
// weight past the caches: 116 us. A workgroup has R * 16 of its rows and 16 tokens, its wavefronts a part of the groups each; operands come straight from memory,
// a row's 128 codes as two halves that four lanes read side by side, and the wavefronts' sums meet in LDS. UNROLL groups are asked for at once.
template <int R, int WAVES, int UNROLL>
__global__ __launch_bounds__(64 * WAVES) void few_kernel(onebit_block_product p, BlockGrid grid) {
  typedef Operand<false> Values;
  constexpr int kRows = R * 16, kPitch = kRows + 1;
  __shared__ float sums[WAVES][16][kPitch];
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), r = lane % 16, q = lane / 16;
  const int tile = blockIdx.x / grid.tiles_n, first_row = tile * kRows, first_token = (blockIdx.x - tile * grid.tiles_n) * 16, split = blockIdx.y;
  const int low = split * grid.groups_per_split, high = min(low + grid.groups_per_split, p.columns / ONEBIT_CODE_GROUP);
  const int each = (high - low + WAVES - 1) / WAVES, begin = min(low + wave * each, high), end = min(begin + each, high);
  const uint8_t* w[R];
#pragma unroll
  for (int i = 0; i < R; ++i) w[i] = (const uint8_t*)p.weight.codes + min(first_row + i * 16 + r, p.rows - 1) * p.weight.row_stride + q * 16;
  const int token = min(first_token + r, p.tokens - 1);
  const uint8_t* const x = (const uint8_t*)p.x.codes + token * p.x.row_stride + q * 16;
  const float* const x_scale = p.x.scales + token * p.x.scale_stride;
  const float* const w_scale = p.weight.scales + first_row / ONEBIT_CODE_GROUP * p.weight.scale_stride;
  f4_t sum[R] = {};
  auto groups = [&](int g, auto count) {
    constexpr int kCount = decltype(count)::value;
    u4_t a[kCount][R][2], b[kCount][2];
    float scale[kCount];
#pragma unroll
    for (int u = 0; u < kCount; ++u)
#pragma unroll
      for (int i = 0; i < R; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) a[u][i][h] = *(const u4_t*)(w[i] + (long long)(g + u) * ONEBIT_CODE_GROUP + h * 64);
#pragma unroll
    for (int u = 0; u < kCount; ++u) {
#pragma unroll
      for (int h = 0; h < 2; ++h) b[u][h] = *(const u4_t*)(x + (long long)(g + u) * ONEBIT_CODE_GROUP + h * 64);
      scale[u] = x_scale[g + u];
    }
#pragma unroll
    for (int u = 0; u < kCount; ++u) {
      const Values bv(b[u][0], b[u][1]);
      const float s = scale[u] * w_scale[g + u];
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const f4_t part = Values(a[u][i][0], a[u][i][1]) * bv;
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[i][e] = __builtin_fmaf(part[e], s, sum[i][e]);
      }
    }
  };
  int g = begin;
  for (; g + UNROLL <= end; g += UNROLL) groups(g, std::integral_constant<int, UNROLL>());
  for (; g < end; ++g) groups(g, std::integral_constant<int, 1>());
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) sums[wave][r][i * 16 + q * 4 + e] = sum[i][e];
  __syncthreads();
  const Result result(p, grid, split);
  const int tokens = min(16, p.tokens - first_token);
  for (int at = threadIdx.x; at < tokens * kRows; at += 64 * WAVES) {
    const int t = at / kRows, row = at % kRows;
    float total = 0.f;
#pragma unroll
    for (int s = 0; s < WAVES; ++s) total += sums[s][t][row];
    result.put_one(first_token + t, first_row + row, total + result.bias_of(first_row + row));
  }
}

// Sums of the splits, in their order, with the bias. One thread: eight rows of a token.
__global__ __launch_bounds__(256) void add_splits_kernel(onebit_block_product p, BlockGrid grid) {
  const int units = (p.rows + 7) / 8;
  const long long at = (long long)blockIdx.x * 256 + threadIdx.x;
  if (at >= (long long)p.tokens * units) return;
  const int token = (int)(at / units), row = (int)(at % units) * 8;
  const long long apart = (long long)p.tokens * p.rows;
  const float* from = grid.partial + (long long)token * p.rows + row;
  const BlockGrid whole = {0, 0, 0, 1, 0, 0, nullptr};
  const Result result(p, whole, 0);
  float sum[8];
  result.load_bias(row, sum);
  // (four splits' loads under way, whole vectors from any place; a row's last few one by one)
  typedef float vector __attribute__((ext_vector_type(4), aligned(4)));
  const bool whole_unit = row + 8 <= p.rows;
  f4_t low = {}, high = {};
#pragma unroll 4
  for (int s = 0; s < grid.splits; ++s) {
    const float* const of_split = from + s * apart;
    if (whole_unit) {
      low += ((const vector*)of_split)[0], high += ((const vector*)of_split)[1];
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        low[i] += row + i < p.rows ? of_split[i] : 0.f;
        high[i] += row + 4 + i < p.rows ? of_split[4 + i] : 0.f;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) sum[i] += low[i], sum[i + 4] += high[i];
  result.put(token, row, sum);
}

template <int R, int WAVES, int UNROLL>
hipError_t launch_few_as(const onebit_block_product& p, BlockGrid grid, hipStream_t stream) {
  grid.tiles_n = (p.tokens + 15) / 16;
  const long long tiles = (p.rows + R * 16 - 1) / (R * 16) * (long long)grid.tiles_n;
  if (tiles * 64 * WAVES >= 1ll << 32) return hipErrorInvalidConfiguration;
  return launch_kernel(few_kernel<R, WAVES, UNROLL>, dim3((unsigned)tiles, grid.splits), dim3(64 * WAVES), 0, stream, p, grid);
}

}  // namespace

BlockGrid plan_block(const onebit_block_product& p, int compute_units) {
  const int groups = p.columns / ONEBIT_CODE_GROUP;
  BlockGrid grid = {0, kBlock16, 0, 1, groups, compute_units / 32 < 1 ? 1 : std::min(compute_units / 32, 8), nullptr};
  auto split = [&](int splits) {
    grid.groups_per_split = (groups + splits - 1) / splits;
    grid.splits = (groups + grid.groups_per_split - 1) / grid.groups_per_split;
  };
  // (a tile's copies know a row's distance in 32 bits)
  auto near = [](const onebit_codes& c) { return c.row_stride >= 0 && c.row_stride < 1 << 23; };
  const bool tiles_may = groups >= kLeastTileGroups && near(p.x) && near(p.weight);
  double least = 1e30;
  auto consider = [&](int kernel, int splits, double time) {
    // another launch, which waits for the sums of other compute units' caches; sums out and in again, at 3 TB/s
    if (splits > 1) time += 4.0 + 0.4 * splits + 8e-6 * splits * p.tokens * p.rows / 3.0;
    if (time < least) {
      least = time;
      grid.kernel = kernel;
      split(splits);
    }
  };
  // 16 tokens to a workgroup: a wavefront's groups one behind the other, or the bytes that the caches and the memory deliver (the tokens' codes for each workgroup again). Measured: 16
  // tokens on 131072 x 4096 with 64 rows 109 us (4.9 TB/s), with 32 rows 136, with 16 rows 163; 11008 x 4096 13.0, 14.6, 14.6 (one token 10.7, 11.5, 10.0); 4096 x 4096
  // 12.7, 8.9, 7.3 (eight wavefronts 6.7); 4096 x 512 3.6, 3.9, 2.7; 300 x 28672 67, 44, 36 (29.5, in two splits 16.2).
  struct Few {
    int kernel, rows, wavefronts;
    double start, step;
  };
  static const Few few[] = {{kBlock16, 16, 4, 2.2, 0.40}, {kBlock16Wide, 16, 8, 2.0, 0.80}, {kBlock64, 64, 4, 2.9, 1.05}};
  const long long token_tiles = (p.tokens + 15) / 16;
  const double weight_bytes = (double)p.rows * p.columns;
  for (const Few& kind : few) {
    // (eight wavefronts where each has more than eight groups, four steps of two: one token on 11008 x 16384 38 us, with four 46. Up to there either is at most a tenth ahead: 11008 x 8192 18.2
    // and 19.1, 11008 x 4096 10.6 and 10.2, sixteen tokens on 4096 x 4096 6.7 and 7.3.)
    if (kind.kernel == (groups > 64 ? kBlock16 : kBlock16Wide) || (kind.kernel == kBlock64 && token_tiles > 1 && tiles_may)) continue;
    const double blocks = (double)((p.rows + kind.rows - 1) / kind.rows) * token_tiles;
    const double through = 2.2 + std::max(weight_bytes / 4.9e6, (weight_bytes * token_tiles + blocks * std::min(p.tokens, 16) * p.columns) / 7e6);
    for (int splits = 1; splits <= 16 && (splits == 1 || groups / splits >= kind.wavefronts); ++splits) {
      if (splits > 1 && blocks * splits > 2 * compute_units) break;
      const int steps = ((groups + splits - 1) / splits + kind.wavefronts - 1) / kind.wavefronts;
      consider(kind.kernel, splits, std::max(kind.start + steps * kind.step, through));
    }
  }
  if (!tiles_may) return grid;
  // A group's time in a tile where workgroups are few and where every compute unit has its number, and what a tile costs beside them, fitted to 150 random shapes of 1 ... 3000 tokens,
  // 64 ... 60000 rows and 512 ... 14336 columns, which it meets to 3 to 6 %; not less than the weight takes from memory. The kernel that the plan takes is 2 % slower than the best of all in the mean. Products in fp16 are no good for the largest tile, which spills.
  struct Kind {
    int kernel, rows, tokens, on_unit;
    double start, alone, crowded, alone_in_fp16, crowded_in_fp16;
  };
  static const Kind kinds[] = {{kBlock128x32, 128, 32, 1, 3.5, 0.34, 0.55, 0.54, 0.57}, {kBlock64x64, 64, 64, 2, 3.5, 0.33, 0.49, 0.56, 0.80}, {kBlock128x64, 128, 64, 1, 3.8, 0.38, 0.48, 0.63, 0.78},
                               {kBlock256x128, 256, 128, 1, 7.0, 0.68, 0.87, 1.50, 2.10}, {kBlock256x256, 256, 256, 1, 10.0, 1.13, 1.63, 0., 0.}};
  const bool in_fp16 = !narrow_products(p);
  auto rounds_of = [&](const Kind& kind, long long blocks, int steps) {
    const double alone = in_fp16 ? kind.alone_in_fp16 : kind.alone, crowded = in_fp16 ? kind.crowded_in_fp16 : kind.crowded;
    const long long places = (long long)compute_units * kind.on_unit, rest = blocks % places;
    const double filled = kind.on_unit == 1 ? (double)rest / places : rest > compute_units;  // (of two workgroups, one has its compute unit to itself or has not)
    return (double)(blocks / places) * (steps * crowded + kind.start) + (rest ? steps * (alone + (crowded - alone) * filled) + kind.start : 0.);
  };
  for (const Kind& kind : kinds) {
    if ((kind.kernel == kBlock128x32 && p.tokens > 32) || (kind.kernel == kBlock256x256 && in_fp16)) continue;
    const long long tiles = (long long)((p.rows + kind.rows - 1) / kind.rows) * ((p.tokens + kind.tokens - 1) / kind.tokens);
    for (int splits = 1; splits <= 16 && groups / splits >= kLeastTileGroups; ++splits) {
      if (splits > 1 && tiles * splits > (long long)compute_units * kind.on_unit) break;
      consider(kind.kernel, splits, std::max(rounds_of(kind, tiles * splits, (groups + splits - 1) / splits), 3.0 + weight_bytes / 4.9e6));
    }
  }
  // Whole rounds of the largest tiles, and what is left in halves of them
  const Kind &half = kinds[3], &large = kinds[4];
  const long long tiles_n = (p.tokens + large.tokens - 1) / large.tokens, tiles_m = (p.rows + large.rows - 1) / large.rows, rounds = tiles_m * tiles_n / compute_units;
  const long long rows_of_tiles = rounds * compute_units / tiles_n;
  if (!in_fp16 && rounds > 0 && rows_of_tiles < tiles_m) {
    const long long halves = (tiles_m - rows_of_tiles) * ((p.tokens + half.tokens - 1) / half.tokens);
    consider(kBlockMixed, 1, rounds_of(large, rows_of_tiles * tiles_n, groups) + rounds_of(half, halves, groups));
    if (grid.kernel == kBlockMixed) grid.large = (int)(rows_of_tiles * tiles_n);
  }
  return grid;
}

size_t block_workspace(const onebit_block_product& p, const BlockGrid& grid) { return grid.splits > 1 ? (size_t)grid.splits * p.tokens * p.rows * sizeof(float) : 0; }

hipError_t launch_block_linear(const onebit_block_product& p, const BlockGrid& grid, hipStream_t stream) {
  hipError_t status;
  switch (grid.kernel) {
    case kBlock16: status = launch_few_as<1, 4, 2>(p, grid, stream); break;
    case kBlock16Wide: status = launch_few_as<1, 8, 2>(p, grid, stream); break;
    case kBlock64: status = launch_few_as<4, 4, 1>(p, grid, stream); break;
    default: status = launch_block_tiles(p, grid, stream);
  }
  if (status != hipSuccess || grid.splits == 1) return status;
  const long long blocks = ((long long)p.tokens * ((p.rows + 7) / 8) + 255) / 256;
  if (blocks >= 1ll << 24) return hipErrorInvalidConfiguration;
  return launch_kernel(add_splits_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, p, grid);
}

}  // namespace onebit
