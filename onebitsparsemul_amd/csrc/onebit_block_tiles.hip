// The product of 8-bit codes for many tokens: tiles of both operands in LDS.
//
// Bound by the waits between the matrix instructions and by whole rounds of tiles: 2048 tokens x 4096 -> 11008 88 to 91 us, in which the matrix units are busy 45 % of the clocks (2.13 GHz), 4096 x 8192 -> 8192, two
// rounds without a rest, 228 to 238 us = 2.3 to 2.4 PFLOP/s, busy 60 % of them (at 1.91 GHz: the clock falls with the load). Each product of
// 16 x 16 x 128 takes the matrix unit 32 clocks, and its four values per lane four multiply-adds with the scales: two wavefronts to a SIMD hide them, so that eight wavefronts
// have a tile; four with products of 128 x 128 each would read less from LDS, and spill. LDS is read without conflicts.
// In fp16 (fp32 results) 2048 x 4096 -> 11008 198 to 201 us = 0.92 PFLOP/s, 4096 x 8192 -> 8192 490 us = 1.12, busy 40 and 50 %. 333 x 1408 -> 4099 8.6 us, 128 x 4096 -> 11008 17.0.
#include "onebit_block.h"
#include "onebit_device.h"

#include <atomic>

namespace onebit {
namespace {

// Wave tiles of FM x FN products of 16 x 16, WM x WN of them to a workgroup; a ring of STAGES groups in LDS. NARROW: the 8-bit matrix instruction.
template <int WM, int WN, int FM, int FN, int STAGES>
struct Tile {
  static constexpr int kWaves = WM * WN, kRows = WM * FM * 16, kTokens = WN * FN * 16;
  // Scales of a wavefront's own tokens, of four groups at a time, of eight in all
  static constexpr int kStage = (kRows + kTokens) * ONEBIT_CODE_GROUP, kScales = 2 * 64 * 16, kLds = STAGES * kStage + kWaves * kScales;
  static constexpr int kCopies = (kRows + kTokens) / 8 / kWaves;  // of 8 rows of 128 codes, to a wavefront
  // A group in a wavefront's products of FM rows: in front of row kRelease all of it is in registers, and copies may begin to take its place, one to each kApart
  // products from there on; in front of row kLanding the next group is there.
  static constexpr int kRelease = FM / 2, kLanding = FM > 4 ? FM - 2 : kRelease, kSlots = FM > 4 ? 5 : 4;
  static constexpr int kApart = FM * FN >= 2 * kCopies ? 2 : 1, kAtOnce = (kCopies + FM * FN - 1) / (FM * FN);
  static constexpr int copies_before(int row) {  // of those from row kRelease on
    const int copies = ((row - kRelease) * FN + kApart - 1) / kApart * kAtOnce;
    return copies < kCopies ? copies : kCopies;
  }
  static constexpr int kEarly = copies_before(FM);  // the others in the next group's rows, in front of row kRelease
  static_assert((kRows + kTokens) / 8 % kWaves == 0 && kRows / 8 % kWaves == 0 && FM * 16 <= 128 && kLds <= 160 * 1024 && FM >= 2 && FN <= 4, "");
};

// Rows of 128 codes in LDS, their pieces of 16 at their number exclusive-or half of the row's: the sixteen lanes that LDS serves at a time read a piece of sixteen
// neighbouring rows from different banks. A lane takes pieces q and q + 4 of both operands' rows: any order of a group's columns will do, if it is one for both.
template <int WM, int WN, int FM, int FN, int STAGES, bool NARROW>
__device__ __forceinline__ void tile(const onebit_block_product& p, const BlockGrid& grid, int first_row, int m, int n, char* smem) {
  typedef Tile<WM, WN, FM, FN, STAGES> T;
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), wave_m = wave / WN, wave_n = wave % WN;
  const int split = blockIdx.y, all = p.columns / ONEBIT_CODE_GROUP, begin = split * grid.groups_per_split, count = min(grid.groups_per_split, all - begin);

  // copies: eight rows each, the weight's first
  uint32_t offset[T::kCopies];
#pragma unroll
  for (int c = 0; c < T::kCopies; ++c) {
    const int piece = c * T::kWaves + wave, row = piece * 8 + lane / 8, chunk = (lane % 8) ^ (row / 2 % 8);
    const bool of_weight = c < T::kRows / 8 / T::kWaves;
    const int from = of_weight ? min(first_row + m * T::kRows + row, p.rows - 1) - (first_row + m * T::kRows) : min(n * T::kTokens + row - T::kRows, p.tokens - 1) - n * T::kTokens;
    offset[c] = (uint32_t)(from * (int)(of_weight ? p.weight.row_stride : p.x.row_stride) + chunk * 16);
  }
  const char* weight = (const char*)p.weight.codes + (long long)(first_row + m * T::kRows) * p.weight.row_stride + (long long)begin * ONEBIT_CODE_GROUP;
  const char* x = (const char*)p.x.codes + (long long)n * T::kTokens * p.x.row_stride + (long long)begin * ONEBIT_CODE_GROUP;
  const float* x_scale = p.x.scales + (long long)min(n * T::kTokens + wave_n * FN * 16 + lane % (FN * 16), p.tokens - 1) * p.x.scale_stride;
  const float* w_scale = p.weight.scales + (long long)min((first_row + m * T::kRows + wave_m * FM * 16) / ONEBIT_CODE_GROUP, (p.rows - 1) / ONEBIT_CODE_GROUP) * p.weight.scale_stride + begin;
  const uint32_t lds = lds_offset_of(smem);
  auto copy = [&](int c, int g, int stage) {  // of a group beyond the last: of the last again, so that as many copies are under way
    g = min(g, count - 1);
    const uint32_t to = lds + stage * T::kStage;
    lds_dma16_base((c < T::kRows / 8 / T::kWaves ? weight : x) + (long long)g * ONEBIT_CODE_GROUP, offset[c], to + (c * T::kWaves + wave) * 1024);
  };
  // Scales of groups 4 b ... 4 b + 3; where the row ends among them, its last four. Each in a line of its own, they would cost a copy as much of the load path as eight rows of codes.
  const uint32_t scales = STAGES * T::kStage + wave * T::kScales;
  auto first_scale = [&](int b) { return min(begin + 4 * b, all - 4); };
  auto copy_scales = [&](int b) { lds_dma16(x_scale + first_scale(b), lds + scales + b % 2 * 1024); };

  typedef Operand<NARROW> Values;
  f4_t sum[FM][FN] = {}, part[2][FN] = {};
  float scale[FN] = {};
  // this lane's pieces of row lane % 16 of a 16-row part
  const int r = lane % 16, q = lane / 16, low = r * ONEBIT_CODE_GROUP + (q ^ (r / 2)) * 16, high = r * ONEBIT_CODE_GROUP + ((q + 4) ^ (r / 2)) * 16;
  auto read = [&](const char* part) { return Values(*(const u4_t*)(part + low), *(const u4_t*)(part + high)); };
  auto add = [&](f4_t& to, const f4_t& v, float s) {
#pragma unroll
    for (int e = 0; e < 4; ++e) to[e] = __builtin_fmaf(v[e], s, to[e]);
  };
  // Registers hold what the products need next: all of the tokens' values of a group, and some rows of the weight's.
  Values av[T::kSlots], bv[FN];
  float next[FN];
  auto read_weight = [&](int stage, int i) { av[i % T::kSlots] = read(smem + stage * T::kStage + (wave_m * FM + i) * 16 * ONEBIT_CODE_GROUP); };
  auto read_tokens = [&](int stage, int j) { bv[j] = read(smem + stage * T::kStage + (T::kRows + (wave_n * FN + j) * 16) * ONEBIT_CODE_GROUP); };
  auto read_scales = [&](int g) {
    const float* const of_group = (const float*)(smem + scales + g / 4 % 2 * 1024) + (begin + g - first_scale(g / 4));
#pragma unroll
    for (int j = 0; j < FN; ++j) next[j] = of_group[(j * 16 + r) * 4];
  };
  // The weight's scales of 64 groups, one to a lane: a load in the loop would be waited for with the copies in front of it. The first 64 come with the first copies, where the tokens' second ones will be.
  auto read_weight_scales = [&](int g) {
    float w = w_scale[min(g + lane, count - 1)];
    asm volatile("" : "+v"(w));  // (waited for here)
    return w;
  };
  lds_dma16(w_scale - begin + first_scale(lane), lds + scales + 1024);
  copy_scales(0);
#pragma unroll
  for (int s = 0; s < STAGES; ++s)
#pragma unroll
    for (int c = 0; c < (s == STAGES - 1 ? T::kEarly : T::kCopies); ++c) copy(c, s, s);
  wait_vmcnt_lgkm0<(STAGES - 2) * T::kCopies + T::kEarly>();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
#pragma unroll
  for (int j = 0; j < FN; ++j) read_tokens(0, j);
  read_weight(0, 0);
  read_weight(0, 1);
  read_scales(0);
  const int own = min(lane, count - 1);
  float w = ((const float*)(smem + scales + 1024))[own / 4 * 4 + begin + own - first_scale(own / 4)];
  int stage = 0;
  for (int g = 0; g < count; ++g) {
    const int following = stage + 1 == STAGES ? 0 : stage + 1, leading = stage ? stage - 1 : STAGES - 1;
    // the last group's last row; nothing before the first
#pragma unroll
    for (int j = 0; j < FN; ++j) add(sum[FM - 1][j], part[(FM - 1) % 2][j], scale[j]);
#pragma unroll
    for (int j = 0; j < FN; ++j) scale[j] = next[j] * __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), g % 64));
    if (g % 64 == 63) w = read_weight_scales(g + 1);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      if (i == T::kLanding) {
        wait_vmcnt_lgkm0<(STAGES - 2) * T::kCopies + T::copies_before(T::kLanding)>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
      } else if (i == T::kRelease) {
        wait_lgkm0();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
      }
      // rows 2 ... FM - 1 of the weight by row kRelease, two at a time in front and at the end
      if (i < T::kRelease) {
        constexpr int kDouble = FM - 2 - T::kRelease;  // rows of products that read two
        const int first = 2 + i + min(i, (kDouble + 1) / 2) + max(0, i - (T::kRelease - kDouble / 2));
        const bool two = i < (kDouble + 1) / 2 || i >= T::kRelease - kDouble / 2;
        if (first < FM) read_weight(stage, first);
        if (two) read_weight(stage, first + 1);
      }
      if (i == T::kLanding) read_scales(min(g + 1, count - 1));
      if (i == 0 && g % 4 == 0 && g + 4 < count) copy_scales(g / 4 + 1);
      if (i == FM - 1) read_weight(following, 0);
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        part[i % 2][j] = av[i % T::kSlots] * bv[j];
        if (i > 0) add(sum[i - 1][j], part[(i - 1) % 2][j], scale[j]);
        if (i == FM - 1) read_tokens(following, j);
        // products from row kRelease on, in the next group's rows from there on
        const int at = (i >= T::kRelease ? i - T::kRelease : FM - T::kRelease + i) * FN + j;
        if (at % T::kApart == 0) {
#pragma unroll
          for (int c = at / T::kApart * T::kAtOnce; c < min((at / T::kApart + 1) * T::kAtOnce, T::kCopies); ++c) {
            if (i >= T::kRelease) copy(c, g + STAGES, stage);
            else copy(c, g - 1 + STAGES, leading);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    read_weight(following, 1);
    __builtin_amdgcn_sched_barrier(0);
    stage = following;
  }
#pragma unroll
  for (int j = 0; j < FN; ++j) add(sum[FM - 1][j], part[(FM - 1) % 2][j], scale[j]);
  wait_vmcnt<0>();  // none into what follows, nor into LDS that another workgroup has by then
  __syncthreads();

  const Result result(p, grid, split);
  const int row = first_row + m * T::kRows + wave_m * FM * 16;
  auto add_bias = [&](auto zero) {  // (all loads first)
    typedef decltype(zero) T;
    T bias[FM][4];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) bias[i][e] = ((const T*)result.bias)[min(row + i * 16 + q * 4 + e, p.rows - 1)];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[i][j][e] += (float)bias[i][e];
  };
  if (result.bias) {
    if (p.bias_dtype == ONEBIT_DTYPE_F32) add_bias(0.f);
    else if (p.bias_dtype == ONEBIT_DTYPE_F16) add_bias((_Float16)0.f);
    else add_bias((__bf16)0.f);
  }
  // fp32 straight from the matrix instructions' registers; 16 bits through LDS, sixteen tokens at a time: neighbouring lanes then have neighbouring rows
  if (result.type == ONEBIT_DTYPE_F32) {
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int token = n * T::kTokens + (wave_n * FN + j) * 16 + r;
#pragma unroll
      for (int i = 0; i < FM; ++i)
        if (token < p.tokens) result.put_four(token, row + i * 16 + q * 4, sum[i][j]);
    }
    return;
  }
  constexpr int kLanes = FM * 2, kAtOnceTokens = 64 / kLanes, kPitch = FM * 32 + 16;  // lanes to a token, tokens of a store, bytes between tokens
  static_assert(T::kWaves * 2 * 16 * kPitch <= T::kLds, "");
#pragma unroll
  for (int j = 0; j < FN; ++j) {
    char* const rows = smem + (wave * 2 + j % 2) * 16 * kPitch;
#pragma unroll
    for (int i = 0; i < FM; i += 2) *(u4_t*)(rows + r * kPitch + (i + q % 2) * 32 + q / 2 * 16) = result.eight_of(sum[i][j], sum[i + 1][j]);
    __builtin_amdgcn_wave_barrier();
    const int token = (wave_n * FN + j) * 16 + lane / kLanes + n * T::kTokens;
#pragma unroll
    for (int t = 0; t < 16; t += kAtOnceTokens) {
      const u4_t eight = *(const u4_t*)(rows + (lane / kLanes + t) * kPitch + lane % kLanes * 16);
      if (token + t < p.tokens) result.put_eight(token + t, row + lane % kLanes * 8, eight);
    }
  }
}

// Number `block` of `total` tiles in rows of tiles_n, as a row and a column: the tiles of an XCD side by side, four rows of tiles at a time
struct Place {
  int m, n;
};
__device__ inline Place place_of(int block, int total, int tiles_n, int xcds) {
  const int tiles_m = total / tiles_n, x = block % xcds, tile = total / xcds * x + min(x, total % xcds) + block / xcds;
  constexpr int kStrip = 4;
  const int strip = tile / (kStrip * tiles_n), rest = tile - strip * kStrip * tiles_n, high = min(kStrip, tiles_m - strip * kStrip), n = rest / high;
  return {strip * kStrip + rest - n * high, n};
}

template <int WM, int WN, int FM, int FN, int STAGES, bool NARROW>
__global__ __launch_bounds__(64 * WM * WN) void tile_kernel(onebit_block_product p, BlockGrid grid) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const Place at = place_of(blockIdx.x, gridDim.x, grid.tiles_n, grid.xcds);
  tile<WM, WN, FM, FN, STAGES, NARROW>(p, grid, 0, at.m, at.n, smem);
}

// Tiles of 256 x 256 for as many of the weight's rows as whole rounds of the compute units take, the others in tiles of 256 x 128 behind them
typedef Tile<2, 4, 8, 4, 2> Large;
typedef Tile<4, 2, 4, 4, 3> Half;
__global__ __launch_bounds__(512) void mixed_kernel(onebit_block_product p, BlockGrid grid) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int block = blockIdx.x;
  if (block < grid.large) {
    const Place at = place_of(block, grid.large, grid.tiles_n, grid.xcds);
    tile<2, 4, 8, 4, 2, true>(p, grid, 0, at.m, at.n, smem);
  } else {
    const int tiles_n = (p.tokens + Half::kTokens - 1) / Half::kTokens;
    const Place at = place_of(block - grid.large, gridDim.x - grid.large, tiles_n, grid.xcds);
    tile<4, 2, 4, 4, 3, true>(p, grid, grid.large / grid.tiles_n * Large::kRows, at.m, at.n, smem);
  }
}

// The dynamic-LDS limit is a per-device attribute of the kernel; threads that race here set the same value
template <class Kernel>
hipError_t allow_lds(Kernel kernel, int bytes, std::atomic<bool> (&set)[64]) {
  int device = 0;
  if (hipError_t status = hipGetDevice(&device); status != hipSuccess) return status;
  if (device < 0 || device >= 64) return hipErrorInvalidDevice;
  if (set[device].load(std::memory_order_acquire)) return hipSuccess;
  if (hipError_t status = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes); status != hipSuccess) return status;
  set[device].store(true, std::memory_order_release);
  return hipSuccess;
}

template <int WM, int WN, int FM, int FN, int STAGES, bool NARROW>
hipError_t launch_tiles_as(const onebit_block_product& p, BlockGrid grid, hipStream_t stream) {
  typedef Tile<WM, WN, FM, FN, STAGES> T;
  auto kernel = tile_kernel<WM, WN, FM, FN, STAGES, NARROW>;
  static std::atomic<bool> set[64] = {};
  if (hipError_t status = allow_lds(kernel, T::kLds, set); status != hipSuccess) return status;
  const int tiles_m = (p.rows + T::kRows - 1) / T::kRows, tiles_n = (p.tokens + T::kTokens - 1) / T::kTokens;
  grid.tiles_n = tiles_n;
  if ((long long)tiles_m * tiles_n * 64 * T::kWaves >= 1ll << 32) return hipErrorInvalidConfiguration;
  return launch_kernel(kernel, dim3((unsigned)((long long)tiles_m * tiles_n), grid.splits), dim3(64 * T::kWaves), T::kLds, stream, p, grid);
}

template <int WM, int WN, int FM, int FN, int STAGES>
hipError_t launch_tiles(const onebit_block_product& p, const BlockGrid& grid, hipStream_t stream) {
  return narrow_products(p) ? launch_tiles_as<WM, WN, FM, FN, STAGES, true>(p, grid, stream) : launch_tiles_as<WM, WN, FM, FN, STAGES, false>(p, grid, stream);
}

}  // namespace

hipError_t launch_block_tiles(const onebit_block_product& p, const BlockGrid& grid, hipStream_t stream) {
  switch (grid.kernel) {
    case kBlockMixed: {
      static std::atomic<bool> set[64] = {};
      constexpr int kLds = Large::kLds > Half::kLds ? Large::kLds : Half::kLds;
      if (hipError_t status = allow_lds(mixed_kernel, kLds, set); status != hipSuccess) return status;
      BlockGrid mixed = grid;
      mixed.tiles_n = (p.tokens + Large::kTokens - 1) / Large::kTokens;
      const int rows_left = p.rows - grid.large / mixed.tiles_n * Large::kRows;
      const long long half = (long long)((rows_left + Half::kRows - 1) / Half::kRows) * ((p.tokens + Half::kTokens - 1) / Half::kTokens);
      if ((grid.large + half) * 512 >= 1ll << 32) return hipErrorInvalidConfiguration;
      return launch_kernel(mixed_kernel, dim3((unsigned)(grid.large + half)), dim3(512), kLds, stream, p, mixed);
    }
    case kBlock128x32: return launch_tiles<4, 1, 2, 2, 3>(p, grid, stream);
    case kBlock64x64: return launch_tiles<2, 2, 2, 2, 4>(p, grid, stream);
    case kBlock128x64: return launch_tiles<4, 2, 2, 2, 3>(p, grid, stream);
    case kBlock256x128: return launch_tiles<4, 2, 4, 4, 3>(p, grid, stream);
    default: return !narrow_products(p) ? hipErrorInvalidValue : launch_tiles_as<2, 4, 8, 4, 2, true>(p, grid, stream);  // (the plan takes no other)
  }
}

}  // namespace onebit
