// Attention over the 8-bit cache (onebit_decoder.h) for a few rows of q to a key/value head: sixteen rows (tokens x heads of the key/value
// head) to a workgroup, whose wavefronts share its keys out and each keep a running maximum, sum and output of their own.
//
// What bounds it: memory where sequences are long, and the chain of loads in front (lengths and pages, scales, codes) where they are not. One token behind
// 131072, 32 heads of 128 on 8, int8: 54 us for 269 MB = 4.9 TB/s (a large copy reaches 5.1), with the join 59. Sixteen sequences of 500 to 4096
// tokens: 19 to 20 us for 69 MB = 3.5 TB/s, the join 3 to 4; the matrix unit is busy in 5 % of the clocks, wavefronts wait for loads in half of theirs. One token
// behind 1000, heads of 64: 5.5 us and the join 2 to 3, nearly all of it that chain and the two launches.
// Why this split: sixteen rows are the columns of a matrix instruction; columns that few heads leave empty cost nothing beside the loads. Four wavefronts, each
// with the next step's codes asked for as soon as this step's registers are free, keep enough bytes under way with three workgroups to a compute unit
// (one step at a time and one wavefront: 78 us for the long sequence, 38 for the sixteen).
#include "onebit_attention.h"

#include <algorithm>

namespace onebit {
namespace {

constexpr int kRows = 16, kWaves = 4;  // wavefronts of a workgroup: kWaves, or twice as many

template <int D, int CODE, int WAVES>
__global__ __launch_bounds__(WAVES * 64, WAVES == kWaves ? 3 : 2) void few_rows_kernel(AttentionArgs args, int row_tiles) {
  // a step: as many tiles of 16 keys as 2 KiB of keys are, each two of them the K of an fp16 matrix instruction
  constexpr int kTiles = 256 / D, kChunk = 16 * kTiles;
  constexpr int kStride = D + 4;  // floats of a row of sums in LDS
  __shared__ __align__(16) float shared[WAVES * kRows * (kStride + 2)];
  typedef uint32_t value_words __attribute__((ext_vector_type(D / 64)));
  const onebit_cache& cache = args.cache;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64, r = lane % 16, g = lane / 16;
  const int first_tile = row_tiles == 1 ? 0 : blockIdx.x / args.splits, split = blockIdx.x - first_tile * args.splits, head = blockIdx.y, s = blockIdx.z;
  const int block_bits = __builtin_ctz(cache.block), low = split * args.keys_per_split;
  const int* const table = args.sequences.page_table + (long long)s * args.sequences.width;
  // The split's first pages are asked for before its sequence is known.
  Window window = load_pages(low >> block_bits, args.sequences.width, table, cache);
  const Sequence seq = read_sequence(args.sequences, s, cache.block);
  const int rows = seq.fresh * args.group;
  const long long all_rows = (long long)args.sequences.tokens * args.heads;
  float* const pairs = args.workspace + (long long)args.splits * all_rows * D;

  for (int tile = first_tile; tile * kRows < rows; tile += row_tiles) {
    // row of q of this lane's column, and how many keys it sees
    const int row = tile * kRows + r;
    const Rows own_first = first_row(tile * kRows, args.group), own_row = behind(own_first, r, args);
    const int token = own_row.token, query_head = head * args.group + own_row.head;
    const int seen = row < rows ? max(seq.length - seq.fresh + token + 1, 0) : 0;
    const int last_token = behind(own_first, min(kRows, rows - tile * kRows) - 1, args).token;
    const int total = max(seq.length - seq.fresh + last_token + 1, 0);
    const int all_see = tile * kRows + kRows <= rows ? max(seq.length - seq.fresh + own_first.token + 1, 0) : 0;
    const int high = split == args.splits - 1 ? total : min(total, low + args.keys_per_split);
    const int chunks = max(high - low + kChunk - 1, 0) / kChunk, per_wave = (chunks + WAVES - 1) / WAVES;
    const int first = low + min(wave * per_wave, chunks) * kChunk, end = min(low + min((wave + 1) * per_wave, chunks) * kChunk, high);

    u4_t raw[D / 64][2] = {};
    if (row < rows) {
      const uint16_t* const at = (const uint16_t*)args.q.data + (seq.start + token) * args.q.token_stride + query_head * args.q.head_stride + 16 * g;
#pragma unroll
      for (int u = 0; u < D / 64; ++u) raw[u][0] = *(const u4_t*)(at + 64 * u), raw[u][1] = *(const u4_t*)(at + 64 * u + 8);
    }

    f4_t sums[D / 16] = {};
    float most = -INFINITY, total_p = 0.f;
    Exponent v_exponent;  // p takes v_scale 2^(14 - exponent of the step's largest)

    // Codes of a chunk as they come from memory: lane (r, g) takes key r of each tile for the scores (bytes 64 u + 16 g of its row), and keys
    // 4 g ... 4 g + 3 of each tile for the values (D / 16 bytes from r D / 16 on). The next chunk's are asked for as soon as this one's are used.
    u4_t raw_k[kTiles][D / 64];
    value_words raw_v[4 * kTiles];
    int valid[kTiles];  // keys of a tile that are there
    long long place[kTiles];
    int entries[kTiles];
    float k_scale[kTiles], v_scale[kTiles];
    int powers[kTiles];  // exponents of v_scale
    auto find_scales = [&] {
      const int power = exponent_of(magnitude(usable_scale(window.v_scale)));
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        k_scale[t] = lane_value(window.k_scale, entries[t]);
        v_scale[t] = lane_value(window.v_scale, entries[t]);
        powers[t] = __builtin_amdgcn_readlane(power, entries[t]);
      }
    };
    auto find = [&](int key) {
      if ((key + kChunk - 1) >> block_bits >= window.first + 64) {
        window = load_pages(key >> block_bits, args.sequences.width, table, cache);
        drop_pages(window, (end - 1) >> block_bits);
        load_scales(window, cache, head);
      }
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        const int at = key + 16 * t, entry = min((at >> block_bits) - window.first, 63);
        const int page = __builtin_amdgcn_readlane(window.page, entry);
        valid[t] = page < 0 ? 0 : min(max(end - at, 0), 16);
        entries[t] = entry;
        place[t] = valid[t] == 0 ? 0 : (((long long)page * cache.kv_heads + head) * cache.block + (at & (cache.block - 1))) * D;
      }
    };
    auto load_keys = [&] {
#pragma unroll
      for (int t = 0; t < kTiles; ++t)
#pragma unroll
        for (int u = 0; u < D / 64; ++u) raw_k[t][u] = *(const u4_t*)((const uint8_t*)cache.k + place[t] + (r * D + 64 * u + 16 * g));
    };
    auto load_values = [&] {
#pragma unroll
      for (int t = 0; t < kTiles; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) raw_v[4 * t + i] = *(const value_words*)((const uint8_t*)cache.v + place[t] + ((4 * g + i) * D + r * (D / 16)));
    };

    if (first < end) {
      if (tile != first_tile || (first >> block_bits) - window.first >= 32) window = load_pages(first >> block_bits, args.sequences.width, table, cache);
      drop_pages(window, (end - 1) >> block_bits);
      load_scales(window, cache, head);
      find(first);
      load_keys();
      load_values();
      find_scales();  // (behind the first codes' loads: they wait for the pages alone)
    }
    h8_t q[D / 64][2];
    float row_factor = args.scale * kLog2E;
    {
      float factor = 1.f;
      if (args.dtype == ONEBIT_DTYPE_BF16) {  // rows as q 2^(8 - e), e the exponent of their largest value
        uint32_t largest = 0;
#pragma unroll
        for (int u = 0; u < D / 64; ++u) largest = max(largest, max(magnitude_bf16(raw[u][0]), magnitude_bf16(raw[u][1])));
        largest = __float_as_uint(max_over_16(__uint_as_float(min(largest, 0x7f800000u))));
        const int e = max(exponent_of(largest), -100);
        factor = power_of_two(8 - e);
        row_factor *= power_of_two(e - 8);
      }
#pragma unroll
      for (int u = 0; u < D / 64; ++u) q[u][0] = q_to_f16(raw[u][0], args.dtype, factor), q[u][1] = q_to_f16(raw[u][1], args.dtype, factor);
    }

    for (int key = first; key < end; key += kChunk) {
      f4_t scores[kTiles] = {};
#pragma unroll
      for (int t = 0; t < kTiles; ++t)
#pragma unroll
        for (int u = 0; u < D / 64; ++u) {
          scores[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes_to_f16<CODE>(raw_k[t][u].x, raw_k[t][u].y), q[u][0], scores[t], 0, 0, 0);
          scores[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes_to_f16<CODE>(raw_k[t][u].z, raw_k[t][u].w), q[u][1], scores[t], 0, 0, 0);
        }
      int there[kTiles], there_all = 0;
      float k_factor[kTiles], own_v[kTiles];
      int power = -1000;
      // of the least v_scale, above -99; what is as good as 0, or not finite and so reaches the sums by itself, wraps round and is none
      uint32_t least = ~0u;
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        there[t] = valid[t];
        there_all += valid[t];
        k_factor[t] = row_factor * k_scale[t];
        own_v[t] = v_scale[t];
        power = max(power, powers[t]);
        least = min(least, (uint32_t)(powers[t] + 99));
      }
      const bool more = key + kChunk < end;
      if (more) {
        find(key + kChunk);
        find_scales();
        load_keys();
      }
      const bool masked = key + kChunk > all_see || there_all < kChunk;
#pragma unroll
      for (int t = 0; t < kTiles; ++t) scores[t] *= k_factor[t];
      if (masked) {
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int left = min(seen - key - 16 * t, there[t]) - 4 * g;
            scores[t][i] = i < left ? scores[t][i] : -INFINITY;
            // codes of keys that are not there may be NaN, which a p of 0 would not hide
            if (4 * g + i >= there[t]) raw_v[4 * t + i] = 0;
          }
      }
      float top = scores[0][0];
#pragma unroll
      for (int i = 1; i < 4 * kTiles; ++i) top = fmaxf(top, scores[i / 4][i % 4]);
      top = max_over_16(top);
      const float v_keep = v_exponent.follow(power);
      if (__any(top > most) || v_keep != 1.f) {
        const float next = fmaxf(top, most), keep = most == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(most - next);
        most = next;
        total_p *= keep;
#pragma unroll
        for (int j = 0; j < D / 16; ++j) sums[j] *= keep * v_keep;
      }
      const float base = most == -INFINITY ? 0.f : most, v_factor = power_of_two(14 - v_exponent.now);
      // the values of 32 keys, four dims at a time, as the left operands of D / 16 products
      auto multiply_values = [&](int c, auto read, auto product) {
#pragma unroll
        for (int w = 0; w < D / 64; ++w) {
          uint32_t near[4], far[4];
          const value_words* const v = raw_v + 8 * c;
          transpose_bytes(read(v[0][w]), read(v[1][w]), read(v[2][w]), read(v[3][w]), near);
          transpose_bytes(read(v[4][w]), read(v[5][w]), read(v[6][w]), read(v[7][w]), far);
#pragma unroll
          for (int i = 0; i < 4; ++i) product(sums[4 * w + i], codes_to_f16<CODE>(near[i], far[i]));
        }
      };
      if (least < (uint32_t)max(v_exponent.now - 6 + 99, 0)) {
        // Pages of one step whose scales are far apart: p of the smaller ones would lose its bits beside the largest, which not all rows need see. By
        // themselves, in their own power, and then no more.
        auto apart = [](uint32_t word) {  // for which the compiler does not keep what the products below need too
          asm("" : "+v"(word));
          return word;
        };
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
          const int own_power = exponent_of(magnitude(usable_scale(own_v[t])));
          if (own_power <= -100 || own_power >= v_exponent.now - 6) continue;
          const float factor = own_v[t] * power_of_two(14 - own_power), down = power_or_zero(own_power - v_exponent.now);
          h8_t high = {}, low = {};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float weighted = __builtin_amdgcn_exp2f(scores[t][i] - base) * factor;
            high[t % 2 * 4 + i] = (_Float16)weighted;
            low[t % 2 * 4 + i] = (_Float16)(weighted - (float)high[t % 2 * 4 + i]);
          }
          multiply_values(t / 2, apart, [&](f4_t& sum, h8_t codes) {
            f4_t own = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes, high, f4_t{}, 0, 0, 0);
            own = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes, low, own, 0, 0, 0);
            sum += own * down;
          });
          own_v[t] = 0.f;
        }
      }
      h8_t p_high[kTiles / 2], p_low[kTiles / 2];  // together 22 bits of p: the products wait for the codes, a second one is hidden
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        const float factor = own_v[t] * v_factor;
        float weighted[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float p = __builtin_amdgcn_exp2f(scores[t][i] - base);
          total_p += p;
          weighted[i] = p * factor;
        }
        if (masked && magnitude(factor) >= 0x7f800000u) {  // a row that does not see the key does not see its page's scale
#pragma unroll
          for (int i = 0; i < 4; ++i) weighted[i] = scores[t][i] == -INFINITY ? 0.f : weighted[i];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          p_high[t / 2][t % 2 * 4 + i] = (_Float16)weighted[i];
          p_low[t / 2][t % 2 * 4 + i] = (_Float16)(weighted[i] - (float)p_high[t / 2][t % 2 * 4 + i]);
        }
      }
#pragma unroll
      for (int c = 0; c < kTiles / 2; ++c)
        multiply_values(c, [](uint32_t word) { return word; }, [&](f4_t& sum, h8_t codes) {
          sum = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes, p_high[c], sum, 0, 0, 0);
          sum = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes, p_low[c], sum, 0, 0, 0);
        });
      if (more) load_values();
    }

    // the wavefronts' sums in the largest of their maxima, one behind the other, then added in their order
    float* const tops = shared + WAVES * kRows * kStride;
    float* const totals = tops + WAVES * kRows;
    total_p = sum_over_16(total_p);
    if (g == 0) tops[wave * kRows + r] = most;
    __syncthreads();
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) top = fmaxf(top, tops[w * kRows + r]);
    // (NaN goes on: a maximum that is none has no keys, or a NaN in its sum)
    const float share = most == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(most - top), v_factor = power_of_two(v_exponent.now - 14);
    if (row < rows) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < D / 16; j += 4)
          *(f4_t*)(shared + (wave * kRows + r) * kStride + (4 * g + i) * (D / 16) + j) =
              f4_t{sums[j][i], sums[j + 1][i], sums[j + 2][i], sums[j + 3][i]} * (share * v_factor);
      if (g == 0) totals[wave * kRows + r] = total_p * share;
    }
    __syncthreads();
    const int here = min(rows - tile * kRows, kRows);
    for (int item = threadIdx.x; item < here * (D / 4); item += WAVES * 64) {
      const int column = item / (D / 4), dim = item % (D / 4) * 4;
      float sum = 0.f, top = -INFINITY;
      f4_t out = {};
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        sum += totals[w * kRows + column];
        top = fmaxf(top, tops[w * kRows + column]);
        out += *(const f4_t*)(shared + (w * kRows + column) * kStride + dim);
      }
      const Rows of = behind(own_first, column, args);
      const long long own_token = seq.start + of.token;
      const int own_head = head * args.group + of.head;
      if (args.splits > 1) {
        const long long place = split * all_rows + own_token * args.heads + own_head;
        if (sum != 0.f) *(f4_t*)(args.workspace + place * D + dim) = out;
        if (dim == 0) *(f2_t*)(pairs + 2 * place) = f2_t{top, sum};
      } else {
        if (sum != 0.f) out /= sum;  // (a row that sees nothing: 0)
        const float values[4] = {out.x, out.y, out.z, out.w};
        const long long at = own_token * args.out.token_stride + own_head * args.out.head_stride + dim;
        if (args.dtype == ONEBIT_DTYPE_F16) store_values<ONEBIT_DTYPE_F16, 4>(args.out.data, at, values);
        else store_values<ONEBIT_DTYPE_BF16, 4>(args.out.data, at, values);
      }
    }
    __syncthreads();
  }
}

// Joins the splits of a row: one workgroup to a row, in the same order whatever order the splits ended in. The first splits' sums are asked for
// together with the maxima that weigh them.
template <int D, int THREADS>
__global__ __launch_bounds__(THREADS) void join_kernel(AttentionArgs args) {
  constexpr int kLanes = D / 4, kGroups = THREADS / kLanes, kAhead = 4;
  static_assert(kAhead * kGroups <= THREADS, "the splits ahead are weighed with the first");
  __shared__ float weights[THREADS];  // of as many splits at a time
  __shared__ float tops[THREADS / 64], totals[THREADS / 64];
  __shared__ f4_t parts[kGroups][kLanes];
  const long long row = blockIdx.x, all_rows = (long long)args.sequences.tokens * args.heads;
  const float* const pairs = args.workspace + (long long)args.splits * all_rows * D;
  const int group = threadIdx.x / kLanes, lane = threadIdx.x % kLanes, wave = threadIdx.x / 64;
  f4_t ahead[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    const int split = group + i * kGroups;
    if (split < args.splits) ahead[i] = *(const f4_t*)(args.workspace + (split * all_rows + row) * D + 4 * lane);
  }
  f2_t pair = {-INFINITY, 0.f};
  if (threadIdx.x < args.splits) pair = *(const f2_t*)(pairs + 2 * (threadIdx.x * all_rows + row));
  float top = pair.y != 0.f ? pair.x : -INFINITY;
  for (int split = threadIdx.x + THREADS; split < args.splits; split += THREADS) {
    const f2_t more = *(const f2_t*)(pairs + 2 * (split * all_rows + row));
    if (more.y != 0.f) top = fmaxf(top, more.x);
  }
  top = wave_max(top);
  if (THREADS > 64) {
    if (threadIdx.x % 64 == 0) tops[wave] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) top = fmaxf(top, tops[w]);
  }
  // (a split in which the row sees nothing has written no sums; NaN goes on)
  auto weigh = [&](f2_t p, float& total) {
    const float weight = p.y == 0.f ? 0.f : __builtin_amdgcn_exp2f(p.x - top);
    total += p.y == 0.f ? 0.f : weight * p.y;
    return weight;
  };
  float total = 0.f;
  weights[threadIdx.x] = weigh(pair, total);
  __syncthreads();
  f4_t out = {};
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    const int split = group + i * kGroups;
    if (split < args.splits && weights[split] != 0.f) out += ahead[i] * weights[split];
  }
  for (int begin = 0; begin < args.splits; begin += THREADS) {
    if (begin > 0) {
      __syncthreads();
      const int split = begin + threadIdx.x;
      if (split < args.splits) weights[threadIdx.x] = weigh(*(const f2_t*)(pairs + 2 * (split * all_rows + row)), total);
      __syncthreads();
    }
    const int from = begin == 0 ? kAhead * kGroups : begin, to = min(begin + THREADS, args.splits);
    for (int split = from + group; split < to; split += kGroups) {
      const float weight = weights[split - begin];
      if (weight != 0.f) out += *(const f4_t*)(args.workspace + (split * all_rows + row) * D + 4 * lane) * weight;
    }
  }
  total = wave_sum(total);
  if (threadIdx.x % 64 == 0) totals[wave] = total;
  parts[group][lane] = out;
  __syncthreads();
  if (group > 0) return;
  total = 0.f;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) total += totals[w];
  f4_t all = {};
#pragma unroll
  for (int i = 0; i < kGroups; ++i) all += parts[i][lane];
  if (total != 0.f) all /= total;
  const float values[4] = {all.x, all.y, all.z, all.w};
  const long long at = row / args.heads * args.out.token_stride + row % args.heads * args.out.head_stride + 4 * lane;
  if (args.dtype == ONEBIT_DTYPE_F16) store_values<ONEBIT_DTYPE_F16, 4>(args.out.data, at, values);
  else store_values<ONEBIT_DTYPE_BF16, 4>(args.out.data, at, values);
}

template <int D, int CODE>
hipError_t launch_few_rows(const AttentionArgs& args, hipStream_t stream) {
  const onebit_sequences& q = args.sequences;
  const int row_tiles = (int)(((long long)q.max_new * args.group + kRows - 1) / kRows);
  const dim3 grid(row_tiles * args.splits, args.cache.kv_heads, q.count);
  if (args.wide) return launch_kernel(few_rows_kernel<D, CODE, 2 * kWaves>, grid, dim3(128 * kWaves), 0, stream, args, row_tiles);
  return launch_kernel(few_rows_kernel<D, CODE, kWaves>, grid, dim3(64 * kWaves), 0, stream, args, row_tiles);
}
template <int D>
hipError_t launch_as(const AttentionArgs& args, hipStream_t stream) {
  const bool int8 = args.cache.code == ONEBIT_CODE_INT8;
  const hipError_t status = args.rows > kRows ? launch_many_rows(args, stream)
                            : int8            ? launch_few_rows<D, ONEBIT_CODE_INT8>(args, stream)
                                              : launch_few_rows<D, ONEBIT_CODE_E4M3>(args, stream);
  if (status != hipSuccess || args.splits == 1) return status;
  const dim3 rows((unsigned)((long long)args.sequences.tokens * args.heads));
  if (args.splits <= 4) return launch_kernel(join_kernel<D, 64>, rows, dim3(64), 0, stream, args);
  if (args.splits <= 32) return launch_kernel(join_kernel<D, 256>, rows, dim3(256), 0, stream, args);
  return launch_kernel(join_kernel<D, 1024>, rows, dim3(1024), 0, stream, args);
}

}  // namespace

// Rows of q to a workgroup, and how its keys are split over workgroups where a call has fewer of them than the device holds at once.
//
// few_rows_kernel reads the keys for every 16 rows again but starts and ends quickly and fills the device with few rows; many_rows_kernel does
// with a quarter of the work. The rule's numbers stand between what was measured, no quantity of the device among them, and calls near them may be better off
// on the other side. Both sides, few | many, us: one prompt of 512, 8 heads of 64 on 4 (256 workgroups) 6.8 | 13.7; one of 1024, 8 of 128 on 4
// (512) 17.9 | 26.3; one of 512, 32 of 128 on 8 (1024) 19.5 | 23.0; eight of 128, 16 of 64 on 16 (1024, but of 64 keys) 10.2 | 7.4; two of 512, 32 of 64 on 8 (2048)
// 21.2 | 14.4; 64 tokens behind 1936 in four sequences, 16 of 128 on 16 (256, 65 million values) 30.1 | 22.0; five of 37 to 512, 8 of 64 on 4 (1280, of which
// 756 have rows) 12.4 | 14.7.
// A split costs its join, some 3 us: few rows go unsplit up to three steps (500 keys, heads of 64: 6.5 us, 7.8 in two splits), four where a quarter of the device
// has work (16 sequences of 1000 on 8 heads of 64: 9.9 us, 10.8 in splits; 4 sequences on 4: 9.0, 8.5). Where a compute unit has no second workgroup to wait
// for and the steps are even, twice as many wavefronts take half of them each: 500 keys, heads of 64 6.7 us for 7.2, 64 sequences on 4 of them 7.7 for 8.3,
// 1000 keys 11.6 for 12.8; three steps gain nothing (8.9), and 512 workgroups of 500 keys take 14.5 for 11.5.
void plan_attention(AttentionArgs& args, int compute_units) {
  const onebit_sequences& q = args.sequences;
  const long long rows = (long long)q.max_new * args.group, room = (long long)q.width * args.cache.block;
  const long long most = std::max(1ll, q.max_length > 0 ? std::min(room, (long long)q.max_length) : room);
  auto workgroups = [&](int of) { return (rows + of - 1) / of * args.cache.kv_heads * q.count; };
  // that have rows, and the keys that one sees: half of its own tokens are behind it
  const long long busy = std::min(workgroups(kRows), ((long long)q.tokens * args.group / kRows + q.count) * args.cache.kv_heads);
  const long long keys_seen = most - std::min<long long>(q.max_new, most) / 2;
  const bool few = rows <= 32 || (busy <= (keys_seen >= 256 ? 4ll : 3ll) * compute_units && busy * keys_seen * args.cache.head_dim <= 148000ll * compute_units);
  args.rows = few ? kRows : many_rows(args.cache.head_dim);
  const long long units = workgroups(args.rows);
  // workgroups that splits are made for (of many_rows_kernel's for heads of 64 the device would hold a third to a compute unit)
  const long long slots = (few ? 3ll : args.rows == 128 ? 2ll : 1ll) * compute_units;
  // (the join has a workgroup of up to 1024 threads to each row, and a launch less than 2^32 of them)
  const long long splits = (long long)q.tokens * args.heads < 1 << 22 ? std::max(1ll, slots / units) : 1;
  // few rows: one step of each wavefront
  const long long least = few ? kWaves * 4096 / args.cache.head_dim : 8 * units <= compute_units && most >= 1024 ? 256 : 512;
  long long keys = std::max(least, ((most + splits - 1) / splits + least - 1) / least * least);
  if (few && most <= (4 * units > compute_units ? 4 : 3) * least) keys = most;
  args.wide = few && keys >= most && units <= compute_units && (most + least - 1) / least % 2 == 0;
  args.splits = (int)((most + keys - 1) / keys);
  args.keys_per_split = (int)keys;
}

size_t attention_workspace(const AttentionArgs& args) {
  return args.splits == 1 ? 0 : (size_t)args.splits * args.sequences.tokens * args.heads * (args.cache.head_dim + 2) * sizeof(float);
}

hipError_t launch_attention(const AttentionArgs& args, hipStream_t stream) {
  return args.cache.head_dim == 64 ? launch_as<64>(args, stream) : launch_as<128>(args, stream);
}

}  // namespace onebit
