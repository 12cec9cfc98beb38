// Attention over the 8-bit cache (onebit_decoder.h) for a few rows of q to a key/value head: sixteen rows (tokens x heads of the key/value
// head) to a workgroup, whose wavefronts share its keys out and each keep a running maximum, sum and output of their own.
#include "onebit_attention.h"

#include <algorithm>

namespace onebit {
namespace {

constexpr int kChunk = 32;  // keys of one step: two tiles of 16, the K of one fp16 matrix instruction
constexpr int kRows = 16;

// Codes of a chunk as they come from memory: lane (r = lane % 16, g = lane / 16) takes key r of each tile for the scores (bytes 64 u + 16 g
// of its row), and keys 4 g ... 4 g + 3 of each tile for the values (D / 16 bytes from r D / 16 on)
template <int D>
struct Chunk {
  typedef uint32_t value_words __attribute__((ext_vector_type(D / 64)));
  u4_t k[2][D / 64];
  value_words v[8];
  float k_scale[2], v_scale[2];
  int valid[2];  // keys of the tile that are there
};

template <int D, int CODE, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void few_rows_kernel(AttentionArgs args, int row_tiles) {
  constexpr int kStride = D + 4;  // floats of a row of sums in LDS
  __shared__ __align__(16) float shared[WAVES * kRows * (kStride + 2)];
  const onebit_cache& cache = args.cache;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64, r = lane % 16, g = lane / 16;
  const int split = blockIdx.x % args.splits, head = blockIdx.y, s = blockIdx.z;
  const Sequence seq = read_sequence(args.sequences, s, cache.block);
  const int rows = seq.fresh * args.group, block_bits = __builtin_ctz(cache.block);
  const int* const table = args.sequences.page_table + (long long)s * args.sequences.width;
  const long long all_rows = (long long)args.sequences.tokens * args.heads;
  float* const pairs = args.workspace + (long long)args.splits * all_rows * D;

  for (int tile = blockIdx.x / args.splits; tile * kRows < rows; tile += row_tiles) {
    // row of q of this lane's column, and how many keys it sees
    const int row = tile * kRows + r, token = row / args.group, query_head = head * args.group + row % args.group;
    const int seen = row < rows ? max(seq.length - seq.fresh + token + 1, 0) : 0;
    const int last_token = min(tile * kRows + kRows, rows) - 1;
    const int total = max(seq.length - seq.fresh + last_token / args.group + 1, 0);
    const int all_see = tile * kRows + kRows <= rows ? max(seq.length - seq.fresh + tile * kRows / args.group + 1, 0) : 0;
    const int low = split * args.keys_per_split, high = split == args.splits - 1 ? total : min(total, low + args.keys_per_split);
    const int chunks = max(high - low + kChunk - 1, 0) / kChunk, per_wave = (chunks + WAVES - 1) / WAVES;
    const int first = low + min(wave * per_wave, chunks) * kChunk, end = min(low + min((wave + 1) * per_wave, chunks) * kChunk, high);

    h8_t q[D / 64][2];
    float row_factor = args.scale * kLog2E;
    {
      u4_t raw[D / 64][2] = {};
      if (row < rows) {
        const uint16_t* const at = (const uint16_t*)args.q.data + (seq.start + token) * args.q.token_stride + query_head * args.q.head_stride + 16 * g;
#pragma unroll
        for (int u = 0; u < D / 64; ++u) raw[u][0] = *(const u4_t*)(at + 64 * u), raw[u][1] = *(const u4_t*)(at + 64 * u + 8);
      }
      float factor = 1.f;
      if (args.dtype == ONEBIT_DTYPE_BF16) {  // rows as q 2^(8 - e), e the exponent of their largest value
        uint32_t most = 0;
#pragma unroll
        for (int u = 0; u < D / 64; ++u) most = max(most, max(magnitude_bf16(raw[u][0]), magnitude_bf16(raw[u][1])));
        most = __float_as_uint(max_over_16(__uint_as_float(min(most, 0x7f800000u))));
        const int e = exponent_of(most, -100);
        factor = power_of_two(8 - e);
        row_factor *= power_of_two(e - 8);
      }
#pragma unroll
      for (int u = 0; u < D / 64; ++u) q[u][0] = q_to_f16(raw[u][0], args.dtype, factor), q[u][1] = q_to_f16(raw[u][1], args.dtype, factor);
    }

    f4_t sums[D / 16] = {};
    float most = -INFINITY, total_p = 0.f;
    int v_exponent = -100;  // p takes v_scale 2^(14 - v_exponent)

    Window window = {0, -1, 0.f, 0.f};
    auto refill = [&](int entry) {
      const int e = fill_window(window, entry, (end - 1) >> block_bits, table, cache, head);
      if (e > v_exponent) {
        const float down = v_exponent == -100 ? 0.f : power_of_two(max(v_exponent - e, -126));
#pragma unroll
        for (int j = 0; j < D / 16; ++j) sums[j] *= down;
        v_exponent = e;
      }
    };
    auto load = [&](int key) {
      Chunk<D> c;
      if ((key + kChunk - 1) >> block_bits >= window.first + 64) refill(key >> block_bits);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int at = key + 16 * t, entry = min((at >> block_bits) - window.first, 63);
        const int page = __builtin_amdgcn_readlane(window.page, entry);
        c.valid[t] = page < 0 ? 0 : min(max(end - at, 0), 16);
        c.k_scale[t] = lane_value(window.k_scale, entry);
        c.v_scale[t] = lane_value(window.v_scale, entry);
        const long long place = c.valid[t] == 0 ? 0 : (((long long)page * cache.kv_heads + head) * cache.block + (at & (cache.block - 1))) * D;
        const uint8_t* const k = (const uint8_t*)cache.k + place;
        const uint8_t* const v = (const uint8_t*)cache.v + place;
#pragma unroll
        for (int u = 0; u < D / 64; ++u) c.k[t][u] = *(const u4_t*)(k + (r * D + 64 * u + 16 * g));
#pragma unroll
        for (int i = 0; i < 4; ++i) c.v[4 * t + i] = *(const typename Chunk<D>::value_words*)(v + ((4 * g + i) * D + r * (D / 16)));
      }
      return c;
    };
    auto multiply = [&](Chunk<D>& c, int key) {
      f4_t scores[2] = {};
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int u = 0; u < D / 64; ++u) {
          scores[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes_to_f16<CODE>(c.k[t][u].x, c.k[t][u].y), q[u][0], scores[t], 0, 0, 0);
          scores[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes_to_f16<CODE>(c.k[t][u].z, c.k[t][u].w), q[u][1], scores[t], 0, 0, 0);
        }
      const bool masked = key + kChunk > all_see || c.valid[0] + c.valid[1] < kChunk;
#pragma unroll
      for (int t = 0; t < 2; ++t) scores[t] *= row_factor * c.k_scale[t];
      if (masked) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (key + 16 * t + 4 * g + i >= seen || 4 * g + i >= c.valid[t]) scores[t][i] = -INFINITY;
        // codes of keys that are not there may be NaN, which a p of 0 would not hide
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (4 * g + i % 4 >= c.valid[i / 4]) c.v[i] = 0;
      }
      float top = fmaxf(fmaxf(fmaxf(scores[0][0], scores[0][1]), fmaxf(scores[0][2], scores[0][3])),
                        fmaxf(fmaxf(scores[1][0], scores[1][1]), fmaxf(scores[1][2], scores[1][3])));
      top = max_over_16(top);
      if (__any(top > most)) {
        const float next = fmaxf(top, most), keep = most == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(most - next);
        most = next;
        total_p *= keep;
#pragma unroll
        for (int j = 0; j < D / 16; ++j) sums[j] *= keep;
      }
      const float base = most == -INFINITY ? 0.f : most, v_factor = power_of_two(14 - v_exponent);
      h8_t p_high, p_low;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const float v_scale = c.v_scale[t] * v_factor;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float p = __builtin_amdgcn_exp2f(scores[t][i] - base);
          total_p += p;
          float weighted = p * v_scale;
          if (masked && scores[t][i] == -INFINITY) weighted = 0.f;  // whatever the scale of a page that the row does not see
          p_high[4 * t + i] = (_Float16)weighted;
          p_low[4 * t + i] = (_Float16)(weighted - (float)p_high[4 * t + i]);
        }
      }
#pragma unroll
      for (int w = 0; w < D / 64; ++w) {  // four dims at a time
        uint32_t near[4], far[4];
        transpose_bytes(c.v[0][w], c.v[1][w], c.v[2][w], c.v[3][w], near);
        transpose_bytes(c.v[4][w], c.v[5][w], c.v[6][w], c.v[7][w], far);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const h8_t v = codes_to_f16<CODE>(near[i], far[i]);
          sums[4 * w + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, p_high, sums[4 * w + i], 0, 0, 0);
          sums[4 * w + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, p_low, sums[4 * w + i], 0, 0, 0);
        }
      }
    };

    if (first < end) {
      refill(first >> block_bits);
      Chunk<D> current = load(first);
      for (int key = first; key < end; key += kChunk) {
        Chunk<D> next = current;
        if (key + kChunk < end) next = load(key + kChunk);
        multiply(current, key);
        current = next;
      }
    }

    // the wavefronts' sums, one behind the other
    float* const own = shared + wave * kRows * kStride;
    float* const tops = shared + WAVES * kRows * kStride;
    float* const totals = tops + WAVES * kRows;
    const float v_factor = power_of_two(v_exponent - 14);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < D / 16; j += 4)
        *(f4_t*)(own + r * kStride + (4 * g + i) * (D / 16) + j) =
            f4_t{sums[j][i], sums[j + 1][i], sums[j + 2][i], sums[j + 3][i]} * v_factor;
    total_p = sum_over_16(total_p);
    if (g == 0) tops[wave * kRows + r] = most, totals[wave * kRows + r] = total_p;
    __syncthreads();
    for (int item = threadIdx.x; item < kRows * (D / 4); item += WAVES * 64) {
      const int column = item / (D / 4), dim = item % (D / 4) * 4, own_row = tile * kRows + column;
      if (own_row >= rows) continue;
      float top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) top = fmaxf(top, tops[w * kRows + column]);
      f4_t out = {};
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        const float own_top = tops[w * kRows + column];
        const float share = own_top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(own_top - top);
        sum += share * totals[w * kRows + column];
        if (own_top != -INFINITY) out += *(const f4_t*)(shared + (w * kRows + column) * kStride + dim) * share;
      }
      const long long own_token = seq.start + own_row / args.group;
      const int own_head = head * args.group + own_row % args.group;
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

// Joins the splits of a row: one workgroup to a row, in the order of the splits whatever order they ended in.
template <int D, int THREADS>
__global__ __launch_bounds__(THREADS) void join_kernel(AttentionArgs args) {
  constexpr int kLanes = D / 4, kGroups = THREADS / kLanes;
  __shared__ float tops[kGroups], totals[kGroups];
  __shared__ f4_t parts[kGroups][kLanes];
  const long long row = blockIdx.x, all_rows = (long long)args.sequences.tokens * args.heads;
  const float* const pairs = args.workspace + (long long)args.splits * all_rows * D;
  const int group = threadIdx.x / kLanes, lane = threadIdx.x % kLanes;
  float top = -INFINITY, sum = 0.f;
  f4_t out = {};
  for (int split = group; split < args.splits; split += kGroups) {
    const long long place = split * all_rows + row;
    const f2_t pair = *(const f2_t*)(pairs + 2 * place);
    if (pair.y == 0.f) continue;
    const f4_t own = *(const f4_t*)(args.workspace + place * D + 4 * lane);
    const float next = fmaxf(top, pair.x), keep = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - next);
    const float share = __builtin_amdgcn_exp2f(pair.x - next);
    out = out * keep + own * share;
    sum = sum * keep + pair.y * share;
    top = next;
  }
  parts[group][lane] = out;
  if (lane == 0) tops[group] = top, totals[group] = sum;
  __syncthreads();
  if (group > 0) return;
  float most = -INFINITY;
  for (int i = 0; i < kGroups; ++i) most = fmaxf(most, tops[i]);
  f4_t all = {};
  float total = 0.f;
  for (int i = 0; i < kGroups; ++i) {
    if (tops[i] == -INFINITY && totals[i] == 0.f) continue;
    const float share = __builtin_amdgcn_exp2f(tops[i] - most);
    all += parts[i][lane] * share;
    total += totals[i] * share;
  }
  if (total != 0.f) all /= total;
  const float values[4] = {all.x, all.y, all.z, all.w};
  const long long at = row / args.heads * args.out.token_stride + row % args.heads * args.out.head_stride + 4 * lane;
  if (args.dtype == ONEBIT_DTYPE_F16) store_values<ONEBIT_DTYPE_F16, 4>(args.out.data, at, values);
  else store_values<ONEBIT_DTYPE_BF16, 4>(args.out.data, at, values);
}

template <int D, int CODE>
hipError_t launch_few_rows(const AttentionArgs& args, hipStream_t stream) {
  constexpr int kWaves = 8;
  const onebit_sequences& q = args.sequences;
  const int row_tiles = (int)(((long long)q.max_new * args.group + kRows - 1) / kRows);
  const dim3 grid(row_tiles * args.splits, args.cache.kv_heads, q.count);
  return launch_kernel(few_rows_kernel<D, CODE, kWaves>, grid, dim3(kWaves * 64), 0, stream, args, row_tiles);
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
  return launch_kernel(join_kernel<D, 256>, rows, dim3(256), 0, stream, args);
}

}  // namespace

// Rows of q to a workgroup, and how its keys are split over workgroups where a call has fewer of them than the device holds at once.
void plan_attention(AttentionArgs& args, int compute_units) {
  const onebit_sequences& q = args.sequences;
  const long long rows = (long long)q.max_new * args.group, room = (long long)q.width * args.cache.block;
  const long long most = std::max(1ll, q.max_length > 0 ? std::min(room, (long long)q.max_length) : room);
  args.rows = rows <= 32 ? kRows : 128;
  const long long units = (rows + args.rows - 1) / args.rows * args.cache.kv_heads * q.count;
  const long long splits = std::max(1ll, (args.rows == kRows ? 4ll : 2ll) * compute_units / units);
  const long long keys = std::max(args.rows == kRows ? 256ll : 512ll, ((most + splits - 1) / splits + 255) / 256 * 256);
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
