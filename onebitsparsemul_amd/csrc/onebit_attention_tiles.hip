// Attention over the 8-bit cache (onebit_decoder.h) for many rows of q to a key/value head: prompts.
//
// A workgroup takes 256 rows (128 where heads are of 64; tokens x heads of the key/value head), 32 to a wavefront, and walks over the keys in tiles
// of 64. Each tile's codes are read once, turned into fp16 by the wavefronts together, and lie in LDS twice (one tile in use, one being written): keys
// by rows of dims, values by rows of keys, so that both matrix products (32x32x16, fp16) read their left operand with one 16-byte load a lane.
//
// What bounds it: the matrix unit and the vector unit one after the other. Of a tile's 32 products a wavefront (1024 clocks) and some 200 vector
// instructions (32 exponentials among them; 16 conversions and 8 byte permutations bring in its share of the next tile) the two wavefronts of a SIMD
// overlap little: the matrix unit is busy in 37 % of the clocks, LDS in 27 %, and power takes 6 % (zeros: 139 us for 149 on one card). 4096 tokens, 32 heads of
// 128 on 8, e4m3, bf16: 152 us (149 to 156 on different cards) = 900 TFLOP/s of the causal half, where a large bf16 matrix product of the library reaches 1330;
// 500 tokens behind 7500, 32 heads on 32, int8, pages of 32: 98 us with 9 of the join = 650.
// Why this tile: 128 rows (four wavefronts) read and convert each tile twice as often, 167 us for 149; 64 rows to a wavefront do not fit its registers.
// Measured and not kept: the wavefronts of a SIMD in turn, one multiplying while the other weighs, with a barrier at each change (148 us for 149, the second
// call 100 for 97: each is then bound by its own instructions' latencies); the loads two tiles ahead, 167; wave priorities, nothing.
// p goes into the second product as one fp16: a second for the bits below, as where rows are few, would be half as many matrix instructions again, and the sum
// of p is taken from the same rounded values. That costs up to 2^-11 of sum p |v| (the second call above stands 2.9e-4 from 64 bits, with p in fp32 2.1e-4: the
// result's own rounding).
#include "onebit_attention.h"

#include <type_traits>

namespace onebit {
namespace {

typedef float f16x_t __attribute__((ext_vector_type(16)));
constexpr int kTile = 64;  // keys
constexpr int kSchedProduct = 0x8, kSchedRead = 0x100;  // kinds of instructions for the scheduler

// Where 16-byte pieces lie: moved within their rows by an exclusive or (other pieces of a row are one such operation away), so that the sixteen lanes that
// LDS serves at a time fall on different banks: keys' rows (tokens) in reads of one piece of sixteen rows, and in writes of whole rows.
template <int PIECES>
__device__ inline int key_place(int row, int piece) {
  return row * PIECES + (piece ^ (PIECES == 16 ? row & 15 : row >> 1 & 7));
}
// The values' rows (dims, of eight pieces) are read as the keys', but written at every fourth row by neighbouring lanes: bits 0 and 2 of the row are exchanged.
// 32 rows further on the piece moves by 2.
__device__ inline int value_place(int row, int piece) {
  const int r = (row & ~5) | (row >> 2 & 1) | (row & 1) << 2;
  return r * 8 + (piece ^ (r >> 1 & 7) ^ (r >> 4 & 3));
}
// The same value, for which the compiler keeps no register with what a loop makes of it
__device__ inline int made_here(int x) {
  asm("" : "+v"(x));
  return x;
}

template <int D, int CODE, bool ONE_PAGE>
__global__ __launch_bounds__(many_rows(D) * 2, 2) void many_rows_kernel(AttentionArgs args, int row_tiles) {
  constexpr int kRows = many_rows(D), kWaves = kRows / 32;
  constexpr int kOwn = kTile / kWaves;  // keys a wavefront brings in
  constexpr int kKeyBytes = kOwn * D / 64, kValueBytes = D * kOwn / 256;
  typedef uint32_t key_words __attribute__((ext_vector_type(kKeyBytes / 4)));
  static_assert(kValueBytes == 4, "a lane takes four dims of four keys");
  __shared__ __align__(16) h8_t keys[2][kTile * D / 8];
  __shared__ __align__(16) h8_t values[2][kTile * D / 8];
  const onebit_cache& cache = args.cache;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64, r = lane % 32, h = lane / 32;
  const int head = blockIdx.x % cache.kv_heads, split = blockIdx.x / cache.kv_heads % args.splits, s = blockIdx.z;
  const Sequence seq = read_sequence(args.sequences, s, cache.block);
  const int rows = seq.fresh * args.group, block_bits = __builtin_ctz(cache.block);
  const int* const table = args.sequences.page_table + (long long)s * args.sequences.width;
  const long long all_rows = (long long)args.sequences.tokens * args.heads;
  float* const pairs = args.workspace + (long long)args.splits * all_rows * D;

  // the last rows see the most keys: first
  for (int tile = row_tiles - 1 - (int)blockIdx.y + (rows > row_tiles * kRows ? ((rows + kRows - 1) / kRows - 1) / row_tiles * row_tiles : 0); tile >= 0; tile -= row_tiles) {
    if (tile * kRows >= rows) continue;
    const Rows own_first = first_row(tile * kRows, args.group);
    const int last_token = behind(own_first, min(kRows, rows - tile * kRows) - 1, args).token;
    const int total = max(seq.length - seq.fresh + last_token + 1, 0);
    const int low = split * args.keys_per_split, high = split == args.splits - 1 ? total : min(total, low + args.keys_per_split);
    const int tiles = max(high - low + kTile - 1, 0) / kTile;
    const int wave_row = tile * kRows + wave * 32;
    // keys that all rows of the wavefront see, and that one of them sees
    const int before = seq.length - seq.fresh + 1, here = min(max(rows - wave_row, 0), 32);
    const int all_see = here == 32 ? max(before + behind(own_first, wave * 32, args).token, 0) : 0;
    const int one_sees = here > 0 ? max(before + behind(own_first, wave * 32 + here - 1, args).token, 0) : 0;
    // the row of this lane's column
    const int row = wave_row + r;
    const Rows own_row = behind(own_first, wave * 32 + r, args);
    const int token = seq.start + own_row.token;
    const int query_head = head * args.group + own_row.head;
    const int seen = row < rows ? max(before + own_row.token, 0) : 0;

    h8_t q[D / 16];
    float row_factor = args.scale * kLog2E;
    {
      u4_t raw[D / 16] = {};
      if (row < rows) {
        const uint16_t* const at = (const uint16_t*)args.q.data + token * args.q.token_stride + query_head * args.q.head_stride + 8 * h;
#pragma unroll
        for (int c = 0; c < D / 16; ++c) raw[c] = *(const u4_t*)(at + 16 * c);
      }
      if (args.scale < 0.f) {  // the sign into q: multiply() takes maxima of products and multiplies them by row_factor afterwards
        row_factor = -row_factor;
#pragma unroll
        for (int c = 0; c < D / 16; ++c) raw[c] ^= 0x80008000u;
      }
      float factor = 1.f;
      if (args.dtype == ONEBIT_DTYPE_BF16) {  // rows as q 2^(8 - e), e the exponent of their largest value
        uint32_t most = 0;
#pragma unroll
        for (int c = 0; c < D / 16; ++c) most = max(most, magnitude_bf16(raw[c]));
        most = max(most, (uint32_t)__shfl_xor((int)most, 32));
        const int e = max(exponent_of(most), -100);
        factor = power_of_two(8 - e);
        row_factor *= power_of_two(e - 8);
      }
#pragma unroll
      for (int c = 0; c < D / 16; ++c) q[c] = q_to_f16(raw[c], args.dtype, factor);
    }

    f16x_t sums[D / 32] = {};
    float most = -INFINITY, total_p = 0.f;
    Exponent v_exponent;  // p takes v_scale 2^(8 - exponent of the tile's largest)

    Window window = {0, -1, 0.f, 0.f};
    // of the window's v_scale: exponent, logarithm and reciprocal
    int v_power = 0;
    float v_log = 0.f, v_inverse = 0.f;
    uint64_t bad = 0;  // entries whose scale is not finite
    auto refill = [&](int entry) {
      window = load_pages(entry, args.sequences.width, table, cache);
      drop_pages(window, (high - 1) >> block_bits);
      load_scales(window, cache, head);
      bad = __ballot(magnitude(window.v_scale) >= 0x7f800000u);
      const float scale = usable_scale(window.v_scale);
      v_power = exponent_of(magnitude(scale));
      v_log = __builtin_amdgcn_logf(scale);
      v_inverse = 1.f / scale;
    };

    // the wavefront's share of a tile: kOwn keys, in one page
    key_words raw_k;
    uint32_t raw_v[4];
    auto load = [&](int key) {
      const int own = key + wave * kOwn, entry = min((own >> block_bits) - window.first, 63);
      const int page = __builtin_amdgcn_readlane(window.page, entry);
      const int valid = page < 0 ? 0 : min(max(high - own, 0), kOwn);
      const long long at = valid == 0 ? 0 : (((long long)page * cache.kv_heads + head) * cache.block + (own & (cache.block - 1))) * D;
      raw_k = *(const key_words*)((const uint8_t*)cache.k + at + lane * kKeyBytes);
      constexpr int kLanes = D / kValueBytes;  // of a token
      const int first = lane / kLanes * 4;
      const uint8_t* const v = (const uint8_t*)cache.v + at + first * D + lane % kLanes * kValueBytes;
#pragma unroll
      for (int i = 0; i < 4; ++i) raw_v[i] = *(const uint32_t*)(v + i * D);
      if (valid < kOwn) {  // codes of keys that are not there may be NaN, which a p of 0 would not hide
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (first + i >= valid) raw_v[i] = 0;
      }
    };
    auto put = [&](auto buffer) {
      constexpr int to = decltype(buffer)::value;
      constexpr int kKeyLanes = D / kKeyBytes, kLanes = D / kValueBytes;
      const int key_at = made_here(key_place<D / 8>(wave * kOwn + lane / kKeyLanes, lane % kKeyLanes * (kKeyBytes / 8)));
#pragma unroll
      for (int i = 0; i < kKeyBytes / 8; ++i) keys[to][key_at ^ i] = codes_to_f16<CODE>(raw_k[2 * i], raw_k[2 * i + 1]);
      // four keys are half a piece of each dim's row; pieces are in the order in which the products want them
      const int group = (wave * kOwn + lane / kLanes * 4) / 4, half = group >> 1 & 1;
      const int value_at = made_here(value_place(lane % kLanes * kValueBytes, (group >> 2) * 2 + (group & 1)));
      uint32_t by_dim[4];
      transpose_bytes(raw_v[0], raw_v[1], raw_v[2], raw_v[3], by_dim);
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // the row's bits 0 and 1 in value_place()
        h2_t a, b;
        codes_to_f16<CODE>(by_dim[i], a, b);
        ((h4_t*)&values[to][(value_at ^ (i >> 1 | (i & 1) << 1)) + ((i & 2) + (i & 1) * 4) * 8])[half] = h4_t{a.x, a.y, b.x, b.y};
      }
    };

    auto multiply = [&](auto buffer, int key) {
      constexpr int kFrom = decltype(buffer)::value;
      f16x_t scores[2] = {};
      const int own_key = made_here(key_place<D / 8>(r, h)), own_value = made_here(value_place(r, h));
      constexpr int kAhead = 6;  // LDS reads in front of the first product: their latency is that of several
#pragma unroll
      for (int c = 0; c < D / 16; ++c)
#pragma unroll
        for (int half = 0; half < 2; ++half)
          scores[half] = __builtin_amdgcn_mfma_f32_32x32x16_f16(keys[kFrom][32 * (D / 8) * half + (own_key ^ 2 * c)], q[c], scores[half], 0, 0, 0);
      __builtin_amdgcn_sched_group_barrier(kSchedRead, kAhead, 0);
#pragma unroll
      for (int i = 0; i < D / 8 - kAhead; ++i) {
        __builtin_amdgcn_sched_group_barrier(kSchedProduct, 1, 0);
        __builtin_amdgcn_sched_group_barrier(kSchedRead, 1, 0);
      }
      __builtin_amdgcn_sched_group_barrier(kSchedProduct, kAhead, 0);
      // a lane's scores: key 32 i + 8 a + 4 h + e of the tile is scores[i][4 a + e]; 16 keys are eight of them
      int entry[4];
      float k_scale[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        entry[i] = ONE_PAGE && i > 0 ? entry[0] : min(((key + 16 * i) >> block_bits) - window.first, 63);
        k_scale[i] = ONE_PAGE && i > 0 ? k_scale[0] : lane_value(window.k_scale, entry[i]);
      }
      float factor[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) factor[i] = ONE_PAGE && i > 0 ? factor[0] : row_factor * k_scale[i];
      bool masked = key + kTile > all_see, any_bad = false;
      int power = -1000, powers[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (ONE_PAGE && i > 0) {
          powers[i] = powers[0];
          continue;
        }
        masked |= __builtin_amdgcn_readlane(window.page, entry[i]) < 0;
        any_bad |= bad >> entry[i] & 1;
        powers[i] = __builtin_amdgcn_readlane(v_power, entry[i]);
        power = max(power, powers[i]);
      }
      if (masked) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // the row sees this many of the tile's keys from here on; none of a page that is not there
          const int left = __builtin_amdgcn_readlane(window.page, entry[i]) < 0 ? 0 : seen - (key + i / 2 * 32 + i % 2 * 16 + 4 * h);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float score = scores[i / 2][i % 2 * 8 + e] * factor[i];
            scores[i / 2][i % 2 * 8 + e] = e / 4 * 8 + e % 4 < left ? score : -INFINITY;
          }
          factor[i] = 1.f;
        }
      }
      float top = -INFINITY;
      if (ONE_PAGE) {
#pragma unroll
        for (int i = 0; i < 32; ++i) top = fmaxf(top, scores[i / 16][i % 16]);
        top *= factor[0];
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float own = scores[i / 2][i % 2 * 8];
#pragma unroll
          for (int e = 1; e < 8; ++e) own = fmaxf(own, scores[i / 2][i % 2 * 8 + e]);
          top = fmaxf(top, own * factor[i]);
        }
      }
      const auto swapped = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
      top = fmaxf(__uint_as_float(swapped[0]), __uint_as_float(swapped[1]));
      // p up to 2^6 is fine: where the maximum grows by less, the sums stay as they are
      const float v_keep = v_exponent.follow(power);
      if (__any(top > most + 6.f) || v_keep != 1.f) {
        const float next = fmaxf(top, most), keep = most == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(most - next);
        most = next;
        total_p *= keep;
#pragma unroll
        for (int j = 0; j < D / 32; ++j) sums[j] *= keep * v_keep;
      }
      const float base = most == -INFINITY ? 0.f : most;
      // rows 32 j + r of the values, pieces 2 i + h
      auto value = [&](int i, int j) { return values[kFrom][32 * 8 * j + (own_value ^ 2 * i ^ 2 * (j & 1))]; };
      const h2_t ones = {(_Float16)1.f, (_Float16)1.f};
      float sum = 0.f;
      // p of 16 keys, with v_scale as a part of the exponent, beside 2^(exponent - 8)
      auto weigh = [&](int i, float log, int exponent) {
        const float shift = log + (float)(8 - exponent) - base;
        h8_t p;
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const float a = __builtin_amdgcn_exp2f(__builtin_fmaf(scores[i / 2][i % 2 * 8 + e], factor[i], shift));
          const float b = __builtin_amdgcn_exp2f(__builtin_fmaf(scores[i / 2][i % 2 * 8 + e + 1], factor[i], shift));
          const h2_t pair = {(_Float16)a, (_Float16)b};
          sum = __builtin_amdgcn_fdot2(pair, ones, sum, false);
          p[e] = pair.x, p[e + 1] = pair.y;
        }
        return p;
      };
      int least = powers[0];
#pragma unroll
      for (int i = 1; i < (ONE_PAGE ? 1 : 4); ++i) least = min(least, powers[i]);
      float v_total[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v_total[i] = lane_value(v_inverse, entry[i]);
      if (least < v_exponent.now - 6) {
        // Pages of one tile whose scales are far apart (p of the smaller ones would lose its bits beside the largest, which not all rows need see), or a scale
        // too small for the sums to follow. By themselves, in their own power, and then no more; a scale that is as good as 0 adds nothing.
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (powers[i] >= v_exponent.now - 6) continue;
          const float down = powers[i] > -100 ? power_or_zero(powers[i] - v_exponent.now) : 0.f;
          const h8_t p = weigh(i, lane_value(v_log, entry[i]), powers[i]);
          total_p += sum * (lane_value(v_inverse, entry[i]) * power_of_two(powers[i] - 8));
          sum = 0.f;
#pragma unroll
          for (int j = 0; j < D / 32; ++j) {
            sums[j] += __builtin_amdgcn_mfma_f32_32x32x16_f16(value(i, j), p, f16x_t{}, 0, 0, 0) * down;
            // one after the other; without it the build of e4m3 codes, heads of 64 and pages from 64 on takes 169 registers, and two workgroups to a compute
            // unit for three: 64 prompts of 256 44.5 us for 37.3 (smaller pages are better off without: int8 168 registers for 169)
            if (ONE_PAGE) __builtin_amdgcn_sched_barrier(0);
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) scores[i / 2][i % 2 * 8 + e] = -INFINITY;
          factor[i] = 1.f;
          v_total[i] = 0.f;  // (beside the large exponent it need not be finite)
        }
      }
      h8_t p[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p[i] = weigh(i, lane_value(v_log, entry[i]), v_exponent.now);
        if (!ONE_PAGE || i == 3) {
          total_p += sum * (v_total[i] * power_of_two(v_exponent.now - 8));
          sum = 0.f;
        }
      }
      if (any_bad) {
#pragma unroll
        for (int i = 0; i < 4; ++i)  // a row sees the scale of a page if it sees one of its keys
          if ((bad >> entry[i] & 1) && key + 16 * i < seen) total_p = __builtin_nanf("");
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < D / 32; ++j) sums[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(value(i, j), p[i], sums[j], 0, 0, 0);
      __builtin_amdgcn_sched_group_barrier(kSchedRead, kAhead, 0);
#pragma unroll
      for (int i = 0; i < D / 8 - kAhead; ++i) {
        __builtin_amdgcn_sched_group_barrier(kSchedProduct, 1, 0);
        __builtin_amdgcn_sched_group_barrier(kSchedRead, 1, 0);
      }
      __builtin_amdgcn_sched_group_barrier(kSchedProduct, kAhead, 0);
    };

    auto step = [&](auto buffer, int t) {
      constexpr int kFrom = decltype(buffer)::value;
      const int key = low + t * kTile;
      __syncthreads();
      const bool more = t + 1 < tiles;
      const bool turn = more && (key + 2 * kTile - 1) >> block_bits >= window.first + 64;
      if (more && !turn) load(key + kTile);
      if (key < one_sees) multiply(buffer, key);
      if (turn) {
        refill((key + kTile) >> block_bits);
        load(key + kTile);
      }
      if (more) put(std::integral_constant<int, 1 - kFrom>());
    };
    if (tiles > 0) {
      refill(low >> block_bits);
      load(low);
      put(std::integral_constant<int, 0>());
      for (int t = 0; t < tiles; t += 2) {
        step(std::integral_constant<int, 0>(), t);
        if (t + 1 < tiles) step(std::integral_constant<int, 1>(), t + 1);
      }
    }

    const auto swapped = __builtin_amdgcn_permlane32_swap(__float_as_uint(total_p), __float_as_uint(total_p), false, false);
    const float sum = __uint_as_float(swapped[0]) + __uint_as_float(swapped[1]), v_factor = v_exponent.largest > -100 ? power_of_two(v_exponent.now - 8) : 0.f;
    if (row < rows) {
      if (args.splits > 1) {
        const long long at = split * all_rows + (long long)token * args.heads + query_head;
        if (sum != 0.f) {
#pragma unroll
          for (int j = 0; j < D / 32; ++j)
#pragma unroll
            for (int a = 0; a < 4; ++a)
              *(f4_t*)(args.workspace + at * D + 32 * j + 8 * a + 4 * h) =
                  f4_t{sums[j][4 * a], sums[j][4 * a + 1], sums[j][4 * a + 2], sums[j][4 * a + 3]} * v_factor;
        }
        if (h == 0) *(f2_t*)(pairs + 2 * at) = f2_t{most, sum};
      } else {
        const float factor = sum != 0.f ? v_factor / sum : 0.f;  // (a row that sees nothing: 0)
        const long long at = token * args.out.token_stride + query_head * args.out.head_stride;
#pragma unroll
        for (int j = 0; j < D / 32; ++j)
#pragma unroll
          for (int a = 0; a < 4; ++a) {
            const float out[4] = {sums[j][4 * a] * factor, sums[j][4 * a + 1] * factor, sums[j][4 * a + 2] * factor, sums[j][4 * a + 3] * factor};
            if (args.dtype == ONEBIT_DTYPE_F16) store_values<ONEBIT_DTYPE_F16, 4>(args.out.data, at + 32 * j + 8 * a + 4 * h, out);
            else store_values<ONEBIT_DTYPE_BF16, 4>(args.out.data, at + 32 * j + 8 * a + 4 * h, out);
          }
      }
    }
    __syncthreads();
  }
}

template <int D, int CODE>
hipError_t launch_as(const AttentionArgs& args, hipStream_t stream) {
  const onebit_sequences& q = args.sequences;
  constexpr int kRows = many_rows(D);
  const int tiles = (int)(((long long)q.max_new * args.group + kRows - 1) / kRows);
  const dim3 grid(args.cache.kv_heads * args.splits, tiles, q.count);
  const auto kernel = args.cache.block >= kTile ? many_rows_kernel<D, CODE, true> : many_rows_kernel<D, CODE, false>;
  return launch_kernel(kernel, grid, dim3(kRows * 2), 0, stream, args, tiles);
}

}  // namespace

hipError_t launch_many_rows(const AttentionArgs& args, hipStream_t stream) {
  const bool int8 = args.cache.code == ONEBIT_CODE_INT8;
  if (args.cache.head_dim == 64) return int8 ? launch_as<64, ONEBIT_CODE_INT8>(args, stream) : launch_as<64, ONEBIT_CODE_E4M3>(args, stream);
  return int8 ? launch_as<128, ONEBIT_CODE_INT8>(args, stream) : launch_as<128, ONEBIT_CODE_E4M3>(args, stream);
}

}  // namespace onebit
