// Rotary positions, and the write side of the 8-bit cache (onebit_decoder.h).
//
// A head's elements are handled in units of two vectors of P values: the two halves of P pairs (half layout), P interleaved
// pairs, or 2 P elements that are not turned. Both operators move each value once and are bound by memory, small calls by the launch and
// the chain of loads in front of a store (position, table row).
#include "onebit_decoder_device.h"
#include "onebit_decoder_launch.h"

#include <algorithm>

namespace onebit {
namespace {

// Where a unit of a head lies, and its pairs in the table
struct Unit {
  int low, high;  // elements: P from each on
  bool turned;
};
template <int P>
__device__ inline Unit unit_of(int u, int rotary_dim, int interleaved) {
  const int half = rotary_dim / 2;
  if (u * P < half && !interleaved) return {u * P, half + u * P, true};
  return {2 * P * u, 2 * P * u + P, u * P < half};
}

// The cosines and sines of a unit's pairs
template <int P>
struct Angles {
  float c[P], s[P];
};
template <int P>
__device__ inline Angles<P> load_angles(const float* table, long long position, int table_rows, int rotary_dim, int u) {
  Angles<P> r;
  if (position >= 0 && position < table_rows) {
    const long long at = position * rotary_dim + u * P;
    load_values<ONEBIT_DTYPE_F32, P>(table, at, r.c);
    load_values<ONEBIT_DTYPE_F32, P>(table, at + rotary_dim / 2, r.s);
  } else {
#pragma unroll
    for (int i = 0; i < P; ++i) r.c[i] = r.s[i] = __builtin_nanf("");
  }
  return r;
}

// Each product and each sum is rounded: contracted forms would differ from it in the last place, and the codes of a cache with them.
__device__ inline void turn_pair(float& a, float& b, float c, float s) {
#pragma clang fp contract(off)
  const float ac = a * c, bs = b * s, bc = b * c, as = a * s;
  a = ac - bs;
  b = bc + as;
}
template <int P>
__device__ inline void turn(float (&low)[P], float (&high)[P], const Angles<P>& angles, int interleaved) {
  if (!interleaved || P == 1) {
#pragma unroll
    for (int i = 0; i < P; ++i) turn_pair(low[i], high[i], angles.c[i], angles.s[i]);
  } else {
#pragma unroll
    for (int i = 0; i < P / 2; ++i) {
      turn_pair(low[2 * i], low[2 * i + 1], angles.c[i], angles.s[i]);
      turn_pair(high[2 * i], high[2 * i + 1], angles.c[P / 2 + i], angles.s[P / 2 + i]);
    }
  }
}

// One thread: one unit of one head, so that a wavefront has its loads of x out at once; the table's rows, which the heads of a token share, come
// from the caches. 4001 tokens x 32 heads of 128, bf16, half turned: 11.7 us as halves, 12.3 interleaved (66 MB, 5.4 to 5.7 TB/s); with two heads to
// a thread, whose angles are then read once, 13.2 and 14.4, with four 13.6 and 14.5. 16 tokens: 2.6 us, of which the launch is most.
template <int TYPE, int P>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs args, int units, int per_token) {
  const int tokens_per_block = max(1, (int)blockDim.x / per_token);
  const int at = blockIdx.y * blockDim.x + threadIdx.x;
  const int token = blockIdx.x * tokens_per_block + at / per_token, rest = at % per_token;
  if (token >= args.tokens || at >= tokens_per_block * per_token) return;
  const int u = rest % units, head = rest / units;
  const long long position = args.wide_positions ? ((const long long*)args.positions)[token] : ((const int*)args.positions)[token];
  const Unit unit = unit_of<P>(u, args.rotary_dim, args.interleaved);
  const long long from = token * args.x.token_stride + head * args.x.head_stride;
  const long long to = token * args.out.token_stride + head * args.out.head_stride;
  float low[P], high[P];
  load_values<TYPE, P>(args.x.data, from + unit.low, low);
  load_values<TYPE, P>(args.x.data, from + unit.high, high);
  if (unit.turned) turn<P>(low, high, load_angles<P>(args.table, position, args.table_rows, args.rotary_dim, u), args.interleaved);
  store_values<TYPE, P>(args.out.data, to + unit.low, low);
  store_values<TYPE, P>(args.out.data, to + unit.high, high);
}

template <int TYPE, int P>
hipError_t launch_rotary_as(const RotaryArgs& args, hipStream_t stream) {
  const int units = args.head_dim / (2 * P), per_token = units * args.heads;
  constexpr int threads = 256;
  const int tokens_per_block = std::max(1, threads / per_token);
  const dim3 grid((args.tokens + tokens_per_block - 1) / tokens_per_block, (tokens_per_block * per_token + threads - 1) / threads);
  return launch_kernel(rotary_kernel<TYPE, P>, grid, dim3(threads), 0, stream, args, units, per_token);
}

bool in_vectors(const onebit_heads& x) {
  return reinterpret_cast<uintptr_t>(x.data) % 16 == 0 && x.token_stride % 8 == 0 && x.head_stride % 8 == 0;
}

template <int TYPE>
hipError_t launch_rotary_type(const RotaryArgs& args, hipStream_t stream) {
  if (args.head_dim % 16 || args.rotary_dim % 16 || !in_vectors(args.x) || !in_vectors(args.out) || reinterpret_cast<uintptr_t>(args.table) % 16)
    return launch_rotary_as<TYPE, 1>(args, stream);
  return launch_rotary_as<TYPE, 8>(args, stream);
}

// ---- the write side of the cache

template <int CODE>
__device__ inline void decode4(uint32_t word, float* x) {
  if (CODE == ONEBIT_CODE_INT8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (float)(int8_t)(word >> (8 * i));
  } else {
    const f2_t low = __builtin_amdgcn_cvt_pk_f32_fp8((int)word, false), high = __builtin_amdgcn_cvt_pk_f32_fp8((int)word, true);
    x[0] = low.x, x[1] = low.y, x[2] = high.x, x[3] = high.y;
  }
}

constexpr int kUnit = 8;  // P of the cache's kernel

// Keys or values of one page and head, in registers from the first read to the codes: THREADS x PASSES units. The scale is that of all the page's new tokens,
// so a workgroup takes a page and head whole and no value is read twice. 2048 tokens, 32 heads of 128 on 8, fp16: 10.6 us for 47 MB = 4.4 TB/s (8192 tokens in
// four sequences 41 us, 4.6); int8 codes take 2 % more. Sixteen sequences' single tokens: 4.4 us, the launch and the chain lengths, page, scale, codes; 14 us where
// scales grow: the codes of a page's older tokens, up to 63 here, then go through the workgroup four to a thread, one round behind the other. With tokens of one
// distribution that is so for some 15 of the 256 pages and heads of such a call.
template <int TYPE, int CODE, int THREADS, int PASSES>
__device__ inline void append_page(const AppendArgs& args, const Sequence& seq, int s, int slot, int head, bool values) {
  __shared__ uint32_t most[THREADS / 64];
  const onebit_cache& cache = args.cache;
  const int first = seq.length - seq.fresh;  // position of the first new token; before the sequence where there are too many
  const int end = first + min(seq.fresh, args.sequences.max_new);  // what is beyond is left out
  const int j = max(first, 0) / cache.block + slot, begin = j * cache.block;
  if (begin >= end) return;
  const int page = args.sequences.page_table[(long long)s * args.sequences.width + j];
  if (page < 0 || page >= cache.pages) return;
  const int units = cache.head_dim / (2 * kUnit), tokens_per_pass = THREADS / units;
  const int low_position = max(max(first, 0), begin);
  const int count = min(end, begin + cache.block) - low_position;  // above 0, at most PASSES * tokens_per_pass
  const onebit_heads& x = values ? args.v : args.k;
  const long long place = (long long)page * cache.kv_heads + head;
  float* const scale_at = (values ? cache.v_scale : cache.k_scale) + place;
  const float held = low_position > begin ? __uint_as_float(magnitude(*scale_at)) : 0.f;
  const int u = threadIdx.x % units, own = threadIdx.x / units;
  const bool turns = !values && args.table;
  const Unit unit = unit_of<kUnit>(u, turns ? args.rotary_dim : 0, args.interleaved);

  float low[PASSES][kUnit], high[PASSES][kUnit];
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int token = p * tokens_per_pass + own;
    if (token < count) {
      const long long at = (long long)(seq.start + low_position - first + token) * x.token_stride + head * x.head_stride;
      load_values<TYPE, kUnit>(x.data, at + unit.low, low[p]);
      load_values<TYPE, kUnit>(x.data, at + unit.high, high[p]);
    }
  }
  uint32_t largest = 0;
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int token = p * tokens_per_pass + own;
    if (token < count) {
      if (unit.turned)
        turn<kUnit>(low[p], high[p], load_angles<kUnit>(args.table, low_position + token, args.table_rows, args.rotary_dim, u), args.interleaved);
#pragma unroll
      for (int i = 0; i < kUnit; ++i) largest = max(largest, max(magnitude(low[p][i]), magnitude(high[p][i])));
    }
  }
  largest = wave_max(largest);
  if (THREADS > 64) {
    if (threadIdx.x % 64 == 0) most[threadIdx.x / 64] = largest;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) largest = max(largest, most[w]);
  }
  // (as integers: NaN stays the largest)
  const float scale = __uint_as_float(max(magnitude(held), magnitude(__uint_as_float(largest) / most_code<CODE>())));
  const bool inside = scale > 0.f && magnitude(scale) < 0x7f800000u;
  uint8_t* const codes = (uint8_t*)(values ? cache.v : cache.k) + place * cache.block * cache.head_dim;
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int token = p * tokens_per_pass + own;
    if (token < count) {
      uint8_t* const at = codes + (low_position - begin + token) * cache.head_dim;
      *(u2_t*)(at + unit.low) = u2_t{encode4<CODE>(low[p], scale, inside), encode4<CODE>(low[p] + 4, scale, inside)};
      *(u2_t*)(at + unit.high) = u2_t{encode4<CODE>(high[p], scale, inside), encode4<CODE>(high[p] + 4, scale, inside)};
    }
  }
  if (low_position > begin && magnitude(scale) != magnitude(held)) {  // the older tokens of the page in the new scale
    for (int i = threadIdx.x; i < (low_position - begin) * cache.head_dim / 4; i += THREADS) {
      float x4[4];
      decode4<CODE>(((uint32_t*)codes)[i], x4);
#pragma unroll
      for (int e = 0; e < 4; ++e) x4[e] *= held;
      ((uint32_t*)codes)[i] = encode4<CODE>(x4, scale, inside);
    }
  }
  if (threadIdx.x == 0) *scale_at = scale;
}

// grid.y: sequences; grid.x: pages that new tokens may touch x heads x (keys, values), then units of the queries.
template <int TYPE, int CODE, int THREADS, int PASSES>
__global__ __launch_bounds__(THREADS) void append_kernel(AppendArgs args, int page_tasks) {
  const int s = blockIdx.y, task = blockIdx.x;
  const Sequence seq = read_sequence(args.sequences, s, args.cache.block);
  if (seq.fresh == 0) return;
  if (task < page_tasks) {
    const int pair = task % (2 * args.cache.kv_heads);
    append_page<TYPE, CODE, THREADS, PASSES>(args, seq, s, task / (2 * args.cache.kv_heads), pair >> 1, pair & 1);
    return;
  }
  const int units = args.cache.head_dim / (2 * kUnit), per_token = units * args.heads;
  const long long step = (long long)(gridDim.x - page_tasks) * THREADS;
  for (long long i = (long long)(task - page_tasks) * THREADS + threadIdx.x; i < (long long)seq.fresh * per_token; i += step) {
    const int token = (int)(i / per_token), rest = (int)(i % per_token), u = rest % units, head = rest / units;
    const Unit unit = unit_of<kUnit>(u, args.rotary_dim, args.interleaved);
    const long long from = (long long)(seq.start + token) * args.q.token_stride + head * args.q.head_stride;
    const long long to = (long long)(seq.start + token) * args.q_out.token_stride + head * args.q_out.head_stride;
    float low[kUnit], high[kUnit];
    load_values<TYPE, kUnit>(args.q.data, from + unit.low, low);
    load_values<TYPE, kUnit>(args.q.data, from + unit.high, high);
    if (unit.turned)
      turn<kUnit>(low, high, load_angles<kUnit>(args.table, seq.length - seq.fresh + token, args.table_rows, args.rotary_dim, u), args.interleaved);
    store_values<TYPE, kUnit>(args.q_out.data, to + unit.low, low);
    store_values<TYPE, kUnit>(args.q_out.data, to + unit.high, high);
  }
}

template <int TYPE, int CODE>
hipError_t launch_append_as(AppendArgs args, hipStream_t stream) {
  const int units = args.cache.head_dim / (2 * kUnit);
  const onebit_sequences& q = args.sequences;
  const int most = q.max_new, in_page = std::min(most, args.cache.block) * units;
  args.slots = (most + args.cache.block - 2) / args.cache.block + 1;
  const long long page_tasks = 2ll * args.slots * args.cache.kv_heads;
  auto launch = [&](auto kernel, int threads) {
    const long long turned = (long long)most * args.heads * units, tasks = page_tasks + (turned + threads - 1) / threads;
    if (tasks * threads >= 1ll << 32) return hipErrorInvalidConfiguration;
    return launch_kernel(kernel, dim3((unsigned)tasks, q.count), dim3(threads), 0, stream, args, (int)page_tasks);
  };
  // A page and head in one pass of a workgroup; where there are more of them than compute units, a few passes of 256 threads, whose loads then
  // cover for each other: 512 tokens 8 heads of 128 in pages of 64, 5.6 us in one pass and 6.4 in two, 2048 tokens 12.5 and 11.8.
  const bool alone = page_tasks * q.count <= device_compute_units();
  if (in_page <= 64) return launch(append_kernel<TYPE, CODE, 64, 1>, 64);
  if (in_page <= 128) return launch(append_kernel<TYPE, CODE, 128, 1>, 128);
  if (in_page <= 256) return launch(append_kernel<TYPE, CODE, 256, 1>, 256);
  if (in_page <= 512) return alone ? launch(append_kernel<TYPE, CODE, 512, 1>, 512) : launch(append_kernel<TYPE, CODE, 256, 2>, 256);
  return alone ? launch(append_kernel<TYPE, CODE, 1024, 1>, 1024) : launch(append_kernel<TYPE, CODE, 256, 4>, 256);
}
template <int TYPE>
hipError_t launch_append_type(const AppendArgs& args, hipStream_t stream) {
  return args.cache.code == ONEBIT_CODE_INT8 ? launch_append_as<TYPE, ONEBIT_CODE_INT8>(args, stream) : launch_append_as<TYPE, ONEBIT_CODE_E4M3>(args, stream);
}

}  // namespace

hipError_t launch_rotary(const RotaryArgs& args, int dtype, hipStream_t stream) {
  if (dtype == ONEBIT_DTYPE_F32) return launch_rotary_type<ONEBIT_DTYPE_F32>(args, stream);
  return dtype == ONEBIT_DTYPE_F16 ? launch_rotary_type<ONEBIT_DTYPE_F16>(args, stream) : launch_rotary_type<ONEBIT_DTYPE_BF16>(args, stream);
}

hipError_t launch_append(AppendArgs args, int dtype, hipStream_t stream) {
  if (dtype == ONEBIT_DTYPE_F32) return launch_append_type<ONEBIT_DTYPE_F32>(args, stream);
  return dtype == ONEBIT_DTYPE_F16 ? launch_append_type<ONEBIT_DTYPE_F16>(args, stream) : launch_append_type<ONEBIT_DTYPE_BF16>(args, stream);
}

}  // namespace onebit
