// What the kernels around the one-bit projections share (internal to libonebitmul): element types, 8-bit codes, reductions.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "onebit_decoder.h"

namespace onebit {

typedef _Float16 h2_t __attribute__((ext_vector_type(2)));
typedef _Float16 h4_t __attribute__((ext_vector_type(4)));
typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef float f2_t __attribute__((ext_vector_type(2)));
typedef float f4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u4_t __attribute__((ext_vector_type(4)));

// Values as they lie in memory; `type` is a dtype code of the C ABI.
template <int TYPE>
struct Stored;
template <>
struct Stored<ONEBIT_DTYPE_F32> { typedef float type; };
template <>
struct Stored<ONEBIT_DTYPE_F16> { typedef _Float16 type; };
template <>
struct Stored<ONEBIT_DTYPE_BF16> { typedef __bf16 type; };

// N consecutive values (16-byte aligned where N is 8) as fp32, and back, rounded to nearest even; FAR: past the caches
template <int TYPE, int N>
__device__ inline void load_values(const void* base, long long at, float (&x)[N]) {
  typedef typename Stored<TYPE>::type T;
  typedef T vector __attribute__((ext_vector_type(N)));
  if constexpr (N == 1) {
    x[0] = (float)((const T*)base)[at];
  } else {
    const vector v = *(const vector*)((const T*)base + at);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = (float)v[i];
  }
}
template <int TYPE, int N, bool FAR = false>
__device__ inline void store_values(void* base, long long at, const float (&x)[N]) {
  typedef typename Stored<TYPE>::type T;
  typedef T vector __attribute__((ext_vector_type(N)));
  if constexpr (N == 1) {
    ((T*)base)[at] = (T)x[0];
  } else {
    vector v;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (T)x[i];
    if constexpr (FAR) __builtin_nontemporal_store(v, (vector*)((T*)base + at));
    else *(vector*)((T*)base + at) = v;
  }
}

constexpr float kMostE4M3 = 448.f, kMostInt8 = 127.f;

// Magnitudes as integers: their order is that of the floats, and NaN is the largest, so that a maximum does not lose it.
__device__ inline uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// Over the 64 lanes, the same in each: neighbours, pairs, halves of a row of 16 and rows by cross-lane moves, then rows and halves by swaps.
template <class Value, class Combine>
__device__ inline Value over_wave(Value x, Combine combine) {
  auto moved = [&](auto pattern) {
    return __builtin_bit_cast(Value, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), decltype(pattern)::value, 0xf, 0xf, true));
  };
  x = combine(x, moved(std::integral_constant<int, 0xb1>()));   // lane ^ 1
  x = combine(x, moved(std::integral_constant<int, 0x4e>()));   // lane ^ 2
  x = combine(x, moved(std::integral_constant<int, 0x141>()));  // the other four of eight
  x = combine(x, moved(std::integral_constant<int, 0x140>()));  // the other eight of sixteen
  auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
  x = combine(__builtin_bit_cast(Value, (uint32_t)r[0]), __builtin_bit_cast(Value, (uint32_t)r[1]));
  r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
  return combine(__builtin_bit_cast(Value, (uint32_t)r[0]), __builtin_bit_cast(Value, (uint32_t)r[1]));
}
__device__ inline uint32_t wave_max(uint32_t x) {
  return over_wave(x, [](uint32_t a, uint32_t b) { return max(a, b); });
}
__device__ inline float wave_max(float x) {
  return over_wave(x, [](float a, float b) { return fmaxf(a, b); });
}
__device__ inline float wave_sum(float x) {
  return over_wave(x, [](float a, float b) { return a + b; });
}

// A sequence of a call, its numbers brought into range.
struct Sequence {
  int start, fresh, length;  // first row, new tokens, tokens with them (all non-negative; fresh <= length is not implied)
};
__device__ inline Sequence read_sequence(const onebit_sequences& q, int s, int block) {
  Sequence r;
  const long long room = (long long)q.width * block;
  r.length = (int)min((long long)max(q.lengths[s], 0), room);
  if (q.starts) {
    r.start = min(max(q.starts[s], 0), q.tokens);
    r.fresh = max(min(q.starts[s + 1], q.tokens) - r.start, 0);
  } else {
    r.fresh = q.tokens / q.count;
    r.start = s * r.fresh;
  }
  return r;
}

}  // namespace onebit
