// What the kernels around the one-bit projections share (internal to libonebitmul): element types, 8-bit codes, reductions.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

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

inline int bytes_of(int type) { return type == ONEBIT_DTYPE_F32 ? 4 : 2; }

// N consecutive values (16-byte aligned where N is 8) as fp32, and back, rounded to nearest even
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
template <int TYPE, int N>
__device__ inline void store_values(void* base, long long at, const float (&x)[N]) {
  typedef typename Stored<TYPE>::type T;
  typedef T vector __attribute__((ext_vector_type(N)));
  if constexpr (N == 1) {
    ((T*)base)[at] = (T)x[0];
  } else {
    vector v;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (T)x[i];
    *(vector*)((T*)base + at) = v;
  }
}

constexpr float kMostE4M3 = 448.f, kMostInt8 = 127.f;

// Magnitudes as integers: their order is that of the floats, and NaN is the largest, so that a maximum does not lose it.
__device__ inline uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

__device__ inline uint32_t wave_max(uint32_t x) {
#pragma unroll
  for (int step = 1; step < 64; step *= 2) x = max(x, (uint32_t)__shfl_xor((int)x, step));
  return x;
}
__device__ inline float wave_sum(float x) {
#pragma unroll
  for (int step = 1; step < 64; step *= 2) x += __shfl_xor(x, step);
  return x;
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
