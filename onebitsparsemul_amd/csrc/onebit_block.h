// What the products of 8-bit codes share (internal to libonebitmul): operands of the matrix instructions, results.
#pragma once
#include "onebit_codes.h"
#include "onebit_head_launch.h"

namespace onebit {

__device__ inline float value_at(const void* base, int type, long long at) {
  if (type == ONEBIT_DTYPE_F32) return ((const float*)base)[at];
  return type == ONEBIT_DTYPE_F16 ? (float)((const _Float16*)base)[at] : (float)((const __bf16*)base)[at];
}

typedef int i8_t __attribute__((ext_vector_type(8)));

// A lane's 32 codes of a group, and the products of 16 x 128 with 128 x 16 of them
template <bool NARROW>
struct Operand {
  h8_t v[4];
  Operand() = default;
  __device__ Operand(const u4_t& a, const u4_t& b)
      : v{codes_to_f16<ONEBIT_CODE_E4M3>(a.x, a.y), codes_to_f16<ONEBIT_CODE_E4M3>(a.z, a.w), codes_to_f16<ONEBIT_CODE_E4M3>(b.x, b.y), codes_to_f16<ONEBIT_CODE_E4M3>(b.z, b.w)} {}
  __device__ f4_t operator*(const Operand& other) const {
    f4_t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < 4; ++k) sum = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[k], other.v[k], sum, 0, 0, 0);
    return sum;
  }
};
template <>
struct Operand<true> {
  i8_t v;
  Operand() = default;
  __device__ Operand(const u4_t& a, const u4_t& b) : v{(int)a.x, (int)a.y, (int)a.z, (int)a.w, (int)b.x, (int)b.y, (int)b.z, (int)b.w} {}
  __device__ f4_t operator*(const Operand& other) const {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(v, other.v, f4_t{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
  }
};

// Eight values from any place on: rows of 4099 as fast as of 4096
template <int TYPE>
__device__ inline void store_eight(void* base, long long at, const float (&x)[8]) {
  typedef typename Stored<TYPE>::type T;
  typedef T vector __attribute__((ext_vector_type(8), aligned(sizeof(T))));
  vector v;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (T)x[i];
  *(vector*)((T*)base + at) = v;
}

// Where sums go: to the split's partial sums or, with the bias, to y
struct Result {
  void* base;
  long long stride;
  int type, rows;
  const void* bias;
  int bias_type;
  __device__ Result(const onebit_block_product& p, const BlockGrid& grid, int split)
      : base(grid.splits > 1 ? (void*)(grid.partial + (long long)split * p.tokens * p.rows) : p.y),
        stride(grid.splits > 1 ? p.rows : p.y_stride),
        type(grid.splits > 1 ? ONEBIT_DTYPE_F32 : p.y_dtype),
        rows(p.rows),
        bias(grid.splits > 1 ? nullptr : p.bias),
        bias_type(p.bias_dtype) {}
  __device__ float bias_of(int row) const { return bias && row < rows ? value_at(bias, bias_type, row) : 0.f; }
  __device__ void load_bias(int row, float (&v)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = bias_of(row + i);
  }
  // sums with the bias: one
  __device__ void put_one(int token, int row, float v) const {
    if (row >= rows) return;
    const float one[1] = {v};
    if (type == ONEBIT_DTYPE_F32) store_values<ONEBIT_DTYPE_F32, 1>(base, token * stride + row, one);
    else if (type == ONEBIT_DTYPE_F16) store_values<ONEBIT_DTYPE_F16, 1>(base, token * stride + row, one);
    else store_values<ONEBIT_DTYPE_BF16, 1>(base, token * stride + row, one);
  }
  // The sums of a matrix instruction's rows 4 q ... 4 q + 3, of lanes 16 q ... 16 q + 15, of two neighbouring parts of 16 rows, in 16 bits: the second and fourth 16 lanes' values of
  // the first part change places with the first and third 16 lanes' of the second, after which a lane has eight neighbouring rows, from q / 2 * 8 of part q % 2 on.
  __device__ u4_t eight_of(const f4_t& first, const f4_t& second) const {
    u2_t a, b;
    if (type == ONEBIT_DTYPE_F16) a = packed<_Float16>(first), b = packed<_Float16>(second);
    else a = packed<__bf16>(first), b = packed<__bf16>(second);
    const auto x = __builtin_amdgcn_permlane16_swap(a.x, b.x, false, false), y = __builtin_amdgcn_permlane16_swap(a.y, b.y, false, false);
    return u4_t{x[0], y[0], x[1], y[1]};
  }
  __device__ void put_eight(int token, int row, const u4_t& eight) const {
    typedef uint32_t vector __attribute__((ext_vector_type(4), aligned(2)));
    uint16_t* const to = (uint16_t*)base + token * stride + row;
    if (row + 8 <= rows) {
      *(vector*)to = eight;
    } else {
#pragma unroll
      for (int i = 0; i < 7; ++i)
        if (row + i < rows) to[i] = (uint16_t)(eight[i / 2] >> i % 2 * 16);
    }
  }
  template <class T>
  static __device__ u2_t packed(const f4_t& v) {
    typedef T four __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(u2_t, four{(T)v.x, (T)v.y, (T)v.z, (T)v.w});
  }
  __device__ void put_four(int token, int row, const f4_t& v) const {
    typedef float vector __attribute__((ext_vector_type(4), aligned(4)));
    float* const to = (float*)base + token * stride + row;
    if (row + 4 <= rows) {
      *(vector*)to = v;
    } else {
#pragma unroll
      for (int i = 0; i < 3; ++i)
        if (row + i < rows) to[i] = v[i];
    }
  }
  // and eight of a token from weight row `row` on, a multiple of eight
  __device__ void put(int token, int row, const float (&v)[8]) const {
    const long long at = token * stride + row;
    if (row + 8 <= rows) {
      if (type == ONEBIT_DTYPE_F32) store_eight<ONEBIT_DTYPE_F32>(base, at, v);
      else if (type == ONEBIT_DTYPE_F16) store_eight<ONEBIT_DTYPE_F16>(base, at, v);
      else store_eight<ONEBIT_DTYPE_BF16>(base, at, v);
      return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (row + i >= rows) break;
      const float one[1] = {v[i]};
      if (type == ONEBIT_DTYPE_F32) store_values<ONEBIT_DTYPE_F32, 1>(base, at + i, one);
      else if (type == ONEBIT_DTYPE_F16) store_values<ONEBIT_DTYPE_F16, 1>(base, at + i, one);
      else store_values<ONEBIT_DTYPE_BF16, 1>(base, at + i, one);
    }
  }
};

}  // namespace onebit
