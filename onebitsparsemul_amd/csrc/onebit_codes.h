// Rows of e4m3 codes with a scale for each 128 values (onebit_head.h): the way from values in registers to memory (internal to libonebitmul).
#pragma once
#include "onebit_decoder_device.h"
#include "onebit_head.h"

namespace onebit {

__host__ __device__ inline int padded_columns(int columns) { return (columns + ONEBIT_CODE_GROUP - 1) / ONEBIT_CODE_GROUP * ONEBIT_CODE_GROUP; }

// Eight values at column `at` of a row, the group's others in the 15 lanes beside; all lanes of the wavefront take part, those without `inside` write nothing.
__device__ inline void store_codes(const onebit_codes& out, long long row, int at, bool inside, const float (&x)[8]) {
  uint32_t largest = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) largest = max(largest, magnitude(x[i]));
  const float scale = __uint_as_float(row_max(largest)) / kMostE4M3;  // (as integers: NaN stays the largest)
  if (!inside) return;
  const bool finite = scale > 0.f && magnitude(scale) < 0x7f800000u;
  *(u2_t*)((uint8_t*)out.codes + row * out.row_stride + at) =
      u2_t{encode4<ONEBIT_CODE_E4M3>(x, scale, finite), encode4<ONEBIT_CODE_E4M3>(x + 4, scale, finite)};
  if (at % ONEBIT_CODE_GROUP == 0) out.scales[row * out.scale_stride + at / ONEBIT_CODE_GROUP] = scale;
}

}  // namespace onebit
