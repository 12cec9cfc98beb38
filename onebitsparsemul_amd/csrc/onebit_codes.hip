// Rows of values as 8-bit codes with a scale for each 128 (onebit_head.h). Each value is moved once: bound by memory, small calls by the launch. 4001 x 5000 of 16 bits 13.5 us for
// 61 MB = 4.5 TB/s, 16 x 11008 2.3. Rows that do not begin at whole vectors go by single values: 4001 x 5001 28.0 us, 2.2 TB/s, 16 x 5001 2.7 (16 x 5000 2.3).
#include "onebit_codes.h"
#include "onebit_head_launch.h"

namespace onebit {
namespace {

// One thread: eight values; 16 of them a group. Groups of all rows one behind the other.
template <int TYPE, bool WHOLE>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const void* x, long long x_stride, int columns, int groups_per_row, int groups, onebit_codes out) {
  const int group = blockIdx.x * (256 / 16) + threadIdx.x / 16;
  const int row = group / groups_per_row, at = (group - row * groups_per_row) * ONEBIT_CODE_GROUP + threadIdx.x % 16 * 8;
  float v[8] = {};
  if (group < groups) {
    if (WHOLE) {
      if (at < columns) load_values<TYPE, 8>(x, row * x_stride + at, v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float one[1] = {0.f};
        if (at + i < columns) load_values<TYPE, 1>(x, row * x_stride + at + i, one);
        v[i] = one[0];
      }
    }
  }
  store_codes(out, row, at, group < groups, v);
}

template <int TYPE>
hipError_t launch_as(const void* x, long long x_stride, int rows, int columns, const onebit_codes& out, hipStream_t stream) {
  const int groups_per_row = padded_columns(columns) / ONEBIT_CODE_GROUP;
  const long long groups = (long long)rows * groups_per_row;
  const bool whole = columns % 8 == 0 && x_stride % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0;
  if (groups * 16 >= 1ll << 32 || groups >= 1ll << 31) return hipErrorInvalidConfiguration;
  const dim3 grid((unsigned)((groups + 15) / 16));
  return launch_kernel(whole ? quantize_rows_kernel<TYPE, true> : quantize_rows_kernel<TYPE, false>, grid, dim3(256), 0, stream, x, x_stride, columns,
                       groups_per_row, (int)groups, out);
}

}  // namespace

hipError_t launch_quantize_rows(const void* x, int dtype, long long x_stride, int rows, int columns, const onebit_codes& out, hipStream_t stream) {
  if (dtype == ONEBIT_DTYPE_F32) return launch_as<ONEBIT_DTYPE_F32>(x, x_stride, rows, columns, out, stream);
  return dtype == ONEBIT_DTYPE_F16 ? launch_as<ONEBIT_DTYPE_F16>(x, x_stride, rows, columns, out, stream)
                                   : launch_as<ONEBIT_DTYPE_BF16>(x, x_stride, rows, columns, out, stream);
}

}  // namespace onebit
