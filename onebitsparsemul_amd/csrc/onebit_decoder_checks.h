// What the entry points of onebit_decoder.h and onebit_head.h share: messages, statuses, checks of operands (internal to libonebitmul). Host code only.
#pragma once
#include "onebit_head.h"
#include "onebit_launch.h"

#include <cstdarg>
#include <cstdio>

namespace onebit {

inline int fail(int code, const char* fmt, ...) {
  char text[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(text, sizeof text, fmt, ap);
  va_end(ap);
  return report(code, text);
}
template <class... Values>
inline int refuse(const char* fmt, Values... values) { return fail(ONEBIT_ERR_ARGUMENT, fmt, values...); }
inline int launched(hipError_t status, const char* what) {
  return status == hipSuccess ? ONEBIT_OK : fail(ONEBIT_ERR_HIP, "HIP error '%s' from %s", hipGetErrorString(status), what);
}

inline bool aligned(const void* p, int to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }
inline bool is_type(int dtype) { return dtype == ONEBIT_DTYPE_F32 || dtype == ONEBIT_DTYPE_F16 || dtype == ONEBIT_DTYPE_BF16; }

inline int check_codes(const onebit_codes* c, const char* name) {
  if (!c || !c->codes || !c->scales) return refuse("null pointer in the codes of %s", name);
  if (!aligned(c->codes, 16) || !aligned(c->scales, 4) || c->row_stride % 16)
    return refuse("the codes of %s must be 16-byte aligned, with rows a multiple of 16 apart", name);
  return ONEBIT_OK;
}
// Rows that are written must not overlap
inline int check_apart(const onebit_codes& c, int rows, int columns) {
  const long long groups = ((long long)columns + ONEBIT_CODE_GROUP - 1) / ONEBIT_CODE_GROUP;
  if (rows > 1 && (c.row_stride < groups * ONEBIT_CODE_GROUP || c.scale_stride < groups))
    return refuse("rows of the result's codes and scales must not overlap (strides %lld, %lld)", c.row_stride, c.scale_stride);
  return ONEBIT_OK;
}

}  // namespace onebit

#define CHECKED(call) \
  if (const int code_ = (call)) return code_
