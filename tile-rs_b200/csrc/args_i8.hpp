// Which calls of the 8-bit operators are refused, and with what words: host arithmetic only, so that it can be looked at without a
// GPU (tests/test_args_i8.py).
#pragma once

#include <cstddef>
#include <cstdint>

#include "../../include/tile_sm100.h"

namespace tsm100 {
namespace args {

inline size_t elem_bytes(int32_t dtype) { return dtype == TSM100_F32 ? 4 : dtype == TSM100_F16 || dtype == TSM100_BF16 ? 2 : 0; }
inline bool off(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes != 0; }

// What is wrong with a call, or null.  *nothing: there is nothing to do.
inline const char* quantise_rows(const tsm100_quantise_rows_desc* d, const void* x, const void* up, const void* y, const float* scales, bool* nothing) {
  *nothing = false;
  if (!d) return "null descriptor";
  if (!elem_bytes(d->dtype)) return "unknown dtype";
  if (d->rows < 0 || d->cols < 0 || d->rows > 0x7fffffff || d->cols > 0x7fff0000 || d->pitch < 0) return "bad shape";
  if (d->rows == 0 || d->cols == 0) {
    *nothing = true;
    return nullptr;
  }
  const int64_t pitch = d->pitch ? d->pitch : d->cols;
  if (pitch < d->cols) return "pitch is less than cols";
  if (pitch > INT64_MAX / 8 / d->rows) return "bad shape";
  if (!x || !y || !scales) return "null buffer";
  if (off(x, elem_bytes(d->dtype)) || off(up, elem_bytes(d->dtype))) return "a buffer does not start on an element boundary";
  if (off(scales, 4)) return "scales do not start on an element boundary";
  return nullptr;
}

// 16384 * 131071 is the largest sum that K numbers of -128 can make, and fits 32 bits.
constexpr int64_t kMaxGemmI8K = 131071;
inline const char* gemm_i8(const tsm100_gemm_i8_desc* d, const void* a, const float* a_scales, const void* w, const float* w_scales, const void* c, bool* nothing) {
  *nothing = false;
  if (!d) return "null descriptor";
  if (!elem_bytes(d->dtype)) return "dtype must be TSM100_F32, TSM100_F16 or TSM100_BF16";
  constexpr int64_t kMost = 0x7fffffff - 1024, kPitch = 1ll << 32;
  if (d->m < 0 || d->n < 0 || d->k < 0 || d->m > kMost || d->n > kMost || d->lda < 0 || d->ldw < 0 || d->ldc < 0) return "bad shape";
  if (d->k > kMaxGemmI8K) return "k must be less than 131072";
  if (d->m == 0 || d->n == 0) {
    *nothing = true;
    return nullptr;
  }
  if ((d->lda && d->lda < d->k) || (d->ldw && d->ldw < d->k) || (d->ldc && d->ldc < d->n)) return "a pitch is less than its row";
  if (d->lda > kPitch || d->ldw > kPitch || d->ldc > kPitch) return "bad shape";
  // CTAs of a launch: tiles of 16 rows or more by 128 columns, up to eight to each
  if ((d->m + 15) / 16 * ((d->n + 127) / 128) > 0x7fffffff / 8) return "too many rows times columns for one launch";
  if (!c || (d->k > 0 && (!a || !w || !a_scales || !w_scales))) return "null buffer";
  if (off(c, elem_bytes(d->dtype)) || off(a_scales, 4) || off(w_scales, 4)) return "a buffer does not start on an element boundary";
  return nullptr;
}

}  // namespace args
}  // namespace tsm100
