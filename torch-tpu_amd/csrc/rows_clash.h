// Whether two sets of rows share memory (host arithmetic).
#pragma once
#include <cstdint>

namespace moe {

// a_rows rows of a_bytes bytes, a_stride bytes apart, and the same of b.  Rows of one lie between those of the other where the distance is the
// same, as two halves of a wider buffer; of two distances the whole stretches count.
inline bool rows_clash(const void *a, int64_t a_stride, int64_t a_bytes, int64_t a_rows, const void *b, int64_t b_stride, int64_t b_bytes, int64_t b_rows) {
  if (!a || !b || a_rows <= 0 || b_rows <= 0 || a_bytes <= 0 || b_bytes <= 0) return false;
  const int64_t p = (int64_t)(uintptr_t)a, q = (int64_t)(uintptr_t)b;
  if (p + (a_rows - 1) * a_stride + a_bytes <= q || q + (b_rows - 1) * b_stride + b_bytes <= p) return false;
  const int64_t stride = a_rows == 1 ? b_stride : a_stride;
  if ((a_rows == 1 && b_rows == 1) || (a_rows > 1 && b_rows > 1 && a_stride != b_stride) || stride <= 0) return true;
  const int64_t off = ((q - p) % stride + stride) % stride;              // from a row of a to the next one of b
  return off < a_bytes || stride - off < b_bytes;
}

}  // namespace moe
