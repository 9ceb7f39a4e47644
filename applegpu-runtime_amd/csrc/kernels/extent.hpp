// How far a matrix operand's values reach in memory, for the bounds of its
// buffer resources.  Plain C++, so that it can be checked without a device.
#pragma once

#include <cstdint>

namespace agpu {
namespace k {
namespace t16 {

// Counts are of 16-bit values.  A row of `n` values: plain ones (planes 1) in
// whole 16-byte chunks, or (planes 2) every 32 of them as high and low halves
// with zeros behind the last.
constexpr int64_t row_values(int64_t n, int planes) {
  return planes == 1 ? (n + 7) / 8 * 8 : (n + 31) / 32 * 64;
}
// `rows` rows, `ld` apart, from their column `first` on: up to the last row's
// own last value.  Rows of a view of columns end short of the next one's start,
// and the storage may end with the last one.
constexpr int64_t extent_of_columns(int64_t rows, int64_t n, int64_t first, int64_t ld, int planes) {
  return (rows - 1) * ld + row_values(n, planes) - first * planes;
}

}  // namespace t16
}  // namespace k
}  // namespace agpu
