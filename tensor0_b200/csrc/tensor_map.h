// TMA tensor maps with 128-byte rows, swizzled.
#pragma once

#include <cuda.h>

#include <cstdint>

namespace t0b {

// A 16-bit operand [depth, rows, columns] (depth 0: two dimensions): boxes of
// 64 columns and `box` rows.  The strides are in elements, multiples of 8.
CUtensorMap EncodeHalves(bool bf16, const void* data, int64_t columns, int64_t rows, int64_t depth,
                         int64_t row_stride, int64_t depth_stride, int box);

// Packed rows of bytes: boxes of `box_columns` (at most 128) and `box_rows`.
CUtensorMap EncodeBytes(const void* data, int64_t columns, int64_t rows, int box_columns, int box_rows);

}  // namespace t0b
