// TMA tensor maps with 128-byte rows, swizzled.
#pragma once

#include <cuda.h>

#include <cstdint>

namespace t0b {

// A 16-bit operand [depth, rows, columns] (depth 0: two dimensions): boxes of
// 64 columns and `box` rows.  The strides are in elements, multiples of 8.
CUtensorMap EncodeHalves(bool bf16, const void* data, int64_t columns, int64_t rows, int64_t depth,
                         int64_t row_stride, int64_t depth_stride, int box);

// The same operand as blocks of 64 columns, [depth, block, row, 64]: boxes of
// `box_blocks` blocks of `box_rows` rows, which land block by block.  64 divides
// the columns.
CUtensorMap EncodeBlocks(bool bf16, const void* data, int64_t columns, int64_t rows, int64_t depth,
                         int64_t row_stride, int64_t depth_stride, int box_rows, int box_blocks);

// Packed rows of bytes: boxes of `box_columns` (at most 128) and `box_rows`.
CUtensorMap EncodeBytes(const void* data, int64_t columns, int64_t rows, int box_columns, int box_rows);

}  // namespace t0b
