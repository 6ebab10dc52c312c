// TMA tensor maps (encoded by the driver; defined in conv_tc.cu).
#pragma once

#include <cstdint>
#include <cuda.h>

namespace spconv {

// 2-D row-major tensor of 16-bit elements: `cols` x `rows`, rows `row_stride` bytes apart;
// box = box_cols x box_rows; swizzle width = box_cols * 2 bytes. Sets the error message and
// returns false where the driver refuses it.
bool make_tmap_2d(CUtensorMap *map, const void *ptr, uint64_t cols, uint64_t rows,
                  uint64_t row_stride, uint32_t box_cols, uint32_t box_rows);
// The same in three dimensions, x contiguous, 128-byte swizzle (box_x * 2 bytes = 128); boxes past an end are filled with
// zeros. Strides in bytes, multiples of 16.
bool make_tmap_3d(CUtensorMap *map, const void *ptr, uint64_t x, uint64_t y, uint64_t z, uint64_t y_stride, uint64_t z_stride,
                  uint32_t box_x, uint32_t box_y, uint32_t box_z);

}  // namespace spconv
