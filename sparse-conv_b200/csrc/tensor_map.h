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

}  // namespace spconv
