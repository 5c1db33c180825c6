// Host side of TMA: building the CUtensorMap a kernel reads its (bh, rows, width) operand through.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include "common.h"

namespace limn_b200 {

// A 4-D map (column, row, head, batch) over an operand of 2-byte elements, fetched in boxes of `box_rows`
// rows by 64 elements (128 bytes) of one (batch, head) problem, written to shared memory with the 128-byte
// swizzle the tcgen05 operand descriptors expect. Rows past `rows` read as zero, so a ragged last tile
// never reaches another problem's rows.
int make_tile_map(CUtensorMap* map, const void* base, bool fp16, int batch, int heads, int rows, int width, int box_rows,
                  const Strides& strides);

// A 5-D map of 2-byte elements with any extents and boxes: dims and box innermost first, strides in bytes of dims 1 to 4 (multiples of 16). The
// box's first extent is 64 elements; the same swizzle, and zeros outside. Errors name `name`.
struct BoxShape {
  unsigned long long dims[5];
  long long strides[4];
  unsigned box[5];
};
int make_box_map(const char* name, CUtensorMap* map, const void* base, bool fp16, const BoxShape& shape);

}  // namespace limn_b200
