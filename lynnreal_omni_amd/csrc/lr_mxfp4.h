// lr_mxfp4.h - where the scale bytes of MXFP4 rows lie.
//
// v_mfma_scale_f32_16x16x128_f8f6f4 takes, for the 16 rows x 128 columns of an
// operand, row l % 16 and columns 32 * (l / 16) .. + 31 from lane l, and that
// block's E8M0 byte from a byte (0..3, chosen by the instruction) of a register
// of lane l. A tile of 64 rows x 8 blocks (256 columns) has its bytes so that
// lane l reads the eight that it needs with one 8-byte load: byte 2 * f + h is
// row 16 * f + l % 16, block 4 * h + l / 16. Tiles: [ceil(rows / 64)]
// [ceil(blocks / 8)], 512 bytes each, row tiles outermost. Bytes of blocks past
// the last one are 0 (their codes read as zero).
#pragma once

#include <stdint.h>

namespace lr {

// Tiles along a row of `width` columns.
__host__ __device__ inline int64_t mxfp4_scale_tiles(int64_t width) { return (width + 255) / 256; }

// Byte of (row, block) among tiles of which a row has `col_tiles`.
__host__ __device__ inline int64_t mxfp4_scale_at(int64_t row, int64_t block, int64_t col_tiles) {
  const int b = (int)(block & 7), r = (int)(row & 63);
  return ((row >> 6) * col_tiles + (block >> 3)) * 512 + (16 * (b & 3) + (r & 15)) * 8 + 2 * (r >> 4) + (b >> 2);
}

}  // namespace lr
