// The 4-bit block formats and their storage, shared by the quantisation and
// product kernels.
//
// A value is an e2m1 code (two to a byte, the even element in the low half)
// times a scale shared by a block of a row:
//   TM_FP4_NV  16 values, e4m3 scale, times an fp32 scale of the row (or tensor)
//   TM_FP4_MX  32 values, e8m0 (power of two) scale
// Block scales are stored the way the tensor cores take them: tiles of 128
// rows x 4 blocks in 512 bytes, row r and block c of a tile at byte
// (r % 32) * 16 + (r / 32) * 4 + c -- 32 lanes of 16 bytes, each holding four
// rows' four scales -- and a row of tiles is contiguous.  Rows and blocks that
// pad the last tiles hold 0.
#pragma once

#include <cstdint>

#include "common.h"

namespace tmw {

constexpr int fp4_block(int format) { return format == TM_FP4_NV ? 16 : 32; }

inline int64_t round_up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

// Byte of the scale of (row, block) when a row of tiles has `ktiles` tiles.
__host__ __device__ __forceinline__ int64_t fp4_scale_offset(int64_t row, int64_t block,
                                                             int64_t ktiles) {
  return ((row >> 7) * ktiles + (block >> 2)) * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4 +
         (block & 3);
}

}  // namespace tmw
