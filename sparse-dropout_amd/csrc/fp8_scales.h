// Where the scales of a matrix in 1 x 128 blocks end.  Plain integer code, the same on the host and in the kernels.
#pragma once
#include <stdint.h>

#ifdef __HIPCC__
#define SD_HOST_DEVICE __host__ __device__ inline
#else
#define SD_HOST_DEVICE inline
#endif

namespace sd {

// Bytes that may be read behind the scale of row `first` (a multiple of 4) in 128-block 0, where scale (row, block k) of `rows` rows and nk blocks
// lies at [k * ld + row], ld a multiple of 4 and at least `rows`, on 4 bytes: up to the word that holds the last row's scale in the last
// block.  The row of that block need not be ld bytes long: the scales may be those of some rows of a larger matrix.
SD_HOST_DEVICE int64_t row_scales_left(int64_t nk, int64_t ld, int64_t rows, int64_t first) { return (nk - 1) * ld + (rows + 3) / 4 * 4 - first; }

}  // namespace sd
