// Microscaled 4-bit tensors as the kernels hold them.
//
// A tensor of R rows of K elements, quantised along K in blocks of 32: an element is a 4-bit float (sign, two exponent
// bits, one mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6), a block has one scale byte s that stands for 2^(s - 127) (255: NaN).
// K is padded to whole slabs of 256 with codes of zero and scales of 127, so that no kernel has a tail along K:
//   codes   row-major, 128 bytes per row and slab; the even element of a byte in its low half
//   scales  8 bytes per row and slab, those of two slabs together, 32 rows together: [row / 32][slab / 2][row % 32][slab % 2][8].  A direct load
//           of 16 bytes per lane brings a row's scales of two slabs, wherever the row lies; 64 neighbouring rows are 1 KiB in a
//           piece (row-major, each row's 16 bytes would be a cache line of their own)
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "gemm_tile.h"

namespace tnx {

constexpr int MX_SLAB = 256, MX_ROWB = 128, MX_SCALEB = 8, MX_GROUP = 32;

__host__ __device__ inline int64_t mx_slabs(int64_t k) { return (k + MX_SLAB - 1) / MX_SLAB; }
__host__ __device__ inline int64_t mx_code_bytes(int64_t rows, int64_t k) { return rows * mx_slabs(k) * MX_ROWB; }
__host__ __device__ inline int64_t mx_pairs(int64_t slabs) { return (slabs + 1) / 2; }
__host__ __device__ inline int64_t mx_scale_bytes(int64_t rows, int64_t k) {
  return (rows + MX_GROUP - 1) / MX_GROUP * mx_pairs(mx_slabs(k)) * (MX_GROUP * 2 * MX_SCALEB);
}
// where the eight scales of (row, slab) start
__device__ __forceinline__ int64_t mx_scale_at(int64_t row, int64_t slab, int64_t slabs) {
  return ((row >> 5) * ((slabs + 1) >> 1) + (slab >> 1)) * (MX_GROUP * 2 * MX_SCALEB) + (row & 31) * (2 * MX_SCALEB) + (slab & 1) * MX_SCALEB;
}

// a launch's own error, noted for tnx_last_hip_error
void note_hip_error(int err);

inline int mx_launched() {
  const hipError_t err = hipGetLastError();
  if (err == hipSuccess) return 0;
  note_hip_error((int)err);
  return 5;                                              // TNX_E_HIP
}

}  // namespace tnx
