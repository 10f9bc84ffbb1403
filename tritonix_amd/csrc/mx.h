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

// ---- quantisation of a block (see mx_quant.hip for the definition)
template <class T> struct Elem;
template <> struct Elem<float> {
  static __device__ __forceinline__ float get(uint32_t v) { return __builtin_bit_cast(float, v); }
  typedef uint32_t raw;
  static __device__ __forceinline__ raw put(float v) { return __builtin_bit_cast(uint32_t, v); }
};
template <> struct Elem<__bf16> {
  typedef uint16_t raw;
  static __device__ __forceinline__ float get(raw v) { return __builtin_bit_cast(float, (uint32_t)v << 16); }
  static __device__ __forceinline__ raw put(float v) { return f32_to_bf16(v); }
};
template <> struct Elem<_Float16> {
  typedef uint16_t raw;
  static __device__ __forceinline__ float get(raw v) { return (float)__builtin_bit_cast(_Float16, v); }
  static __device__ __forceinline__ raw put(float v) { return __builtin_bit_cast(uint16_t, (_Float16)v); }
};

// magnitude of an element as an integer (these order as the magnitudes do, infinities and NaNs last), and the binary32 bits of one
template <class R> __device__ __forceinline__ R magnitude(R v) { return v & (R)(sizeof(R) == 4 ? 0x7fffffffu : 0x7fffu); }
template <class T> __device__ __forceinline__ uint32_t top_bits(typename Elem<T>::raw m) { return __builtin_bit_cast(uint32_t, Elem<T>::get(m)); }

// scale byte of a block whose largest magnitude has the binary32 bits `top`, and the factor 2^-e (0 for a block without finite values: its codes are zero)
__device__ __forceinline__ uint32_t scale_byte(uint32_t top, float* factor) {
  const int exponent = (int)(top >> 23);                 // biased; 0: zero or subnormal, below 2^-126: e is -127 there
  if (exponent == 255) { *factor = 0.0f; return 255; }
  const int s = exponent > 2 ? exponent - 2 : 0;         // e + 127
  *factor = __builtin_bit_cast(float, (uint32_t)(254 - s) << 23);      // s <= 252: a normal number
  return (uint32_t)s;
}

__device__ __forceinline__ float scale_value(uint32_t s) {
  return __builtin_bit_cast(float, s == 255 ? 0x7fc00000u : s == 0 ? 0x00400000u : s << 23);
}

// eight values already divided by the scale -> eight codes; the first in the low bits
__device__ __forceinline__ uint32_t codes8(const float* v) {
  uint32_t r = 0;
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[0], v[1], 1.0f, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[2], v[3], 1.0f, 1);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[4], v[5], 1.0f, 2);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[6], v[7], 1.0f, 3);
  return r;
}

// an element times the block's factor; in a block without finite values everything becomes 0
__device__ __forceinline__ float scaled(float x, float factor) { return factor == 0.0f ? 0.0f : x * factor; }

// the largest of the four lanes that share a block
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
  const uint32_t a = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, true);      // lane ^ 1
  v = v > a ? v : a;
  const uint32_t b = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, true);      // lane ^ 2
  return v > b ? v : b;
}

// the largest of the N lanes (8 or 16) that share a block
template <int N> __device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
  v = quad_max(v);
  const uint32_t a = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xF, 0xF, true);     // the mirrored lane of eight: of the other quad
  v = v > a ? v : a;
  if (N == 16) {
    const uint32_t b = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xF, 0xF, true);   // of sixteen
    v = v > b ? v : b;
  }
  return v;
}

// eight neighbouring elements, at any alignment of an element
template <class T> struct __attribute__((packed, aligned(sizeof(T)))) Run8 { typename Elem<T>::raw v[8]; };

// a launch's own error, noted for tnx_last_hip_error
void note_hip_error(int err);

inline int mx_launched() {
  const hipError_t err = hipGetLastError();
  if (err == hipSuccess) return 0;
  note_hip_error((int)err);
  return 5;                                              // TNX_E_HIP
}

}  // namespace tnx
