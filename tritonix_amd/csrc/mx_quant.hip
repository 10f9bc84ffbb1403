// Quantisation to microscaled 4-bit floats and back.
//
// A block of 32 elements with largest magnitude a gets the scale 2^e, e = floor(log2 a) - 2 (the exponent of 6, the
// largest 4-bit value, is 2), clamped to [-127, 127], and each element x the 4-bit float nearest to x / 2^e, ties to the even
// code, magnitudes above 6 to 6.  The division is a multiplication by 2^-e, exact in binary32 but for results below
// its smallest normal number, which round to code 0 either way.  A block that holds an infinity or a NaN gets the NaN scale.
//
// Both directions are bound by memory: 2 (4) bytes and 17/32 of one per element.  Two layouts of the source:
//   k contiguous   a lane takes 8 neighbouring elements (16 or 32 bytes), four lanes share a block, and the largest magnitude goes round the
//                  four in two DPP steps; the codes of a lane are one aligned word, so loads and stores are whole runs of a row
//   anything else  (rows contiguous: a matrix quantised down its columns.)  A lane takes two neighbouring rows and walks
//                  the 32 k of its block, loads of 64 neighbouring pairs; the largest magnitude needs no other lane.  The codes of
//                  128 rows x 256 k meet in LDS and leave as rows of 128 bytes.
#include <hip/hip_runtime.h>

#include "../../include/tritonix_hip.h"
#include "mx.h"

using namespace tnx;

namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void values8(uint32_t c, float scale, float* v) {
  const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 1);
  const f32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 2), f = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 3);
  v[0] = a.x * scale; v[1] = a.y * scale; v[2] = b.x * scale; v[3] = b.y * scale;
  v[4] = d.x * scale; v[5] = d.y * scale; v[6] = f.x * scale; v[7] = f.y * scale;
}

struct QuantParams {
  const uint8_t* src;
  uint8_t *dst, *codes, *scales;
  int64_t rows, k, slabs, batch;
  int64_t stride_b, stride_r, stride_k;                  // elements of src / dst
  int64_t codes_b, scales_b;                             // bytes from one matrix of the batch to the next
};

constexpr int ROW_ITEMS = 4;                             // runs of 8 elements a lane takes, 256 lanes apart


template <class T>
__global__ __launch_bounds__(256) void quantize_rows_kernel(QuantParams p) {
  typedef typename Elem<T>::raw raw;
  const int64_t total = p.rows * p.slabs * 32;           // runs of one matrix
  const int64_t first = (int64_t)blockIdx.x * (256 * ROW_ITEMS) + threadIdx.x;
  const raw* src = (const raw*)p.src + (int64_t)blockIdx.y * p.stride_b;
  uint8_t* codes = p.codes + (int64_t)blockIdx.y * p.codes_b;
  uint8_t* scales = p.scales + (int64_t)blockIdx.y * p.scales_b;
  Run8<T> x[ROW_ITEMS];
  int64_t row[ROW_ITEMS];
  int at[ROW_ITEMS];
#pragma unroll
  for (int u = 0; u < ROW_ITEMS; ++u) {
    const int64_t i = first + u * 256;
    const int64_t item = i < total ? i : 0;
    row[u] = total < 0x7fffffff ? (int64_t)((uint32_t)item / (uint32_t)(p.slabs * 32)) : item / (p.slabs * 32);
    at[u] = (int)(item - row[u] * p.slabs * 32);
    const int64_t left = p.k - (int64_t)at[u] * 8;
    const raw* s = src + row[u] * p.stride_r + (int64_t)at[u] * 8;
    if (left >= 8) x[u] = *(const Run8<T>*)s;
    else {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[u].v[e] = e < left ? s[e] : (raw)0;
    }
  }
#pragma unroll
  for (int u = 0; u < ROW_ITEMS; ++u) {
    float v[8];
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] = Elem<T>::get(x[u].v[e]);
      const uint32_t b = __builtin_bit_cast(uint32_t, v[e]) & 0x7fffffffu;
      top = top > b ? top : b;
    }
    top = quad_max(top);                                 // (all four lanes of a block are here: runs come in whole slabs)
    float factor;
    uint32_t s = scale_byte(top, &factor);
    if ((int64_t)(at[u] & ~3) * 8 >= p.k) s = 127;       // a block of padding
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = scaled(v[e], factor);
    if (first + u * 256 >= total) continue;
    *(uint32_t*)(codes + (row[u] * p.slabs * 32 + at[u]) * 4) = codes8(v);
    if ((at[u] & 3) == 0) scales[mx_scale_at(row[u], at[u] >> 5, p.slabs) + ((at[u] >> 2) & 7)] = (uint8_t)s;
  }
}

template <class T>
__global__ __launch_bounds__(256) void dequantize_rows_kernel(QuantParams p) {
  typedef typename Elem<T>::raw raw;
  const int64_t total = p.rows * p.slabs * 32;
  const int64_t first = (int64_t)blockIdx.x * (256 * ROW_ITEMS) + threadIdx.x;
  raw* dst = (raw*)p.dst + (int64_t)blockIdx.y * p.stride_b;
  const uint8_t* codes = p.codes + (int64_t)blockIdx.y * p.codes_b;
  const uint8_t* scales = p.scales + (int64_t)blockIdx.y * p.scales_b;
  uint32_t c[ROW_ITEMS], s[ROW_ITEMS];
  int64_t row[ROW_ITEMS];
  int at[ROW_ITEMS];
#pragma unroll
  for (int u = 0; u < ROW_ITEMS; ++u) {
    const int64_t i = first + u * 256;
    const int64_t item = i < total ? i : 0;
    row[u] = total < 0x7fffffff ? (int64_t)((uint32_t)item / (uint32_t)(p.slabs * 32)) : item / (p.slabs * 32);
    at[u] = (int)(item - row[u] * p.slabs * 32);
    c[u] = *(const uint32_t*)(codes + (row[u] * p.slabs * 32 + at[u]) * 4);
    s[u] = scales[mx_scale_at(row[u], at[u] >> 5, p.slabs) + ((at[u] >> 2) & 7)];
  }
#pragma unroll
  for (int u = 0; u < ROW_ITEMS; ++u) {
    const int64_t left = p.k - (int64_t)at[u] * 8;
    if (first + u * 256 >= total || left <= 0) continue;
    float v[8];
    values8(c[u], scale_value(s[u]), v);
    Run8<T> out;
#pragma unroll
    for (int e = 0; e < 8; ++e) out.v[e] = Elem<T>::put(v[e]);
    raw* d = dst + row[u] * p.stride_r + (int64_t)at[u] * 8;
    if (left >= 8) *(Run8<T>*)d = out;
    else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < left) d[e] = out.v[e];
    }
  }
}

// Columns: a workgroup takes 128 rows and one slab, wave b the block b of it, a lane the rows 2 lane and 2 lane + 1.
// Pitch of a row of codes in LDS: 16 bytes more than 128, so that the lanes' 16-byte pieces of neighbouring rows fall on
// different banks.
constexpr int COL_ROWS = 128, COL_PITCH = MX_ROWB + 16;

template <class T> struct __attribute__((packed, aligned(sizeof(T)))) Pair { typename Elem<T>::raw v[2]; };

// PAIRED: rows are neighbours in memory (stride_r == 1); otherwise any strides, an element at a time
template <class T, bool PAIRED>
__global__ __launch_bounds__(512) void quantize_columns_kernel(QuantParams p) {
  typedef typename Elem<T>::raw raw;
  __shared__ __attribute__((aligned(16))) uint8_t tile[COL_ROWS * COL_PITCH];
  __shared__ __attribute__((aligned(16))) uint8_t tile_s[COL_ROWS * MX_SCALEB];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t slab = blockIdx.y, row0 = (int64_t)blockIdx.x * COL_ROWS;
  const raw* src = (const raw*)p.src + (int64_t)blockIdx.z * p.stride_b;
  uint8_t* codes = p.codes + (int64_t)blockIdx.z * p.codes_b;
  uint8_t* scales = p.scales + (int64_t)blockIdx.z * p.scales_b;
  const int64_t k0 = slab * MX_SLAB + wave * 32, left = p.k - k0;
  const int64_t r = row0 + 2 * lane;
  const bool have0 = r < p.rows, have1 = r + 1 < p.rows;
  raw x0[32], x1[32];
  const raw* s = src + k0 * p.stride_k + r * p.stride_r;
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    x0[i] = x1[i] = 0;
    if (i < left) {
      if (PAIRED && have1) {
        const Pair<T> t = *(const Pair<T>*)(s + i * p.stride_k);
        x0[i] = t.v[0];
        x1[i] = t.v[1];
      } else {
        if (have0) x0[i] = s[i * p.stride_k];
        if (have1) x1[i] = s[i * p.stride_k + p.stride_r];
      }
    }
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const uint32_t b = __builtin_bit_cast(uint32_t, Elem<T>::get(h ? x1[i] : x0[i])) & 0x7fffffffu;
      top = top > b ? top : b;
    }
    float factor;
    const uint32_t sb = left <= 0 ? 127u : scale_byte(top, &factor);
    if (left <= 0) factor = 0.0f;
    i32x4 c;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = scaled(Elem<T>::get(h ? x1[q * 8 + e] : x0[q * 8 + e]), factor);
      c[q] = (int)codes8(v);
    }
    *(i32x4*)(tile + (2 * lane + h) * COL_PITCH + wave * 16) = c;
    tile_s[(2 * lane + h) * MX_SCALEB + wave] = (uint8_t)sb;
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < COL_ROWS * 8 / 512; ++u) {
    const int i = u * 512 + tid, row = i >> 3, chunk = i & 7;
    if (row0 + row < p.rows)
      *(i32x4*)(codes + ((row0 + row) * p.slabs + slab) * MX_ROWB + chunk * 16) = *(const i32x4*)(tile + row * COL_PITCH + chunk * 16);
  }
  // (the scales of the whole groups of 32 rows that the tensor's allocation has)
  if (tid < COL_ROWS && row0 + (tid & ~31) < p.rows)
    *(uint64_t*)(scales + mx_scale_at(row0 + tid, slab, p.slabs)) = *(const uint64_t*)(tile_s + tid * MX_SCALEB);
}

template <class T, bool PAIRED>
__global__ __launch_bounds__(512) void dequantize_columns_kernel(QuantParams p) {
  typedef typename Elem<T>::raw raw;
  __shared__ __attribute__((aligned(16))) uint8_t tile[COL_ROWS * COL_PITCH];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t slab = blockIdx.y, row0 = (int64_t)blockIdx.x * COL_ROWS;
  raw* dst = (raw*)p.dst + (int64_t)blockIdx.z * p.stride_b;
  const uint8_t* codes = p.codes + (int64_t)blockIdx.z * p.codes_b;
  const uint8_t* scales = p.scales + (int64_t)blockIdx.z * p.scales_b;
#pragma unroll
  for (int u = 0; u < COL_ROWS * 8 / 512; ++u) {
    const int i = u * 512 + tid, row = i >> 3, chunk = i & 7;
    if (row0 + row < p.rows)
      *(i32x4*)(tile + row * COL_PITCH + chunk * 16) = *(const i32x4*)(codes + ((row0 + row) * p.slabs + slab) * MX_ROWB + chunk * 16);
  }
  __syncthreads();
  const int64_t k0 = slab * MX_SLAB + wave * 32, left = p.k - k0;
  const int64_t r = row0 + 2 * lane;
  const bool have0 = r < p.rows, have1 = r + 1 < p.rows;
  if (!have0 || left <= 0) return;
  const float f0 = scale_value(scales[mx_scale_at(r, slab, p.slabs) + wave]);
  const float f1 = have1 ? scale_value(scales[mx_scale_at(r + 1, slab, p.slabs) + wave]) : 0.0f;
  const i32x4 c0 = *(const i32x4*)(tile + 2 * lane * COL_PITCH + wave * 16);
  const i32x4 c1 = *(const i32x4*)(tile + (2 * lane + (have1 ? 1 : 0)) * COL_PITCH + wave * 16);
  raw* d = dst + k0 * p.stride_k + r * p.stride_r;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    float v0[8], v1[8];
    values8((uint32_t)c0[q], f0, v0);
    values8((uint32_t)c1[q], f1, v1);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int i = q * 8 + e;
      if (i >= left) continue;
      if (PAIRED && have1) {
        Pair<T> t;
        t.v[0] = Elem<T>::put(v0[e]);
        t.v[1] = Elem<T>::put(v1[e]);
        *(Pair<T>*)(d + i * p.stride_k) = t;
      } else {
        d[i * p.stride_k] = Elem<T>::put(v0[e]);
        if (have1) d[i * p.stride_k + p.stride_r] = Elem<T>::put(v1[e]);
      }
    }
  }
}

// Codes and scales as files hold them (row-major, ceil(k / 2) and ceil(k / 32) bytes a row) into the layout above.  A
// thread per block: 16 bytes of codes and a scale.
__global__ __launch_bounds__(256) void import_kernel(const uint8_t* codes, const uint8_t* scales, uint8_t* out_codes, uint8_t* out_scales,
                                                     int64_t rows, int64_t k, int64_t slabs) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = i / (slabs * 8);
  if (row >= rows) return;
  const int64_t block = i - row * slabs * 8, cb = (k + 1) / 2, sb = (k + 31) / 32, left = k - block * 32;
  codes += (int64_t)blockIdx.y * rows * cb;
  scales += (int64_t)blockIdx.y * rows * sb;
  out_codes += (int64_t)blockIdx.y * mx_code_bytes(rows, k);
  out_scales += (int64_t)blockIdx.y * mx_scale_bytes(rows, k);
  uint8_t c[16];
  const uint8_t* s = codes + row * cb + block * 16;
#pragma unroll
  for (int b = 0; b < 16; ++b) {
    c[b] = 2 * b < left ? s[b] : 0;
    if (2 * b + 1 == left) c[b] &= 15;                   // an odd k: the last byte has one element
  }
  i32x4 v;
  __builtin_memcpy(&v, c, 16);
  *(i32x4*)(out_codes + (row * slabs * 8 + block) * 16) = v;
  out_scales[mx_scale_at(row, block >> 3, slabs) + (block & 7)] = left > 0 ? scales[row * sb + block] : 127;
}

template <class T, bool BACK> int launch(const QuantParams& p, hipStream_t stream) {
  if (p.stride_k == 1) {
    const int64_t blocks = (p.rows * p.slabs * 32 + 256 * ROW_ITEMS - 1) / (256 * ROW_ITEMS);
    if (blocks > 0x7fffffff) return TNX_E_UNSUPPORTED;
    const dim3 grid((unsigned)blocks, (unsigned)p.batch);
    if (BACK) hipLaunchKernelGGL((dequantize_rows_kernel<T>), grid, dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((quantize_rows_kernel<T>), grid, dim3(256), 0, stream, p);
    return mx_launched();
  }
  const int64_t tiles = (p.rows + COL_ROWS - 1) / COL_ROWS;
  if (tiles > 0x7fffff || p.slabs > 65535) return TNX_E_UNSUPPORTED;
  const dim3 grid((unsigned)tiles, (unsigned)p.slabs, (unsigned)p.batch);
  const bool paired = p.stride_r == 1;
  if (BACK && paired) hipLaunchKernelGGL((dequantize_columns_kernel<T, true>), grid, dim3(512), 0, stream, p);
  else if (BACK) hipLaunchKernelGGL((dequantize_columns_kernel<T, false>), grid, dim3(512), 0, stream, p);
  else if (paired) hipLaunchKernelGGL((quantize_columns_kernel<T, true>), grid, dim3(512), 0, stream, p);
  else hipLaunchKernelGGL((quantize_columns_kernel<T, false>), grid, dim3(512), 0, stream, p);
  return mx_launched();
}

template <bool BACK> int convert(const tnx_mx_args* a) {
  if (!a || a->rows < 0 || a->k < 0 || a->batch < 0) return TNX_E_INVALID;
  if (a->rows == 0 || a->k == 0 || a->batch == 0) return TNX_OK;
  if (!a->data || !a->codes || !a->scales || ((uintptr_t)a->codes & 15) || ((uintptr_t)a->scales & 15)) return TNX_E_INVALID;
  if (a->k > TNX_MX_MAX_K || a->batch > 65535) return TNX_E_UNSUPPORTED;
  const unsigned size = a->dtype == TNX_F32 ? 4 : 2;
  if ((uintptr_t)a->data & (size - 1)) return TNX_E_INVALID;
  QuantParams p;
  p.src = (const uint8_t*)a->data;
  p.dst = (uint8_t*)a->data;
  p.codes = (uint8_t*)a->codes;
  p.scales = (uint8_t*)a->scales;
  p.rows = a->rows; p.k = a->k; p.slabs = mx_slabs(a->k); p.batch = a->batch;
  p.stride_b = a->stride_batch; p.stride_r = a->stride_row; p.stride_k = a->k == 1 ? 1 : a->stride_k;
  p.codes_b = mx_code_bytes(a->rows, a->k);
  p.scales_b = mx_scale_bytes(a->rows, a->k);
  const hipStream_t stream = (hipStream_t)a->stream;
  switch (a->dtype) {
    case TNX_BF16: return launch<__bf16, BACK>(p, stream);
    case TNX_F16: return launch<_Float16, BACK>(p, stream);
    case TNX_F32: return launch<float, BACK>(p, stream);
    default: return TNX_E_UNSUPPORTED;
  }
}

}  // namespace

extern "C" size_t tnx_mx_code_bytes(int64_t rows, int64_t k) { return rows > 0 && k > 0 ? (size_t)mx_code_bytes(rows, k) : 0; }
extern "C" size_t tnx_mx_scale_bytes(int64_t rows, int64_t k) { return rows > 0 && k > 0 ? (size_t)mx_scale_bytes(rows, k) : 0; }

extern "C" int tnx_mx_quantize(const tnx_mx_args* a) { return convert<false>(a); }
extern "C" int tnx_mx_dequantize(const tnx_mx_args* a) { return convert<true>(a); }

extern "C" int tnx_mx_import(const void* codes, const void* scales, int64_t batch, int64_t rows, int64_t k, void* out_codes, void* out_scales,
                             void* stream) {
  if (rows < 0 || k < 0 || batch < 0) return TNX_E_INVALID;
  if (rows == 0 || k == 0 || batch == 0) return TNX_OK;
  if (!codes || !scales || !out_codes || !out_scales || (((uintptr_t)out_codes | (uintptr_t)out_scales) & 15)) return TNX_E_INVALID;
  if (k > TNX_MX_MAX_K || batch > 65535) return TNX_E_UNSUPPORTED;
  const int64_t slabs = mx_slabs(k), blocks = (rows * slabs * 8 + 255) / 256;
  if (blocks > 0x7fffffff) return TNX_E_UNSUPPORTED;
  hipLaunchKernelGGL(import_kernel, dim3((unsigned)blocks, (unsigned)batch), dim3(256), 0, (hipStream_t)stream, (const uint8_t*)codes, (const uint8_t*)scales,
                     (uint8_t*)out_codes, (uint8_t*)out_scales, rows, k, slabs);
  return mx_launched();
}
