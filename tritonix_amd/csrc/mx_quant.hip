// Quantisation to microscaled 4-bit floats and back.
//
// A block of 32 elements with largest magnitude a gets the scale 2^e, e = floor(log2 a) - 2 (the exponent of 6, the
// largest 4-bit value, is 2) but at least -127, and each element x the 4-bit float nearest to x / 2^e, ties to the even
// code, magnitudes above 6 to 6.  The division is a multiplication by 2^-e, exact in binary32 but for results below
// its smallest normal number, which round to code 0 either way.  A block that holds an infinity or a NaN gets the NaN scale.
//
// Both directions are bound by memory: 2 (4) bytes and 17/32 of one per element.  Two layouts of the source:
//   k contiguous   a lane takes 8 neighbouring elements (16 or 32 bytes), four lanes share a block, and the largest magnitude goes round the
//                  four in two DPP steps; the codes of a lane are one aligned word, so loads and stores are whole runs of a row
//   anything else  (rows contiguous: a matrix quantised down its columns.)  A lane takes 8 bytes of neighbouring rows and walks
//                  the 32 k of its block; the largest magnitude needs no other lane.  The codes of the rows x 256 k meet in LDS
//                  and leave as rows of 128 bytes.
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
  uint8_t *codes2, *scales2;                             // the same matrix quantised along its rows instead (quantize_columns_kernel)
};

// Runs that a lane takes, 256 lanes apart.  8192 x 8192 bfloat16: quantising 30.9 us with two, 35.6 with four (the next workgroups' loads begin sooner).
constexpr int QUANT_RUNS = 2, BACK_RUNS = 4;


// STREAM: a source that the memory-side cache of 256 MiB cannot hold is read past the caches (8192 x 28672 bfloat16: 108 us, so 123; a smaller one
// that was just written is there: 8192 x 8192 31 us, past the caches 34).  For 2-byte elements; float32 is the same either way.
template <class T, bool STREAM>
__global__ __launch_bounds__(256) void quantize_rows_kernel(QuantParams p) {
  typedef typename Elem<T>::raw raw;
  const int64_t total = p.rows * p.slabs * 32;           // runs of one matrix
  const int64_t first = (int64_t)blockIdx.x * (256 * QUANT_RUNS) + threadIdx.x;
  const raw* src = (const raw*)p.src + (int64_t)blockIdx.y * p.stride_b;
  uint8_t* codes = p.codes + (int64_t)blockIdx.y * p.codes_b;
  uint8_t* scales = p.scales + (int64_t)blockIdx.y * p.scales_b;
  Run8<T> x[QUANT_RUNS];
  int64_t row[QUANT_RUNS];
  int at[QUANT_RUNS];
#pragma unroll
  for (int u = 0; u < QUANT_RUNS; ++u) {
    const int64_t i = first + u * 256;
    const int64_t item = i < total ? i : 0;
    row[u] = total < 0x7fffffff ? (int64_t)((uint32_t)item / (uint32_t)(p.slabs * 32)) : item / (p.slabs * 32);
    at[u] = (int)(item - row[u] * p.slabs * 32);
    const int64_t left = p.k - (int64_t)at[u] * 8;
    const raw* s = src + row[u] * p.stride_r + (int64_t)at[u] * 8;
    if (left >= 8) {
      if constexpr (STREAM && sizeof(raw) == 2) {
        const i32x4 w = __builtin_nontemporal_load((const i32x4_loose*)s);
        __builtin_memcpy(&x[u], &w, 16);
      } else x[u] = *(const Run8<T>*)s;
    }
    else {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[u].v[e] = e < left ? s[e] : (raw)0;
    }
  }
#pragma unroll
  for (int u = 0; u < QUANT_RUNS; ++u) {
    float v[8];
    raw top = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const raw b = magnitude(x[u].v[e]);
      top = top > b ? top : b;
    }
    top = (raw)quad_max(top);                            // (all four lanes of a block are here: runs come in whole slabs)
    float factor;
    uint32_t s = scale_byte(top_bits<T>(top), &factor);
    if ((int64_t)(at[u] & ~3) * 8 >= p.k) s = 127;       // a block of padding
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = scaled(Elem<T>::get(x[u].v[e]), factor);
    if (first + u * 256 >= total) continue;
    *(uint32_t*)(codes + (row[u] * p.slabs * 32 + at[u]) * 4) = codes8(v);
    if ((at[u] & 3) == 0) scales[mx_scale_at(row[u], at[u] >> 5, p.slabs) + ((at[u] >> 2) & 7)] = (uint8_t)s;
  }
}

// Back: a lane's run is 16 bytes of the result (8 elements of 2 bytes, 4 of 4), stored past the caches: written through them, the lines that
// the stores only fill in part for a while push out the codes (8192 x 28672: 197 us, so 128; float32 with 32 bytes a lane 339 us).
template <class T>
__global__ __launch_bounds__(256) void dequantize_rows_kernel(QuantParams p) {
  typedef typename Elem<T>::raw raw;
  constexpr int RUN = 16 / sizeof(raw), PER_SLAB = MX_SLAB / RUN;
  const int64_t per_row = p.slabs * PER_SLAB, total = p.rows * per_row;
  const int64_t first = (int64_t)blockIdx.x * (256 * BACK_RUNS) + threadIdx.x;
  raw* dst = (raw*)p.dst + (int64_t)blockIdx.y * p.stride_b;
  const uint8_t* codes = p.codes + (int64_t)blockIdx.y * p.codes_b;
  const uint8_t* scales = p.scales + (int64_t)blockIdx.y * p.scales_b;
  uint32_t c[BACK_RUNS], s[BACK_RUNS];
  int64_t row[BACK_RUNS];
  int at[BACK_RUNS];
#pragma unroll
  for (int u = 0; u < BACK_RUNS; ++u) {
    const int64_t i = first + u * 256;
    const int64_t item = i < total ? i : 0;
    row[u] = total < 0x7fffffff ? (int64_t)((uint32_t)item / (uint32_t)per_row) : item / per_row;
    at[u] = (int)(item - row[u] * per_row);
    const uint8_t* from = codes + (row[u] * per_row + at[u]) * (RUN / 2);
    c[u] = RUN == 8 ? *(const uint32_t*)from : *(const uint16_t*)from;
    s[u] = scales[mx_scale_at(row[u], at[u] / PER_SLAB, p.slabs) + (at[u] / (32 / RUN)) % 8];
  }
#pragma unroll
  for (int u = 0; u < BACK_RUNS; ++u) {
    const int64_t left = p.k - (int64_t)at[u] * RUN;
    if (first + u * 256 >= total || left <= 0) continue;
    float v[8];
    values8(c[u], scale_value(s[u]), v);
    raw o[RUN];
#pragma unroll
    for (int e = 0; e < RUN; ++e) o[e] = Elem<T>::put(v[e]);
    raw* d = dst + row[u] * p.stride_r + (int64_t)at[u] * RUN;
    if (left >= RUN) {
      i32x4 w;
      __builtin_memcpy(&w, o, 16);
      store16_stream_loose(d, w);
    } else {
#pragma unroll
      for (int e = 0; e < RUN; ++e)
        if (e < left) d[e] = o[e];
    }
  }
}

// Columns: wave b of a workgroup takes the b-th 32 k of its part of a slab, a lane LANE neighbouring rows, which it reads 32 times: a load
// instruction is one k.  Two shapes.  WIDE: a whole slab by 8 bytes a lane, 256 rows (128 of float32), so that loads are runs of 512 bytes (4 bytes a lane:
// 8192 x 8192 bfloat16 57 us, with 8 37) and stores whole rows of a slab.  Small, where that makes too few workgroups for the card:
// 64 k by 128 rows (512 x 512 bfloat16, quantised, back and both ways at once: 3.0, 6.0 and 5.8 us, wide 5.9, 10.4 and 11.0;
// 8192 x 4096: 18.8, 17.4 and 27.3, wide 16.4, 16.2 and 24.3).  Pitch of a row of codes in LDS: 16 bytes more, so that the lanes' 16-byte pieces fall on different banks.
template <class T, bool WIDE> struct Columns {
  static constexpr int LANE = WIDE ? 8 / sizeof(typename Elem<T>::raw) : 2, WAVES = WIDE ? 8 : 2, THREADS = 64 * WAVES;
  static constexpr int ROWS = 64 * LANE, K = 32 * WAVES, PARTS = 8 / WAVES;      // of a workgroup; workgroups along a slab
  static constexpr int CHUNKS = WAVES, PITCH = 16 * WAVES + 16;                   // a row's 16-byte pieces
  static constexpr int WORDS = LANE * (int)sizeof(typename Elem<T>::raw) / 4;     // of a lane and k
};
template <class T, int N> struct __attribute__((packed, aligned(sizeof(T)))) RunC { typename Elem<T>::raw v[N]; };

// RUNS: rows are neighbours in memory (stride_r == 1); otherwise any strides, an element at a time
// BOTH: the matrix quantised along its rows as well, from the registers: a block of 32 neighbouring rows is 8 lanes (16 with two rows each), whose
// largest magnitude goes round them for each k.  In the words of the other tensor, a row's codes are 2 bytes (1) a lane.  8192 x 4096 bfloat16: 24.3 us,
// one after the other 18.6 + 16.4.
template <class T, bool WIDE, bool RUNS, bool BOTH>
__global__ __launch_bounds__((Columns<T, WIDE>::THREADS)) void quantize_columns_kernel(QuantParams p) {
  typedef typename Elem<T>::raw raw;
  typedef Columns<T, WIDE> C;
  constexpr int LANE = C::LANE, W = C::WORDS, BITS = 8 * sizeof(raw);
  constexpr int BYTES2 = C::ROWS / 2, PITCH2 = BYTES2 + 16, BLOCKS2 = C::ROWS / 32;
  __shared__ __attribute__((aligned(16))) uint8_t tile[C::ROWS * C::PITCH];
  __shared__ __attribute__((aligned(16))) uint8_t tile_s[C::ROWS * C::WAVES];
  __shared__ __attribute__((aligned(16))) uint8_t tile2[BOTH ? C::K * PITCH2 : 16];
  __shared__ __attribute__((aligned(16))) uint8_t tile2_s[BOTH ? C::K * BLOCKS2 : 16];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t slab = blockIdx.y / C::PARTS, row0 = (int64_t)blockIdx.x * C::ROWS;
  const int part = blockIdx.y % C::PARTS;
  const raw* src = (const raw*)p.src + (int64_t)blockIdx.z * p.stride_b;
  uint8_t* codes = p.codes + (int64_t)blockIdx.z * p.codes_b;
  uint8_t* scales = p.scales + (int64_t)blockIdx.z * p.scales_b;
  const int64_t k0 = slab * MX_SLAB + part * C::K + wave * 32, left = p.k - k0;
  const int64_t r = row0 + LANE * lane, rows_left = p.rows - r;
  // the lane's rows of each k, as words (the empty asm keeps them so: 32 x 4 unpacked elements spill)
  uint32_t x[32][W];
  // 2-byte elements past the caches: a source that is not in them comes at 2 TB/s otherwise (8192 x 4096 bfloat16 42 us, so 17; float32 is the same
  // either way from memory, and 53 us or 70 for 8192 x 8192 where it is in the caches)
  auto load = [&](int i, const raw* at) __attribute__((always_inline)) {
    typedef i32x2 __attribute__((aligned(2))) loose2;
    typedef int __attribute__((aligned(2))) loose1;
    if constexpr (W == 2) {
      const i32x2 w = sizeof(raw) == 2 ? __builtin_nontemporal_load((const loose2*)at) : *(const loose2*)at;
      x[i][0] = (uint32_t)w[0];
      x[i][1] = (uint32_t)w[1];
    } else {
      x[i][0] = (uint32_t)__builtin_nontemporal_load((const loose1*)at);
    }
  };
  if (RUNS && row0 + C::ROWS <= p.rows && left >= 32) {
    const raw* s = src + k0 * p.stride_k + r;
#pragma unroll
    for (int i = 0; i < 32; ++i) load(i, s + i * p.stride_k);
  } else if (RUNS && p.rows >= LANE && left > 0) {
    // An edge: every lane reads whole runs inside the matrix, the last rows' moved up to end with it, k past the end the last one again; then the rows
    // that the lane does not have are shifted out and the k cleared.  (Element by element, each load waits for the one before.)
    const int64_t run = rows_left >= LANE ? r : p.rows - LANE;
    const int drop = rows_left >= LANE ? 0 : rows_left > 0 ? (int)(r - run) * BITS : 64;
    const raw* s = src + k0 * p.stride_k + run;
#pragma unroll
    for (int i = 0; i < 32; ++i) load(i, s + (i < left ? i : left - 1) * p.stride_k);
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      uint64_t v = x[i][0];
      if (W == 2) v |= (uint64_t)x[i][W - 1] << 32;
      v = drop < 64 && i < left ? v >> drop : 0;
      x[i][0] = (uint32_t)v;
      if (W == 2) x[i][W - 1] = (uint32_t)(v >> 32);
    }
  } else {
    const raw* s = src + k0 * p.stride_k + r * p.stride_r;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      RunC<T, LANE> t;
#pragma unroll
      for (int h = 0; h < LANE; ++h) t.v[h] = i < left && h < rows_left ? s[i * p.stride_k + h * p.stride_r] : (raw)0;
      __builtin_memcpy(x[i], &t, 4 * W);
      if (sizeof(raw) == 2 && i % 8 == 7) {               // (eight k at a time: the elements of all 32 spill before they are packed)
#pragma unroll
        for (int q = i - 7; q <= i; ++q)
#pragma unroll
          for (int w = 0; w < W; ++w) asm volatile("" : "+v"(x[q][w]));
      }
    }
  }
  auto pin = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 32; ++i)
#pragma unroll
      for (int w = 0; w < W; ++w) asm volatile("" : "+v"(x[i][w]));
  };
  pin();
  auto element = [&](int i, int h) __attribute__((always_inline)) { return sizeof(raw) == 4 ? (raw)x[i][h % W] : (raw)(x[i][(h >> 1) % W] >> (h & 1) * 16); };
#pragma unroll
  for (int h = 0; h < LANE; ++h) {
    raw top = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const raw b = magnitude(element(i, h));
      top = top > b ? top : b;
    }
    float factor;
    const uint32_t sb = left <= 0 ? 127u : scale_byte(top_bits<T>(top), &factor);
    if (left <= 0) factor = 0.0f;
    i32x4 c;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = scaled(Elem<T>::get(element(q * 8 + e, h)), factor);
      c[q] = (int)codes8(v);
    }
    *(i32x4*)(tile + (LANE * lane + h) * C::PITCH + wave * 16) = c;
    tile_s[(LANE * lane + h) * C::WAVES + wave] = (uint8_t)sb;
    __builtin_amdgcn_sched_barrier(0);                   // (one row's 32 floats at a time: all four at once spill)
  }
  if (BOTH) {
    pin();                                               // (unpacked once more, not kept unpacked)
    const bool padding = row0 + (LANE * lane & ~31) >= p.rows;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      raw top = 0;
#pragma unroll
      for (int h = 0; h < LANE; ++h) {
        const raw b = magnitude(element(i, h));
        top = top > b ? top : b;
      }
      top = (raw)lanes_max<32 / LANE>(top);
      float factor;
      const uint32_t sb = scale_byte(top_bits<T>(top), &factor);
      uint32_t c = 0;
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, scaled(Elem<T>::get(element(i, 0)), factor), scaled(Elem<T>::get(element(i, 1)), factor), 1.0f, 0);
      if (LANE == 4)
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, scaled(Elem<T>::get(element(i, 2)), factor), scaled(Elem<T>::get(element(i, 3)), factor), 1.0f, 1);
      uint8_t* at = tile2 + (wave * 32 + i) * PITCH2 + lane * (LANE / 2);
      if (LANE == 4) *(uint16_t*)at = (uint16_t)c;
      else *at = (uint8_t)c;
      if (lane % (32 / LANE) == 0) tile2_s[(wave * 32 + i) * BLOCKS2 + lane / (32 / LANE)] = (uint8_t)(padding ? 127u : sb);
      if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);
    }
  }
  __syncthreads();
  if (BOTH) {
    const int64_t slabs2 = mx_slabs(p.rows), slab2 = row0 / MX_SLAB, k2 = slab * MX_SLAB + part * C::K;
    const int part2 = (int)(row0 % MX_SLAB) / C::ROWS;
#pragma unroll
    for (int u = 0; u < C::K * (BYTES2 / 16) / C::THREADS; ++u) {
      const int i = u * C::THREADS + tid, row = i / (BYTES2 / 16), chunk = i % (BYTES2 / 16);
      if (k2 + row < p.k)
        *(i32x4*)(p.codes2 + ((k2 + row) * slabs2 + slab2) * MX_ROWB + part2 * BYTES2 + chunk * 16) = *(const i32x4*)(tile2 + row * PITCH2 + chunk * 16);
    }
    if (tid < C::K && k2 + tid < p.k) {
      uint8_t* at = p.scales2 + mx_scale_at(k2 + tid, slab2, slabs2) + part2 * BLOCKS2;
      if (BLOCKS2 == 8) *(uint64_t*)at = *(const uint64_t*)(tile2_s + tid * 8);
      else *(uint32_t*)at = *(const uint32_t*)(tile2_s + tid * 4);
    }
  }
#pragma unroll
  for (int u = 0; u < C::ROWS * C::CHUNKS / C::THREADS; ++u) {
    const int i = u * C::THREADS + tid, row = i / C::CHUNKS, chunk = i % C::CHUNKS;
    if (row0 + row < p.rows)
      *(i32x4*)(codes + ((row0 + row) * p.slabs + slab) * MX_ROWB + (part * C::CHUNKS + chunk) * 16) = *(const i32x4*)(tile + row * C::PITCH + chunk * 16);
  }
  // (the scales of the whole groups of 32 rows that the tensor's allocation has)
  if (tid < C::ROWS && row0 + (tid & ~31) < p.rows) {
    uint8_t* at = scales + mx_scale_at(row0 + tid, slab, p.slabs) + part * C::WAVES;
    if (C::WAVES == 8) *(uint64_t*)at = *(const uint64_t*)(tile_s + tid * C::WAVES);
    else *(uint16_t*)at = *(const uint16_t*)(tile_s + tid * C::WAVES);
  }
}

template <class T, bool WIDE, bool RUNS>
__global__ __launch_bounds__((Columns<T, WIDE>::THREADS)) void dequantize_columns_kernel(QuantParams p) {
  typedef typename Elem<T>::raw raw;
  typedef Columns<T, WIDE> C;
  constexpr int LANE = C::LANE;
  __shared__ __attribute__((aligned(16))) uint8_t tile[C::ROWS * C::PITCH];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t slab = blockIdx.y / C::PARTS, row0 = (int64_t)blockIdx.x * C::ROWS;
  const int part = blockIdx.y % C::PARTS;
  raw* dst = (raw*)p.dst + (int64_t)blockIdx.z * p.stride_b;
  const uint8_t* codes = p.codes + (int64_t)blockIdx.z * p.codes_b;
  const uint8_t* scales = p.scales + (int64_t)blockIdx.z * p.scales_b;
  const int64_t k0 = slab * MX_SLAB + part * C::K + wave * 32, left = p.k - k0;
  const int64_t r = row0 + LANE * lane, rows_left = p.rows - r;
  float f[LANE];
#pragma unroll
  for (int h = 0; h < LANE; ++h) f[h] = h < rows_left ? scale_value(scales[mx_scale_at(r + h, slab, p.slabs) + part * C::WAVES + wave]) : 0.0f;
#pragma unroll
  for (int u = 0; u < C::ROWS * C::CHUNKS / C::THREADS; ++u) {
    const int i = u * C::THREADS + tid, row = i / C::CHUNKS, chunk = i % C::CHUNKS;
    if (row0 + row < p.rows)
      *(i32x4*)(tile + row * C::PITCH + chunk * 16) = *(const i32x4*)(codes + ((row0 + row) * p.slabs + slab) * MX_ROWB + (part * C::CHUNKS + chunk) * 16);
  }
  __syncthreads();
  if (rows_left <= 0 || left <= 0) return;
  raw* d = dst + k0 * p.stride_k + r * p.stride_r;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    float v[LANE][8];
#pragma unroll
    for (int h = 0; h < LANE; ++h)                       // (rows past the end: what LDS holds, times 0, and not stored)
      values8(*(const uint32_t*)(tile + (LANE * lane + h) * C::PITCH + wave * 16 + q * 4), f[h], v[h]);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int i = q * 8 + e;
      if (i >= left) continue;
      if (RUNS && rows_left >= LANE) {
        RunC<T, LANE> t;
#pragma unroll
        for (int h = 0; h < LANE; ++h) t.v[h] = Elem<T>::put(v[h][e]);
        typedef i32x2 __attribute__((aligned(2))) loose2;
        typedef int __attribute__((aligned(2))) loose1;
        if constexpr (C::WORDS == 2) {
          i32x2 w;
          __builtin_memcpy(&w, &t, 8);
          __builtin_nontemporal_store(w, (loose2*)(d + i * p.stride_k));
        } else {
          int w;
          __builtin_memcpy(&w, &t, 4);
          __builtin_nontemporal_store(w, (loose1*)(d + i * p.stride_k));
        }
      } else {
#pragma unroll
        for (int h = 0; h < LANE; ++h)
          if (h < rows_left) d[i * p.stride_k + h * p.stride_r] = Elem<T>::put(v[h][e]);
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

// Whether the wide shape has a workgroup for every CU, or for every other of float32, whose lanes have half the work.  (Quantising, small and wide: bfloat16 3000 x 2001,
// 96 workgroups, 6.3 and 9.1 us, 4096 x 4096, 256 of them, 10.3 and 10.2; float32 1024 x 2048, 64, 4.1 and 4.8, 2048 x 2048, 128, 5.8 and 5.3.  The way back
// takes the same shape.)
template <class T> bool columns_wide(int64_t rows, const QuantParams& p) {
  typedef Columns<T, true> C;
  return (rows + C::ROWS - 1) / C::ROWS * p.slabs * p.batch >= 64 * C::LANE;
}

template <class C> bool columns_grid(int64_t rows, const QuantParams& p, dim3* grid) {
  const int64_t tiles = (rows + C::ROWS - 1) / C::ROWS, parts = p.slabs * C::PARTS;
  *grid = dim3((unsigned)tiles, (unsigned)parts, (unsigned)p.batch);
  return tiles <= 0x7fffff && parts <= 65535;
}

template <class T, bool BACK, bool WIDE> int launch_columns(const QuantParams& p, hipStream_t stream) {
  typedef Columns<T, WIDE> C;
  dim3 grid;
  if (!columns_grid<C>(p.rows, p, &grid)) return TNX_E_UNSUPPORTED;
  const bool runs = p.stride_r == 1;
  if (BACK && runs) hipLaunchKernelGGL((dequantize_columns_kernel<T, WIDE, true>), grid, dim3(C::THREADS), 0, stream, p);
  else if (BACK) hipLaunchKernelGGL((dequantize_columns_kernel<T, WIDE, false>), grid, dim3(C::THREADS), 0, stream, p);
  else if (runs) hipLaunchKernelGGL((quantize_columns_kernel<T, WIDE, true, false>), grid, dim3(C::THREADS), 0, stream, p);
  else hipLaunchKernelGGL((quantize_columns_kernel<T, WIDE, false, false>), grid, dim3(C::THREADS), 0, stream, p);
  return mx_launched();
}

// both quantisations; p: the matrix's columns, neighbours in memory.  (Whole slabs of the rows too: the padding of the other tensor)
template <class T, bool WIDE> int launch_both(const QuantParams& p, hipStream_t stream) {
  typedef Columns<T, WIDE> C;
  dim3 grid;
  if (!columns_grid<C>(mx_slabs(p.rows) * MX_SLAB, p, &grid)) return TNX_E_UNSUPPORTED;
  hipLaunchKernelGGL((quantize_columns_kernel<T, WIDE, true, true>), grid, dim3(C::THREADS), 0, stream, p);
  return mx_launched();
}
template <class T> int launch_both(const QuantParams& p, hipStream_t stream) {
  return columns_wide<T>(p.rows, p) ? launch_both<T, true>(p, stream) : launch_both<T, false>(p, stream);
}

template <class T, bool BACK> int launch(const QuantParams& p, hipStream_t stream) {
  if (p.stride_k == 1) {
    const int64_t per_block = 256 * (BACK ? BACK_RUNS : QUANT_RUNS), runs = p.rows * p.slabs * (BACK && sizeof(typename Elem<T>::raw) == 4 ? 64 : 32);
    const int64_t blocks = (runs + per_block - 1) / per_block;
    if (blocks > 0x7fffffff) return TNX_E_UNSUPPORTED;
    const dim3 grid((unsigned)blocks, (unsigned)p.batch);
    if (BACK) hipLaunchKernelGGL((dequantize_rows_kernel<T>), grid, dim3(256), 0, stream, p);
    else if (sizeof(typename Elem<T>::raw) == 2 && p.batch * p.rows * p.k > (256 << 20) / 2) hipLaunchKernelGGL((quantize_rows_kernel<T, true>), grid, dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((quantize_rows_kernel<T, false>), grid, dim3(256), 0, stream, p);
    return mx_launched();
  }
  return columns_wide<T>(p.rows, p) ? launch_columns<T, BACK, true>(p, stream) : launch_columns<T, BACK, false>(p, stream);
}

void fill(const tnx_mx_args* a, QuantParams* p) {
  p->src = (const uint8_t*)a->data;
  p->dst = (uint8_t*)a->data;
  p->codes = (uint8_t*)a->codes;
  p->scales = (uint8_t*)a->scales;
  p->rows = a->rows; p->k = a->k; p->slabs = mx_slabs(a->k); p->batch = a->batch;
  p->stride_b = a->stride_batch; p->stride_r = a->stride_row; p->stride_k = a->k == 1 ? 1 : a->stride_k;
  p->codes_b = mx_code_bytes(a->rows, a->k);
  p->scales_b = mx_scale_bytes(a->rows, a->k);
  p->codes2 = p->scales2 = nullptr;
}

template <bool BACK> int convert(const tnx_mx_args* a) {
  if (!a || a->rows < 0 || a->k < 0 || a->batch < 0) return TNX_E_INVALID;
  if (a->rows == 0 || a->k == 0 || a->batch == 0) return TNX_OK;
  if (!a->data || !a->codes || !a->scales || ((uintptr_t)a->codes & 15) || ((uintptr_t)a->scales & 15)) return TNX_E_INVALID;
  if (a->k > TNX_MX_MAX_K || a->batch > 65535) return TNX_E_UNSUPPORTED;
  const unsigned size = a->dtype == TNX_F32 ? 4 : 2;
  if ((uintptr_t)a->data & (size - 1)) return TNX_E_INVALID;
  QuantParams p;
  fill(a, &p);
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
extern "C" int tnx_mx_quantize_both(const tnx_mx_args* a, void* codes2, void* scales2) {
  if (!a || a->batch != 1 || a->rows < 0 || a->k < 0) return TNX_E_INVALID;
  if (a->rows == 0 || a->k == 0) return TNX_OK;
  if (!codes2 || !scales2 || ((uintptr_t)codes2 & 15) || ((uintptr_t)scales2 & 15)) return TNX_E_INVALID;
  if (a->rows > TNX_MX_MAX_K) return TNX_E_UNSUPPORTED;
  tnx_mx_args other = *a;                                // the same matrix with the parts of its two dimensions exchanged
  other.codes = codes2; other.scales = scales2;
  other.rows = a->k; other.k = a->rows;
  other.stride_row = a->stride_k; other.stride_k = a->stride_row;
  const bool along = a->stride_k == 1 && a->rows > 1 && a->k > 1;      // k is the contiguous one: the columns are the other tensor's
  const tnx_mx_args *columns = along ? &other : a, *rows = along ? a : &other;
  if (columns->stride_row != 1 || columns->rows == 1 || columns->k == 1) {       // neither is, or a vector
    const int status = tnx_mx_quantize(a);
    return status != TNX_OK ? status : tnx_mx_quantize(&other);
  }
  if (!a->data || !a->codes || !a->scales || ((uintptr_t)a->codes & 15) || ((uintptr_t)a->scales & 15)) return TNX_E_INVALID;
  if (a->k > TNX_MX_MAX_K) return TNX_E_UNSUPPORTED;
  if ((uintptr_t)a->data & (a->dtype == TNX_F32 ? 3 : 1)) return TNX_E_INVALID;
  QuantParams p;
  fill(columns, &p);
  p.codes2 = (uint8_t*)rows->codes;
  p.scales2 = (uint8_t*)rows->scales;
  const hipStream_t stream = (hipStream_t)a->stream;
  switch (a->dtype) {
    case TNX_BF16: return launch_both<__bf16>(p, stream);
    case TNX_F16: return launch_both<_Float16>(p, stream);
    case TNX_F32: return launch_both<float>(p, stream);
    default: return TNX_E_UNSUPPORTED;
  }
}
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
