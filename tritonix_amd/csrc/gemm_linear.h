// The tile kernels with a linear layer's epilogue: y = act(x w + bias) + residual, and z = x w + bias beside it where the backward
// pass will ask for it.
//
// y, z and residual are row-major without gaps.  The sums pass a wave's LDS strip in 32 bits and are read back row by row, eight
// neighbouring columns a lane (float32: four): there the bias is the lane's own for all its rows, and residual, z and y are 16-byte
// runs.  Each output is rounded once, from 32 bits.  Bound by what it moves: the residual is asked for a row-block ahead.
// 8192 x 4096 x 4096 bf16 with z and gelu_tanh 261 us, the product alone 217, y and z 27 at a copy's rate.
#pragma once
#include "activation.h"

namespace tnx {

struct LinearParts {
  const uint8_t* bias;       // [n] of bias_dtype, or null
  const uint8_t* residual;   // [m, n] of the output's type, or null
  uint8_t* z;                // [m, n] of the output's type, or null
  int bias_dtype, act;
};

// As PlainParams, in its 112 bytes: the outputs' rows have no gaps, the operands' pitches are below 2^31 elements.
struct LinearParams {
  const uint8_t* a;
  const uint8_t* b;
  uint8_t* c;
  uint8_t* ws;
  const uint8_t* bias;
  const uint8_t* residual;
  uint8_t* z;
  int32_t lda, ldb;
  int32_t m, n, k;
  int32_t group_m, split_k, split_tile0, ktiles_per_split;
  uint32_t mul_tiles, mul_group, mul_rows, mul_rows_last;
  uint32_t flags;            // PF_*, and the activation
};
static_assert(sizeof(LinearParams) == 112, "a longer argument list costs every launch 0.7 us");
constexpr uint32_t PF_ACT_SHIFT = 17;

inline bool linear_params(const GemmParams& p, const LinearParts& x, bool bt, int es, LinearParams* q) {
  PlainParams d;
  if (!plain_params(p, bt, false, es, &d)) return false;
  if (d.lda > 0x7fffffff || d.ldb > 0x7fffffff || p.scm != p.n || p.scn != 1 || p.atomic_reduce || p.batch > 1) return false;
  q->a = p.a; q->b = p.b; q->c = p.c; q->ws = p.ws;
  q->bias = x.bias; q->residual = x.residual; q->z = x.z;
  q->lda = (int32_t)d.lda; q->ldb = (int32_t)d.ldb;
  q->m = d.m; q->n = d.n; q->k = d.k;
  q->group_m = d.group_m; q->split_k = d.split_k; q->split_tile0 = d.split_tile0; q->ktiles_per_split = d.ktiles_per_split;
  q->mul_tiles = d.mul_tiles; q->mul_group = d.mul_group; q->mul_rows = d.mul_rows; q->mul_rows_last = d.mul_rows_last;
  q->flags = d.flags | (uint32_t)x.bias_dtype << PF_BIAS_SHIFT | (uint32_t)x.act << PF_ACT_SHIFT;
  return true;
}

// N neighbouring 16- or 32-bit floats in 32 bits
template <class O, int N> struct Run {
  typedef typename O::raw raw;
  static __device__ __forceinline__ float widen(raw v) {
    if constexpr (std::is_same<O, OutBF16>::value) return __builtin_bit_cast(float, (uint32_t)v << 16);
    else if constexpr (std::is_same<O, OutF16>::value) return (float)__builtin_bit_cast(_Float16, v);
    else return v;
  }
};

struct LinearFamily {
  static constexpr bool LINEAR = true, GROUPED = false, SUMS = false;
  template <bool> using params = LinearParams;

  template <class C, bool BT, bool AT> static __device__ __forceinline__ GemmParams expand(const LinearParams& q) {
    PlainParams d;
    d.a = q.a; d.b = q.b; d.c = q.c; d.ws = q.ws;
    d.lda = q.lda; d.ldb = q.ldb;
    d.scm = q.n; d.scn = 1;
    d.m = q.m; d.n = q.n; d.k = q.k;
    d.group_m = q.group_m; d.split_k = q.split_k; d.split_tile0 = q.split_tile0; d.ktiles_per_split = q.ktiles_per_split;
    d.mul_tiles = q.mul_tiles; d.mul_group = q.mul_group; d.mul_rows = q.mul_rows; d.mul_rows_last = q.mul_rows_last;
    d.flags = q.flags & ~PF_MANY;
    return expand_params<C, BT, AT>(d);
  }

  // One wave's part of a tile.  The loop over row-blocks is rolled and only the write to the strip picks its accumulators by the
  // block's number: the activation is there once, not once per row-block (five of them on eight values each, times eight).
  template <class C, class O, class ACC>
  static __device__ __forceinline__ void store(const LinearParams& q, ACC (&acc)[C::TM][C::TN], const GemmParams& p, uint32_t strip, int lane, int64_t gm0,
                                               int64_t gc0) {
    typedef typename O::raw raw;
    constexpr int MI = C::MI, NGRP = C::ACC_N / 4;
    constexpr int V = 16 / sizeof(raw);                   // columns of a lane
    constexpr int PITCH = C::WTN * 4 + 16;
    constexpr int CPRW = C::WTN / V;
    typedef RowPasses<MI, CPRW> RP;
    static_assert(PITCH <= EpiStage<C>::PITCH && C::WTN % V == 0, "strip too small");
    if (gm0 >= p.m) return;
    const int rows_left = p.m - gm0 < C::WTM ? (int)(p.m - gm0) : C::WTM;
    const int act = (int)(q.flags >> PF_ACT_SHIFT & 7u), bias_dtype = (int)(q.flags >> PF_BIAS_SHIFT & 7u);
    const uint32_t wbase = strip + (lane % MI) * PITCH + (lane / MI) * 16;
    raw* const y = (raw*)q.c;
    raw* const z = (raw*)q.z;
    const raw* const res = (const raw*)q.residual;
    typedef f32x4 acc4;

    int l_row[RP::NL], l_cols[RP::NL];
    uint32_t l_lds[RP::NL];
    int64_t l_at[RP::NL];
    float bias[RP::NL][V];
#pragma unroll
    for (int t = 0; t < RP::NL; ++t) {
      const int u = t * 64 + lane, row = u / CPRW, cc = u % CPRW;
      const int64_t col = gc0 + cc * V, left = p.n - col;
      const bool idle = MI * CPRW % 64 != 0 && row >= MI;
      l_row[t] = row;
      l_cols[t] = idle || left <= 0 ? 0 : left < V ? (int)left : V;
      l_lds[t] = strip + (idle ? MI - 1 : row) * PITCH + cc * (V * 4);
      l_at[t] = (gm0 + row) * p.n + col;
#pragma unroll
      for (int e = 0; e < V; ++e) bias[t][e] = 0.0f;
      if (q.bias) {
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (e < l_cols[t]) bias[t][e] = bias_value(q.bias, (int)(col + e), bias_dtype);
      }
    }
    auto fetch = [&](int i, i32x4 (&r)[RP::ITERS]) __attribute__((always_inline)) {
#pragma unroll
      for (int it = 0; it < RP::ITERS; ++it) {
        const int t = RP::EVEN ? 0 : it, step = RP::EVEN ? it * RP::RSTEP : 0;
        r[it] = i32x4{0, 0, 0, 0};
        if (l_row[t] >= rows_left - (i * MI + step) || l_cols[t] == 0) continue;
        const raw* src = res + l_at[t] + (int64_t)(i * MI + step) * p.n;
        if (l_cols[t] == V) {
          r[it] = *(const i32x4_loose*)src;
        } else {
          raw e[V];
#pragma unroll
          for (int x = 0; x < V; ++x) e[x] = x < l_cols[t] ? src[x] : (raw)0;
          __builtin_memcpy(&r[it], e, 16);
        }
      }
    };
    auto put = [&](raw* dst, int cols, const raw (&out)[V]) __attribute__((always_inline)) {
      if (cols == V) {
        i32x4 v;
        __builtin_memcpy(&v, out, 16);
        store16_stream_loose(dst, v);
      } else {
#pragma unroll
        for (int x = 0; x < V; ++x)
          if (x < cols) dst[x] = out[x];
      }
    };
    i32x4 r[RP::ITERS];
    if (res) fetch(0, r);
#pragma unroll 1
    for (int i = 0; i * MI < rows_left; ++i) {
#pragma unroll
      for (int ii = 0; ii < C::TM; ++ii) {
        if (ii != i) continue;
#pragma unroll
        for (int j = 0; j < C::TN; ++j)
#pragma unroll
          for (int g = 0; g < NGRP; ++g)
            *TNX_LDS(acc4, wbase + (j * MI + g * 8) * 4) =
                acc4{acc[ii][j][4 * g + 0], acc[ii][j][4 * g + 1], acc[ii][j][4 * g + 2], acc[ii][j][4 * g + 3]};
        // (branches that end alike are made one with an index into the accumulators, which then live in memory: 8192 x 4096 x 4096 1239 us instead of 273)
        asm volatile("; row-block %0" : : "i"(ii));
      }
      i32x4 now[RP::ITERS];
#pragma unroll
      for (int it = 0; it < RP::ITERS; ++it) now[it] = r[it];
      if (res && (i + 1) * MI < rows_left) fetch(i + 1, r);
#pragma unroll
      for (int it = 0; it < RP::ITERS; ++it) {
        const int t = RP::EVEN ? 0 : it, step = RP::EVEN ? it * RP::RSTEP : 0;
        float f[V];
#pragma unroll
        for (int x = 0; x < V / 4; ++x) {
          const i32x4 v = *TNX_LDS(i32x4, l_lds[t] + step * PITCH + 16 * x);
          __builtin_memcpy(&f[4 * x], &v, 16);
        }
        if (l_row[t] >= rows_left - (i * MI + step) || l_cols[t] == 0) continue;
        const int64_t at = l_at[t] + (int64_t)(i * MI + step) * p.n;
        raw out[V];
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] += bias[t][e];
        if (z) {
          // (rounded to the output's type, as y is: the backward pass takes the derivative there.  In 32 bits it would take dx and dw from 2.40e-3 to 2.34e-3 of their 2-norm (bf16, silu or gelu; the
          // rest is dz's rounding and their own), for twice the memory that a layer holds between its passes and, at a copy's rate, 13 us more in both passes of 8192 x 4096)
#pragma unroll
          for (int e = 0; e < V; ++e) out[e] = O::cvt(f[e]);
          put(z + at, l_cols[t], out);
        }
        if (act != ACT_NONE) {
#pragma unroll
          for (int e = 0; e < V; ++e) f[e] = activate(f[e], act);
        }
        if (res) {
          raw s[V];
          __builtin_memcpy(s, &now[it], 16);
#pragma unroll
          for (int e = 0; e < V; ++e) f[e] += Run<O, V>::widen(s[e]);
        }
#pragma unroll
        for (int e = 0; e < V; ++e) out[e] = O::cvt(f[e]);
        put(y + at, l_cols[t], out);
      }
    }
  }
};

constexpr int LINEAR_PAIR = 7;   // LinearEntry::dtype of the kernels on head and tail slabs of float32 operands
typedef hipError_t (*linear_fn)(const GemmParams& p, const LinearParts& x, unsigned grid, hipStream_t stream);
struct LinearEntry {
  int dtype, bm, bn, nw, stages;
  linear_fn nn, bt;           // row-major and k-contiguous w
};
struct LinearGroup {
  LinearEntry* entries;
  int count;
};

template <class T, class C, bool BT, bool PAIR> hipError_t launch_linear(const GemmParams& p, const LinearParts& x, unsigned grid, hipStream_t stream) {
  LinearParams q;
  if (!linear_params(p, x, BT, C::ES, &q)) return hipErrorInvalidValue;
  return launch_kernel((const void*)&gemm_tile_kernel<T, C, true, false, BT, false, false, false, PAIR, LinearFamily>, grid, C::THREADS, 0, stream, &q);
}

// tiles as the built-in choice names them, 128 bytes of k to a slab
#define TNX_LINEAR_ENTRY(TAG, ID, BM, BN, NW, ST, PAIR)                                                            \
  {ID, BM, BN, NW, ST, &launch_linear<TAG, TileCfg<TAG, BM, BN, 128 / TAG::ES, NW, ST>, false, PAIR>,              \
   &launch_linear<TAG, TileCfg<TAG, BM, BN, 128 / TAG::ES, NW, ST>, true, PAIR>}

}  // namespace tnx
