// Layer normalisation: y = (x - mean) rstd weight + bias by rows, and its gradients.
//
//   unit = (x - mean) rstd,  g = dy weight
//   dx = rstd (g - mean(g) - unit mean(g unit)),  dweight = sum over rows of dy unit,  dbias = sum over rows of dy
//
// Bound by memory: forward reads x and writes y, backward reads x and dy and writes dx.  A row is read once, into registers (16-byte runs,
// one after another over the threads), the mean before the variance from the same registers: no difference of large squares.  16384 x 8192
// bf16: 107 us (5.0 TB/s; a copy reaches 5.1), backward 182 (4.4 TB/s, 5 of them for the parameters' shares).  In the backward pass a workgroup
// keeps its rows' share of dweight and dbias, in 32 bits per column, and a second launch adds the workgroups' shares up in order.
#include <hip/hip_runtime.h>

#include "../../include/tritonix_hip.h"
#include "registry.h"
#include "gemm_linear.h"

using namespace tnx;

namespace {

struct NormParams {
  const uint8_t *x, *weight, *bias, *dy;
  uint8_t *y, *dx;
  float *mean, *rstd;
  float* parts;                  // backward: [workgroups][2][n], or null where neither weight nor bias asks
  int64_t rows, n, stride_x, stride_dy;
  int weight_dtype, bias_dtype;
  float eps;
  int block;                     // rows of a workgroup that sums columns alone
};


// the sum over 2, 4, 8, 16, 32 or 64 neighbouring lanes, in each of them, without LDS: exchanges within a row of 16 lanes (from 4 on mirrored,
// which is the same once the smaller groups agree), then of rows and of halves
template <int L> __device__ __forceinline__ float lanes_sum(float v) {
  auto with = [&](int other) __attribute__((always_inline)) { v += __builtin_bit_cast(float, other); };
  const auto bits = [&]() __attribute__((always_inline)) { return __builtin_bit_cast(int, v); };
  if constexpr (L >= 2) with(__builtin_amdgcn_update_dpp(0, bits(), 0xB1, 0xF, 0xF, true));
  if constexpr (L >= 4) with(__builtin_amdgcn_update_dpp(0, bits(), 0x4E, 0xF, 0xF, true));
  if constexpr (L >= 8) with(__builtin_amdgcn_update_dpp(0, bits(), 0x141, 0xF, 0xF, true));
  if constexpr (L >= 16) with(__builtin_amdgcn_update_dpp(0, bits(), 0x140, 0xF, 0xF, true));
  if constexpr (L >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap((unsigned)bits(), (unsigned)bits(), false, false);
    const unsigned one = r[0], other = r[1];             // (__builtin_bit_cast of a vector's element reads its first)
    v = __builtin_bit_cast(float, one) + __builtin_bit_cast(float, other);
  }
  if constexpr (L >= 64) {
    const auto r = __builtin_amdgcn_permlane32_swap((unsigned)bits(), (unsigned)bits(), false, false);
    const unsigned one = r[0], other = r[1];             // (__builtin_bit_cast of a vector's element reads its first)
    v = __builtin_bit_cast(float, one) + __builtin_bit_cast(float, other);
  }
  return v;
}

// Sums over the TPR threads of a row of NS values; every thread gets them.  TPR is a part of a wave, a wave or the whole workgroup.  `slot` alternates from call
// to call, so that one barrier does.  The waves' sums are read a lane each and added up over lanes: read by every thread in turn they took 64
// registers of 16 waves' four sums (16384 x 8192 bf16 backward: 1142 us, now 182).
template <int TPR, int NS> __device__ __forceinline__ void row_sums(float (&v)[NS], float* lds, int slot) {
#pragma unroll
  for (int s = 0; s < NS; ++s) v[s] = lanes_sum<(TPR < 64 ? TPR : 64)>(v[s]);
  if constexpr (TPR > 64) {
    constexpr int W = TPR / 64;
    float* at = lds + slot * W * NS;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int s = 0; s < NS; ++s) at[(threadIdx.x >> 6) * NS + s] = v[s];
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < NS; ++s) v[s] = lanes_sum<W>(at[(threadIdx.x & (W - 1)) * NS + s]);
  }
}

// V columns as they lie in memory, `cols` of which exist; past the row's end zeros.  WHOLE: all or none, since n is a multiple of V.  A run that is cut off
// is the end of the 16 bytes that end with the row, shifted down (9613 x 4082 f16 forward 33.7 us by elements, 28.9 so; the backward pass of float32 and of
// 1024 threads has no registers for it: 9613 x 6002 bf16 110 us by elements, 128 so); where it is the row's first (`first`: the row is shorter than a run) it
// is loaded by elements.
template <class O, bool WHOLE, bool SHIFT = true> __device__ __forceinline__ i32x4 load_packed(const typename O::raw* src, int cols, bool first) {
  typedef typename O::raw raw;
  constexpr int V = 16 / sizeof(raw);
  if (WHOLE) return cols ? *(const i32x4_loose*)src : i32x4{0, 0, 0, 0};
  i32x4 v = {0, 0, 0, 0};
  auto elements = [&]() __attribute__((always_inline)) {
    raw e[V];
#pragma unroll
    for (int x = 0; x < V; ++x) e[x] = x < cols ? src[x] : (raw)0;
    __builtin_memcpy(&v, e, 16);
    return v;
  };
  if (!SHIFT) return cols == V ? (i32x4)*(const i32x4_loose*)src : elements();
  if (cols == V || (cols > 0 && !first)) {
    v = *(const i32x4_loose*)(src + cols - V);
    if (cols < V) v = __builtin_bit_cast(i32x4, __builtin_bit_cast(unsigned __int128, v) >> ((V - cols) * 8 * (int)sizeof(raw)));
  } else if (cols > 0) {
    elements();
  }
  return v;
}
template <class O, int V> __device__ __forceinline__ void unpack(i32x4 v, float (&f)[V]) {
  typename O::raw e[V];
  __builtin_memcpy(e, &v, 16);
#pragma unroll
  for (int x = 0; x < V; ++x) f[x] = Run<O, V>::widen(e[x]);
}
template <class O, int V, bool WHOLE = false, bool SHIFT = true> __device__ __forceinline__ void load_run(const typename O::raw* src, int cols, bool first, float (&f)[V]) {
  unpack<O, V>(load_packed<O, WHOLE, SHIFT>(src, cols, first), f);
}
template <class O, int V, bool WHOLE = false, bool SHIFT = true> __device__ __forceinline__ void store_run(typename O::raw* dst, int cols, const float (&f)[V]) {
  typedef typename O::raw raw;
  raw e[V];
#pragma unroll
  for (int x = 0; x < V; ++x) e[x] = O::cvt(f[x]);
  if (WHOLE && cols == 0) return;
  if (WHOLE || cols == V) {
    i32x4 v;
    __builtin_memcpy(&v, e, 16);
    *(i32x4_loose*)dst = v;
  } else if (!SHIFT) {
#pragma unroll
    for (int x = 0; x < V; ++x)
      if (x < cols) dst[x] = e[x];
  } else {
    // in pieces of half a run, a quarter and, of 16 bits, an eighth
    struct __attribute__((packed, aligned(2))) Eight { uint64_t v; };
    struct __attribute__((packed, aligned(2))) Four { uint32_t v; };
    uint64_t half[2];
    __builtin_memcpy(half, e, 16);
    uint64_t left = half[0];
    if (cols & V / 2) {
      ((Eight*)dst)->v = left;
      left = half[1];
      dst += V / 2;
    }
    if (cols & V / 4) {
      ((Four*)dst)->v = (uint32_t)left;
      left >>= 32;
      dst += V / 4;
    }
    if (V == 8 && cols & 1) *(uint16_t*)dst = (uint16_t)left;
  }
}

// V columns of weight or bias, of the rows' type or float32; null: `none` throughout
template <class O, int V, bool WHOLE = false, bool SHIFT = true> __device__ __forceinline__ void load_param(const uint8_t* p, int dtype, int64_t col, int cols, float none, float (&f)[V]) {
  if (!p) {
#pragma unroll
    for (int x = 0; x < V; ++x) f[x] = none;
  } else if (dtype != DT_F32) {
    load_run<O, V, WHOLE, SHIFT>((const typename O::raw*)p + col, cols, col == 0, f);
  } else {
    const float* src = (const float*)p + col;
#pragma unroll
    for (int h = 0; h < V / 4; ++h) {
      float q[4];
      load_run<OutF32, 4, WHOLE, SHIFT>(src + 4 * h, cols - 4 * h >= 4 ? 4 : cols - 4 * h > 0 ? cols - 4 * h : 0, col + h == 0, q);
#pragma unroll
      for (int x = 0; x < 4; ++x) f[4 * h + x] = q[x];
    }
  }
}

// TPR threads to a row, each with up to CH runs of V columns
template <class O, int TPR, int CH, bool WHOLE> __global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void norm_kernel(NormParams p) {
  typedef typename O::raw raw;
  constexpr int V = 16 / sizeof(raw), THREADS = TPR < 256 ? 256 : TPR;
  __shared__ float lds[2 * THREADS / 64];
  const int t = threadIdx.x % TPR;
  const int64_t row = (int64_t)blockIdx.x * (THREADS / TPR) + threadIdx.x / TPR;
  if (row >= p.rows) return;                             // (all lanes of a row together, and no sum leaves a row's lanes; with TPR = THREADS whole workgroups)
  const raw* src = (const raw*)p.x + row * p.stride_x;
  float f[CH][V];
  float s[1] = {0.0f};
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int64_t col = (int64_t)(c * TPR + t) * V, left = p.n - col;
    load_run<O, V, WHOLE>(src + (left > 0 ? col : 0), left >= V ? V : left > 0 ? (int)left : 0, col == 0, f[c]);
#pragma unroll
    for (int e = 0; e < V; ++e) s[0] += f[c][e];
  }
  row_sums<TPR, 1>(s, lds, 0);
  const float mean = s[0] / (float)p.n;
  float q[1] = {0.0f};
#pragma unroll
  for (int c = 0; c < CH; ++c)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float d = f[c][e] - mean;
      q[0] += (c * TPR + t) * V + (WHOLE ? 0 : e) < (int)p.n ? d * d : 0.0f;
    }
  row_sums<TPR, 1>(q, lds, 1);
  const float rstd = 1.0f / sqrtf(q[0] / (float)p.n + p.eps);
  if (p.mean && t == 0) {
    p.mean[row] = mean;
    p.rstd[row] = rstd;
  }
  raw* dst = (raw*)p.y + row * p.n;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int64_t col = (int64_t)(c * TPR + t) * V, left = p.n - col;
    if (left <= 0) break;
    const int cols = left >= V ? V : (int)left;
    float w[V], b[V];
    load_param<O, V, WHOLE>(p.weight, p.weight_dtype, col, cols, 1.0f, w);
    load_param<O, V, WHOLE>(p.bias, p.bias_dtype, col, cols, 0.0f, b);
#pragma unroll
    for (int e = 0; e < V; ++e) f[c][e] = (f[c][e] - mean) * rstd * w[e] + b[e];
    store_run<O, V, WHOLE>(dst + col, cols, f[c]);
  }
}

// A workgroup walks over rows, R of them at a step (one barrier for their sums; two where a workgroup is alone on its CU or the
// values are few: 16384 x 8192 bf16 214 us with one, 182 with two, float32 65536 x 1024 172 and 154; elsewhere two spill); x and dy of these and of the next R are in registers as they
// lie in memory (widened twice: for the sums, then for dx), which leaves room for two sums per column and lets the loads run ahead of the
// barrier.  Columns past the row's end are zeros in dy and weight and so add nothing.
template <class O, int TPR, int CH, bool PARTS, bool WHOLE> __global__ __launch_bounds__(TPR < 128 ? 256 : TPR, 4) void norm_backward_kernel(NormParams p) {
  typedef typename O::raw raw;
  constexpr int V = 16 / sizeof(raw), THREADS = TPR < 128 ? 256 : TPR, LINES = THREADS / TPR, R = CH == 1 && (V == 4 || TPR == 1024) ? 2 : 1;
  constexpr bool AHEAD = CH <= 2, SHIFT = V == 8 && TPR < 1024;
  __shared__ float lds[2 * 2 * R * THREADS / 64];
  const int t = threadIdx.x % TPR, line = threadIdx.x / TPR;
  float dw[PARTS ? CH : 1][V], db[PARTS ? CH : 1][V];
  int cols[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int64_t left = p.n - (int64_t)(c * TPR + t) * V;
    cols[c] = left >= V ? V : left > 0 ? (int)left : 0;
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (PARTS) dw[c][e] = db[c][e] = 0.0f;
  }
  i32x4 x[R][CH], g[R][CH];
  float mean[R], rstd[R];
  const int64_t step = (int64_t)gridDim.x * LINES;       // from one of a line's rows to its next
  auto fetch = [&](int64_t first, i32x4 (&fx)[R][CH], i32x4 (&fg)[R][CH], float (&fmean)[R], float (&frstd)[R]) __attribute__((always_inline)) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = first + r * step;
      const bool there = row < p.rows;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const int64_t at = cols[c] ? (int64_t)(c * TPR + t) * V : 0;
        const int count = there ? cols[c] : 0;
        fx[r][c] = load_packed<O, WHOLE, SHIFT>((const raw*)p.x + (there ? row : 0) * p.stride_x + at, count, at == 0);
        fg[r][c] = load_packed<O, WHOLE, SHIFT>((const raw*)p.dy + (there ? row : 0) * p.stride_dy + at, count, at == 0);
      }
      fmean[r] = there ? p.mean[row] : 0.0f;
      frstd[r] = there ? p.rstd[row] : 0.0f;
    }
  };
  int64_t row = (int64_t)blockIdx.x * LINES + line;
  const float share = 1.0f / (float)p.n;
  int slot = 0;
  if (AHEAD && row < p.rows) fetch(row, x, g, mean, rstd);
  for (; row < p.rows; row += R * step) {                // (a wave's own rows; with TPR = THREADS the workgroup's)
    i32x4 nx[R][CH], ng[R][CH];
    float nmean[R] = {}, nrstd[R] = {};
    if (!AHEAD) fetch(row, x, g, mean, rstd);
    else if (row + R * step < p.rows) fetch(row + R * step, nx, ng, nmean, nrstd);
    float s[2 * R];
#pragma unroll
    for (int i = 0; i < 2 * R; ++i) s[i] = 0.0f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      float w[V];
      load_param<O, V, WHOLE, SHIFT>(p.weight, p.weight_dtype, cols[c] ? (int64_t)(c * TPR + t) * V : 0, cols[c], 1.0f, w);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float u[V], d[V];
        unpack<O, V>(x[r][c], u);
        unpack<O, V>(g[r][c], d);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          u[e] = (u[e] - mean[r]) * rstd[r];
          if (PARTS) {
            dw[c][e] += d[e] * u[e];
            db[c][e] += d[e];
          }
          d[e] *= w[e];
          s[2 * r] += d[e];
          s[2 * r + 1] += d[e] * u[e];
        }
      }
    }
    if (p.dx) {
      row_sums<TPR, 2 * R>(s, lds, slot);
      slot ^= 1;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        float w[V];
        load_param<O, V, WHOLE, SHIFT>(p.weight, p.weight_dtype, cols[c] ? (int64_t)(c * TPR + t) * V : 0, cols[c], 1.0f, w);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          float u[V], d[V];
          asm("" : "+v"(x[r][c]), "+v"(g[r][c]));         // (widened again, not kept wide since the sums)
          unpack<O, V>(x[r][c], u);
          unpack<O, V>(g[r][c], d);
          const float a = s[2 * r] * share, b = s[2 * r + 1] * share;
#pragma unroll
          for (int e = 0; e < V; ++e) d[e] = rstd[r] * (d[e] * w[e] - a - (u[e] - mean[r]) * rstd[r] * b);
          if (cols[c] && (R == 1 || row + r * step < p.rows))
            store_run<O, V, WHOLE, SHIFT>((raw*)p.dx + (row + r * step) * p.n + (int64_t)(c * TPR + t) * V, cols[c], d);
        }
      }
    }
    if (AHEAD) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          x[r][c] = nx[r][c];
          g[r][c] = ng[r][c];
        }
        mean[r] = nmean[r];
        rstd[r] = nrstd[r];
      }
    }
  }
  if constexpr (PARTS) {
    // the workgroup's share: its lines meet in LDS, in order
    float* const out = p.parts + (int64_t)blockIdx.x * 2 * p.n;
    if constexpr (LINES > 1) {
      __shared__ float meet[LINES][2][CH * V * TPR];
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          meet[line][0][(c * TPR + t) * V + e] = dw[c][e];
          meet[line][1][(c * TPR + t) * V + e] = db[c][e];
        }
      __syncthreads();
      for (int i = threadIdx.x; i < 2 * CH * V * TPR; i += THREADS) {
        const int which = i / (CH * V * TPR), col = i % (CH * V * TPR);
        float sum = 0.0f;
#pragma unroll
        for (int l = 0; l < LINES; ++l) sum += meet[l][which][col];
        if (col < p.n) out[which * p.n + col] = sum;
      }
    } else {
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const int64_t col = (int64_t)(c * TPR + t) * V;
#pragma unroll
        for (int h = 0; h < V / 4; ++h) {
          const int left = cols[c] - 4 * h;
          float q[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) q[e] = dw[c][4 * h + e];
          store_run<OutF32, 4, WHOLE, SHIFT>(out + col + 4 * h, left >= 4 ? 4 : left > 0 ? left : 0, q);
#pragma unroll
          for (int e = 0; e < 4; ++e) q[e] = db[c][4 * h + e];
          store_run<OutF32, 4, WHOLE, SHIFT>(out + p.n + col + 4 * h, left >= 4 ? 4 : left > 0 ? left : 0, q);
        }
      }
    }
  }
}

// Rows longer than the registers hold: read again for each of the passes.  A workgroup of 1024 threads to a row, whose loads, reductions and stores take turns (2048 x 65536 bf16:
// 160 us forward, 3.4 TB/s of x and y once; 4096 x 32768, in registers by the same workgroups, 142).
template <class O, bool BACKWARD> __global__ __launch_bounds__(1024) void norm_long_kernel(NormParams p) {
  typedef typename O::raw raw;
  constexpr int V = 16 / sizeof(raw), TPR = 1024;
  __shared__ float lds[2 * 2 * 16];
  const int64_t row = blockIdx.x;
  const raw* src = (const raw*)p.x + row * p.stride_x;
  auto over = [&](auto f) __attribute__((always_inline)) {
    for (int64_t col = (int64_t)threadIdx.x * V; col < p.n; col += TPR * V) f(col, p.n - col >= V ? V : (int)(p.n - col));
  };
  if constexpr (!BACKWARD) {
    float s[1] = {0.0f}, q[1] = {0.0f}, f[V];
    over([&](int64_t col, int cols) __attribute__((always_inline)) {
      load_run<O, V>(src + col, cols, col == 0, f);
      for (int e = 0; e < V; ++e) s[0] += f[e];
    });
    row_sums<TPR, 1>(s, lds, 0);
    const float mean = s[0] / (float)p.n;
    over([&](int64_t col, int cols) __attribute__((always_inline)) {
      load_run<O, V>(src + col, cols, col == 0, f);
      for (int e = 0; e < V; ++e) q[0] += e < cols ? (f[e] - mean) * (f[e] - mean) : 0.0f;
    });
    row_sums<TPR, 1>(q, lds, 1);
    const float rstd = 1.0f / sqrtf(q[0] / (float)p.n + p.eps);
    if (p.mean && threadIdx.x == 0) {
      p.mean[row] = mean;
      p.rstd[row] = rstd;
    }
    over([&](int64_t col, int cols) __attribute__((always_inline)) {
      load_run<O, V>(src + col, cols, col == 0, f);
      float w[V], b[V];
      load_param<O, V>(p.weight, p.weight_dtype, col, cols, 1.0f, w);
      load_param<O, V>(p.bias, p.bias_dtype, col, cols, 0.0f, b);
      for (int e = 0; e < V; ++e) f[e] = (f[e] - mean) * rstd * w[e] + b[e];
      store_run<O, V>((raw*)p.y + row * p.n + col, cols, f);
    });
  } else {
    const float mean = p.mean[row], rstd = p.rstd[row];
    const raw* dy = (const raw*)p.dy + row * p.stride_dy;
    float s[2] = {0.0f, 0.0f}, u[V], g[V];
    auto both = [&](int64_t col, int cols) __attribute__((always_inline)) {
      load_run<O, V>(src + col, cols, col == 0, u);
      load_run<O, V>(dy + col, cols, col == 0, g);
      float w[V];
      load_param<O, V>(p.weight, p.weight_dtype, col, cols, 1.0f, w);
      for (int e = 0; e < V; ++e) {
        u[e] = e < cols ? (u[e] - mean) * rstd : 0.0f;
        g[e] *= w[e];
      }
    };
    over([&](int64_t col, int cols) __attribute__((always_inline)) {
      both(col, cols);
      for (int e = 0; e < V; ++e) {
        s[0] += g[e];
        s[1] += g[e] * u[e];
      }
    });
    row_sums<TPR, 2>(s, lds, 0);
    const float a = s[0] / (float)p.n, b = s[1] / (float)p.n;
    over([&](int64_t col, int cols) __attribute__((always_inline)) {
      both(col, cols);
      for (int e = 0; e < V; ++e) g[e] = rstd * (g[e] - a - u[e] * b);
      store_run<O, V>((raw*)p.dx + row * p.n + col, cols, g);
    });
  }
}

// dweight and dbias of such rows, and of those too long for a thread to keep its columns' sums too (sums_apart): a workgroup's 32 runs of columns down 32 to 256 rows (columns_rows), its 8 rows of
// threads meet in LDS.  x and dy are read a second time for them: 10 bytes an element of 16 bits where 6 would do (8192 x 16384 bf16 265 us backward, 160 at a copy's rate)
template <class O> __global__ __launch_bounds__(256) void norm_columns_kernel(NormParams p) {
  typedef typename O::raw raw;
  constexpr int V = 16 / sizeof(raw);
  __shared__ float sums[2][8][32 * V + 4];
  const int lane = threadIdx.x & 31, line = threadIdx.x >> 5;
  const int64_t col = ((int64_t)blockIdx.x * 32 + lane) * V, row0 = (int64_t)blockIdx.y * p.block, end = row0 + p.block < p.rows ? row0 + p.block : p.rows;
  const int cols = p.n - col >= V ? V : p.n > col ? (int)(p.n - col) : 0;
  float dw[V] = {}, db[V] = {};
  constexpr int AHEAD = 4;                                // rows of a thread whose loads are on their way together
  for (int64_t row = row0 + line; row < end && cols > 0; row += 8 * AHEAD) {
    i32x4 x[AHEAD], d[AHEAD];
    float mean[AHEAD], rstd[AHEAD];
#pragma unroll
    for (int r = 0; r < AHEAD; ++r) {
      const bool there = row + 8 * r < end;
      const int64_t at = there ? row + 8 * r : row;
      x[r] = load_packed<O, false>((const raw*)p.x + at * p.stride_x + col, cols, col == 0);
      d[r] = load_packed<O, false>((const raw*)p.dy + at * p.stride_dy + col, there ? cols : 0, col == 0);
      mean[r] = p.mean[at];
      rstd[r] = there ? p.rstd[at] : 0.0f;
    }
#pragma unroll
    for (int r = 0; r < AHEAD; ++r) {
      float u[V], g[V];
      unpack<O, V>(x[r], u);
      unpack<O, V>(d[r], g);
      if (row + 8 * r >= end) break;                      // (a row that is not there has no part, not even of a NaN)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        dw[e] += e < cols ? g[e] * (u[e] - mean[r]) * rstd[r] : 0.0f;
        db[e] += g[e];
      }
    }
  }
#pragma unroll
  for (int e = 0; e < V; ++e) {
    sums[0][line][lane * V + e] = dw[e];
    sums[1][line][lane * V + e] = db[e];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * 32 * V; i += 256) {
    const int which = i / (32 * V), c = i % (32 * V);
    const int64_t at = (int64_t)blockIdx.x * 32 * V + c;
    if (at >= p.n) continue;
    float s = 0.0f;
#pragma unroll
    for (int l = 0; l < 8; ++l) s += sums[which][l][c];
    p.parts[((int64_t)blockIdx.y * 2 + which) * p.n + at] = s;
  }
}

// out[c] = the sum of parts[i][c] in the order of i, from column `first` on: the first n columns are dweight, the others dbias
template <int ACROSS> __global__ __launch_bounds__(1024) void norm_parts_kernel(const float* parts, int64_t count, int64_t n, int64_t first, uint8_t* dweight, int weight_dtype,
                                                                                 uint8_t* dbias, int bias_dtype) {
  constexpr int LINES = 1024 / ACROSS;
  __shared__ float sums[LINES][ACROSS];
  const int lane = threadIdx.x % ACROSS, line = threadIdx.x / ACROSS;
  const int64_t col = first + (int64_t)blockIdx.x * ACROSS + lane;
  float s = 0.0f;
  if (col < 2 * n) {
#pragma unroll 8
    for (int64_t i = line; i < count; i += LINES) s += parts[i * 2 * n + col];
  }
  sums[line][lane] = s;
  __syncthreads();
  if (line == 0 && col < 2 * n) {
#pragma unroll
    for (int l = 1; l < LINES; ++l) s += sums[l][lane];
    if (col < n && dweight) store_out<float>(dweight, col, s, weight_dtype);
    if (col >= n && dbias) store_out<float>(dbias, col - n, s, bias_dtype);
  }
}

// Threads and runs of a row; 0: longer than the registers hold.  Several short rows share a wave (45231 x 67 f16: a wave to a row 24 us forward, 42
// backward, 16 lanes 9 and 23; 65536 x 128 bf16 22, 32 and 9, 23).
struct Shape {
  int tpr, ch;
};
Shape shape_of(const Shape* shapes, int count, int64_t n, int v) {
  for (int i = 0; i < count; ++i)
    if (n <= (int64_t)shapes[i].tpr * shapes[i].ch * v) return shapes[i];
  return {0, 0};
}
const Shape FORWARD[] = {{8, 1}, {16, 1}, {32, 1}, {64, 1}, {64, 2}, {64, 4}, {256, 2}, {256, 4}, {512, 4}, {1024, 4}};
const Shape BACKWARD[] = {{8, 1}, {16, 1}, {32, 1}, {64, 1}, {128, 1}, {256, 1}, {512, 1}, {1024, 1}, {1024, 2}, {1024, 4}};
#define TNX_NORM_FORWARD_SHAPES(DO) DO(8, 1) DO(16, 1) DO(32, 1) DO(64, 1) DO(64, 2) DO(64, 4) DO(256, 2) DO(256, 4) DO(512, 4) DO(1024, 4)
#define TNX_NORM_BACKWARD_SHAPES(DO) DO(8, 1) DO(16, 1) DO(32, 1) DO(64, 1) DO(128, 1) DO(256, 1) DO(512, 1) DO(1024, 1) DO(1024, 2) DO(1024, 4)
Shape forward_shape(int64_t n, int v) { return shape_of(FORWARD, sizeof FORWARD / sizeof *FORWARD, n, v); }
Shape backward_shape(int64_t n, int v) { return shape_of(BACKWARD, sizeof BACKWARD / sizeof *BACKWARD, n, v); }
// rows that a workgroup has at a time
int64_t lines_of(const Shape& s) { return s.tpr > 0 && s.tpr < 256 ? 256 / s.tpr : 1; }
int64_t backward_lines(const Shape& s) { return s.tpr > 0 && s.tpr < 128 ? 256 / s.tpr : 1; }
// more columns' sums than that a thread's registers do not hold: they are a launch of their own
bool sums_apart(const Shape& s, int v) { return s.tpr == 0 || s.ch * v > 8; }
// Workgroups of the backward pass.  Each costs a share of 8 n bytes, written and read, where a row of 16 bits costs 6 n: so 16 rows or
// more to a line where that leaves every CU a workgroup, and not more than run together.
int64_t groups_of(const tnx_norm_args* a, const Shape& s) {
  const int64_t lines = backward_lines(s), most = (a->rows + lines - 1) / lines, together = 256 * 16 / (s.tpr < 128 ? 4 : s.tpr / 64);
  int64_t groups = most / 16;
  groups = groups < 256 ? 256 : groups > together ? together : groups;
  return groups < most ? groups : most;
}
// Rows of a workgroup of the launch of their own: 256, fewer while CUs are left without one (874 x 11520 bf16: 256 rows, loaded one after another, 20.0 us, 64 rows by fours 8.6).
int columns_rows(const tnx_norm_args* a) {
  const int64_t span = a->dtype == TNX_F32 ? 128 : 256, across = (a->n + span - 1) / span;
  int rows = 256;
  while (rows > 32 && (a->rows + rows - 1) / rows * across < 512) rows /= 2;
  return rows;
}
int64_t shares_of(const tnx_norm_args* a) {
  const Shape s = backward_shape(a->n, a->dtype == TNX_F32 ? 4 : 8);
  return sums_apart(s, a->dtype == TNX_F32 ? 4 : 8) ? (a->rows + columns_rows(a) - 1) / columns_rows(a) : groups_of(a, s);
}

int check(const tnx_norm_args* a) {
  if (!a || a->rows < 0 || a->n < 0 || !(a->eps >= 0.0f)) return TNX_E_INVALID;
  if (a->dtype != TNX_F16 && a->dtype != TNX_BF16 && a->dtype != TNX_F32) return TNX_E_UNSUPPORTED;
  // (of a parameter's gradient too, which may be asked for where the parameter itself is not given)
  if (((a->weight || a->dweight) && a->weight_dtype != a->dtype && a->weight_dtype != TNX_F32) ||
      ((a->bias || a->dbias) && a->bias_dtype != a->dtype && a->bias_dtype != TNX_F32))
    return TNX_E_UNSUPPORTED;
  if (a->rows > 0x7fffffff || a->n > 0x3fffffff) return TNX_E_UNSUPPORTED;
  return TNX_OK;
}
NormParams params_of(const tnx_norm_args* a) {
  NormParams p;
  p.x = (const uint8_t*)a->x; p.weight = (const uint8_t*)a->weight; p.bias = (const uint8_t*)a->bias; p.dy = (const uint8_t*)a->dy;
  p.y = (uint8_t*)a->y; p.dx = (uint8_t*)a->dx;
  p.mean = a->mean; p.rstd = a->rstd;
  p.parts = nullptr;
  p.rows = a->rows; p.n = a->n; p.stride_x = a->stride_x; p.stride_dy = a->stride_dy;
  p.weight_dtype = a->weight_dtype; p.bias_dtype = a->bias_dtype;
  p.eps = a->eps;
  p.block = columns_rows(a);
  return p;
}
int launched() {
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess) { note_hip_error((int)err); return TNX_E_HIP; }
  return TNX_OK;
}

// One launch's rows: the threads of a grid are counted in 32 bits.
template <class O> int forward_rows(const NormParams& p, hipStream_t stream) {
  const Shape s = forward_shape(p.n, 16 / sizeof(typename O::raw));
  const unsigned grid = (unsigned)((p.rows + lines_of(s) - 1) / lines_of(s));
  const bool whole = p.n % (16 / sizeof(typename O::raw)) == 0;
#define TNX_NORM_FORWARD(TPR, CH)                                                                                       \
  if (s.tpr == TPR && s.ch == CH) {                                                                                     \
    if (whole) hipLaunchKernelGGL((norm_kernel<O, TPR, CH, true>), dim3(grid), dim3(TPR < 256 ? 256 : TPR), 0, stream, p); \
    else hipLaunchKernelGGL((norm_kernel<O, TPR, CH, false>), dim3(grid), dim3(TPR < 256 ? 256 : TPR), 0, stream, p);   \
    return launched();                                                                                                  \
  }
  TNX_NORM_FORWARD_SHAPES(TNX_NORM_FORWARD)
  hipLaunchKernelGGL((norm_long_kernel<O, false>), dim3((unsigned)p.rows), dim3(1024), 0, stream, p);
  return launched();
}

// 16 columns to a workgroup while 64 leave CUs without one (25953 x 978 bf16, 1024 shares: 64 columns 8.5 us, 16 columns 5.5).  In several launches where one has
// not threads for all columns: a grid's are counted in 32 bits.
void launch_parts(const NormParams& p, int64_t shares, const tnx_norm_args* a, hipStream_t stream) {
  const int across = 2 * p.n <= 64 * 128 ? 16 : 64;
  constexpr int64_t MOST = 0xffffffffll / 1024;
  for (int64_t first = 0; first < 2 * p.n; first += MOST * across) {
    const int64_t left = (2 * p.n - first + across - 1) / across;
    hipLaunchKernelGGL((across == 16 ? norm_parts_kernel<16> : norm_parts_kernel<64>), dim3((unsigned)(left < MOST ? left : MOST)), dim3(1024), 0, stream, p.parts, shares, p.n,
                       first, (uint8_t*)a->dweight, a->weight_dtype, (uint8_t*)a->dbias, a->bias_dtype);
  }
}

template <class O> int forward(NormParams p, hipStream_t stream) {
  constexpr int64_t MOST = (1 << 22) - 4, ES = sizeof(typename O::raw);       // of 1024 threads, if a row takes that many
  const int64_t at_once = p.n <= 64 * 4 * (16 / ES) ? MOST * 4 : MOST;
  for (int64_t left = p.rows; left > 0; left -= at_once) {
    p.rows = left < at_once ? left : at_once;
    if (const int status = forward_rows<O>(p, stream)) return status;
    p.x += p.rows * p.stride_x * ES;
    p.y += p.rows * p.n * ES;
    if (p.mean) {
      p.mean += p.rows;
      p.rstd += p.rows;
    }
  }
  return TNX_OK;
}

template <class O> int backward(const tnx_norm_args* a, NormParams p, hipStream_t stream) {
  const Shape s = backward_shape(p.n, 16 / sizeof(typename O::raw));
  const int64_t shares = shares_of(a);
  const bool wanted = a->dweight || a->dbias, whole = p.n % (16 / sizeof(typename O::raw)) == 0;
  constexpr int V = 16 / sizeof(typename O::raw);
  const bool apart = sums_apart(s, V);
  const unsigned grid = (unsigned)(s.tpr ? groups_of(a, s) : 0);
  if (s.tpr == 0 && p.dx) hipLaunchKernelGGL((norm_long_kernel<O, true>), dim3((unsigned)p.rows), dim3(1024), 0, stream, p);
#define TNX_NORM_BACKWARD(TPR, CH)                                                                                      \
  if (s.tpr == TPR && s.ch == CH && (p.dx || !apart)) {                                                                 \
    constexpr bool SUMS = CH * V <= 8;                                                                                  \
    const dim3 threads(TPR < 128 ? 256 : TPR);                                                                          \
    if (SUMS && wanted && whole) hipLaunchKernelGGL((norm_backward_kernel<O, TPR, CH, SUMS, true>), dim3(grid), threads, 0, stream, p);  \
    else if (SUMS && wanted) hipLaunchKernelGGL((norm_backward_kernel<O, TPR, CH, SUMS, false>), dim3(grid), threads, 0, stream, p);     \
    else if (whole) hipLaunchKernelGGL((norm_backward_kernel<O, TPR, CH, false, true>), dim3(grid), threads, 0, stream, p);       \
    else hipLaunchKernelGGL((norm_backward_kernel<O, TPR, CH, false, false>), dim3(grid), threads, 0, stream, p);       \
  }
  TNX_NORM_BACKWARD_SHAPES(TNX_NORM_BACKWARD)
  constexpr int SPAN = 32 * V;
  if (apart && wanted)
    hipLaunchKernelGGL((norm_columns_kernel<O>), dim3((unsigned)((p.n + SPAN - 1) / SPAN), (unsigned)shares), dim3(256), 0, stream, p);
  if (wanted)
    launch_parts(p, shares, a, stream);
  return launched();
}

}  // namespace

extern "C" int tnx_layer_norm(const tnx_norm_args* a) {
  const int st = check(a);
  if (st != TNX_OK) return st;
  if (a->rows == 0 || a->n == 0) return TNX_OK;
  if (!a->x || !a->y || !a->mean != !a->rstd) return TNX_E_INVALID;
  const NormParams p = params_of(a);
  const hipStream_t stream = (hipStream_t)a->stream;
  return a->dtype == TNX_BF16 ? forward<OutBF16>(p, stream) : a->dtype == TNX_F16 ? forward<OutF16>(p, stream) : forward<OutF32>(p, stream);
}

extern "C" size_t tnx_layer_norm_workspace_bytes(const tnx_norm_args* a) {
  return check(a) != TNX_OK || !(a->dweight || a->dbias) ? 0 : (size_t)shares_of(a) * 2 * a->n * 4;
}

extern "C" int tnx_layer_norm_backward(const tnx_norm_args* a) {
  const int st = check(a);
  if (st != TNX_OK) return st;
  if (a->n == 0 || (!a->dx && !a->dweight && !a->dbias) || (a->rows == 0 && !a->dweight && !a->dbias)) return TNX_OK;
  if (a->rows > 0 && (!a->x || !a->dy || !a->mean || !a->rstd)) return TNX_E_INVALID;
  const size_t need = tnx_layer_norm_workspace_bytes(a);
  if (need && (!a->workspace || a->workspace_bytes < need || ((uintptr_t)a->workspace & 15))) return TNX_E_WORKSPACE;
  if (shares_of(a) > 65535) return TNX_E_UNSUPPORTED;
  NormParams p = params_of(a);
  p.parts = (float*)a->workspace;
  const hipStream_t stream = (hipStream_t)a->stream;
  if (a->rows == 0) {                                     // sums of no rows
    launch_parts(p, 0, a, stream);
    return launched();
  }
  return a->dtype == TNX_BF16 ? backward<OutBF16>(a, p, stream) : a->dtype == TNX_F16 ? backward<OutF16>(a, p, stream) : backward<OutF32>(a, p, stream);
}
