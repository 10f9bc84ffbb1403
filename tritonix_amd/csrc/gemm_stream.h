// Linear layers of few rows with a k-contiguous weight (the transpose of a row-major one): single tokens and small decode batches.
//
// Bound by reading the weight once, and a CU alone takes in little over 20 GB/s of it whatever its waves have in flight, so that all CUs have to
// read all the time: small blocks of columns, no step that waits for another workgroup.  A workgroup owns C columns (NT times, for more use of a
// row of x), its waves take turns along k, and the weight goes from memory straight into the registers that v_mfma_f32_16x16x32 reads: no LDS and no
// barrier in the loop.  Of the 16 rows and columns of a matrix instruction a block needs C columns of the weight and at most C rows; the 16 / C
// groups of them take different parts of k, and of the 16 x 16 sums the blocks on the diagonal count.  That narrows a workgroup without an idle lane
// among the loads, and a row's part of an instruction is 32 x 16 / C elements: from C = 8 on down whole lines of memory.  Rows of x come from the
// caches.  The waves' and groups' sums meet in LDS, in order, where the epilogue runs on them: one launch, no workspace, the same bits every time.
// bf16, cold weights, us: 1 x 4096 x 4096 7.7 (4.4 TB/s; the tile kernels, which cut k and hand slices over, 9.5), 1 x 14336 x 4096 19 to 21 (22),
// 1 x 16384 x 16384 78 (6.9 TB/s), 1 x 1000 x 704 3.1 (4.9), 8 x 1814 x 2752 5.5 (7.5).
#pragma once
#include "gemm_grouped.h"
#include "gemm_linear.h"

namespace tnx {

struct StreamParams {
  const uint8_t* x;
  const uint8_t* w;
  uint8_t* y;
  uint8_t* z;
  const uint8_t* bias;
  const uint8_t* residual;
  int64_t ldx, ldw;
  int32_t m, n, k;
  int32_t act, bias_dtype;
};
static_assert(sizeof(StreamParams) <= 112, "a longer argument list costs every launch 0.7 us");

// C: columns of the weight and rows of x at most; W: waves; U: steps of 64 x 16 / C of k in flight; LINES: rows of the weight begin on lines of memory,
// of which nothing is left for another instruction to read (float32: half of these numbers, and the binary32 instruction four times; with C = 8, us: 1 x 4096 x 4096 7.6 past the caches and 8.1 through them; rows that begin
// anywhere, 1 x 2050 x 4100 7.5 and 6.4).
template <class T, int C, int NT, int W, int U, bool LINES> __device__ __forceinline__ void stream_block(const StreamParams& p, int block) {
  typedef Mma<T, 16> MMA;
  typedef typename OutOf<T>::type O;
  typedef typename O::raw raw;
  constexpr int V = 16 / T::ES, G = 16 / C, HALF = 4 * V * G, STEP = 2 * HALF;
  __shared__ f32x4 sums[W][NT][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int li = lane & 15, kg = lane >> 4;
  const int n0 = block * (C * NT);
  const int koff = li / C * (4 * V) + kg * V;
  const raw* const xp = (const raw*)p.x + (int64_t)(li % C < p.m ? li % C : p.m - 1) * p.ldx + koff;
  const raw* wp[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int col = n0 + t * C + li % C;
    wp[t] = (const raw*)p.w + (int64_t)(col < p.n ? col : p.n - 1) * p.ldw + koff;      // (what does not exist is not stored)
  }
  f32x4 acc[NT][2] = {};
  const int whole = p.k / STEP;
  auto steps = [&](int s, auto count) __attribute__((always_inline)) {
    constexpr int N = decltype(count)::value;
    i32x4 b[N][NT][2], a[N][2];
#pragma unroll
    for (int u = 0; u < N; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const i32x4_loose* const at = (const i32x4_loose*)(wp[t] + (int64_t)(s + u * W) * STEP + h * HALF);
          b[u][t][h] = LINES ? (i32x4)__builtin_nontemporal_load(at) : (i32x4)*at;
        }
        a[u][h] = *(const i32x4_loose*)(xp + (int64_t)(s + u * W) * STEP + h * HALF);
      }
#pragma unroll
    for (int u = 0; u < N; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[t][h] = MMA::run(b[u][t][h], a[u][h], acc[t][h]);
  };
  int s = wave;
  for (; s + (U - 1) * W < whole; s += U * W) steps(s, std::integral_constant<int, U>());
  if constexpr (U > 2)
    if (s + W < whole) {
      steps(s, std::integral_constant<int, 2>());
      s += 2 * W;
    }
  for (; s < whole; s += W) steps(s, std::integral_constant<int, 1>());
  if (s == whole && whole * STEP < p.k) {
    // the wave whose turn it is takes the short last step: what lies past k is zero on both sides
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int64_t at = (int64_t)whole * STEP + h * HALF;
      const int left = p.k - (int)at - koff;
      auto fetch = [&](const raw* from) __attribute__((always_inline)) {
        i32x4 v = {};
        if (left >= V) return (i32x4)*(const i32x4_loose*)(from + at);
        raw e[V];
#pragma unroll
        for (int i = 0; i < V; ++i) e[i] = i < left ? from[at + i] : (raw)0;
        __builtin_memcpy(&v, e, 16);
        return v;
      };
      const i32x4 a = fetch(xp);
#pragma unroll
      for (int t = 0; t < NT; ++t) acc[t][h] = MMA::run(fetch(wp[t]), a, acc[t][h]);
    }
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) sums[wave][t][lane] = acc[t][0] + acc[t][1];
  __syncthreads();
  for (int o = threadIdx.x; o < p.m * C * NT; o += W * 64) {
    const int n = o % (C * NT), m = o / (C * NT);
    if (n0 + n >= p.n) continue;
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w)
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const int r = g * C + n % C;
        v += ((const float*)&sums[w][n / C][(r >> 2) * 16 + g * C + m])[r & 3];
      }
    const int64_t at = (int64_t)m * p.n + n0 + n;
    if (p.bias) v += bias_value(p.bias, n0 + n, p.bias_dtype);
    if (p.z) ((raw*)p.z)[at] = O::cvt(v);
    v = activate(v, p.act);
    if (p.residual) v += Run<O, V>::widen(((const raw*)p.residual)[at]);
    ((raw*)p.y)[at] = O::cvt(v);
  }
}

template <class T, int C, int NT, int W, int U, bool LINES> __global__ __launch_bounds__(W * 64) void gemm_stream_kernel(StreamParams p) {
  stream_block<T, C, NT, W, U, LINES>(p, xcd_remap(blockIdx.x, (p.n + C * NT - 1) / (C * NT), 8));
}

template <class T, int C, int NT, int W, int U, bool LINES> hipError_t stream_launch(const StreamParams& p, hipStream_t stream) {
  StreamParams q = p;
  return launch_kernel((const void*)&gemm_stream_kernel<T, C, NT, W, U, LINES>, (unsigned)((p.n + C * NT - 1) / (C * NT)), W * 64, 0, stream, &q);
}

// waves: 4 where k has no step for each of 8 (1 x 30000 x 512, us: 7.1 and 8.1)
template <class T, int C, int NT, int U, bool LINES> hipError_t stream_waves(const StreamParams& p, hipStream_t stream) {
  if (p.k < 8 * (128 / T::ES) * (16 / C)) return stream_launch<T, C, NT, 4, U, LINES>(p, stream);
  return stream_launch<T, C, NT, 8, U, LINES>(p, stream);
}

template <class T, int C, int NT, int U> hipError_t stream_lines(const StreamParams& p, hipStream_t stream) {
  if constexpr (C < 16)
    if (p.ldw % (128 / T::ES) == 0 && ((uintptr_t)p.w & 127) == 0) return stream_waves<T, C, NT, U, true>(p, stream);
  return stream_waves<T, C, NT, U, false>(p, stream);
}

// Columns of a workgroup: 4 while 8 give fewer than 512 workgroups (1 x 512 x 8192, us: 4.9 and 7.0; 1 x 4096 x 4096 8.7 and 7.6), which have room for
// 4 rows; 8 for up to 8 rows, in pairs of blocks where there are many rows and columns (8 x 4096 x 4096: 9.9, with pairs 9.2); 16 beyond.
template <class T> hipError_t stream_columns(const StreamParams& p, hipStream_t stream) {
  if (p.m <= 4 && p.n < 4096) return stream_lines<T, 4, 1, 4>(p, stream);
  if (p.m <= 8 && (p.m <= 4 || p.n < 4096)) return stream_lines<T, 8, 1, 4>(p, stream);
  if constexpr (T::ES == 2)
    if (p.m > 8) return stream_lines<T, 16, 1, 4>(p, stream);
  return stream_lines<T, 8, 2, 2>(p, stream);
}

// The same for a row-major weight, up to 8 rows.  A workgroup owns 64 columns (float32: 32; a line of memory of each row of the weight), a step is 64 of k: a lane
// reads 8 columns of 8 rows of the weight and picks the 8 numbers of a column together with v_perm_b32, half an instruction a number.  Column e of
// every lane makes one matrix instruction: 8 columns in two groups, as C = 8 above.  64 columns are few workgroups (narrower ones would leave parts of
// lines), so that `parts` of them share a block's k: each writes its sums through its L2, and the one that arrives last adds them up in the order of the parts.
// That costs 3 us, less than a CU's slow pace.  bf16, cold weights, us, against the tile kernels': 1 x 512 x 8192 6.5 and 8.2, 1 x 1024 x 8192 8.6 and 10.2,
// 8 x 128 x 4096 5.7 and 6.3.
struct StreamRowsParams {
  const uint8_t* x;
  const uint8_t* w;
  uint8_t* y;
  uint8_t* z;
  const uint8_t* bias;
  const uint8_t* residual;
  uint8_t* workspace;        // counters, all zero, then the parts' sums; null without parts
  int64_t ldx, ldw;
  int32_t m, n, k, parts;
  int32_t flags;             // activation | bias_dtype << 8
};
static_assert(sizeof(StreamRowsParams) <= 112, "a longer argument list costs every launch 0.7 us");

// APART: the sums of a part go to y as they are, in 32 bits, for a launch that adds them up.
template <class T, int W, int U, bool APART> __device__ __forceinline__ void stream_rows_block(const StreamRowsParams& p, int id) {
  typedef Mma<T, 16> MMA;
  typedef typename OutOf<T>::type O;
  typedef typename O::raw raw;
  constexpr int V = 16 / T::ES, COLUMNS = 8 * V, STEP = 8 * V;
  __shared__ f32x4 sums[W][V][32];
  __shared__ int arrived;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int li = lane & 15, octet = (li >> 3) * 4 + (lane >> 4), c = li & 7;
  const int tile = id / p.parts, part = id - tile * p.parts, n0 = tile * COLUMNS;
  // (the last run of columns begins where it ends with the row)
  const int col = n0 + c * V < p.n - V ? n0 + c * V : p.n - V;
  const raw* const xp = (const raw*)p.x + (int64_t)(c < p.m ? c : p.m - 1) * p.ldx + octet * V;
  const raw* const wp = (const raw*)p.w + (int64_t)(octet * V) * p.ldw + col;
  f32x4 acc[V] = {};
  auto multiply = [&](const i32x4 (&b)[V], i32x4 a) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      i32x4 v;
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        if constexpr (T::ES == 4) v[d] = b[d][e];
        else v[d] = (int)__builtin_amdgcn_perm((uint32_t)b[2 * d + 1][e / 2], (uint32_t)b[2 * d][e / 2], e & 1 ? 0x07060302u : 0x05040100u);
      }
      acc[e] = MMA::run(v, a, acc[e]);
    }
  };
  const int whole = p.k / STEP, turn = W * p.parts;
  auto steps = [&](int s, auto count) __attribute__((always_inline)) {
    constexpr int N = decltype(count)::value;
    i32x4 b[N][V], a[N];
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const raw* const from = wp + (int64_t)(s + u * turn) * STEP * p.ldw;
#pragma unroll
      for (int j = 0; j < V; ++j) b[u][j] = (i32x4)__builtin_nontemporal_load((const i32x4_loose*)(from + j * p.ldw));
      a[u] = *(const i32x4_loose*)(xp + (int64_t)(s + u * turn) * STEP);
    }
#pragma unroll
    for (int u = 0; u < N; ++u) multiply(b[u], a[u]);
  };
  int s = part * W + wave;
  for (; s + (U - 1) * turn < whole; s += U * turn) steps(s, std::integral_constant<int, U>());
  for (; s < whole; s += turn) steps(s, std::integral_constant<int, 1>());
  if (s == whole && whole * STEP < p.k) {
    const int left = p.k - whole * STEP - octet * V;
    i32x4 b[V], a = {};
#pragma unroll
    for (int j = 0; j < V; ++j) {
      b[j] = i32x4{0, 0, 0, 0};
      if (j < left) b[j] = *(const i32x4_loose*)(wp + ((int64_t)whole * STEP + j) * p.ldw);
    }
    const raw* const from = xp + (int64_t)whole * STEP;
    if (left >= V) a = *(const i32x4_loose*)from;
    else {
      raw e[V];
#pragma unroll
      for (int i = 0; i < V; ++i) e[i] = i < left ? from[i] : (raw)0;
      __builtin_memcpy(&a, e, 16);
    }
    multiply(b, a);
  }
  // rows 0 to 7 of the sums are the first group's columns, whose x is in columns 0 to 7, the others the second's
  if ((lane >> 5) == (li >> 3)) {
#pragma unroll
    for (int e = 0; e < V; ++e) sums[wave][e][(lane >> 4) * 8 + c] = acc[e];
  }
  __syncthreads();
  auto sum_of = [&](int o) __attribute__((always_inline)) {
    const int m = o / COLUMNS, cc = o / V % 8, e = o % V;
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w)
#pragma unroll
      for (int g = 0; g < 2; ++g) v += ((const float*)&sums[w][e][(g * 2 + (cc >> 2)) * 8 + m])[cc & 3];
    return v;
  };
  // the column of an output, or -1: not there, or another run's
  auto column_of = [&](int o) __attribute__((always_inline)) {
    const int own = n0 + o % COLUMNS / V * V, n = (own < p.n - V ? own : p.n - V) + o % V;
    return n >= own && own < p.n ? n : -1;
  };
  if constexpr (APART) {
    for (int o = threadIdx.x; o < p.m * COLUMNS; o += W * 64) {
      const int n = column_of(o);
      if (n >= 0) ((float*)p.y)[(int64_t)(o / COLUMNS) * p.n + n] = sum_of(o);
    }
    return;
  }
  float* const slab = p.workspace ? (float*)(p.workspace + WS_COUNTER_BYTES) + (int64_t)tile * p.parts * p.m * COLUMNS : nullptr;
  if (p.parts > 1) {
    for (int o = threadIdx.x; o < p.m * COLUMNS; o += W * 64)
      __hip_atomic_store(slab + (int64_t)part * p.m * COLUMNS + o, sum_of(o), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (threadIdx.x == 0) {
      int* const counter = (int*)p.workspace + tile;
      const int before = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      // the last arrival re-arms the counter for the next launch
      if (before == p.parts - 1) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      arrived = before;
    }
    __syncthreads();
    if (arrived != p.parts - 1) return;
  }
  const int act = p.flags & 255, bias_dtype = p.flags >> 8;
  for (int o = threadIdx.x; o < p.m * COLUMNS; o += W * 64) {
    const int m = o / COLUMNS, n = column_of(o);
    if (n < 0) continue;
    float v = 0.0f;
    if (p.parts > 1) {
#pragma unroll 8
      for (int q = 0; q < p.parts; ++q) v += __hip_atomic_load(slab + (int64_t)q * p.m * COLUMNS + o, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    } else {
      v = sum_of(o);
    }
    const int64_t at = (int64_t)m * p.n + n;
    if (p.bias) v += bias_value(p.bias, n, bias_dtype);
    if (p.z) ((raw*)p.z)[at] = O::cvt(v);
    v = activate(v, act);
    if (p.residual) v += Run<O, V>::widen(((const raw*)p.residual)[at]);
    ((raw*)p.y)[at] = O::cvt(v);
  }
}

template <class T, int W, int U> __global__ __launch_bounds__(W * 64) void gemm_stream_rows_kernel(StreamRowsParams p) {
  stream_rows_block<T, W, U, false>(p, xcd_remap(blockIdx.x, (p.n + 128 / T::ES - 1) / (128 / T::ES) * p.parts, 8));
}

// Workgroups to a block of columns: a step for each of their waves, and not more than two workgroups to a CU (1 x 512 x 8192: 8 parts 1.2 us more than 16).
constexpr int STREAM_ROWS_WAVES = 8;
inline int stream_rows_parts(int64_t n, int64_t k, int es) {
  const int64_t step = 128 / es, tiles = (n + step - 1) / step, most = k / (step * STREAM_ROWS_WAVES), room = 512 / tiles, parts = most < room ? most : room;
  return parts < 1 ? 1 : (int)parts;
}
inline size_t stream_rows_workspace(int64_t m, int64_t n, int64_t k, int es) {
  const int64_t columns = 128 / es, parts = stream_rows_parts(n, k, es);
  return parts > 1 ? WS_COUNTER_BYTES + (size_t)((n + columns - 1) / columns) * parts * m * columns * 4 : 0;
}

template <class T> hipError_t stream_rows(const StreamRowsParams& p, hipStream_t stream) {
  StreamRowsParams q = p;
  return launch_kernel((const void*)&gemm_stream_rows_kernel<T, STREAM_ROWS_WAVES, 2>, (unsigned)((p.n + 128 / T::ES - 1) / (128 / T::ES) * p.parts), STREAM_ROWS_WAVES * 64, 0, stream, &q);
}

// The k-contiguous one by groups of rows, a weight to each (gemm_grouped.h): 8 rows of a group at a time, for few rows in all or few to a group.  A workgroup
// finds its rows in the bounds, which are all that it waits for.  bf16, cold weights, us, against the tile kernels': 2 rows, 64 groups, 4096 x 2048 8.5 and 15.1,
// 4 rows, 128 groups, 2048 x 768 5.5 and 11.8, 16 rows, 64 groups, 4096 x 2048 38 and 40, 64 rows, 128 groups, 2048 x 768 27 and 37.
template <class T, int NT, int W, int U, bool LINES> __global__ __launch_bounds__(W * 64) void grouped_stream_kernel(GroupedParams q) {
  constexpr int ES = T::ES, COLUMNS = 8 * NT;
  const int across = (int)(((uint32_t)q.n + COLUMNS - 1) / COLUMNS), id = windowed<64>(blockIdx.x, gridDim.x), want = id / across, block = id - want * across;
  int total = 0;
  const GroupedFamily<false>::Stretch s = GroupedFamily<false>::stretch_of<8>(q, threadIdx.x & 63, want, &total);
  if (s.number < 0) return;
  const int skip = (want - s.before) * 8, m = s.rows - skip < 8 ? s.rows - skip : 8;
  const int64_t row = s.first + skip;
  uint8_t* const y = q.c + row * q.n * ES;
  if (s.number == 0 || s.number == q.groups + 1) {
    typedef typename OutOf<T>::type::raw raw;
    for (int o = threadIdx.x; o < m * COLUMNS; o += W * 64) {
      const int n = block * COLUMNS + o % COLUMNS;
      if (n < q.n) ((raw*)y)[(int64_t)(o / COLUMNS) * q.n + n] = 0;
    }
    return;
  }
  const uint8_t* const x = q.a + row * q.lda * ES;
  const uint8_t* const w = q.b + (int64_t)(s.number - 1) * q.group_stride * ES;
  stream_block<T, 8, NT, W, U, LINES>({x, w, y, nullptr, nullptr, nullptr, q.lda, q.ldb, m, q.n, q.k, ACT_NONE, 0}, block);
}

// the most runs of 8 rows that there can be
inline int64_t stream_runs(int64_t rows, int64_t groups) { return rows / 8 + (groups + 2 < rows ? groups + 2 : rows); }
template <class T, int NT, int W, int U> hipError_t grouped_stream_launch(const GroupedParams& p, hipStream_t stream) {
  GroupedParams q = p;
  const unsigned grid = (unsigned)(stream_runs(p.rows, p.groups) * ((p.n + 8 * NT - 1) / (8 * NT)));
  const bool lines = p.ldb % (128 / T::ES) == 0 && p.group_stride % (128 / T::ES) == 0 && ((uintptr_t)p.b & 127) == 0;
  if (lines) return launch_kernel((const void*)&grouped_stream_kernel<T, NT, W, U, true>, grid, W * 64, 0, stream, &q);
  return launch_kernel((const void*)&grouped_stream_kernel<T, NT, W, U, false>, grid, W * 64, 0, stream, &q);
}
// Columns and waves of a workgroup: blocks of 8 columns in pairs where workgroups are many and k is short, or where a group has two rows or more (us, single
// and in pairs: 64 rows, 128 groups, 2048 x 768 29 and 27, 128 rows, 64 groups, 4096 x 2048 141 and 131; 8 rows, 32 groups, 4096 x 4096 38 and 41); 8 waves
// for a long k (4 rows, 8 groups, 14336 x 4096: 4 waves 70, 8 waves 66; 4 rows, 128 groups, 2048 x 768 5.5 and 6.0).
template <class T> hipError_t grouped_stream(const GroupedParams& p, hipStream_t stream) {
  const int64_t used = p.rows < p.groups ? p.rows : p.groups;
  const bool pairs = p.rows >= 2 * (int64_t)p.groups || (p.k < 4096 && used * p.n > 16384);
  if (p.k >= 8192) return pairs ? grouped_stream_launch<T, 2, 8, 2>(p, stream) : grouped_stream_launch<T, 1, 8, 4>(p, stream);
  return pairs ? grouped_stream_launch<T, 2, 4, 4>(p, stream) : grouped_stream_launch<T, 1, 4, 4>(p, stream);
}

// Row-major weights of a few groups, in parts of k whose sums another launch adds up.
template <class T> __global__ __launch_bounds__(STREAM_ROWS_WAVES * 64) void grouped_stream_rows_kernel(GroupedParams q) {
  constexpr int ES = T::ES, COLUMNS = 128 / ES;
  const int across = (int)(((uint32_t)q.n + COLUMNS - 1) / COLUMNS) * q.parts, id = windowed<64>(blockIdx.x, gridDim.x), want = id / across, block = id - want * across;
  int total = 0;
  const GroupedFamily<false>::Stretch s = GroupedFamily<false>::stretch_of<8>(q, threadIdx.x & 63, want, &total);
  if (s.number < 0) return;
  const int skip = (want - s.before) * 8, m = s.rows - skip < 8 ? s.rows - skip : 8, part = block % q.parts;
  const int64_t row = s.first + skip;
  float* const y = (float*)q.c + part * q.part_stride + row * q.n;
  if (s.number == 0 || s.number == q.groups + 1) {
    for (int o = threadIdx.x; o < m * COLUMNS; o += STREAM_ROWS_WAVES * 64) {
      const int n = block / q.parts * COLUMNS + o % COLUMNS;
      if (n < q.n) y[(int64_t)(o / COLUMNS) * q.n + n] = 0.0f;
    }
    return;
  }
  const uint8_t* const x = q.a + row * q.lda * ES;
  const uint8_t* const w = q.b + (int64_t)(s.number - 1) * q.group_stride * ES;
  stream_rows_block<T, STREAM_ROWS_WAVES, 2, true>({x, w, (uint8_t*)y, nullptr, nullptr, nullptr, nullptr, q.lda, q.ldb, m, q.n, q.k, q.parts, ACT_NONE}, block);
}
template <class T> hipError_t grouped_stream_rows(const GroupedParams& p, hipStream_t stream) {
  GroupedParams q = p;
  const unsigned grid = (unsigned)(stream_runs(p.rows, p.groups) * ((p.n + 128 / T::ES - 1) / (128 / T::ES)) * p.parts);
  return launch_kernel((const void*)&grouped_stream_rows_kernel<T>, grid, STREAM_ROWS_WAVES * 64, 0, stream, &q);
}

}  // namespace tnx
