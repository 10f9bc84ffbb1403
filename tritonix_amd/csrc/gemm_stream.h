// Linear layers of few rows with a k-contiguous weight (the transpose of a row-major one): single tokens and small decode batches.
//
// Bound by reading the weight once, and a CU alone takes in little over 20 GB/s of it whatever its waves have in flight, so that all CUs have to
// read all the time: small blocks of columns, no step that waits for another workgroup.  A workgroup owns C columns (NT times, for more use of a
// row of x), its waves take turns along k, and the weight goes from memory straight into the registers that v_mfma_f32_16x16x32 reads: no LDS and no
// barrier in the loop.  Of the 16 rows and columns of a matrix instruction a block needs C columns of the weight and at most C rows; the 16 / C
// groups of them take different parts of k, and of the 16 x 16 sums the blocks on the diagonal count.  That narrows a workgroup without an idle lane
// among the loads, and a row's part of an instruction is 32 x 16 / C elements: from C = 8 on down whole lines of memory.  Rows of x come from the
// caches.  The waves' and groups' sums meet in LDS, in order, where the epilogue runs on them: one launch, no workspace, the same bits every time.
// bf16, cold weights, us: 1 x 4096 x 4096 7.6 (4.4 TB/s; the tile kernels, which cut k and hand slices over, 12.4), 1 x 14336 x 4096 19 (6.2 TB/s; 25),
// 1 x 1024 x 1024 2.5 (7.4), 8 x 4096 x 4096 9.2 (12.5), 16 x 1024 x 1024 3.9 (7.5).
#pragma once
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
// of which nothing is left for another instruction to read (with C = 8, us: 1 x 4096 x 4096 7.6 past the caches and 8.1 through them; rows that begin
// anywhere, 1 x 2050 x 4100 7.5 and 6.4).
template <class T, int C, int NT, int W, int U, bool LINES> __global__ __launch_bounds__(W * 64) void gemm_stream_kernel(StreamParams p) {
  static_assert(T::ES == 2, "16-bit element types only");
  typedef Mma<T, 16> MMA;
  typedef typename OutOf<T>::type O;
  typedef typename O::raw raw;
  constexpr int G = 16 / C, STEP = 64 * G, HALF = 32 * G;
  __shared__ f32x4 sums[W][NT][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int li = lane & 15, kg = lane >> 4;
  const int tiles = (p.n + C * NT - 1) / (C * NT), n0 = xcd_remap(blockIdx.x, tiles, 8) * (C * NT);
  const int koff = li / C * 32 + kg * 8;
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
        if (left >= 8) return (i32x4)*(const i32x4_loose*)(from + at);
        raw e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = i < left ? from[at + i] : (raw)0;
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
    if (p.residual) v += Run<O, 8>::widen(((const raw*)p.residual)[at]);
    ((raw*)p.y)[at] = O::cvt(v);
  }
}

template <class T, int C, int NT, int W, int U, bool LINES> hipError_t stream_launch(const StreamParams& p, hipStream_t stream) {
  StreamParams q = p;
  return launch_kernel((const void*)&gemm_stream_kernel<T, C, NT, W, U, LINES>, (unsigned)((p.n + C * NT - 1) / (C * NT)), W * 64, 0, stream, &q);
}

// waves: 4 where k has no step for each of 8 (1 x 30000 x 512, us: 7.1 and 8.1)
template <class T, int C, int NT, int U, bool LINES> hipError_t stream_waves(const StreamParams& p, hipStream_t stream) {
  if (p.k < 8 * 64 * (16 / C)) return stream_launch<T, C, NT, 4, U, LINES>(p, stream);
  return stream_launch<T, C, NT, 8, U, LINES>(p, stream);
}

template <class T, int C, int NT, int U> hipError_t stream_lines(const StreamParams& p, hipStream_t stream) {
  if constexpr (C < 16)
    if (p.ldw % 64 == 0 && ((uintptr_t)p.w & 127) == 0) return stream_waves<T, C, NT, U, true>(p, stream);
  return stream_waves<T, C, NT, U, false>(p, stream);
}

// Columns of a workgroup: 4 while 8 give fewer than 512 workgroups (1 x 512 x 8192, us: 4.9 and 7.0; 1 x 4096 x 4096 8.7 and 7.6), which have room for
// 4 rows; 8 for up to 8 rows, in pairs of blocks where there are many rows and columns (8 x 4096 x 4096: 9.9, with pairs 9.2); 16 beyond.
template <class T> hipError_t stream_columns(const StreamParams& p, hipStream_t stream) {
  if (p.m <= 4 && p.n < 4096) return stream_lines<T, 4, 1, 4>(p, stream);
  if (p.m <= 8 && (p.m <= 4 || p.n < 4096)) return stream_lines<T, 8, 1, 4>(p, stream);
  if (p.m <= 8) return stream_lines<T, 8, 2, 2>(p, stream);
  return stream_lines<T, 16, 1, 4>(p, stream);
}

}  // namespace tnx
