// Linear layers: the product with its epilogue, and what the backward pass needs beside products.
//
//   y = act(z) + residual,  z = x w + bias          dz = dy act'(z),  dbias = the columns' sums of dz
//
// The product runs on the tile kernels with the epilogue of gemm_linear.h, float32 on the same kernels by heads and tails or, small ones, on
// the binary32 matrix instruction.  Where no such kernel takes the operands as they lie (an x that is contiguous along m, rows shorter
// than a 16-byte chunk, k = 0) the sums go to scratch in 32 bits and the epilogue is a launch of its own.  Few rows: gemm_stream.h.  dx = dz w^T and dw = x^T dz are
// products without an epilogue.
#include <hip/hip_runtime.h>
#include <string.h>

#include <unordered_map>

#include "../../include/tritonix_hip.h"
#include "registry.h"
#include "gemm_linear.h"
#include "gemm_stream.h"

using namespace tnx;

namespace {

__device__ __forceinline__ float load_float(const uint8_t* p, int64_t i, int dtype) {
  if (dtype == DT_F32) return ((const float*)p)[i];
  const uint16_t v = ((const uint16_t*)p)[i];
  return dtype == DT_BF16 ? __builtin_bit_cast(float, (uint32_t)v << 16) : (float)__builtin_bit_cast(_Float16, v);
}

// The epilogue alone, of sums in 32 bits (null: zeros); y may be the sums themselves.
__global__ __launch_bounds__(256) void epilogue_kernel(const float* sums, LinearParts x, uint8_t* y, int64_t m, int64_t n, int dtype) {
  const int64_t col = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (col >= n) return;
  const float bias = x.bias ? load_float(x.bias, col, x.bias_dtype) : 0.0f;
  for (int64_t row = blockIdx.y; row < m; row += gridDim.y) {
    const int64_t at = row * n + col;
    float v = (sums ? sums[at] : 0.0f) + bias;
    if (x.z) store_out<float>(x.z, at, v, dtype);
    v = activate(v, x.act);
    if (x.residual) v += load_float(x.residual, at, dtype);
    store_out<float>(y, at, v, dtype);
  }
}

struct GradParams {
  const uint8_t *dy, *z;
  uint8_t *dz, *dbias;         // dz null: dy as it is; dbias null: not wanted
  float* parts;                // [row blocks][n]; null: one row block, which writes dbias itself
  int64_t m, n;
  int act, bias_dtype, block;  // block: rows of a workgroup
};

// A workgroup takes a block of rows of 32 runs of V columns; its 8 lines of threads take a row in turn, add up their columns and meet in
// LDS.  Bound by memory: 8192 x 4096 bf16, dz of relu 38 us (5.3 TB/s).
//
// dz is rounded to the operands' type, for that is what the matrix instructions of dx = dz w^T and dw = x^T dz take; dbias sums it unrounded.  This rounding costs dx and dw as much as their own: off
// by 2.4e-3 (2-norm, bf16; f16 3.0e-4) against 1.66e-3 (2.1e-4) for a result that is rounded once.  dz in two terms would halve the rate of both products, which are two thirds of a step.
template <class O> __global__ __launch_bounds__(256) void grad_kernel(GradParams p) {
  typedef typename O::raw raw;
  constexpr int V = 16 / sizeof(raw);
  __shared__ float sums[8][32 * V + 4];
  const int lane = threadIdx.x & 31, line = threadIdx.x >> 5;
  const int64_t col = ((int64_t)blockIdx.x * 32 + lane) * V, row0 = (int64_t)blockIdx.y * p.block;
  const int cols = p.n - col >= V ? V : p.n > col ? (int)(p.n - col) : 0;
  float acc[V] = {};
  auto fetch = [&](const uint8_t* from, int64_t at, raw (&out)[V]) __attribute__((always_inline)) {
    if (cols == V) {
      const i32x4 v = *(const i32x4_loose*)((const raw*)from + at);
      __builtin_memcpy(out, &v, 16);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) out[e] = e < cols ? ((const raw*)from)[at + e] : (raw)0;
    }
  };
#pragma unroll 2
  for (int r = line; r < p.block; r += 8) {
    const int64_t row = row0 + r;
    if (row >= p.m || cols == 0) break;
    const int64_t at = row * p.n + col;
    raw g[V], z[V], out[V];
    fetch(p.dy, at, g);
    if (p.act != ACT_NONE) fetch(p.z, at, z);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      float v = Run<O, V>::widen(g[e]);
      if (p.act != ACT_NONE) v *= activation_slope(Run<O, V>::widen(z[e]), p.act);
      acc[e] += e < cols ? v : 0.0f;
      out[e] = O::cvt(v);
    }
    if (p.dz) {
      raw* dst = (raw*)p.dz + at;
      if (cols == V) {
        i32x4 v;
        __builtin_memcpy(&v, out, 16);
        *(i32x4_loose*)dst = v;
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (e < cols) dst[e] = out[e];
      }
    }
  }
  if (!p.dbias) return;
#pragma unroll
  for (int e = 0; e < V; ++e) sums[line][lane * V + e] = acc[e];
  __syncthreads();
  for (int c = threadIdx.x; c < 32 * V; c += 256) {
    const int64_t at = (int64_t)blockIdx.x * 32 * V + c;
    if (at >= p.n) continue;
    float s = 0.0f;
#pragma unroll
    for (int l = 0; l < 8; ++l) s += sums[l][c];
    if (p.parts) p.parts[(int64_t)blockIdx.y * p.n + at] = s;
    else store_out<float>(p.dbias, at, s, p.bias_dtype);
  }
}

// out[c] = the sum of parts[i][c] in the order of i, 64 columns from the `first` on and 16 lines of threads to a workgroup
__global__ __launch_bounds__(1024) void parts_kernel(const float* parts, int64_t count, int64_t n, int64_t first, uint8_t* out, int dtype) {
  __shared__ float sums[16][64];
  const int lane = threadIdx.x & 63, line = threadIdx.x >> 6;
  const int64_t col = first + (int64_t)blockIdx.x * 64 + lane;
  float s = 0.0f;
  if (col < n) {
#pragma unroll 8
    for (int64_t i = line; i < count; i += 16) s += parts[i * n + col];
  }
  sums[line][lane] = s;
  __syncthreads();
  if (line == 0 && col < n) {
#pragma unroll
    for (int l = 1; l < 16; ++l) s += sums[l][lane];
    store_out<float>(out, col, s, dtype);
  }
}

enum Route { ROUTE_PRODUCT = 0, ROUTE_FUSED = 1, ROUTE_APART = 2, ROUTE_STREAM = 3, ROUTE_STREAM_ROWS = 4 };
struct Plan {
  tnx_gemm_args g;             // of the product, without pointers
  Route route;
  bool f32;
  size_t workspace, scratch, sums;       // sums: the part of scratch that holds them in 32 bits, ahead of the float32 terms
  int status;
};

bool with_epilogue(const tnx_linear_args* a) { return a->bias || a->residual || a->z || a->activation != TNX_ACT_NONE; }

// an activation of an exponential and a division
bool curved(const tnx_linear_args* a) { return a->activation > TNX_ACT_RELU; }

// rows that begin at whole words: 16-byte loads of others take twice the time
bool whole_words(const tnx_linear_args* a) {
  if (a->dtype == TNX_F32) return true;
  return !(((uintptr_t)a->x | (uintptr_t)a->w) & 3) && a->stride_wn % 2 == 0 && (a->m == 1 || a->stride_xm % 2 == 0);
}

// Few rows, k-contiguous on both sides: gemm_stream.h.  Rows of x are fetched for every block of columns, which counts the more the more rows there are and
// the more blocks, and a long k by few workgroups is slower than the tile kernels' parts of it.  us, against the tile kernels', bf16: one row 1 x 1000 x 704
// 3.1 and 4.9, 1 x 4096 x 4096 7.7 and 9.5, 1 x 8192 x 8192 25.4 and 26.7, 1 x 4096 x 14336 21.9 and 20.8; 4 x 4096 x 4096 9.1 and 9.4, 4 x 512 x 8192 6.0 and
// 7.6, 4 x 14336 x 4096 25.2 and 21.2; 8 x 4096 x 4098 9.5 and 10.9, 8 x 512 x 8192 9.3 and 7.7; 16 x 1814 x 2746 7.2 and 8.1, 16 x 1024 x 4096 9.3 and 7.4.  Rows
// of the weight off whole words: 4 x 1000 x 701 3.4 and 6.8, 1 x 4096 x 4097 16.4 and 10.8.  float32: 1 x 14336 x 4096 46 and 122 (whose operands are cut into
// terms first), 4 x 8192 x 8192 52 and 56, 4 x 4096 x 14336 47 and 44, 8 x 4096 x 4096 13.9 and 18.1, 8 x 14336 x 4096 47 and 46.
bool takes_stream(const tnx_linear_args* a) {
  if (a->stride_xk != 1 || a->stride_wk != 1 || a->m > 16 || a->n > 0x1000000 || a->k > 0x40000000) return false;
  const bool f32 = a->dtype == TNX_F32;
  const int64_t weight = a->n * a->k;
  if (!whole_words(a) && weight > 1 << 20) return false;
  if (a->m == 1) return f32 || weight <= 1 << 24 || a->k <= 8192;
  if (a->m <= 4) return a->k <= 8192 && (f32 || weight <= 1 << 24);
  if (a->m <= 8) return a->k <= 4608 && weight <= 1 << 24;
  return !f32 && a->k <= 2816 && weight <= 6 << 20;
}

// The same by a row-major weight.  Its blocks have 64 columns, which pays against the tile kernels where columns are few and k is long: bf16, us, 1 x 512 x 8192
// 6.5 and 8.2, 8 x 512 x 8192 7.5 and 8.3, 1 x 1024 x 4096 6.4 and 7.5, 1 x 64 x 16384 6.1 and 8.6; 1 x 256 x 2048 5.5 and 5.3, 1 x 4096 x 4096 10.0 and 10.3,
// 1 x 14336 x 4096 26.7 and 23.1.  float32, whose operands the tile kernels cut into terms where columns are many: 1 x 14336 x 4096 47 and 115, 4 x 30000 x 512
// 22 and 38, 4 x 14336 x 4096 48 and 45; 1 x 1000 x 704 6.7 and 6.6.
bool takes_stream_rows(const tnx_linear_args* a) {
  if (a->stride_xk != 1 || a->stride_wn != 1 || a->n < 8 || a->k > 0x40000000) return false;
  if (a->dtype == TNX_F32) return a->m <= 4 && a->n > 8192 && a->n <= 0x1000000 && a->k <= 4096;
  return a->m <= 8 && a->n <= 1024 && a->k >= 4096;
}

Plan make_plan(const tnx_linear_args* a) {
  Plan p;
  memset(&p, 0, sizeof p);
  tnx_gemm_args& g = p.g;
  g.a = a->x; g.b = a->w;
  g.m = a->m; g.n = a->n; g.k = a->k;
  g.stride_am = a->stride_xm; g.stride_ak = a->stride_xk; g.stride_bk = a->stride_wk; g.stride_bn = a->stride_wn;
  g.stride_cm = a->n; g.stride_cn = 1;
  g.in_dtype = g.out_dtype = a->dtype;
  p.f32 = a->dtype == TNX_F32;
  if (a->k == 0) {               // no product
    p.route = ROUTE_APART;
    return p;
  }
  if (takes_stream(a)) {
    p.route = ROUTE_STREAM;
    return p;
  }
  if (takes_stream_rows(a)) {
    p.route = ROUTE_STREAM_ROWS;
    p.workspace = stream_rows_workspace(a->m, a->n, a->k, a->dtype == TNX_F32 ? 4 : 2);
    return p;
  }
  p.route = with_epilogue(a) ? ROUTE_FUSED : ROUTE_PRODUCT;
  p.status = p.f32 ? tnx_gemm_f32_config(&g) : tnx_gemm_default_config(&g);
  if (p.status != TNX_OK) return p;
  // (256x256 on four waves, the choice for long sums, has no registers left for this epilogue: 129 spilled, none on eight)
  if (p.route == ROUTE_FUSED && !p.f32 && g.block_m == 256 && g.block_n == 256) g.num_warps = 8;
  // Of a short k the epilogue's arithmetic is the time: two workgroups to a CU, whose epilogues and products overlap (bf16, gelu, us, 256x256 and 128x128: 8192 x
  // 4096 x 128 56 and 44, 4708 x 5248 x 352 63 and 49, 8192 x 4096 x 512 68 and 63, x 1024 84 and 88; writing z too 61 and 55 of a k of 256, 75 and 72, silu
  // 63 and 70, of one of 512; bias alone 4708 x 5248 x 352 38 and 38)
  if (p.route == ROUTE_FUSED && !p.f32 && curved(a) && a->k <= 384 && g.split_k <= 1 && g.block_m * g.block_n > 128 * 128) {
    g.block_m = g.block_n = 128;
    g.num_warps = 8;
    g.num_stages = 2;
    g.tail_tiles = 0;
  }
  if (p.route == ROUTE_FUSED && !(p.f32 ? gemm_f32_linear_fused(&g) : gemm_linear_fused(&g, GEMM_PLAIN))) {
    p.route = ROUTE_APART;
    if (!p.f32) {
      g.out_dtype = TNX_F32;
      p.status = tnx_gemm_default_config(&g);
      if (p.status != TNX_OK) return p;
      p.sums = ((size_t)a->m * a->n * 4 + 255) / 256 * 256;
    }
  }
  p.scratch = p.sums + (p.f32 ? tnx_gemm_f32_scratch_bytes(&g) : 0);
  p.workspace = g.split_k > 1 ? tnx_gemm_workspace_bytes(&g) : 0;
  return p;
}

struct Key {
  int64_t v[12];
  bool operator==(const Key& o) const { return memcmp(this, &o, sizeof *this) == 0; }
};
struct KeyHash {
  size_t operator()(const Key& k) const {
    uint64_t h = 0x9e3779b97f4a7c15ull;
    for (int64_t w : k.v) h = ((h ^ (uint64_t)w) * 0xff51afd7ed558ccdull) ^ (h >> 29);
    return (size_t)h;
  }
};

// what is decided about a layer's sizes, kept by thread: the choice takes longer than a launch
const Plan& plan_of(const tnx_linear_args* a) {
  static thread_local std::unordered_map<Key, Plan, KeyHash> plans;
  int device = 0;
  (void)hipGetDevice(&device);
  const Key k = {{a->m, a->n, a->k, a->stride_xm, a->stride_xk, a->stride_wk, a->stride_wn, a->dtype, with_epilogue(a) ? 1 : 0,
                  (int64_t)(((uintptr_t)a->x & 15) << 4 | ((uintptr_t)a->w & 15)), device, curved(a) ? 1 : 0}};
  const auto hit = plans.find(k);
  if (hit != plans.end()) return hit->second;
  if (plans.size() >= 512) plans.clear();
  return plans[k] = make_plan(a);
}

int check(const tnx_linear_args* a) {
  if (!a || a->m < 0 || a->n < 0 || a->k < 0) return TNX_E_INVALID;
  if (a->dtype != TNX_F16 && a->dtype != TNX_BF16 && a->dtype != TNX_F32) return TNX_E_UNSUPPORTED;
  if (a->activation < TNX_ACT_NONE || a->activation > TNX_ACT_GELU_TANH) return TNX_E_INVALID;
  if (a->bias && a->bias_dtype != a->dtype && a->bias_dtype != TNX_F32) return TNX_E_UNSUPPORTED;
  if (a->m > 0x7fffffff || a->n > 0x7fffffff || a->k > 0x7fffffff) return TNX_E_UNSUPPORTED;
  return TNX_OK;
}

int launched() {
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess) { note_hip_error((int)err); return TNX_E_HIP; }
  return TNX_OK;
}

}  // namespace

extern "C" size_t tnx_linear_workspace_bytes(const tnx_linear_args* a) {
  if (check(a) != TNX_OK || a->m == 0 || a->n == 0) return 0;
  const Plan& p = plan_of(a);
  return p.status == TNX_OK ? p.workspace : 0;
}
extern "C" size_t tnx_linear_scratch_bytes(const tnx_linear_args* a) {
  if (check(a) != TNX_OK || a->m == 0 || a->n == 0) return 0;
  const Plan& p = plan_of(a);
  return p.status == TNX_OK ? p.scratch : 0;
}
extern "C" int tnx_linear_route(const tnx_linear_args* a, int32_t info[5]) {
  if (check(a) != TNX_OK || a->m == 0 || a->n == 0) return 0;
  const Plan& p = plan_of(a);
  if (p.status != TNX_OK) return 0;
  if (info) {
    info[0] = p.g.block_m; info[1] = p.g.block_n; info[2] = p.g.num_warps; info[3] = p.g.num_stages; info[4] = p.g.split_k;
  }
  return 1 + (int)p.route;
}

extern "C" int tnx_linear(const tnx_linear_args* a) {
  const int st = check(a);
  if (st != TNX_OK) return st;
  if (a->m == 0 || a->n == 0) return TNX_OK;
  if (!a->y || (a->k > 0 && (!a->x || !a->w))) return TNX_E_INVALID;
  const Plan& p = plan_of(a);
  if (p.status != TNX_OK) return p.status;
  const int bias_dtype = a->bias ? a->bias_dtype : a->dtype;          // (packed beside other flags: without a bias it may hold anything)
  if (p.route == ROUTE_STREAM) {
    const StreamParams q = {(const uint8_t*)a->x, (const uint8_t*)a->w, (uint8_t*)a->y, (uint8_t*)a->z, (const uint8_t*)a->bias, (const uint8_t*)a->residual,
                            a->stride_xm, a->stride_wn, (int32_t)a->m, (int32_t)a->n, (int32_t)a->k, a->activation, bias_dtype};
    const hipStream_t s = (hipStream_t)a->stream;
    const hipError_t err = a->dtype == TNX_BF16 ? stream_columns<TagBF16>(q, s) : a->dtype == TNX_F16 ? stream_columns<TagF16>(q, s) : stream_columns<TagF32>(q, s);
    if (err != hipSuccess) { note_hip_error((int)err); return TNX_E_HIP; }
    return TNX_OK;
  }
  if (p.route == ROUTE_STREAM_ROWS) {
    if (p.workspace > 0 && (!a->workspace || a->workspace_bytes < p.workspace || ((uintptr_t)a->workspace & 15))) return TNX_E_WORKSPACE;
    const StreamRowsParams q = {(const uint8_t*)a->x, (const uint8_t*)a->w, (uint8_t*)a->y, (uint8_t*)a->z, (const uint8_t*)a->bias, (const uint8_t*)a->residual,
                                p.workspace > 0 ? (uint8_t*)a->workspace : nullptr, a->stride_xm, a->stride_wk, (int32_t)a->m, (int32_t)a->n, (int32_t)a->k,
                                stream_rows_parts(a->n, a->k, a->dtype == TNX_F32 ? 4 : 2), a->activation | bias_dtype << 8};
    const hipStream_t s = (hipStream_t)a->stream;
    const hipError_t err = a->dtype == TNX_BF16 ? stream_rows<TagBF16>(q, s) : a->dtype == TNX_F16 ? stream_rows<TagF16>(q, s) : stream_rows<TagF32>(q, s);
    if (err != hipSuccess) { note_hip_error((int)err); return TNX_E_HIP; }
    return TNX_OK;
  }
  if (p.scratch > 0 && (!a->scratch || a->scratch_bytes < p.scratch || ((uintptr_t)a->scratch & 255))) return TNX_E_WORKSPACE;
  tnx_gemm_args g = p.g;
  g.a = a->x; g.b = a->w;
  g.c = p.sums ? a->scratch : a->y;
  g.workspace = a->workspace; g.workspace_bytes = a->workspace_bytes;
  g.stream = a->stream;
  uint8_t* terms = (uint8_t*)a->scratch + p.sums;
  const LinearParts x = {(const uint8_t*)a->bias, (const uint8_t*)a->residual, (uint8_t*)a->z, bias_dtype, a->activation};
  const LinearParts* fused = p.route == ROUTE_FUSED ? &x : nullptr;
  const int status = a->k == 0 ? TNX_OK : p.f32 ? gemm_f32(&g, p.scratch > p.sums ? terms : nullptr, p.scratch - p.sums, fused) : gemm_launch(&g, nullptr, GEMM_PLAIN, fused);
  if (status != TNX_OK || p.route != ROUTE_APART) return status;
  const unsigned cols = (unsigned)((a->n + 255) / 256);
  hipLaunchKernelGGL(epilogue_kernel, dim3(cols, (unsigned)(a->m < 65535 ? a->m : 65535)), dim3(256), 0, (hipStream_t)a->stream, a->k == 0 ? nullptr : (const float*)g.c, x,
                     (uint8_t*)a->y, a->m, a->n, a->dtype);
  return launched();
}

// Rows of a workgroup of the gradient's pass: 64, fewer while that leaves CUs without one (1025 x 770 f16, both launches: 68 workgroups of 64 rows
// 15 us, 516 of 8 rows 5.6); each block of rows is a row of partial sums for the second launch to add up.  A grid has at most 65535 blocks of rows.
static int block_rows(int64_t m, int64_t n, int dtype) {
  const int64_t span = 32 * (dtype == TNX_F32 ? 4 : 8), across = (n + span - 1) / span;
  int rows = 64;
  while (rows > 8 && (m + rows - 1) / rows * across < 512) rows /= 2;
  while (rows < 0x40000000 && (m + rows - 1) / rows > 65535) rows *= 2;
  return rows;
}
static int64_t row_blocks(const tnx_linear_gradient_args* a) { return (a->m + block_rows(a->m, a->n, a->dtype) - 1) / block_rows(a->m, a->n, a->dtype); }

extern "C" size_t tnx_linear_gradient_bytes(const tnx_linear_gradient_args* a) {
  return !a || !a->dbias || a->m <= 0 || a->n <= 0 || row_blocks(a) <= 1 ? 0 : (size_t)row_blocks(a) * a->n * 4;
}

extern "C" int tnx_linear_gradient(const tnx_linear_gradient_args* a) {
  if (!a || a->m < 0 || a->n < 0 || a->activation < TNX_ACT_NONE || a->activation > TNX_ACT_GELU_TANH) return TNX_E_INVALID;
  if (a->dtype != TNX_F16 && a->dtype != TNX_BF16 && a->dtype != TNX_F32) return TNX_E_UNSUPPORTED;
  if (a->dbias && a->bias_dtype != a->dtype && a->bias_dtype != TNX_F32) return TNX_E_UNSUPPORTED;
  if (a->n == 0 || (!a->dz && !a->dbias) || (a->m == 0 && !a->dbias)) return TNX_OK;
  if ((a->m > 0 && !a->dy) || (a->m > 0 && a->activation != TNX_ACT_NONE && !a->z)) return TNX_E_INVALID;
  const int64_t blocks = a->m > 0 ? row_blocks(a) : 1, span = 32 * (a->dtype == TNX_F32 ? 4 : 8), cols = (a->n + span - 1) / span;
  if (blocks > 65535 || cols > 0xffffffffll / 256) return TNX_E_UNSUPPORTED;           // (a grid's threads are counted in 32 bits)
  const size_t need = tnx_linear_gradient_bytes(a);
  if (need && (!a->workspace || a->workspace_bytes < need || ((uintptr_t)a->workspace & 15))) return TNX_E_WORKSPACE;
  GradParams p = {(const uint8_t*)a->dy, (const uint8_t*)a->z, (uint8_t*)a->dz, (uint8_t*)a->dbias, need ? (float*)a->workspace : nullptr, a->m, a->n,
                  a->activation, a->bias_dtype, block_rows(a->m, a->n, a->dtype)};
  const dim3 grid((unsigned)cols, (unsigned)blocks);
  const hipStream_t stream = (hipStream_t)a->stream;
  if (a->dtype == TNX_BF16) hipLaunchKernelGGL(grad_kernel<OutBF16>, grid, dim3(256), 0, stream, p);
  else if (a->dtype == TNX_F16) hipLaunchKernelGGL(grad_kernel<OutF16>, grid, dim3(256), 0, stream, p);
  else hipLaunchKernelGGL(grad_kernel<OutF32>, grid, dim3(256), 0, stream, p);
  if (need) {
    constexpr int64_t MOST = 0xffffffffll / 1024;
    for (int64_t first = 0; first < a->n; first += MOST * 64) {
      const int64_t left = (a->n - first + 63) / 64;
      hipLaunchKernelGGL(parts_kernel, dim3((unsigned)(left < MOST ? left : MOST)), dim3(1024), 0, stream, (const float*)a->workspace, blocks, a->n, first,
                         (uint8_t*)a->dbias, a->bias_dtype);
    }
  }
  return launched();
}
