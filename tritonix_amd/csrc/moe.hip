// Routing of tokens to experts: scores, choice, the plan of the experts' rows, the join of their outputs, and the gradient
// of the logits.
#include <hip/hip_runtime.h>

#include "../../include/tritonix_hip.h"
#include "mx.h"

using namespace tnx;

namespace {

struct RouteParams {
  const uint8_t* logits;
  const float* bias;
  float* weights;
  int32_t* experts;
  const float* grad;
  uint8_t* grad_logits;
  int64_t tokens, stride;
  int e, k, dtype, scoring, groups, top_groups, group_top, renorm, group_size;
  float scale;
};

struct PlanParams {
  const int32_t* experts;
  int32_t *offsets, *order, *rows;
  int32_t *counts, *totals;                // workspace: [experts][blocks] and [experts]
  int64_t pairs;
  int e, blocks;
};

__device__ __forceinline__ float load_logit(const uint8_t* p, int64_t i, int dtype) {
  if (dtype == DT_F32) return ((const float*)p)[i];
  const uint16_t v = ((const uint16_t*)p)[i];
  return dtype == DT_BF16 ? __builtin_bit_cast(float, (uint32_t)v << 16) : (float)__builtin_bit_cast(_Float16, v);
}

// the value of lane ^ D (D a power of two up to 32) as every group of 2 D lanes needs it for a sum or maximum that all
// its lanes end up with: D = 4 and 8 mirror instead, which is the same once the smaller groups agree
template <int D> __device__ __forceinline__ int lane_xor(int v) {
  if constexpr (D == 1) return __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xF, 0xF, true);
  else if constexpr (D == 2) return __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xF, 0xF, true);
  else if constexpr (D == 4) return __builtin_amdgcn_update_dpp(0, v, 0x141, 0xF, 0xF, true);      // mirror of 8
  else if constexpr (D == 8) return __builtin_amdgcn_update_dpp(0, v, 0x140, 0xF, 0xF, true);      // mirror of 16
  else return __shfl_xor(v, D);
}
template <int L, class F> __device__ __forceinline__ void over_lanes(F f) {
  if constexpr (L > 1) f(IntTag<1>());
  if constexpr (L > 2) f(IntTag<2>());
  if constexpr (L > 4) f(IntTag<4>());
  if constexpr (L > 8) f(IntTag<8>());
  if constexpr (L > 16) f(IntTag<16>());
  if constexpr (L > 32) f(IntTag<32>());
}
template <int L> __device__ __forceinline__ float lanes_max(float v) {
  over_lanes<L>([&](auto d) { v = __builtin_fmaxf(v, __builtin_bit_cast(float, lane_xor<decltype(d)::value>(__builtin_bit_cast(int, v)))); });
  return v;
}
template <int L> __device__ __forceinline__ float lanes_sum(float v) {
  over_lanes<L>([&](auto d) { v += __builtin_bit_cast(float, lane_xor<decltype(d)::value>(__builtin_bit_cast(int, v))); });
  return v;
}
template <int L> __device__ __forceinline__ bool lanes_any(bool v) {
  int x = v;
  over_lanes<L>([&](auto d) { x |= lane_xor<decltype(d)::value>(x); });
  return x != 0;
}

__device__ __forceinline__ float sigmoid(float x) { return 1.0f / (1.0f + __expf(-x)); }

constexpr int PLAN_PAIRS = 512;            // pairs of token and slot a workgroup of 256 threads places

// The places of PLAN_PAIRS pairs among their experts, without atomics whose order could show: a bit per pair and expert
// (setting bits commutes); a pair's rank is the number of bits below its own.
struct PairBits {
  unsigned long long* words;               // [experts][PLAN_PAIRS / 64]
  __device__ __forceinline__ int rank(int e, int i) const {
    const unsigned long long* w = words + e * (PLAN_PAIRS / 64);
    int r = 0;
    for (int q = 0; q < i / 64; ++q) r += __popcll(w[q]);
    return r + __popcll(w[i / 64] & ((1ull << (i & 63)) - 1));
  }
  __device__ __forceinline__ int count(int e) const {
    int r = 0;
#pragma unroll
    for (int q = 0; q < PLAN_PAIRS / 64; ++q) r += __popcll(words[e * (PLAN_PAIRS / 64) + q]);
    return r;
  }
};

// the experts of a block's pairs into bits; expert[] of this thread's pairs (-1: none)
__device__ __forceinline__ void mark_pairs(const PlanParams& p, int64_t first, const PairBits& bits, int tid, int (&expert)[PLAN_PAIRS / 256]) {
  for (int i = tid; i < p.e * (PLAN_PAIRS / 64); i += 256) bits.words[i] = 0;
  __syncthreads();
#pragma unroll
  for (int u = 0; u < PLAN_PAIRS / 256; ++u) {
    const int i = u * 256 + tid;
    expert[u] = first + i < p.pairs ? p.experts[first + i] : -1;
    if (expert[u] < 0 || expert[u] >= p.e) expert[u] = -1;
    else atomicOr(bits.words + expert[u] * (PLAN_PAIRS / 64) + (i >> 6), 1ull << (i & 63));
  }
  __syncthreads();
}

// exclusive sums of n values in LDS (n <= TNX_MOE_MAX_EXPERTS) over a workgroup of 256 threads; returns the whole sum
__device__ __forceinline__ int scan_experts(int* v, int n, int tid) {
  __shared__ int waves[4];
  constexpr int PER = TNX_MOE_MAX_EXPERTS / 256;
  int mine[PER], sum = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int at = tid * PER + i;
    mine[i] = at < n ? v[at] : 0;
    sum += mine[i];
  }
  int upto = sum;
  const int lane = tid & 63;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int x = __shfl_up(upto, d);
    if (lane >= d) upto += x;
  }
  if (lane == 63) waves[tid >> 6] = upto;
  __syncthreads();
  int before = upto - sum, total = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (w < (tid >> 6)) before += waves[w];
    total += waves[w];
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int at = tid * PER + i;
    if (at < n) v[at] = before;
    before += mine[i];
  }
  __syncthreads();
  return total;
}

// all of the plan of at most PLAN_PAIRS pairs, by one workgroup.  smem: the pairs' bits, then an int per expert
__device__ __forceinline__ void plan_alone(const PlanParams& p, uint8_t* smem, int tid) {
  const PairBits bits{(unsigned long long*)smem};
  int* base = (int*)(smem + (size_t)p.e * PLAN_PAIRS / 8);
  int expert[PLAN_PAIRS / 256];
  mark_pairs(p, 0, bits, tid, expert);
  for (int e = tid; e < p.e; e += 256) base[e] = bits.count(e);
  __syncthreads();
  const int total = scan_experts(base, p.e, tid);
  for (int e = tid; e <= p.e; e += 256) p.offsets[e] = e < p.e ? base[e] : total;
#pragma unroll
  for (int u = 0; u < PLAN_PAIRS / 256; ++u) {
    const int i = u * 256 + tid;
    if (i >= p.pairs) continue;
    if (expert[u] >= 0) {
      const int at = base[expert[u]] + bits.rank(expert[u], i);
      p.order[at] = i;
      p.rows[i] = at;
    } else p.rows[i] = -1;
    if (i >= total) p.order[i] = -1;
  }
}

// Scores and choice.  L lanes share a token and hold EPL experts each, expert i L + j in lane j: a load instruction reads
// neighbouring logits.  The choice is top_k rounds of a maximum over the lanes' best; a round costs EPL compares and log2 L DPP
// steps, so as few lanes a token as the registers allow are best (128 experts: 8 lanes of 16).
template <int L, int EPL, bool GROUPS>
__device__ __forceinline__ void route_tokens(const RouteParams& p, int tid, int64_t token0, uint8_t* smem) {
  const int j = tid % L, slot = tid / L;
  const int64_t token = token0 + slot;
  const bool live = token < p.tokens;
  const uint8_t* row = p.logits + (live ? token : p.tokens - 1) * p.stride * (p.dtype == DT_F32 ? 4 : 2);
  float l[EPL], key[EPL];
  float top = -INFINITY;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    const int e = i * L + j;
    l[i] = e < p.e ? load_logit(row, e, p.dtype) : -INFINITY;
  }
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    bad |= l[i] != l[i];
    top = __builtin_fmaxf(top, l[i]);
  }
  top = lanes_max<L>(top);
  const bool soft = p.scoring == TNX_MOE_SOFTMAX;
  bad = lanes_any<L>(bad) || (soft && top == INFINITY);
  // softmax: score = exp(l - top) * inv (a row of -inf throughout has no score: nothing is chosen)
  float inv = 0.0f;
  const float off = top == -INFINITY ? 0.0f : top;
  if (soft) {
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < EPL; ++i) sum += __expf(l[i] - off);
    sum = lanes_sum<L>(sum);
    inv = sum > 0.0f ? 1.0f / sum : 0.0f;
  }
  auto score = [&](float x) { return soft ? __expf(x - off) * inv : sigmoid(x); };
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    const int e = i * L + j;
    key[i] = l[i];
    if (p.bias && e < p.e && l[i] > -INFINITY) {
      key[i] = score(l[i]) + p.bias[e];
      if (!(key[i] > -INFINITY)) key[i] = -INFINITY;
    }
    if (bad) key[i] = -INFINITY;
  }
  if (GROUPS) {
    // the keys of the workgroup's tokens in LDS; a lane ranks groups j, j + L, ... of its token
    float* keys = (float*)smem + slot * (p.e + TNX_MOE_MAX_GROUPS);
    float* worth = keys + p.e;
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if (i * L + j < p.e) keys[i * L + j] = key[i];
    __syncthreads();
    for (int g = j; g < p.groups; g += L) {
      // the sum of the group_top (1 or 2) largest keys that can be chosen
      float a = -INFINITY, b = -INFINITY;
      for (int i = 0; i < p.group_size; ++i) {
        const float x = keys[g * p.group_size + i];
        b = __builtin_fmaxf(b, __builtin_fminf(a, x));
        a = __builtin_fmaxf(a, x);
      }
      worth[g] = p.group_top == 2 && b > -INFINITY ? a + b : a;
    }
    __syncthreads();
    unsigned long long stay = 0;           // the groups with fewer than top_groups better ones
    for (int g = j; g < p.groups; g += L) {
      const float w = worth[g];
      int better = 0;
      for (int o = 0; o < p.groups; ++o) better += worth[o] > w || (worth[o] == w && o < g);
      if (better < p.top_groups) stay |= 1ull << g;
    }
    int lo = (int)(uint32_t)stay, hi = (int)(uint32_t)(stay >> 32);
    over_lanes<L>([&](auto d) { lo |= lane_xor<decltype(d)::value>(lo); hi |= lane_xor<decltype(d)::value>(hi); });
    stay = (unsigned long long)(uint32_t)hi << 32 | (uint32_t)lo;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const int e = i * L + j;
      if (e < p.e && !(stay >> (e / p.group_size) & 1)) key[i] = -INFINITY;
    }
    __syncthreads();                       // (the plan's bits take the same memory)
  }
  constexpr int KR = (TNX_MOE_MAX_TOP_K + L - 1) / L;
  float w[KR];
  int id[KR];
  float total = 0.0f;
#pragma unroll
  for (int r = 0; r < KR; ++r) {
    w[r] = 0.0f;
    id[r] = -1;
    for (int q = r * L; q < p.k && q < r * L + L; ++q) {
      float best = key[0], best_l = l[0];
      int best_e = j;
#pragma unroll
      for (int i = 1; i < EPL; ++i)
        if (key[i] > best) { best = key[i]; best_l = l[i]; best_e = i * L + j; }
      over_lanes<L>([&](auto d) {
        constexpr int D = decltype(d)::value;
        const float o = __builtin_bit_cast(float, lane_xor<D>(__builtin_bit_cast(int, best)));
        const float ol = __builtin_bit_cast(float, lane_xor<D>(__builtin_bit_cast(int, best_l)));
        const int oe = lane_xor<D>(best_e);
        if (o > best || (o == best && oe < best_e)) { best = o; best_l = ol; best_e = oe; }
      });
      const bool found = best > -INFINITY;
      const float s = found ? score(best_l) : 0.0f;
      total += s;
      if (j == q - r * L) { w[r] = s; id[r] = found ? best_e : -1; }
      if (best_e % L == j) {
#pragma unroll
        for (int i = 0; i < EPL; ++i)
          if (i * L + j == best_e) key[i] = -INFINITY;
      }
    }
  }
  const float f = p.renorm ? (total > 0.0f ? p.scale / total : 0.0f) : p.scale;
#pragma unroll
  for (int r = 0; r < KR; ++r) {
    const int q = r * L + j;
    if (live && q < p.k) {
      p.weights[token * p.k + q] = bad ? __builtin_nanf("") : w[r] * f;
      p.experts[token * p.k + q] = id[r];
    }
  }
}

// ALONE: one workgroup has all the tokens, and places their pairs too
template <int L, int EPL, bool GROUPS, bool ALONE>
__global__ __launch_bounds__(256) void route_kernel(RouteParams p, PlanParams q) {
  extern __shared__ __attribute__((aligned(16))) uint8_t moe_smem[];
  route_tokens<L, EPL, GROUPS>(p, threadIdx.x, (int64_t)blockIdx.x * (256 / L), moe_smem);
  if (ALONE) {
    __threadfence_block();                 // the experts just written are read back through memory by this workgroup
    __syncthreads();
    plan_alone(q, moe_smem, threadIdx.x);
  }
}

__global__ __launch_bounds__(256) void plan_alone_kernel(PlanParams p) {
  extern __shared__ __attribute__((aligned(16))) uint8_t moe_smem[];
  plan_alone(p, moe_smem, threadIdx.x);
}

// Many pairs, three launches: how many pairs of each block an expert has; sums over the blocks; places.
__global__ __launch_bounds__(256) void plan_count_kernel(PlanParams p) {
  extern __shared__ __attribute__((aligned(16))) uint8_t moe_smem[];
  const PairBits bits{(unsigned long long*)moe_smem};
  int expert[PLAN_PAIRS / 256];
  mark_pairs(p, (int64_t)blockIdx.x * PLAN_PAIRS, bits, threadIdx.x, expert);
  for (int e = threadIdx.x; e < p.e; e += 256) p.counts[(int64_t)e * p.blocks + blockIdx.x] = bits.count(e);
}

__global__ __launch_bounds__(256) void plan_sum_kernel(PlanParams p) {
  __shared__ int waves[4];
  int32_t* c = p.counts + (int64_t)blockIdx.x * p.blocks;
  const int tid = threadIdx.x, lane = tid & 63;
  int carry = 0;
  for (int b0 = 0; b0 < p.blocks; b0 += 256) {
    const int v = b0 + tid < p.blocks ? c[b0 + tid] : 0;
    int upto = v;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int x = __shfl_up(upto, d);
      if (lane >= d) upto += x;
    }
    if (lane == 63) waves[tid >> 6] = upto;
    __syncthreads();
    int before = carry + upto - v, all = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      if (w < (tid >> 6)) before += waves[w];
      all += waves[w];
    }
    if (b0 + tid < p.blocks) c[b0 + tid] = before;
    carry += all;
    __syncthreads();
  }
  if (tid == 0) p.totals[blockIdx.x] = carry;
}

__global__ __launch_bounds__(256) void plan_place_kernel(PlanParams p) {
  extern __shared__ __attribute__((aligned(16))) uint8_t moe_smem[];
  const PairBits bits{(unsigned long long*)moe_smem};
  int* base = (int*)(moe_smem + (size_t)p.e * PLAN_PAIRS / 8);
  const int tid = threadIdx.x;
  const int64_t first = (int64_t)blockIdx.x * PLAN_PAIRS;
  for (int e = tid; e < p.e; e += 256) base[e] = p.totals[e];
  int expert[PLAN_PAIRS / 256];
  mark_pairs(p, first, bits, tid, expert);
  const int total = scan_experts(base, p.e, tid);
  if (blockIdx.x == 0)
    for (int e = tid; e <= p.e; e += 256) p.offsets[e] = e < p.e ? base[e] : total;
#pragma unroll
  for (int u = 0; u < PLAN_PAIRS / 256; ++u) {
    const int i = u * 256 + tid;
    const int64_t pair = first + i;
    if (pair >= p.pairs) continue;
    if (expert[u] >= 0) {
      const int at = base[expert[u]] + p.counts[(int64_t)expert[u] * p.blocks + blockIdx.x] + bits.rank(expert[u], i);
      p.order[at] = (int32_t)pair;
      p.rows[pair] = at;
    } else p.rows[pair] = -1;
    if (pair >= total) p.order[pair] = -1;
  }
}

// Gradient of the logits.  With g_j the gradient of weight j and S the sum of the chosen scores:
//   ds_j = scale g_j, or scale (g_j - sum_i (s_i / S) g_i) / S with renormalised weights
//   softmax: dl_i = s_i (ds_i - sum_j s_j ds_j) over all i; with renormalised weights the sum is zero and s_j / S = weight / scale, so
//            neither the logits nor the other experts enter: dl_j = w_j (g_j - sum_i (w_i / scale) g_i)
//   sigmoid: dl_j = ds_j s_j (1 - s_j), of the chosen alone
template <int L, int EPL>
__global__ __launch_bounds__(256) void route_backward_kernel(RouteParams p) {
  const int tid = threadIdx.x, j = tid % L;
  const int64_t token = (int64_t)blockIdx.x * (256 / L) + tid / L;
  const bool live = token < p.tokens;
  const int64_t t = live ? token : p.tokens - 1;
  const uint8_t* row = p.logits + t * p.stride * (p.dtype == DT_F32 ? 4 : 2);
  const bool soft = p.scoring == TNX_MOE_SOFTMAX;
  float l[EPL], d[EPL];
  float off = 0.0f, inv = 0.0f;
  const bool dense = soft && !p.renorm;
#pragma unroll
  for (int i = 0; i < EPL; ++i) d[i] = 0.0f;
  if (dense) {
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      l[i] = i * L + j < p.e ? load_logit(row, i * L + j, p.dtype) : -INFINITY;
      top = __builtin_fmaxf(top, l[i]);
    }
    top = lanes_max<L>(top);
    off = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < EPL; ++i) sum += l[i] = __expf(l[i] - off);
    sum = lanes_sum<L>(sum);
    inv = sum > 0.0f ? 1.0f / sum : 0.0f;
  }
  // the chosen experts, lane j those of slots j, j + L, ...
  constexpr int KR = (TNX_MOE_MAX_TOP_K + L - 1) / L;
  float g[KR], s[KR], w[KR];
  int id[KR];
  float wg = 0.0f, total = 0.0f;
  bool bad = false;
#pragma unroll
  for (int r = 0; r < KR; ++r) {
    const int q = r * L + j;
    id[r] = -1;
    g[r] = s[r] = w[r] = 0.0f;
    if (q < p.k) {
      w[r] = p.weights[t * p.k + q];
      bad |= w[r] != w[r];
      id[r] = p.experts[t * p.k + q];
      if (id[r] >= p.e) id[r] = -1;
      if (id[r] >= 0) {
        g[r] = p.grad[t * p.k + q];
        if (!soft) s[r] = sigmoid(load_logit(row, id[r], p.dtype));
      } else w[r] = 0.0f;
    }
    total += s[r];
    wg += soft ? w[r] * g[r] : s[r] * g[r];
  }
  bad = lanes_any<L>(bad);
  wg = lanes_sum<L>(wg);
  total = lanes_sum<L>(total);
  float value[KR];                         // of the chosen: dl (dense: without the common term)
#pragma unroll
  for (int r = 0; r < KR; ++r) {
    if (soft && p.renorm) value[r] = w[r] * (g[r] - (p.scale != 0.0f ? wg / p.scale : 0.0f));
    else if (soft) value[r] = w[r] * g[r];                  // s ds: weight is scale s
    else {
      float ds = p.scale * g[r];
      if (p.renorm) ds = total > 0.0f ? p.scale * (g[r] - wg / total) / total : 0.0f;
      value[r] = ds * s[r] * (1.0f - s[r]);
    }
  }
  if (dense) {
#pragma unroll
    for (int i = 0; i < EPL; ++i) d[i] = -(l[i] * inv) * wg;
  }
#pragma unroll
  for (int r = 0; r < KR; ++r) {
    for (int q = r * L; q < p.k && q < r * L + L; ++q) {
      // slot q's expert and value from the lane that has them
      const int from = (tid & 63) - j + (q - r * L);
      const int e = __shfl(id[r], from);
      const float v = __shfl(value[r], from);
#pragma unroll
      for (int i = 0; i < EPL; ++i)
        if (e == i * L + j) d[i] += v;
    }
  }
  if (!live) return;
#pragma unroll
  for (int i = 0; i < EPL; ++i)
    if (i * L + j < p.e) store_out<float>(p.grad_logits, token * p.e + i * L + j, bad ? __builtin_nanf("") : d[i], p.dtype);
}

// The join: 16 bytes of a token's output per lane, the top_k rows one after another.
typedef uint16_t u16x8_loose __attribute__((ext_vector_type(8), aligned(2)));
typedef float f32x8_loose __attribute__((ext_vector_type(8), aligned(4)));

template <int YD> __device__ __forceinline__ float value_at(const uint8_t* y, int64_t i) { return load_logit(y, i, YD); }

template <int YD>
__global__ __launch_bounds__(256) void combine_kernel(const uint8_t* y, const int32_t* rows, const float* weights, uint8_t* out, int64_t tokens, int k,
                                                      int64_t n, int out_dtype) {
  const int64_t t = blockIdx.x;
  const int64_t c = ((int64_t)blockIdx.y * 256 + threadIdx.x) * 8;
  if (c >= n) return;
  float acc[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  const bool whole = c + 8 <= n;
  for (int j = 0; j < k; ++j) {
    const int r = rows[t * k + j];
    if (r < 0) continue;
    const float w = weights[t * k + j];
    const int64_t at = (int64_t)r * n + c;
    if (whole) {
      if constexpr (YD == DT_F32) {
        const f32x8_loose v = *(const f32x8_loose*)((const float*)y + at);
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] += w * v[e];
      } else {
        const u16x8_loose v = *(const u16x8_loose*)((const uint16_t*)y + at);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          acc[e] += w * (YD == DT_BF16 ? __builtin_bit_cast(float, (uint32_t)v[e] << 16) : (float)__builtin_bit_cast(_Float16, (uint16_t)v[e]));
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c + e < n) acc[e] += w * value_at<YD>(y, at + e);
    }
  }
  const int64_t o = t * n + c;
  if (whole && out_dtype != DT_F32) {
    u16x8_loose v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = out_dtype == DT_BF16 ? OutBF16::cvt(acc[e]) : OutF16::cvt(acc[e]);
    *(u16x8_loose*)((uint16_t*)out + o) = v;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c + e < n) store_out<float>(out, o + e, acc[e], out_dtype);
  }
}

// ------------------------------------------------------------------------------------------------------------------
int64_t up16(int64_t v) { return (v + 15) / 16 * 16; }
int64_t plan_blocks(int64_t pairs) { return (pairs + PLAN_PAIRS - 1) / PLAN_PAIRS; }
size_t plan_lds(int e) { return (size_t)e * (PLAN_PAIRS / 8) + (size_t)e * 4; }

int check_plan(const tnx_moe_args* a) {
  if (!a || a->tokens < 0 || a->top_k < 1 || a->num_experts < 1) return TNX_E_INVALID;
  if (a->num_experts > TNX_MOE_MAX_EXPERTS || a->top_k > TNX_MOE_MAX_TOP_K || a->tokens > 0x3fffffff / a->top_k) return TNX_E_UNSUPPORTED;
  if (!a->offsets) return TNX_E_INVALID;
  if (a->tokens > 0 && (!a->experts || !a->order || !a->rows)) return TNX_E_INVALID;
  if (a->tokens * a->top_k > PLAN_PAIRS && (!a->workspace || ((uintptr_t)a->workspace & 15) ||
      a->workspace_bytes < tnx_moe_workspace_bytes(a->tokens, a->top_k, a->num_experts))) return TNX_E_WORKSPACE;
  return TNX_OK;
}

PlanParams plan_params(const tnx_moe_args* a) {
  PlanParams q;
  q.experts = a->experts; q.offsets = a->offsets; q.order = a->order; q.rows = a->rows;
  q.pairs = a->tokens * a->top_k;
  q.e = a->num_experts;
  q.blocks = (int)plan_blocks(q.pairs);
  q.counts = (int32_t*)a->workspace;
  q.totals = q.counts ? (int32_t*)((uint8_t*)q.counts + up16((int64_t)q.e * q.blocks * 4)) : nullptr;
  return q;
}

int launch_plan(const PlanParams& q, hipStream_t stream) {
  if (q.pairs <= PLAN_PAIRS) {
    hipLaunchKernelGGL(plan_alone_kernel, dim3(1), dim3(256), plan_lds(q.e), stream, q);
    return mx_launched();
  }
  hipLaunchKernelGGL(plan_count_kernel, dim3((unsigned)q.blocks), dim3(256), plan_lds(q.e), stream, q);
  int st = mx_launched();
  if (st) return st;
  hipLaunchKernelGGL(plan_sum_kernel, dim3((unsigned)q.e), dim3(256), 0, stream, q);
  if ((st = mx_launched())) return st;
  hipLaunchKernelGGL(plan_place_kernel, dim3((unsigned)q.blocks), dim3(256), plan_lds(q.e), stream, q);
  return mx_launched();
}

int check_route(const tnx_moe_args* a) {
  if (a->top_k > a->num_experts) return TNX_E_INVALID;
  if (a->dtype != TNX_BF16 && a->dtype != TNX_F16 && a->dtype != TNX_F32) return TNX_E_UNSUPPORTED;
  if (a->scoring != TNX_MOE_SOFTMAX && a->scoring != TNX_MOE_SIGMOID) return TNX_E_INVALID;
  if (a->tokens > 0 && (!a->logits || !a->weights || ((uintptr_t)a->logits & (a->dtype == TNX_F32 ? 3 : 1)))) return TNX_E_INVALID;
  if (a->num_groups < 1 || a->num_groups > TNX_MOE_MAX_GROUPS || a->num_experts % a->num_groups || a->top_groups < 1 || a->top_groups > a->num_groups)
    return TNX_E_INVALID;
  if (a->group_top < 1 || a->group_top > 2) return TNX_E_INVALID;
  return TNX_OK;
}

RouteParams route_params(const tnx_moe_args* a) {
  RouteParams p;
  p.logits = (const uint8_t*)a->logits; p.bias = a->bias; p.weights = a->weights; p.experts = a->experts;
  p.grad = a->grad; p.grad_logits = (uint8_t*)a->grad_logits;
  p.tokens = a->tokens; p.stride = a->stride_logits;
  p.e = a->num_experts; p.k = a->top_k; p.dtype = a->dtype; p.scoring = a->scoring;
  p.groups = a->num_groups; p.top_groups = a->top_groups; p.group_top = a->group_top; p.renorm = a->renormalize;
  p.group_size = a->num_experts / a->num_groups;
  p.scale = a->scale;
  return p;
}

template <int L, int EPL> int launch_route(const RouteParams& p, const PlanParams& q, hipStream_t stream) {
  constexpr int TOKENS = 256 / L;
  const unsigned blocks = (unsigned)((p.tokens + TOKENS - 1) / TOKENS);
  const bool groups = p.groups > 1 && p.top_groups < p.groups;
  const bool alone = blocks == 1 && q.pairs <= PLAN_PAIRS;
  const size_t keys = groups ? (size_t)TOKENS * (p.e + TNX_MOE_MAX_GROUPS) * 4 : 0, bits = alone ? plan_lds(p.e) : 0;
  const size_t lds = keys > bits ? keys : bits;
  if (groups && alone) hipLaunchKernelGGL((route_kernel<L, EPL, true, true>), dim3(blocks), dim3(256), lds, stream, p, q);
  else if (groups) hipLaunchKernelGGL((route_kernel<L, EPL, true, false>), dim3(blocks), dim3(256), lds, stream, p, q);
  else if (alone) hipLaunchKernelGGL((route_kernel<L, EPL, false, true>), dim3(blocks), dim3(256), lds, stream, p, q);
  else hipLaunchKernelGGL((route_kernel<L, EPL, false, false>), dim3(blocks), dim3(256), lds, stream, p, q);
  const int st = mx_launched();
  return st || alone ? st : launch_plan(q, stream);
}

template <int L, int EPL> int launch_backward(const RouteParams& p, hipStream_t stream) {
  constexpr int TOKENS = 256 / L;
  hipLaunchKernelGGL((route_backward_kernel<L, EPL>), dim3((unsigned)((p.tokens + TOKENS - 1) / TOKENS)), dim3(256), 0, stream, p);
  return mx_launched();
}

}  // namespace

extern "C" size_t tnx_moe_workspace_bytes(int64_t tokens, int32_t top_k, int32_t num_experts) {
  const int64_t pairs = tokens * top_k;
  if (tokens <= 0 || top_k <= 0 || num_experts <= 0 || pairs <= PLAN_PAIRS) return 0;
  return (size_t)(up16((int64_t)num_experts * plan_blocks(pairs) * 4) + up16((int64_t)num_experts * 4));
}

extern "C" int tnx_moe_plan(const tnx_moe_args* a) {
  const int st = check_plan(a);
  return st ? st : launch_plan(plan_params(a), (hipStream_t)a->stream);
}

extern "C" int tnx_moe_route(const tnx_moe_args* a) {
  int st = check_plan(a);
  if (st || (st = check_route(a))) return st;
  const RouteParams p = route_params(a);
  const PlanParams q = plan_params(a);
  const hipStream_t stream = (hipStream_t)a->stream;
  if (a->tokens == 0) return launch_plan(q, stream);
  if (p.e <= 32) return launch_route<8, 4>(p, q, stream);
  if (p.e <= 64) return launch_route<8, 8>(p, q, stream);
  if (p.e <= 128) return launch_route<8, 16>(p, q, stream);
  if (p.e <= 256) return launch_route<16, 16>(p, q, stream);
  if (p.e <= 512) return launch_route<32, 16>(p, q, stream);
  return launch_route<64, 16>(p, q, stream);
}

extern "C" int tnx_moe_route_backward(const tnx_moe_args* a) {
  if (!a || a->tokens < 0 || a->top_k < 1 || a->num_experts < 1) return TNX_E_INVALID;
  if (a->num_experts > TNX_MOE_MAX_EXPERTS || a->top_k > TNX_MOE_MAX_TOP_K || a->tokens > 0x3fffffff / a->top_k) return TNX_E_UNSUPPORTED;
  const int st = check_route(a);
  if (st) return st;
  if (a->tokens == 0) return TNX_OK;
  if (!a->experts || !a->grad || !a->grad_logits) return TNX_E_INVALID;
  const RouteParams p = route_params(a);
  const hipStream_t stream = (hipStream_t)a->stream;
  if (p.e <= 32) return launch_backward<8, 4>(p, stream);
  if (p.e <= 64) return launch_backward<8, 8>(p, stream);
  if (p.e <= 128) return launch_backward<8, 16>(p, stream);
  if (p.e <= 256) return launch_backward<16, 16>(p, stream);
  if (p.e <= 512) return launch_backward<32, 16>(p, stream);
  return launch_backward<64, 16>(p, stream);
}

extern "C" int tnx_moe_combine(const void* y, const int32_t* rows, const float* weights, void* out, int64_t tokens, int32_t top_k, int64_t n,
                               int32_t y_dtype, int32_t out_dtype, void* stream) {
  if (tokens < 0 || top_k < 1 || n < 0) return TNX_E_INVALID;
  if (tokens == 0 || n == 0) return TNX_OK;
  if (!y || !rows || !weights || !out) return TNX_E_INVALID;
  if (out_dtype != TNX_BF16 && out_dtype != TNX_F16 && out_dtype != TNX_F32) return TNX_E_UNSUPPORTED;
  const int64_t cols = (n + 2047) / 2048;
  if (tokens > 0x7fffffff || cols > 65535) return TNX_E_UNSUPPORTED;
  const dim3 grid((unsigned)tokens, (unsigned)cols);
  switch (y_dtype) {
    case TNX_BF16:
      hipLaunchKernelGGL((combine_kernel<DT_BF16>), grid, dim3(256), 0, (hipStream_t)stream, (const uint8_t*)y, rows, weights, (uint8_t*)out, tokens, top_k, n, out_dtype);
      break;
    case TNX_F16:
      hipLaunchKernelGGL((combine_kernel<DT_F16>), grid, dim3(256), 0, (hipStream_t)stream, (const uint8_t*)y, rows, weights, (uint8_t*)out, tokens, top_k, n, out_dtype);
      break;
    case TNX_F32:
      hipLaunchKernelGGL((combine_kernel<DT_F32>), grid, dim3(256), 0, (hipStream_t)stream, (const uint8_t*)y, rows, weights, (uint8_t*)out, tokens, top_k, n, out_dtype);
      break;
    default: return TNX_E_UNSUPPORTED;
  }
  return mx_launched();
}
