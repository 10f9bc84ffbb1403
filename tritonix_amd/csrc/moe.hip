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
  int runs_at;                             // bytes of LDS before the runs of keys
  bool vec, vec_out;                       // rows of the logits (of their gradient) in aligned runs of four
};

struct PlanParams {
  const int32_t* experts;
  int32_t *offsets, *order, *rows;
  int32_t *counts, *totals;                // workspace: [experts][blocks] where they are summed first, else [blocks][experts]; and [experts]
  int64_t pairs;
  int e, block, blocks, words;             // pairs of a block, blocks, 64-bit words of a block's bits
  bool fused;                              // the routing kernel's workgroups are the blocks, and count
  bool summed;                             // the counts are summed over the blocks by a launch of their own
  __device__ __forceinline__ int64_t count_at(int expert, int at) const { return summed ? (int64_t)expert * blocks + at : (int64_t)at * e + expert; }
};

__device__ __forceinline__ float load_logit(const uint8_t* p, int64_t i, int dtype) {
  if (dtype == DT_F32) return ((const float*)p)[i];
  const uint16_t v = ((const uint16_t*)p)[i];
  return dtype == DT_BF16 ? __builtin_bit_cast(float, (uint32_t)v << 16) : (float)__builtin_bit_cast(_Float16, v);
}

// The value of lane ^ D for sums and maxima that every lane of a group of 2 D ends up with: D = 4 and 8 mirror instead, which is
// the same once the smaller groups agree.  All without LDS: these are the steps of latency in the choice.
template <int D> __device__ __forceinline__ int lane_xor(int v) {
  if constexpr (D == 1) return __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xF, 0xF, true);
  else if constexpr (D == 2) return __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xF, 0xF, true);
  else if constexpr (D == 4) return __builtin_amdgcn_update_dpp(0, v, 0x141, 0xF, 0xF, true);      // mirror of 8
  else if constexpr (D == 8) return __builtin_amdgcn_update_dpp(0, v, 0x140, 0xF, 0xF, true);      // mirror of 16
  else if constexpr (D == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap((unsigned)v, (unsigned)v, false, false);       // even rows twice, odd rows twice
    return (int)(threadIdx.x & 16 ? r[0] : r[1]);
  } else {
    const auto r = __builtin_amdgcn_permlane32_swap((unsigned)v, (unsigned)v, false, false);
    return (int)(threadIdx.x & 32 ? r[0] : r[1]);
  }
}
template <int D> __device__ __forceinline__ float lane_xor(float v) { return __builtin_bit_cast(float, lane_xor<D>(__builtin_bit_cast(int, v))); }
template <int L, class F> __device__ __forceinline__ void over_lanes(F f) {
  if constexpr (L > 1) f(IntTag<1>());
  if constexpr (L > 2) f(IntTag<2>());
  if constexpr (L > 4) f(IntTag<4>());
  if constexpr (L > 8) f(IntTag<8>());
  if constexpr (L > 16) f(IntTag<16>());
  if constexpr (L > 32) f(IntTag<32>());
}
template <int L> __device__ __forceinline__ float lanes_max(float v) {
  over_lanes<L>([&](auto d) { v = __builtin_fmaxf(v, lane_xor<decltype(d)::value>(v)); });
  return v;
}
template <int L> __device__ __forceinline__ float lanes_sum(float v) {
  over_lanes<L>([&](auto d) { v += lane_xor<decltype(d)::value>(v); });
  return v;
}
template <int L> __device__ __forceinline__ int lanes_min(int v) {
  over_lanes<L>([&](auto d) {
    const int o = lane_xor<decltype(d)::value>(v);
    v = o < v ? o : v;
  });
  return v;
}
template <int L> __device__ __forceinline__ int lanes_or(int v) {
  over_lanes<L>([&](auto d) { v |= lane_xor<decltype(d)::value>(v); });
  return v;
}

__device__ __forceinline__ float sigmoid(float x) { return 1.0f / (1.0f + __expf(-x)); }
// exp(x), x <= 0, down to the smallest number: the exponential's instruction itself gives 0 for results next to the subnormal numbers
__device__ __forceinline__ float exp_below(float x) {
  const float h = __expf(0.5f * x);
  return h * h;
}
// What a sum of scores and its terms are multiplied by, so that neither its reciprocal nor a quotient by it leaves the range: 1 but for scores next to nothing
__device__ __forceinline__ float lift_of(float total) { return total < 0x1p-60f ? 0x1p64f : 1.0f; }

// Expert i of lane j where L lanes hold a row: four neighbours a lane, so that a load or store is 16 bytes.
template <int L> __device__ __forceinline__ int expert_of(int i, int j) { return (i >> 2) * (4 * L) + 4 * j + (i & 3); }

// a row of logits; past the end -inf.  vec: four neighbours in one load
template <int L, int EPL> __device__ __forceinline__ void load_row(const uint8_t* row, int e_count, int dtype, bool vec, int j, float (&l)[EPL]) {
#pragma unroll
  for (int i = 0; i < EPL; i += 4) {
    const int e = expert_of<L>(i, j);
    if (vec) {
      if (e < e_count) {
        if (dtype == DT_F32) {
          const f32x4 v = *(const f32x4*)((const float*)row + e);
#pragma unroll
          for (int x = 0; x < 4; ++x) l[i + x] = v[x];
        } else {
          typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
          const u16x4 v = *(const u16x4*)((const uint16_t*)row + e);
#pragma unroll
          for (int x = 0; x < 4; ++x) l[i + x] = dtype == DT_BF16 ? Elem<__bf16>::get(v[x]) : Elem<_Float16>::get(v[x]);
        }
      } else {
#pragma unroll
        for (int x = 0; x < 4; ++x) l[i + x] = -INFINITY;
      }
    } else {
#pragma unroll
      for (int x = 0; x < 4; ++x) l[i + x] = e + x < e_count ? load_logit(row, e + x, dtype) : -INFINITY;
    }
  }
}

// Places of pairs among their experts, without atomics whose order could show: a bit per pair of a block and expert
// (setting bits commutes); a pair's rank is the number of bits below its own.
struct PairBits {
  unsigned long long* words;               // [experts][n]
  int n;
  __device__ __forceinline__ int rank(int e, int i) const {
    const unsigned long long* w = words + e * n;
    int r = 0;
    for (int q = 0; q < i / 64; ++q) r += __popcll(w[q]);
    return r + __popcll(w[i / 64] & ((1ull << (i & 63)) - 1));
  }
  __device__ __forceinline__ int count(int e) const {
    int r = 0;
    for (int q = 0; q < n; ++q) r += __popcll(words[e * n + q]);
    return r;
  }
  __device__ __forceinline__ void clear(int e_count, int tid) const {
    for (int i = tid; i < e_count * n; i += 256) words[i] = 0;
  }
  __device__ __forceinline__ void mark(int e, int i) const { atomicOr(words + e * n + (i >> 6), 1ull << (i & 63)); }
};

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

// All of a plan of at most PLAN_ALONE pairs by one workgroup, from the experts in LDS (ids, -1: none).  A pair's place is the number of pairs
// before it: counted one by one, which for so few is quicker than sums over the experts.
constexpr int PLAN_ALONE = 128;
__device__ __forceinline__ void plan_alone(const PlanParams& p, const int* ids, int tid) {
  const int pairs = (int)p.pairs;
  if (tid < pairs) {
    const int mine = ids[tid];
    int at = 0, total = 0;
    for (int i = 0; i < pairs; ++i) {
      const int e = ids[i];
      total += e >= 0;
      at += e >= 0 && (e < mine || (e == mine && i < tid));
    }
    p.rows[tid] = mine >= 0 ? at : -1;
    if (mine >= 0) p.order[at] = tid;
    if (tid >= total) p.order[tid] = -1;
  }
  for (int e = tid; e <= p.e; e += 256) {
    int before = 0;
    for (int i = 0; i < pairs; ++i) before += ids[i] >= 0 && ids[i] < e;
    p.offsets[e] = before;
  }
}

// Scores and choice.  L lanes share a token and hold EPL experts each.  The choice is top_k rounds of a maximum over all keys, then the lowest expert that
// has it.  Bound by its instructions: eight lanes of sixteen experts where there are tokens enough to fill the card, a wave per token
// where there are few and a token's own time counts.  65536 tokens, 8 of 128 experts: 16.8 us; with a search through all sixteen registers
// each round 22, with the lanes' keys sorted first as doubles that hold key and expert 84 (a compare is one instruction, but not a fast one).
// FULL: with a bias or groups.  smem: a workgroup's own.
template <int L, int EPL, bool FULL>
__device__ __forceinline__ void route_tokens(const RouteParams& p, int tid, int64_t token0, uint8_t* smem, int (&id)[(TNX_MOE_MAX_TOP_K + L - 1) / L]) {
  const int j = tid % L, slot = tid / L;
  const int64_t token = token0 + slot;
  const bool live = token < p.tokens;
  const uint8_t* row = p.logits + (live ? token : p.tokens - 1) * p.stride * (p.dtype == DT_F32 ? 4 : 2);
  float l[EPL];
  load_row<L, EPL>(row, p.e, p.dtype, p.vec, j, l);
  float top = -INFINITY;
  int bad_bit = 0;
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    bad_bit |= l[i] != l[i];
    top = __builtin_fmaxf(top, l[i]);
  }
  top = lanes_max<L>(top);
  const bool soft = p.scoring == TNX_MOE_SOFTMAX;
  const bool bad = lanes_or<L>(bad_bit) || (soft && top == INFINITY);
  // softmax: score = exp(l - top) * inv (a row of -inf throughout has no score: nothing is chosen)
  // Where the weights are divided by their own sum, and no bias asks for the scores themselves, the sum over all falls out.
  float inv = 1.0f;
  const float off = top == -INFINITY ? 0.0f : top;
  if (soft && (!p.renorm || (FULL && p.bias))) {
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < EPL; ++i) sum += __expf(l[i] - off);
    sum = lanes_sum<L>(sum);
    inv = sum > 0.0f ? 1.0f / sum : 0.0f;
  }
  auto score = [&](float x) { return soft ? __expf(x - off) * inv : sigmoid(x); };      // (as keys have it)
  float key[EPL];
  if (FULL) {
    float (&f)[EPL] = key;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const int e = expert_of<L>(i, j);
      f[i] = l[i];
      if (p.bias && e < p.e && l[i] > -INFINITY) {
        f[i] = score(l[i]) + p.bias[e];
        if (!(f[i] > -INFINITY)) f[i] = -INFINITY;
      }
    }
    if (p.top_groups < p.groups) {
      // The token's keys in LDS, its own lanes' only: they are in one wave, whose LDS operations are in order.
      float* keys = (float*)smem + slot * (p.e + TNX_MOE_MAX_GROUPS);
      float* worth = keys + p.e;
#pragma unroll
      for (int i = 0; i < EPL; ++i)
        if (expert_of<L>(i, j) < p.e) keys[expert_of<L>(i, j)] = f[i];
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      // several lanes a group: the sum of the group_top (1 or 2) largest keys that can be chosen
      int per = 1;
      while (per < 16 && 2 * per * p.groups <= L) per *= 2;
      for (int g0 = 0; g0 < p.groups; g0 += L / per) {
        const int g = g0 + j / per;
        float a = -INFINITY, b = -INFINITY;
        if (g < p.groups)
          for (int i = j % per; i < p.group_size; i += per) {
            const float x = keys[g * p.group_size + i];
            b = __builtin_fmaxf(b, __builtin_fminf(a, x));
            a = __builtin_fmaxf(a, x);
          }
        auto merge = [&](auto d) {
          const float oa = lane_xor<decltype(d)::value>(a), ob = lane_xor<decltype(d)::value>(b);
          b = __builtin_fmaxf(__builtin_fminf(a, oa), __builtin_fmaxf(b, ob));
          a = __builtin_fmaxf(a, oa);
        };
        if (per > 1) merge(IntTag<1>());
        if (per > 2) merge(IntTag<2>());
        if (per > 4) merge(IntTag<4>());
        if (per > 8) merge(IntTag<8>());
        if (g < p.groups && j % per == 0) worth[g] = p.group_top == 2 && b > -INFINITY ? a + b : a;
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      int lo = 0, hi = 0;                  // the groups with fewer than top_groups better ones
      for (int g = j; g < p.groups; g += L) {
        const float w = worth[g];
        int better = 0;
        for (int o = 0; o < p.groups; ++o) better += worth[o] > w || (worth[o] == w && o < g);
        if (better < p.top_groups) (g < 32 ? lo : hi) |= 1 << (g & 31);
      }
      lo = lanes_or<L>(lo);
      hi = lanes_or<L>(hi);
#pragma unroll
      for (int i = 0; i < EPL; ++i) {
        const int e = expert_of<L>(i, j), g = e / p.group_size;
        if (e < p.e && !((g < 32 ? lo : hi) >> (g & 31) & 1)) f[i] = -INFINITY;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < EPL; ++i) key[i] = l[i];
  }
  constexpr int KR = (TNX_MOE_MAX_TOP_K + L - 1) / L, NG = EPL / 4;
  float won[KR];
  if constexpr (NG == 1) {
#pragma unroll
    for (int r = 0; r < KR; ++r) {
      won[r] = -INFINITY;
      id[r] = 0;
#pragma unroll 1
      for (int q = r * L; q < p.k && q < r * L + L; ++q) {
        const float best = lanes_max<L>(__builtin_fmaxf(__builtin_fmaxf(key[0], key[1]), __builtin_fmaxf(key[2], key[3])));
        int at = key[3] == best ? 3 : -1;  // this lane's first place that has it
        at = key[2] == best ? 2 : at;
        at = key[1] == best ? 1 : at;
        at = key[0] == best ? 0 : at;
        const int mine = at >= 0 ? 4 * j + at : 0x7fffffff, e = lanes_min<L>(mine);
        if (j == q - r * L) { won[r] = best; id[r] = e; }
        at = mine == e ? at : -1;
#pragma unroll
        for (int i = 0; i < 4; ++i) key[i] = i == at ? -INFINITY : key[i];
      }
    }
  } else {
    // Runs of four keys in LDS, the runs' maxima in registers: run g L + j (experts 4 (g L + j) + 0 .. 3) is lane j's g-th.  Only the lane that holds the
    // round's key looks into its run.  (All in one wave, whose LDS operations are in order.)
    f32x4* runs = (f32x4*)(smem + p.runs_at) + tid;                       // [NG][256]
    int* chosen = (int*)(smem + p.runs_at + NG * 4096) + slot * TNX_MOE_MAX_TOP_K;
    float top4[NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      runs[g * 256] = f32x4{key[4 * g], key[4 * g + 1], key[4 * g + 2], key[4 * g + 3]};
      top4[g] = __builtin_fmaxf(__builtin_fmaxf(key[4 * g], key[4 * g + 1]), __builtin_fmaxf(key[4 * g + 2], key[4 * g + 3]));
    }
#pragma unroll
    for (int r = 0; r < KR; ++r) {
      won[r] = -INFINITY;
#pragma unroll 1
      for (int q = r * L; q < p.k && q < r * L + L; ++q) {
        float best = top4[0];
#pragma unroll
        for (int g = 1; g < NG; ++g) best = __builtin_fmaxf(best, top4[g]);
        best = lanes_max<L>(best);
        int at = -1;
#pragma unroll
        for (int g = NG - 1; g >= 0; --g) at = top4[g] == best ? g : at;
        const int mine = at >= 0 ? at * L + j : 0x7fffffff, run = lanes_min<L>(mine);
        if (j == q - r * L) won[r] = best;
        if (at >= 0 && mine == run) {
          f32x4 v = runs[at * 256];
          const int x = v[0] == best ? 0 : v[1] == best ? 1 : v[2] == best ? 2 : 3;
#pragma unroll
          for (int i = 0; i < 4; ++i) v[i] = i == x ? -INFINITY : v[i];
          const float rest = __builtin_fmaxf(__builtin_fmaxf(v[0], v[1]), __builtin_fmaxf(v[2], v[3]));
          ((float*)(runs + at * 256))[x] = -INFINITY;
          chosen[q] = 4 * run + x;
#pragma unroll
          for (int g = 0; g < NG; ++g) top4[g] = g == at ? rest : top4[g];
        }
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int r = 0; r < KR; ++r) id[r] = r * L + j < p.k ? chosen[r * L + j] : 0;
  }
  float w[KR], total = 0.0f, most = off;
  const bool shares = FULL && p.bias && soft && p.renorm;  // a bias may choose experts far below the row's largest: a softmax of the chosen among themselves
#pragma unroll
  for (int r = 0; r < KR; ++r) {
    const bool found = won[r] > -INFINITY && !bad;        // (a row with a NaN may have chosen nothing at all)
    id[r] = found ? id[r] : -1;
    // (with a bias the key is not the logit: read again)
    w[r] = !found ? -INFINITY : FULL && p.bias ? load_logit(row, id[r], p.dtype) : won[r];
  }
  if (shares) {
    most = -INFINITY;
#pragma unroll
    for (int r = 0; r < KR; ++r) {
      if (w[r] - off < -745.0f) w[r] = -INFINITY;          // (masked by the type's lowest value: no score, in 64 bits neither)
      most = __builtin_fmaxf(most, w[r]);
    }
    most = lanes_max<L>(most);
    if (most == -INFINITY) most = 0.0f;
    inv = 1.0f;
  }
#pragma unroll
  for (int r = 0; r < KR; ++r) {
    w[r] = id[r] < 0 ? 0.0f : soft ? exp_below(w[r] - most) * inv : sigmoid(w[r]);
    total += w[r];
  }
  total = lanes_sum<L>(total);
  const float lift = p.renorm ? lift_of(total) : 1.0f;
  const float f = p.renorm ? (total > 0.0f ? p.scale / (total * lift) : 0.0f) : p.scale;
#pragma unroll
  for (int r = 0; r < KR; ++r) {
    const int q = r * L + j;
    if (live && q < p.k) {
      p.weights[token * p.k + q] = bad ? __builtin_nanf("") : w[r] * lift * f;
      p.experts[token * p.k + q] = id[r];
    }
  }
}

// The block of a workgroup.  Neighbours are on one XCD: an expert's counts and places in neighbouring blocks are neighbours in memory, a few bytes from each, and
// meet in its L2.  (65536 x 8 of 128 experts, spread over the XCDs as they come: the choice 18.3 us instead of 16.8, places 8.6 instead of 5.6.)
__device__ __forceinline__ int plan_block() { return xcd_remap(blockIdx.x, gridDim.x, 8); }

// What a workgroup's tokens chose, for the plan: ALONE places the pairs of the only workgroup, otherwise each counts its own per expert.
template <int L, int EPL, bool FULL, bool ALONE>
__global__ __launch_bounds__(256) void route_kernel(RouteParams p, PlanParams q) {
  extern __shared__ __attribute__((aligned(16))) uint8_t moe_smem[];
  constexpr int KR = (TNX_MOE_MAX_TOP_K + L - 1) / L;
  const int tid = threadIdx.x, j = tid % L, slot = tid / L;
  const int block = plan_block();
  int id[KR];
  route_tokens<L, EPL, FULL>(p, tid, (int64_t)block * (256 / L), moe_smem, id);
  if (FULL || EPL > 4) __syncthreads();    // (the keys lay where the plan's memory is)
  if (ALONE) {
    int* ids = (int*)moe_smem;
#pragma unroll
    for (int r = 0; r < KR; ++r)
      if (slot < p.tokens && r * L + j < p.k) ids[slot * p.k + r * L + j] = id[r];
    __syncthreads();
    plan_alone(q, ids, tid);
  } else if (q.fused) {
    const PairBits bits{(unsigned long long*)moe_smem, q.words};
    bits.clear(q.e, tid);
    __syncthreads();
#pragma unroll
    for (int r = 0; r < KR; ++r)
      if ((int64_t)block * (256 / L) + slot < p.tokens && r * L + j < p.k && id[r] >= 0) bits.mark(id[r], slot * p.k + r * L + j);
    __syncthreads();
    for (int e = tid; e < q.e; e += 256) q.counts[q.count_at(e, block)] = bits.count(e);
  }
}

// a thread's pairs of a block, tid, tid + 256, ..: their experts, -1 where there is none.  Anything outside the range is an empty slot.
constexpr int PLAN_BLOCK = 1024;
__device__ __forceinline__ void load_pairs(const PlanParams& p, int block, int tid, int (&mine)[PLAN_BLOCK / 256]) {
  const int64_t first = (int64_t)block * p.block;
#pragma unroll
  for (int u = 0; u < PLAN_BLOCK / 256; ++u) {
    const int i = tid + u * 256;
    mine[u] = -1;
    if (i < p.block && first + i < p.pairs) mine[u] = p.experts[first + i];
  }
}
// into bits
__device__ __forceinline__ void mark_pairs(const PlanParams& p, const PairBits& bits, int tid, int (&mine)[PLAN_BLOCK / 256]) {
  bits.clear(p.e, tid);
  __syncthreads();
#pragma unroll
  for (int u = 0; u < PLAN_BLOCK / 256; ++u) {
    if (mine[u] >= p.e) mine[u] = -1;
    if (mine[u] >= 0) bits.mark(mine[u], tid + u * 256);
  }
  __syncthreads();
}

__global__ __launch_bounds__(256) void plan_alone_kernel(PlanParams p) {
  __shared__ int ids[PLAN_ALONE];
  if ((int)threadIdx.x < PLAN_ALONE) {
    const int e = (int)threadIdx.x < p.pairs ? p.experts[threadIdx.x] : -1;
    ids[threadIdx.x] = e >= 0 && e < p.e ? e : -1;
  }
  __syncthreads();
  plan_alone(p, ids, threadIdx.x);
}

// Many pairs: how many of each block an expert has (with the routing, or here); sums over the blocks, where there are more than a placing
// workgroup should add up by itself; places.
__global__ __launch_bounds__(256) void plan_count_kernel(PlanParams p) {
  extern __shared__ __attribute__((aligned(16))) uint8_t moe_smem[];
  const PairBits bits{(unsigned long long*)moe_smem, p.words};
  const int block = plan_block();
  int mine[PLAN_BLOCK / 256];
  load_pairs(p, block, threadIdx.x, mine);
  mark_pairs(p, bits, threadIdx.x, mine);
  for (int e = threadIdx.x; e < p.e; e += 256) p.counts[p.count_at(e, block)] = bits.count(e);
}

// counts[e][block] -> pairs of e in the blocks before it; a workgroup per expert, eight neighbouring blocks a thread (65536 tokens of 8 pairs: 2048 blocks,
// one turn).  With the experts next to each other instead, 8.5 us, most of it for lines of which a workgroup uses 16 bytes.
__global__ __launch_bounds__(256) void plan_sum_kernel(PlanParams p) {
  __shared__ int waves[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int32_t* c = p.counts + (int64_t)blockIdx.x * p.blocks;
  int carry = 0;
  for (int b0 = 0; b0 < p.blocks; b0 += 2048) {
    int v[8], sum = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = b0 + tid * 8 + i < p.blocks ? c[b0 + tid * 8 + i] : 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += v[i];
    int upto = sum;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int x = __shfl_up(upto, d);
      if (lane >= d) upto += x;
    }
    __syncthreads();
    if (lane == 63) waves[wave] = upto;
    __syncthreads();
    int before = carry + upto - sum;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      if (w < wave) before += waves[w];
      carry += waves[w];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (b0 + tid * 8 + i < p.blocks) c[b0 + tid * 8 + i] = before;
      before += v[i];
    }
  }
  if (tid == 0) p.totals[blockIdx.x] = carry;
}

// SUMMED: the counts are sums over the blocks before already
template <bool SUMMED>
__global__ __launch_bounds__(256) void plan_place_kernel(PlanParams p) {
  extern __shared__ __attribute__((aligned(16))) uint8_t moe_smem[];
  const PairBits bits{(unsigned long long*)moe_smem, p.words};
  int* base = (int*)(moe_smem + (size_t)p.e * p.words * 8);
  int* own = base + p.e;                   // pairs of the expert in the blocks before this one
  const int tid = threadIdx.x, block = plan_block();
  const int64_t first = (int64_t)block * p.block;
  int mine[PLAN_BLOCK / 256];
  load_pairs(p, block, tid, mine);                // (on their way together with the counts)
  if (SUMMED) {
    for (int e = tid; e < p.e; e += 256) {
      base[e] = p.totals[e];
      own[e] = p.counts[p.count_at(e, block)];
    }
  } else {
    // Neighbouring threads have neighbouring experts, and where there are threads left over, several share an expert's blocks.  129 blocks of 60
    // experts: 5.4 us for all of it; with a thread per expert and the counts of an expert's blocks side by side 8.0.
    for (int e = tid; e < p.e; e += 256) base[e] = own[e] = 0;
    __syncthreads();
    const int shares = p.e < 256 ? 256 / p.e : 1;
    for (int i = tid; i < p.e * shares; i += 256) {
      const int share = i / p.e, e = i - share * p.e;
      int all = 0, before = 0;
      for (int b0 = share; b0 < p.blocks; b0 += 16 * shares) {
        int c[16];
#pragma unroll
        for (int u = 0; u < 16; ++u) {
          const int b = b0 + u * shares;
          c[u] = p.counts[(int64_t)(b < p.blocks ? b : b0) * p.e + e];
        }
#pragma unroll
        for (int u = 0; u < 16; ++u) {
          const int b = b0 + u * shares;
          all += b < p.blocks ? c[u] : 0;
          before += b < block ? c[u] : 0;
        }
      }
      atomicAdd(&base[e], all);                            // (in LDS, and of integers: any order gives the same)
      atomicAdd(&own[e], before);
    }
  }
  mark_pairs(p, bits, tid, mine);
  const int total = scan_experts(base, p.e, tid);
  if (block == 0)
    for (int e = tid; e <= p.e; e += 256) p.offsets[e] = e < p.e ? base[e] : total;
#pragma unroll
  for (int u = 0; u < PLAN_BLOCK / 256; ++u) {
    const int i = tid + u * 256, e = mine[u];
    const int64_t pair = first + i;
    if (i >= p.block || pair >= p.pairs) break;
    const int at = e >= 0 ? base[e] + own[e] + bits.rank(e, i) : -1;
    if (e >= 0) p.order[at] = (int32_t)pair;
    p.rows[pair] = at;
    if (pair >= total) p.order[pair] = -1;
  }
}

// Gradient of the logits.  With g_j the gradient of weight j and S the sum of the chosen scores:
//   ds_j = scale g_j, or scale (g_j - sum_i (s_i / S) g_i) / S with renormalised weights
//   softmax: dl_i = s_i (ds_i - sum_j s_j ds_j) over all i; with renormalised weights the sum is zero and s_j / S = weight / scale, so
//            neither the logits nor the other experts enter: dl_j = w_j (g_j - sum_i (w_i / scale) g_i)
//   sigmoid: dl_j = ds_j s_j (1 - s_j), of the chosen alone (renormalised: the quotient s_j / S first, which is at most 1 where 1 / S may be past the range)
// The chosen experts' values go through a row in LDS that starts as zeros, and the row leaves in runs of four.  Bound by writing the
// gradient: 65536 x 128, float32, renormalised softmax: 7.7 us for 33.5 MB.  (Compared one by one with every lane's experts: 13.6 us.)
template <int L, int EPL>
__global__ __launch_bounds__(256) void route_backward_kernel(RouteParams p) {
  extern __shared__ __attribute__((aligned(16))) uint8_t moe_smem[];
  const int tid = threadIdx.x, j = tid % L;
  const int64_t token = (int64_t)blockIdx.x * (256 / L) + tid / L;
  const bool live = token < p.tokens;
  const int64_t t = live ? token : p.tokens - 1;
  const uint8_t* row = p.logits + t * p.stride * (p.dtype == DT_F32 ? 4 : 2);
  const bool soft = p.scoring == TNX_MOE_SOFTMAX, dense = soft && !p.renorm;
  f32x4* mine = (f32x4*)moe_smem + (tid / L) * (EPL / 4 * L);              // [EPL / 4][L] runs of four
#pragma unroll
  for (int i = 0; i < EPL; i += 4) mine[i / 4 * L + j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  float l[EPL];
  float inv = 0.0f;
  if (dense) {
    load_row<L, EPL>(row, p.e, p.dtype, p.vec, j, l);
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < EPL; ++i) top = __builtin_fmaxf(top, l[i]);
    top = lanes_max<L>(top);
    const float off = top == -INFINITY ? 0.0f : top;
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
  int bad_bit = 0;
#pragma unroll
  for (int r = 0; r < KR; ++r) {
    const int q = r * L + j;
    id[r] = -1;
    g[r] = s[r] = w[r] = 0.0f;
    if (q < p.k) {
      w[r] = p.weights[t * p.k + q];
      bad_bit |= w[r] != w[r];
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
  const bool bad = lanes_or<L>(bad_bit) != 0;
  wg = lanes_sum<L>(wg);
  total = lanes_sum<L>(total);
  const float lift = lift_of(total);
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");      // the row is its own lanes' only, and they are in one wave
#pragma unroll
  for (int r = 0; r < KR; ++r) {
    float value;                           // dl (dense: without the common term)
    if (soft && p.renorm) value = w[r] * (g[r] - (p.scale != 0.0f ? wg / p.scale : 0.0f));
    else if (soft) value = w[r] * g[r];                    // s ds: weight is scale s
    else {
      float ds = p.scale * g[r], share = s[r];
      if (p.renorm) {
        const float by = total > 0.0f ? 1.0f / (total * lift) : 0.0f;
        ds = p.scale * (g[r] - wg * lift * by);
        share = s[r] * lift * by;
      }
      value = ds * share * (1.0f - s[r]);
    }
    if (id[r] >= 0) ((float*)mine)[id[r]] = value;
  }
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  if (!live) return;
#pragma unroll
  for (int i = 0; i < EPL; i += 4) {
    const int e = expert_of<L>(i, j);
    f32x4 d = mine[i / 4 * L + j];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      if (dense) d[x] -= l[i + x] * inv * wg;
      if (bad) d[x] = __builtin_nanf("");
    }
    const int64_t at = token * p.e + e;
    if (e + 4 <= p.e && p.vec_out) {
      if (p.dtype == DT_F32) *(f32x4*)((float*)p.grad_logits + at) = d;
      else {
        const uint32_t a = p.dtype == DT_BF16 ? (uint32_t)OutBF16::cvt(d[0]) | (uint32_t)OutBF16::cvt(d[1]) << 16 : (uint32_t)OutF16::cvt(d[0]) | (uint32_t)OutF16::cvt(d[1]) << 16;
        const uint32_t b = p.dtype == DT_BF16 ? (uint32_t)OutBF16::cvt(d[2]) | (uint32_t)OutBF16::cvt(d[3]) << 16 : (uint32_t)OutF16::cvt(d[2]) | (uint32_t)OutF16::cvt(d[3]) << 16;
        *(i32x2*)((uint16_t*)p.grad_logits + at) = i32x2{(int)a, (int)b};
      }
    } else {
#pragma unroll
      for (int x = 0; x < 4; ++x)
        if (e + x < p.e) store_out<float>(p.grad_logits, at + x, d[x], p.dtype);
    }
  }
}

// The join: 16 bytes of a token's output per lane, the top_k rows one after another.  An empty slot counts for nothing, unless its weight is NaN: that
// is a token whose logits were (route_tokens), and its output says so.
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
    const float w = weights[t * k + j];
    if (r < 0 || r >= tokens * k) {
      if (w != w) {
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] = w;
      }
      continue;
    }
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

// Lanes a token: one wave for few tokens or many experts
int route_lanes(int64_t tokens, int e) {
  if (e > 512 || tokens <= 1024) return 64;
  return e <= 128 ? 8 : e <= 256 ? 16 : 32;
}
// Counts of more blocks, or more of them for a thread, are summed by a launch of their own.  A placing workgroup reads 16 at a time, and that takes what
// memory takes: 161 blocks of 512 experts (322 a thread) 17.5 us, summed first 7.3; 111 of 160 (111 a thread) 7.7, 75 of 256 6.4.
constexpr int SUM_BLOCKS = 256, SUM_LOADS = 160;

// The plan's blocks are the pairs of a routing workgroup's 256 / lanes tokens; many tokens at four a workgroup are counted apart, in larger blocks.
void plan_shape(PlanParams* q, int64_t tokens, int k, int e) {
  const int lanes = route_lanes(tokens, e);
  q->pairs = tokens * k;
  q->e = e;
  q->fused = lanes < 64 || tokens <= 1024;
  q->block = q->fused ? 256 / lanes * k : 512;
  static_assert(256 / 8 * TNX_MOE_MAX_TOP_K <= PLAN_BLOCK && 512 <= PLAN_BLOCK, "a thread's pairs");
  q->blocks = (int)((q->pairs + q->block - 1) / q->block);
  q->words = (q->block + 63) / 64;
  q->summed = q->blocks > SUM_BLOCKS || (int64_t)q->blocks * q->e > SUM_LOADS * 256;
}
bool plan_is_alone(const PlanParams& q) { return q.blocks <= 1 && q.pairs <= PLAN_ALONE; }
size_t bits_lds(const PlanParams& q) { return (size_t)q.e * q.words * 8; }

size_t plan_bytes(const PlanParams& q) {
  if (q.pairs <= PLAN_ALONE && q.blocks <= 1) return 0;
  return (size_t)(up16((int64_t)q.e * q.blocks * 4) + up16((int64_t)q.e * 4));
}

int check_plan(const tnx_moe_args* a) {
  if (!a || a->tokens < 0 || a->top_k < 1 || a->num_experts < 1) return TNX_E_INVALID;
  if (a->num_experts > TNX_MOE_MAX_EXPERTS || a->top_k > TNX_MOE_MAX_TOP_K || a->tokens > 0x3fffffff / a->top_k) return TNX_E_UNSUPPORTED;
  if (!a->offsets) return TNX_E_INVALID;
  if (a->tokens > 0 && (!a->experts || !a->order || !a->rows)) return TNX_E_INVALID;
  const size_t need = tnx_moe_workspace_bytes(a->tokens, a->top_k, a->num_experts);
  if (need && (!a->workspace || ((uintptr_t)a->workspace & 15) || a->workspace_bytes < need)) return TNX_E_WORKSPACE;
  return TNX_OK;
}

PlanParams plan_params(const tnx_moe_args* a) {
  PlanParams q;
  q.experts = a->experts; q.offsets = a->offsets; q.order = a->order; q.rows = a->rows;
  plan_shape(&q, a->tokens, a->top_k, a->num_experts);
  q.counts = (int32_t*)a->workspace;
  q.totals = q.counts ? (int32_t*)((uint8_t*)q.counts + up16((int64_t)q.e * q.blocks * 4)) : nullptr;
  return q;
}

// the launches after the counts
int place_pairs(const PlanParams& q, hipStream_t stream) {
  const size_t lds = bits_lds(q) + (size_t)q.e * 8;
  if (q.summed) {
    hipLaunchKernelGGL(plan_sum_kernel, dim3((unsigned)q.e), dim3(256), 0, stream, q);
    const int st = mx_launched();
    if (st) return st;
    hipLaunchKernelGGL((plan_place_kernel<true>), dim3((unsigned)q.blocks), dim3(256), lds, stream, q);
  } else {
    hipLaunchKernelGGL((plan_place_kernel<false>), dim3((unsigned)q.blocks), dim3(256), lds, stream, q);
  }
  return mx_launched();
}

int launch_plan(const PlanParams& q, hipStream_t stream) {
  if (plan_is_alone(q)) {
    hipLaunchKernelGGL(plan_alone_kernel, dim3(1), dim3(256), 0, stream, q);
    return mx_launched();
  }
  hipLaunchKernelGGL(plan_count_kernel, dim3((unsigned)q.blocks), dim3(256), bits_lds(q), stream, q);
  const int st = mx_launched();
  return st ? st : place_pairs(q, stream);
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
  p.runs_at = 0;
  const int es = a->dtype == TNX_F32 ? 4 : 2;
  p.vec = p.e % 4 == 0 && p.stride % 4 == 0 && ((uintptr_t)a->logits & (4 * es - 1)) == 0;
  p.vec_out = p.e % 4 == 0 && ((uintptr_t)a->grad_logits & (4 * es - 1)) == 0;
  return p;
}

template <int L, int EPL> int launch_route(const RouteParams& in, const PlanParams& q, hipStream_t stream) {
  constexpr int TOKENS = 256 / L;
  const unsigned blocks = (unsigned)((in.tokens + TOKENS - 1) / TOKENS);
  const bool groups = in.top_groups < in.groups, full = groups || in.bias, alone = plan_is_alone(q);
  const size_t keys = groups ? (size_t)up16((int64_t)TOKENS * (in.e + TNX_MOE_MAX_GROUPS) * 4) : 0, plan = alone ? PLAN_ALONE * 4 : bits_lds(q);
  RouteParams p = in;
  p.runs_at = (int)keys;
  const size_t choice = keys + (EPL > 4 ? (size_t)EPL * 1024 + TOKENS * TNX_MOE_MAX_TOP_K * 4 : 0), lds = choice > plan ? choice : plan;
  if (full && alone) hipLaunchKernelGGL((route_kernel<L, EPL, true, true>), dim3(blocks), dim3(256), lds, stream, p, q);
  else if (full) hipLaunchKernelGGL((route_kernel<L, EPL, true, false>), dim3(blocks), dim3(256), lds, stream, p, q);
  else if (alone) hipLaunchKernelGGL((route_kernel<L, EPL, false, true>), dim3(blocks), dim3(256), lds, stream, p, q);
  else hipLaunchKernelGGL((route_kernel<L, EPL, false, false>), dim3(blocks), dim3(256), lds, stream, p, q);
  const int st = mx_launched();
  return st || alone ? st : q.fused ? place_pairs(q, stream) : launch_plan(q, stream);
}

template <int L, int EPL> int launch_backward(const RouteParams& p, hipStream_t stream) {
  constexpr int TOKENS = 256 / L;
  hipLaunchKernelGGL((route_backward_kernel<L, EPL>), dim3((unsigned)((p.tokens + TOKENS - 1) / TOKENS)), dim3(256), (size_t)256 * EPL * 4, stream, p);
  return mx_launched();
}

// f(lanes, experts a lane) of the smallest built pair that holds e experts
template <class F> int with_lanes(int lanes, int e, F f) {
  switch (lanes) {
    case 8: return e <= 32 ? f(IntTag<8>(), IntTag<4>()) : e <= 64 ? f(IntTag<8>(), IntTag<8>()) : f(IntTag<8>(), IntTag<16>());
    case 16: return f(IntTag<16>(), IntTag<16>());
    case 32: return f(IntTag<32>(), IntTag<16>());
    default: return e <= 256 ? f(IntTag<64>(), IntTag<4>()) : f(IntTag<64>(), IntTag<16>());
  }
}

}  // namespace

extern "C" size_t tnx_moe_workspace_bytes(int64_t tokens, int32_t top_k, int32_t num_experts) {
  if (tokens <= 0 || top_k <= 0 || num_experts <= 0) return 0;
  PlanParams q;
  plan_shape(&q, tokens, top_k, num_experts);
  return plan_bytes(q);
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
  return with_lanes(route_lanes(p.tokens, p.e), p.e, [&](auto l, auto n) { return launch_route<decltype(l)::value, decltype(n)::value>(p, q, stream); });
}

extern "C" int tnx_moe_route_backward(const tnx_moe_args* a) {
  if (!a || a->tokens < 0 || a->top_k < 1 || a->num_experts < 1) return TNX_E_INVALID;
  if (a->num_experts > TNX_MOE_MAX_EXPERTS || a->top_k > TNX_MOE_MAX_TOP_K || a->tokens > 0x3fffffff / a->top_k) return TNX_E_UNSUPPORTED;
  const int st = check_route(a);
  if (st) return st;
  if (a->tokens == 0) return TNX_OK;
  if (!a->experts || !a->grad || !a->grad_logits) return TNX_E_INVALID;
  const RouteParams p = route_params(a);
  return with_lanes(route_lanes(p.tokens, p.e), p.e, [&](auto l, auto n) {
    return launch_backward<decltype(l)::value, decltype(n)::value>(p, (hipStream_t)a->stream);
  });
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
