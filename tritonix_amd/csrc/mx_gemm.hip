// Products of microscaled 4-bit tensors, plain and grouped by expert, with the gated epilogue.
//
// out[m, n] = sum over blocks of 32 k of 2^(sa + sb) * (qa . qb): the matrix instruction of CDNA4 for 4-bit floats takes a block per lane
// with the block's scale, so the scales cost no instruction of their own.  The weights are the instruction's first operand:
// a lane then holds four neighbouring columns of one output row, which is what the gate and the stores want.
//
// The order of the blocks along k is free as long as both operands keep it.  A lane half (32x32x64: lanes 0-31 and
// 32-63) takes the blocks 4 h .. 4 h + 3 of a slab of 256 in four steps: the four scales are then one word, of which each step names a byte.
#include <hip/hip_runtime.h>

#include "../../include/tritonix_hip.h"
#include "mx.h"

using namespace tnx;

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));

struct MxParams {
  const uint8_t *a, *as, *b, *bs;
  uint8_t* out;
  const int32_t *offsets, *order;
  int64_t ldo, b_expert, bs_expert;        // elements; bytes from expert to expert
  int m, n, slabs, a_rows;
  int experts, tiles_n, tiles_m;           // experts == 0: one matrix; tiles_m: of one matrix
  FastDiv top_k;
  int out_dtype, epi;
};

__device__ __forceinline__ f32x16 mfma32(i32x4 a, i32x4 b, f32x16 c, int sa, int sb, int step) {
  const i32x8 a8 = {a[0], a[1], a[2], a[3], 0, 0, 0, 0}, b8 = {b[0], b[1], b[2], b[3], 0, 0, 0, 0};
  switch (step) {                          // (a constant after unrolling: the byte of the scale words is part of the instruction)
    case 0: return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a8, b8, c, 4, 4, 0, sa, 0, sb);
    case 1: return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a8, b8, c, 4, 4, 1, sa, 1, sb);
    case 2: return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a8, b8, c, 4, 4, 2, sa, 2, sb);
    default: return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a8, b8, c, 4, 4, 3, sa, 3, sb);
  }
}
template <int STEP> __device__ __forceinline__ f32x4 mfma16(i32x4 a, i32x4 b, f32x4 c, int sa, int sb) {
  const i32x8 a8 = {a[0], a[1], a[2], a[3], 0, 0, 0, 0}, b8 = {b[0], b[1], b[2], b[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a8, b8, c, 4, 4, STEP, sa, STEP, sb);
}

// 16 (4) bytes per lane from a 64-bit address of its own to LDS (base + lane * 16 or 4): see dma16 for M0
__device__ __forceinline__ void dma16_at(const uint8_t* src, uint32_t lds_base) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(__builtin_amdgcn_readfirstlane(lds_base)), "v"(src) : "memory");
}
__device__ __forceinline__ void dma16_from(const uint8_t* sbase, uint32_t voff, uint32_t lds_base) {
  dma16(sbase, voff, __builtin_amdgcn_readfirstlane(lds_base));
}
__device__ __forceinline__ void dma4_at(const uint8_t* src, uint32_t lds_base) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" : : "s"(__builtin_amdgcn_readfirstlane(lds_base)), "v"(src) : "memory");
}

// Which rows a workgroup has: one matrix, or the tile-th tile of BM rows over all experts, each expert's rows cut on their
// own.  All 64 lanes take part; the answer is uniform.  expert == experts: rows past the last expert's; false: no such tile.
struct RowTile { int expert, row0, rows; };

template <int BM> __device__ __forceinline__ int expert_tiles(const MxParams& p, int lane) {
  int total = 0;
  for (int e0 = 0; e0 <= p.experts; e0 += 64) {
    const int e = e0 + lane;
    int t = 0;
    if (e < p.experts) t = (p.offsets[e + 1] - p.offsets[e] + BM - 1) / BM;
    else if (e == p.experts) t = (p.m - p.offsets[e] + BM - 1) / BM;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) t += __shfl_xor(t, d);
    total += t;
  }
  return __builtin_amdgcn_readfirstlane(total);
}

template <int BM> __device__ __forceinline__ bool find_rows(const MxParams& p, int tile, int lane, RowTile* out) {
  int before = 0;
  for (int e0 = 0; e0 <= p.experts; e0 += 64) {
    const int e = e0 + lane;
    int lo = 0, hi = 0;
    if (e <= p.experts) { lo = p.offsets[e]; hi = e < p.experts ? p.offsets[e + 1] : p.m; }
    const int t = (hi - lo + BM - 1) / BM;
    int upto = t;                                        // tiles of the lanes up to this one
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int v = __shfl_up(upto, d);
      if (lane >= d) upto += v;
    }
    const int first = before + upto - t;
    const unsigned long long mine = __ballot(tile >= first && tile < first + t);
    if (mine) {
      const int l = __ffsll(mine) - 1;
      const int lo_l = __shfl(lo, l), hi_l = __shfl(hi, l), first_l = __shfl(first, l);
      const int row0 = lo_l + (tile - first_l) * BM;
      out->expert = __builtin_amdgcn_readfirstlane(e0 + l);
      out->row0 = __builtin_amdgcn_readfirstlane(row0);
      out->rows = __builtin_amdgcn_readfirstlane(hi_l - row0 < BM ? hi_l - row0 : BM);
      return true;
    }
    before += __shfl(upto, 63);
  }
  return false;
}

// row of a that row r of the product takes
__device__ __forceinline__ int source_row(const MxParams& p, int r) {
  if (!p.order) return r;
  const int pair = p.order[r], t = (int)fd_div((uint32_t)(pair < 0 ? 0 : pair), p.top_k);
  return t < p.a_rows ? t : p.a_rows - 1;
}

// `count` of four neighbouring columns of a row (two with the gate), as many as there are
__device__ __forceinline__ void store_columns(const MxParams& p, int64_t row, int col, int cols, const f32x4& v) {
  float o[4];
  int c = col, n = 4;
  if (p.epi != EPI_NONE) {
    o[0] = glu_gate<true>(v[0], p.epi) * v[1];
    o[1] = glu_gate<true>(v[2], p.epi) * v[3];
    o[2] = o[3] = 0.0f;
    c = col >> 1; n = 2; cols >>= 1;
  } else {
    o[0] = v[0]; o[1] = v[1]; o[2] = v[2]; o[3] = v[3];
  }
  const int64_t at = row * p.ldo + c;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < n && c + i < cols) store_out<float>(p.out, at + i, o[i], p.out_dtype);
}

// ------------------------------------------------------------------------------------------------------------------
// Tiles: BN columns of the output (rows of the weights) x BM rows, four waves of half of each, slabs of 256 k in two LDS
// buffers filled by direct loads.  Slab s + 1 has to be there, and slab s be read by all, when the last step of slab s
// begins: one barrier per slab, its wait hidden behind that step's products.
template <int BN, int BM> struct MxTile {
  static constexpr int WTN = BN / 2, WTM = BM / 2, TN = WTN / 32, TM = WTM / 32;
  static constexpr int B_BYTES = BN * MX_ROWB, A_BYTES = BM * MX_ROWB, BS_BYTES = BN * MX_SCALEB, AS_BYTES = BM * MX_SCALEB;
  static constexpr int SLOT = B_BYTES + A_BYTES + BS_BYTES + AS_BYTES;
  static constexpr int B_OPS = B_BYTES / 4096, A_OPS = A_BYTES / 4096;      // 16-byte loads per lane and slab
  // the epilogue's strip of a wave: 32 rows of its columns in binary32 at most
  static constexpr int PITCH = WTN * 4 + 16, STRIP = 32 * PITCH;
  static constexpr int LDS = 2 * SLOT > 4 * STRIP ? 2 * SLOT : 4 * STRIP;
};

template <int BN, int BM, bool EXPERTS>
__global__ __launch_bounds__(256) void mx_tile_kernel(MxParams p) {
  typedef MxTile<BN, BM> C;
  extern __shared__ __attribute__((aligned(1024))) uint8_t mx_smem[];
  const uint32_t lds0 = (uint32_t)(uintptr_t)(uint8_t __attribute__((address_space(3)))*)mx_smem;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  RowTile rt;
  int tn;
  if (EXPERTS) {
    // neighbouring ids share the rows of a; an XCD has a run of them, so an expert's weights meet its tiles in one L2
    const int tiles = expert_tiles<BM>(p, lane) * p.tiles_n;
    if ((int)blockIdx.x >= tiles) return;
    const int id = xcd_remap(blockIdx.x, tiles, 8);
    const int tm = id / p.tiles_n;
    tn = id - tm * p.tiles_n;
    if (!find_rows<BM>(p, tm, lane, &rt)) return;
  } else {
    const int id = xcd_remap(blockIdx.x, p.tiles_m * p.tiles_n, 8);
    int tm;
    swizzle2d(id / p.tiles_n, id % p.tiles_n, p.tiles_m, p.tiles_n, 8, &tm, &tn);
    rt.expert = 0;
    rt.row0 = tm * BM;
    rt.rows = p.m - rt.row0 < BM ? p.m - rt.row0 : BM;
  }
  const int n0 = tn * BN, ncols = p.n - n0 < BN ? p.n - n0 : BN;
  if (EXPERTS && rt.expert == p.experts) {               // rows of no expert
    const int c0 = p.epi != EPI_NONE ? n0 / 2 : n0, nc = p.epi != EPI_NONE ? ncols / 2 : ncols;
    for (int i = tid; i < rt.rows * nc; i += 256) store_out<float>(p.out, (int64_t)(rt.row0 + i / nc) * p.ldo + c0 + i % nc, 0.0f, p.out_dtype);
    return;
  }
  const uint8_t* b = uniform_ptr(p.b + (int64_t)rt.expert * p.b_expert + (int64_t)n0 * p.slabs * MX_ROWB);
  const uint8_t* bs = uniform_ptr(p.bs + (int64_t)rt.expert * p.bs_expert + (int64_t)(n0 >> 5) * p.slabs * 256);

  // Direct loads.  Instruction q of wave w fills rows 8 (4 q + w) .. + 7 of a side, lane l the 16-byte place l % 8 of row l / 8,
  // which holds the chunk place ^ (row / 2 % 8): a fragment read (16 lanes a cycle, rows {0-3, 12-15, 20-27} or the others, one chunk)
  // then falls on 16 different places of 256 bytes.  Rows past the end are the last row again; nobody stores what they give.
  uint32_t b_off[C::B_OPS];
#pragma unroll
  for (int q = 0; q < C::B_OPS; ++q) {
    const int row = 8 * (4 * q + wave) + (lane >> 3), chunk = (lane & 7) ^ ((row >> 1) & 7);
    b_off[q] = (uint32_t)(row < ncols ? row : ncols - 1) * (uint32_t)(p.slabs * MX_ROWB) + chunk * 16;
  }
  uint32_t a_off[C::A_OPS];
  const uint8_t* a_at[EXPERTS ? C::A_OPS : 1];
  const uint8_t* a = nullptr;
  if (EXPERTS) {
#pragma unroll
    for (int q = 0; q < C::A_OPS; ++q) {
      const int row = 8 * (4 * q + wave) + (lane >> 3), chunk = (lane & 7) ^ ((row >> 1) & 7);
      a_at[q] = p.a + (int64_t)source_row(p, rt.row0 + (row < rt.rows ? row : rt.rows - 1)) * p.slabs * MX_ROWB + chunk * 16;
    }
  } else {
    a = uniform_ptr(p.a + (int64_t)rt.row0 * p.slabs * MX_ROWB);
#pragma unroll
    for (int q = 0; q < C::A_OPS; ++q) {
      const int row = 8 * (4 * q + wave) + (lane >> 3), chunk = (lane & 7) ^ ((row >> 1) & 7);
      a_off[q] = (uint32_t)(row < rt.rows ? row : rt.rows - 1) * (uint32_t)(p.slabs * MX_ROWB) + chunk * 16;
    }
  }
  // Scales: 16 lanes a group of 32 rows (256 bytes); a wave's instruction takes four groups.  BN / 128 instructions of 1 KiB in all.  With
  // experts the rows of a lie anywhere: two words per row, 32 rows an instruction.
  constexpr int BS_OPS = (C::BS_BYTES + 1023) / 1024, AS_OPS = EXPERTS ? C::AS_BYTES / 256 : (C::AS_BYTES + 1023) / 1024;
  uint32_t bs_off[BS_OPS];
#pragma unroll
  for (int q = 0; q < BS_OPS; ++q) {
    const int last = (ncols - 1) >> 5, g = 4 * q + (lane >> 4);
    bs_off[q] = (uint32_t)(g < last ? g : last) * (uint32_t)(p.slabs * 256) + (lane & 15) * 16;
  }
  uint32_t as_off[EXPERTS ? 1 : AS_OPS];
  const uint8_t* as_at[EXPERTS ? (AS_OPS + 3) / 4 : 1];
  const uint8_t* as = nullptr;
  if (EXPERTS) {
#pragma unroll
    for (int q = 0; q < (AS_OPS + 3) / 4; ++q) {
      const int row = 32 * (4 * q + wave) + (lane >> 1);
      const int src = source_row(p, rt.row0 + (row < rt.rows ? row : rt.rows - 1));
      as_at[q] = p.as + mx_scale_at(src, 0, p.slabs) + (lane & 1) * 4;
    }
  } else {
    as = uniform_ptr(p.as + (int64_t)(rt.row0 >> 5) * p.slabs * 256);
#pragma unroll
    for (int q = 0; q < AS_OPS; ++q) {
      const int last = (rt.rows - 1) >> 5, g = 4 * q + (lane >> 4);
      as_off[q] = (uint32_t)(g < last ? g : last) * (uint32_t)(p.slabs * 256) + (lane & 15) * 16;
    }
  }

  auto fetch = [&](int slab) __attribute__((always_inline)) {
    const uint32_t slot = lds0 + (slab & 1) * C::SLOT;
    const uint8_t* bk = b + (int64_t)slab * MX_ROWB;
#pragma unroll
    for (int q = 0; q < C::B_OPS; ++q) dma16_from(bk, b_off[q], slot + (4 * q + wave) * 1024);
    if (EXPERTS) {
#pragma unroll
      for (int q = 0; q < C::A_OPS; ++q) dma16_at(a_at[q] + (int64_t)slab * MX_ROWB, slot + C::B_BYTES + (4 * q + wave) * 1024);
    } else {
      const uint8_t* ak = a + (int64_t)slab * MX_ROWB;
#pragma unroll
      for (int q = 0; q < C::A_OPS; ++q) dma16_from(ak, a_off[q], slot + C::B_BYTES + (4 * q + wave) * 1024);
    }
    const uint32_t sb = slot + C::B_BYTES + C::A_BYTES, sa = sb + C::BS_BYTES;
    const uint8_t* bsk = bs + (int64_t)slab * 256;
    // (every branch below is uniform over the wave)
#pragma unroll
    for (int q = 0; q < BS_OPS; ++q)
      if (wave == q) { if (C::BS_BYTES >= 1024 || lane < C::BS_BYTES / 16) dma16_from(bsk, bs_off[q], sb + q * 1024); }
    if (EXPERTS) {
#pragma unroll
      for (int q = 0; q < (AS_OPS + 3) / 4; ++q)
        if (AS_OPS >= 4 || wave < AS_OPS) dma4_at(as_at[q] + (int64_t)slab * 256, sa + (4 * q + wave) * 256);
    } else {
      const uint8_t* ask = as + (int64_t)slab * 256;
#pragma unroll
      for (int q = 0; q < AS_OPS; ++q)
        if (wave == 3 - q) { if (C::AS_BYTES >= 1024 || lane < C::AS_BYTES / 16) dma16_from(ask, as_off[q], sa + q * 1024); }
    }
  };

  const int wn = (wave >> 1) * C::WTN, wm = (wave & 1) * C::WTM, half = lane >> 5, r32 = lane & 31;
  // place of chunk 4 half + step in this lane's row
  const uint32_t place = (uint32_t)r32 * MX_ROWB + (((4 * half) ^ ((r32 >> 1) & 7)) << 4);
  f32x16 acc[C::TN][C::TM];
#pragma unroll
  for (int i = 0; i < C::TN; ++i)
#pragma unroll
    for (int j = 0; j < C::TM; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;
  i32x4 fb[2][C::TN], fa[2][C::TM];
  int sb[2][C::TN], sa[2][C::TM];
  auto read_step = [&](int slab, int step, int set) __attribute__((always_inline)) {
    const uint32_t at = lds0 + (slab & 1) * C::SLOT + (place ^ (step << 4));
#pragma unroll
    for (int i = 0; i < C::TN; ++i) fb[set][i] = *TNX_LDS(i32x4, at + (wn + 32 * i) * MX_ROWB);
#pragma unroll
    for (int j = 0; j < C::TM; ++j) fa[set][j] = *TNX_LDS(i32x4, at + C::B_BYTES + (wm + 32 * j) * MX_ROWB);
  };
  auto read_scales = [&](int slab, int set) __attribute__((always_inline)) {
    const uint32_t at = lds0 + (slab & 1) * C::SLOT + C::B_BYTES + C::A_BYTES + r32 * MX_SCALEB + half * 4;
#pragma unroll
    for (int i = 0; i < C::TN; ++i) sb[set][i] = *TNX_LDS(int, at + (wn + 32 * i) * MX_SCALEB);
#pragma unroll
    for (int j = 0; j < C::TM; ++j) sa[set][j] = *TNX_LDS(int, at + C::BS_BYTES + (wm + 32 * j) * MX_SCALEB);
  };

  const int slabs = p.slabs;
  fetch(0);
  TNX_WAIT_VM(0);
  __syncthreads();
  if (slabs > 1) fetch(1);
  read_scales(0, 0);
  read_step(0, 0, 0);
  for (int s = 0; s < slabs; ++s) {
#pragma unroll
    for (int step = 0; step < 4; ++step) {
      if (step < 3) read_step(s, step + 1, (step + 1) & 1);
      constexpr int HALF = C::TN * C::TM / 2;
#pragma unroll
      for (int e = 0; e < C::TN * C::TM; ++e) {
        if (step == 3 && e == HALF) {
          // The fragments of this slab are in registers and the loads of the next one have landed, in every wave.  (After the
          // last slab the reads fetch what the other buffer still holds, and nothing uses it.)
          __builtin_amdgcn_sched_barrier(0);
          asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
          __builtin_amdgcn_s_barrier();
          asm volatile("" ::: "memory");
          read_step(s + 1, 0, 0);
          read_scales(s + 1, 1);
          if (s + 2 < slabs) fetch(s + 2);
          __builtin_amdgcn_sched_barrier(0);
        }
        const int i = e / C::TM, j = (i & 1) ? C::TM - 1 - e % C::TM : e % C::TM;
        acc[i][j] = mfma32(fb[step & 1][i], fa[step & 1][j], acc[i][j], sb[0][i], sa[0][j], step);
      }
    }
#pragma unroll
    for (int i = 0; i < C::TN; ++i) sb[0][i] = sb[1][i];
#pragma unroll
    for (int j = 0; j < C::TM; ++j) sa[0][j] = sa[1][j];
  }

  // Epilogue.  A lane has, of output row lane % 32 of each 32x32 product, the columns 8 q + 4 half + 0 .. 3: they go to the wave's own strip of
  // LDS (rows of outputs, gated and rounded), and leave as 16-byte pieces of whole rows.
  __syncthreads();
  const uint32_t strip = lds0 + wave * C::STRIP;
  const bool glu = p.epi != EPI_NONE;
  const int es = p.out_dtype == DT_F32 ? 4 : 2;
  const int ocols = glu ? C::WTN / 2 : C::WTN;
  const int row_bytes = ocols * es, pieces = row_bytes / 16;          // a power of two
  const int left_cols = (glu ? ncols / 2 : ncols) - (glu ? wn / 2 : wn);
  const int64_t col0 = (glu ? n0 / 2 : n0) + (glu ? wn / 2 : wn);
  const int shift = 31 - __clz(pieces);
#pragma unroll
  for (int j = 0; j < C::TM; ++j) {
#pragma unroll
    for (int i = 0; i < C::TN; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float v0 = acc[i][j][4 * q], v1 = acc[i][j][4 * q + 1], v2 = acc[i][j][4 * q + 2], v3 = acc[i][j][4 * q + 3];
        const int c = 32 * i + 8 * q + 4 * half;
        const uint32_t at = strip + r32 * C::PITCH;
        if (glu) {
          const float o0 = glu_gate<true>(v0, p.epi) * v1, o1 = glu_gate<true>(v2, p.epi) * v3;
          if (es == 4) *TNX_LDS(i32x2, at + c * 2) = i32x2{__builtin_bit_cast(int, o0), __builtin_bit_cast(int, o1)};
          else if (p.out_dtype == DT_BF16) *TNX_LDS(int, at + c) = (int)((uint32_t)OutBF16::cvt(o0) | (uint32_t)OutBF16::cvt(o1) << 16);
          else *TNX_LDS(int, at + c) = (int)((uint32_t)OutF16::cvt(o0) | (uint32_t)OutF16::cvt(o1) << 16);
        } else if (es == 4) {
          *TNX_LDS(i32x4, at + c * 4) = i32x4{__builtin_bit_cast(int, v0), __builtin_bit_cast(int, v1), __builtin_bit_cast(int, v2), __builtin_bit_cast(int, v3)};
        } else if (p.out_dtype == DT_BF16) {
          *TNX_LDS(i32x2, at + c * 2) = i32x2{(int)((uint32_t)OutBF16::cvt(v0) | (uint32_t)OutBF16::cvt(v1) << 16),
                                              (int)((uint32_t)OutBF16::cvt(v2) | (uint32_t)OutBF16::cvt(v3) << 16)};
        } else {
          *TNX_LDS(i32x2, at + c * 2) = i32x2{(int)((uint32_t)OutF16::cvt(v0) | (uint32_t)OutF16::cvt(v1) << 16),
                                              (int)((uint32_t)OutF16::cvt(v2) | (uint32_t)OutF16::cvt(v3) << 16)};
        }
      }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the strip is the wave's own: its LDS operations are in order
    const int m_left = rt.rows - (wm + 32 * j);
    for (int t = lane; t < 32 * pieces; t += 64) {
      const int row = t >> shift, piece = t & (pieces - 1), c = piece * 16 / es;
      const i32x4 v = *TNX_LDS(i32x4, strip + row * C::PITCH + piece * 16);
      if (row >= m_left || c >= left_cols) continue;
      uint8_t* d = p.out + ((int64_t)(rt.row0 + wm + 32 * j + row) * p.ldo + col0 + c) * es;
      if (c + 16 / es <= left_cols) *(i32x4_loose*)d = v;
      else {
        for (int e = 0; c + e < left_cols; ++e) {        // (constant places of v only: no array in scratch memory)
          const uint32_t w = (uint32_t)(e * es < 4 ? v[0] : e * es < 8 ? v[1] : e * es < 12 ? v[2] : v[3]);
          if (es == 4) ((uint32_t*)d)[e] = w;
          else ((uint16_t*)d)[e] = (uint16_t)(e & 1 ? w >> 16 : w);
        }
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
}

// ------------------------------------------------------------------------------------------------------------------
// Few rows: bound by streaming the weights, so nothing goes through LDS on the way in.  A workgroup has 16 NT rows of the
// weights and up to 16 MT rows of a; its eight waves each take every eighth slab, all of a turn's loads in flight together, and meet in
// LDS.  16x16x128 instructions: lane group g (lane / 16) takes the blocks 2 g and 2 g + 1 of a slab, 32 neighbouring bytes and
// two neighbouring scales.
constexpr int FEW_WAVES = 8;

template <int NT, int MT, bool EXPERTS>
__global__ __launch_bounds__(FEW_WAVES * 64) void mx_few_kernel(MxParams p) {
  __shared__ __attribute__((aligned(16))) f32x4 part[FEW_WAVES][NT * MT][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  RowTile rt;
  if (EXPERTS) {
    if (!find_rows<16 * MT>(p, blockIdx.y, lane, &rt)) return;
  } else {
    rt.expert = 0;
    rt.row0 = blockIdx.y * (16 * MT);
    rt.rows = p.m - rt.row0 < 16 * MT ? p.m - rt.row0 : 16 * MT;
  }
  const int n0 = blockIdx.x * (16 * NT);
  const int row = lane & 15, g = lane >> 4;
  f32x4 acc[NT][MT];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  if (!EXPERTS || rt.expert < p.experts) {
    const uint8_t* b = p.b + (int64_t)rt.expert * p.b_expert;
    const uint8_t* bs = p.bs + (int64_t)rt.expert * p.bs_expert;
    const uint8_t *b_at[NT], *bs_at[NT], *a_at[MT], *as_at[MT];
    bool a_have[MT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int n = n0 + 16 * i + row < p.n ? n0 + 16 * i + row : p.n - 1;
      b_at[i] = b + (int64_t)n * p.slabs * MX_ROWB + 32 * g;
      bs_at[i] = bs + mx_scale_at(n, 0, p.slabs) + 2 * g;
    }
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      a_have[j] = 16 * j + row < rt.rows;
      const int src = EXPERTS ? source_row(p, rt.row0 + (a_have[j] ? 16 * j + row : 0)) : rt.row0 + (a_have[j] ? 16 * j + row : 0);
      a_at[j] = p.a + (int64_t)src * p.slabs * MX_ROWB + 32 * g;
      as_at[j] = p.as + mx_scale_at(src, 0, p.slabs) + 2 * g;
    }
    constexpr int DEPTH = 4;                             // slabs of a turn
    for (int s0 = wave; s0 < p.slabs; s0 += FEW_WAVES * DEPTH) {
      i32x4 fb[DEPTH][NT][2];
      int sb[DEPTH][NT];
#pragma unroll
      for (int d = 0; d < DEPTH; ++d) {
        const int64_t s = s0 + d * FEW_WAVES;
        if (s < p.slabs) {
#pragma unroll
          for (int i = 0; i < NT; ++i) {
            fb[d][i][0] = *(const i32x4*)(b_at[i] + s * MX_ROWB);
            fb[d][i][1] = *(const i32x4*)(b_at[i] + s * MX_ROWB + 16);
            sb[d][i] = *(const uint16_t*)(bs_at[i] + s * 256);
          }
        }
      }
#pragma unroll
      for (int d = 0; d < DEPTH; ++d) {
        const int64_t s = s0 + d * FEW_WAVES;
        if (s < p.slabs) {
#pragma unroll
          for (int j = 0; j < MT; ++j) {
            i32x4 fa0 = {0, 0, 0, 0}, fa1 = {0, 0, 0, 0};
            int sa = 0x7f7f;
            if (a_have[j]) {
              fa0 = *(const i32x4*)(a_at[j] + s * MX_ROWB);
              fa1 = *(const i32x4*)(a_at[j] + s * MX_ROWB + 16);
              sa = *(const uint16_t*)(as_at[j] + s * 256);
            }
#pragma unroll
            for (int i = 0; i < NT; ++i) {
              acc[i][j] = mfma16<0>(fb[d][i][0], fa0, acc[i][j], sb[d][i], sa);
              acc[i][j] = mfma16<1>(fb[d][i][1], fa1, acc[i][j], sb[d][i], sa);
            }
          }
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) part[wave][i * MT + j][lane] = acc[i][j];
  __syncthreads();
  for (int t = tid; t < NT * MT * 64; t += FEW_WAVES * 64) {
    const int ij = t >> 6, l = t & 63;
    f32x4 v = part[0][ij][l];
#pragma unroll
    for (int w = 1; w < FEW_WAVES; ++w) v += part[w][ij][l];
    const int r = 16 * (ij % MT) + (l & 15), c = n0 + 16 * (ij / MT) + 4 * (l >> 4);
    if (r < rt.rows && c < p.n) store_columns(p, rt.row0 + r, c, p.n, v);
  }
}

// ------------------------------------------------------------------------------------------------------------------
template <int BN, int BM, bool EXPERTS> int launch_tile(MxParams p, int64_t row_tiles, hipStream_t stream) {
  typedef MxTile<BN, BM> C;
  p.tiles_n = (p.n + BN - 1) / BN;
  p.tiles_m = (p.m + BM - 1) / BM;
  const int64_t grid = row_tiles * p.tiles_n;
  if (grid > 0x7fffffff) return TNX_E_UNSUPPORTED;
  hipLaunchKernelGGL((mx_tile_kernel<BN, BM, EXPERTS>), dim3((unsigned)grid), dim3(256), C::LDS, stream, p);
  return mx_launched();
}

template <int NT, int MT, bool EXPERTS> int launch_few(MxParams p, int64_t row_tiles, hipStream_t stream) {
  if (row_tiles > 65535) return TNX_E_UNSUPPORTED;
  hipLaunchKernelGGL((mx_few_kernel<NT, MT, EXPERTS>), dim3((unsigned)((p.n + 16 * NT - 1) / (16 * NT)), (unsigned)row_tiles), dim3(FEW_WAVES * 64), 0,
                     stream, p);
  return mx_launched();
}

template <bool EXPERTS> int launch(const MxParams& p, hipStream_t stream) {
  // rows that a workgroup can expect, and how many tiles of BM there are at most
  const int64_t each = EXPERTS ? (p.m + p.experts - 1) / p.experts : p.m;
  auto tiles = [&](int bm) { return EXPERTS ? (int64_t)p.m / bm + 1 + (p.experts < p.m ? p.experts : p.m) : ((int64_t)p.m + bm - 1) / bm; };
  if (each <= 16 && tiles(16) <= 65535) return launch_few<1, 1, EXPERTS>(p, tiles(16), stream);
  if (each <= 32 && tiles(32) <= 65535) return launch_few<2, 2, EXPERTS>(p, tiles(32), stream);
  if (each <= 64 && tiles(64) <= 65535) return launch_few<2, 4, EXPERTS>(p, tiles(64), stream);
  const int64_t big = tiles(256) * ((p.n + 255) / 256);
  if (big >= 200) return launch_tile<256, 256, EXPERTS>(p, tiles(256), stream);
  const int64_t mid = tiles(128) * ((p.n + 127) / 128);
  if (mid >= 256) return launch_tile<128, 128, EXPERTS>(p, tiles(128), stream);
  return launch_tile<64, 64, EXPERTS>(p, tiles(64), stream);
}

}  // namespace

extern "C" int tnx_mx_gemm(const tnx_mx_gemm_args* a) {
  if (!a || a->m < 0 || a->n < 0 || a->k < 0 || a->experts < 0 || a->epilogue < TNX_EPI_NONE || a->epilogue > TNX_EPI_GLU_IDENTITY) return TNX_E_INVALID;
  if (a->m == 0 || a->n == 0) return TNX_OK;
  if (a->out_dtype != TNX_BF16 && a->out_dtype != TNX_F16 && a->out_dtype != TNX_F32) return TNX_E_UNSUPPORTED;
  if (a->epilogue != TNX_EPI_NONE && a->n % 2) return TNX_E_UNSUPPORTED;
  const int64_t cols = a->epilogue != TNX_EPI_NONE ? a->n / 2 : a->n;
  if (!a->out || a->stride_out < cols || ((uintptr_t)a->out & (a->out_dtype == TNX_F32 ? 3 : 1))) return TNX_E_INVALID;
  if (a->k == 0 || a->k > TNX_MX_MAX_K || a->m > 0x3fffffff || a->n > 0x3fffffff || a->a_rows > 0x3fffffff) return TNX_E_UNSUPPORTED;
  if (!a->a_codes || !a->a_scales || !a->b_codes || !a->b_scales) return TNX_E_INVALID;
  if (((uintptr_t)a->a_codes | (uintptr_t)a->a_scales | (uintptr_t)a->b_codes | (uintptr_t)a->b_scales) & 15) return TNX_E_INVALID;
  if (a->experts > 0 ? (!a->offsets || a->experts > TNX_MOE_MAX_EXPERTS) : (a->offsets || a->order)) return TNX_E_INVALID;
  if (a->order ? (a->top_k < 1 || a->a_rows < 1) : a->a_rows != a->m) return TNX_E_INVALID;
  MxParams p;
  p.a = (const uint8_t*)a->a_codes; p.as = (const uint8_t*)a->a_scales;
  p.b = (const uint8_t*)a->b_codes; p.bs = (const uint8_t*)a->b_scales;
  p.out = (uint8_t*)a->out;
  p.offsets = a->offsets; p.order = a->order;
  p.ldo = a->stride_out;
  p.b_expert = mx_code_bytes(a->n, a->k);
  p.bs_expert = mx_scale_bytes(a->n, a->k);
  p.m = (int)a->m; p.n = (int)a->n; p.slabs = (int)mx_slabs(a->k); p.a_rows = (int)a->a_rows;
  p.experts = a->experts; p.tiles_n = p.tiles_m = 0;
  p.top_k = make_fastdiv((uint32_t)(a->order ? a->top_k : 1));
  p.out_dtype = a->out_dtype; p.epi = a->epilogue;
  return a->experts > 0 ? launch<true>(p, (hipStream_t)a->stream) : launch<false>(p, (hipStream_t)a->stream);
}
