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
  int64_t lda;                             // few rows as floats: their stride, type and k; parts of k (log2)
  int a_dtype, k, wk_log;
  int part_slabs;                          // k cut in parts of so many slabs, an even number
  bool stream_b;                           // the weights are read by one tile of rows each: past the caches (tiles of up to 128 rows)
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

// 16 bytes per lane from a 64-bit address of its own to LDS (base + lane * 16): see dma16 for M0
__device__ __forceinline__ void dma16_at(const uint8_t* src, uint32_t lds_base) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(__builtin_amdgcn_readfirstlane(lds_base)), "v"(src) : "memory");
}
__device__ __forceinline__ void dma16_from(const uint8_t* sbase, uint32_t voff, uint32_t lds_base) {
  dma16(sbase, voff, __builtin_amdgcn_readfirstlane(lds_base));
}
// Which rows a workgroup has: one matrix, or the tile-th tile of BM rows over all experts, each expert's rows cut on their
// own.  All 64 lanes take part; the answer is uniform.  expert == experts: rows past the last expert's; false: no such tile.
struct RowTile { int expert, row0, rows; };

// (Offsets are taken inside [0, m] and as not decreasing, whatever they hold: no row outside of the product is touched.)
__device__ __forceinline__ int rows_upto(const MxParams& p, int e) {
  const int v = e > p.experts ? p.m : p.offsets[e];
  return v < 0 ? 0 : v < p.m ? v : p.m;
}

template <int BM> __device__ __forceinline__ int tiles_between(int lo, int hi) { return hi > lo ? (hi - lo + BM - 1) / BM : 0; }

template <int BM> __device__ __forceinline__ int expert_tiles(const MxParams& p, int lane) {
  int total = 0;
  for (int e0 = 0; e0 <= p.experts; e0 += 64) {
    const int e = e0 + lane;
    int t = 0;
    if (e <= p.experts) t = tiles_between<BM>(rows_upto(p, e), rows_upto(p, e + 1));
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
    if (e <= p.experts) { lo = rows_upto(p, e); hi = rows_upto(p, e + 1); }
    const int t = tiles_between<BM>(lo, hi);
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

// act(g) * l, to the bits of the tiles of wider types (glu_gate): a result of 16 bits from the reciprocal corrected to the division's, one of 32 from the
// division.  Without branches, which would take the gates of a product one by one: whatever the activation, it is a factor of 1 or the sigmoid and one of 1 or
// the gate.  SHORT: SiLU of a g that is not below -66, so that 1 + exp(-g) is where the correction needs neither a scale nor a bound and is two
// instructions.  The empty asm makes the product a binary32 number, which is then rounded: the compiler takes it and the conversion to float16 together in
// some of the kernels, and the same operands would give them other bits.
template <bool ROUNDED, bool SHORT> __device__ __forceinline__ float gated(float g, float l, int epi) {
  const float d = 1.0f + __expf(-g);
  float v;
  if (SHORT) {
    const float r = __builtin_amdgcn_rcpf(d);
    v = g * __builtin_fmaf(__builtin_fmaf(-d, r, 1.0f), r, r) * l;
  } else {
    const float s = ROUNDED ? reciprocal_from_one(d) : 1.0f / d;
    v = (epi == EPI_GLU_IDENTITY ? 1.0f : s) * (epi == EPI_GLU_SIGMOID ? 1.0f : g) * l;
  }
  asm("" : "+v"(v));
  return v;
}

// `count` of four neighbouring columns of a row (two with the gate), as many as there are
__device__ __forceinline__ void store_columns(const MxParams& p, int64_t row, int col, int cols, const f32x4& v) {
  float o[4];
  int c = col, n = 4;
  if (p.epi != EPI_NONE) {
    o[0] = gated<false, false>(v[0], v[1], p.epi);         // (few of them: the division for every type)
    o[1] = gated<false, false>(v[2], v[3], p.epi);
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
// Tiles: BN columns of the output (rows of the weights) x BM rows, WGN x WGM waves, slabs of 256 k in a ring of S LDS buffers
// filled by direct loads.  Slab s + 1 has to be there, and slab s be read by all, when the last step of slab s
// begins: one barrier per slab, its wait hidden behind that step's products.  Slab s + S then goes where s was.
//
// What bounds them.  8192 x 8192 x 8192 on tiles of 256: 260 us, 4.2 PFLOP/s, on random values, and 190 to 215 on zeros: the board's power limit.  A tile costs
// 1.8 us a slab and 9 beside its slabs, most of that for the burst of results that all CUs write at the end of a round; so 8192 x 4096 x 4096 74 us, 3.7
// PFLOP/s.  Products of 16x16x128 instead, twice as many instructions for an issue slot that the reads and loads want as well: 295 us on
// zeros.  With few rows of many weights it is the weights' bytes: 64 tokens of 8 through 64 experts' 4096 x 1024 matrices 30.6 us, 4.7 TB/s.
template <int BN_, int BM_, int WGN, int WGM, int S_> struct MxTile {
  static constexpr int BN = BN_, BM = BM_, NW = WGN * WGM, THREADS = NW * 64, WAVES_N = WGN, S = S_;
  static constexpr int WTN = BN / WGN, WTM = BM / WGM, TN = WTN / 32, TM = WTM / 32;
  static constexpr int B_BYTES = BN * MX_ROWB, A_BYTES = BM * MX_ROWB;
  static constexpr int S_WAVES = (BN + BM + 63) / 64;     // waves that bring the scales of 64 rows each
  static constexpr int SLOT = B_BYTES + A_BYTES, S_BYTES = S_WAVES * 64 * 2 * MX_SCALEB;      // codes of a slab; scales of two
  static constexpr int B_OPS = B_BYTES / (1024 * NW), A_OPS = A_BYTES / (1024 * NW);      // 16-byte loads per lane and slab
  static constexpr int LDS = S * (SLOT + S_BYTES);       // (slabs s .. s + S are of S / 2 + 1 pairs: S buffers are enough)
  // waves per SIMD that the LDS leaves room for
  static constexpr int OCC = (163840 / LDS) * NW / 4;
  static_assert((S & (S - 1)) == 0 && S >= 2 && LDS <= 163840, "a ring of 2, 4, 8 buffers");
};

// x: words of an even q, y: of the odd q after it.  Lanes 0-31 keep x and get its upper lanes' as y; lanes 32-63 the same of y.
__device__ __forceinline__ void exchange_halves(uint32_t& x, uint32_t& y) {
  const auto r = __builtin_amdgcn_permlane32_swap(x, y, false, false);
  x = r[0];
  y = r[1];
}
template <class O> __device__ __forceinline__ uint32_t two(float a, float b) { return (uint32_t)O::cvt(a) | (uint32_t)O::cvt(b) << 16; }

// a lane's words of a row, or as many of their elements (of ES bytes) as the row still has
template <bool WHOLE, int ES, int WORDS> __device__ __forceinline__ void store_words(uint8_t* d, const uint32_t (&w)[WORDS], int left) {
  if (WHOLE || left >= WORDS * 4 / ES) {
    typedef i32x2 __attribute__((aligned(2))) loose2;
    if constexpr (WORDS == 4) *(i32x4_loose*)d = i32x4{(int)w[0], (int)w[1], (int)w[2], (int)w[3]};
    else *(loose2*)d = i32x2{(int)w[0], (int)w[1]};
  } else {
#pragma unroll
    for (int e = 0; e < WORDS * 4 / ES; ++e)
      if (e < left) {
        if constexpr (ES == 4) ((uint32_t*)d)[e] = w[e];
        else ((uint16_t*)d)[e] = (uint16_t)(w[e / 2] >> (e & 1) * 16);
      }
  }
}

// One 32x32 product into its place (out: row 0, column 0 of it; m_left, left_cols: what there is of it).  A lane has, of row lane % 32, the columns
// 8 q + 4 half + 0 .. 3.  Rounded, four columns are two words; exchanging the halves' words of an even q with those of the odd q after it leaves
// lanes 0-31 with all eight columns of the one and lanes 32-63 with those of the other: 16 bytes a lane.  (With the gate two columns are a word,
// 8 bytes a lane; binary32 needs no exchange.)
// SHORT: see gated; where that does not do, the product is stored by the other form, chosen once, by a scalar.  (bfloat16 by 4-bit 4096 x 28672 x 512 with
// ordinary gates 69.1 us, always the other form 73.7, the bare reciprocal, whose results are not glu's, 68.0; 8192 tokens' up-projections 343, 351 and 340.)
template <bool WHOLE, class O, bool GLU, bool SHORT = GLU && sizeof(typename O::raw) == 2>
__device__ __forceinline__ void store_product(const f32x16& v, uint8_t* out, int64_t ldo, int r32, int half, int m_left, int left_cols, int epi) {
  constexpr int ES = sizeof(typename O::raw);
  if constexpr (SHORT) {
    float low = v[0];
#pragma unroll
    for (int e = 2; e < 16; e += 2) low = __builtin_fminf(low, v[e]);
    if (epi != EPI_GLU_SILU || __any(low < -66.0f)) return store_product<WHOLE, O, GLU, false>(v, out, ldo, r32, half, m_left, left_cols, epi);
  }
  uint8_t* row = out + (int64_t)r32 * ldo * ES;
  const bool have = WHOLE || r32 < m_left;
#pragma unroll
  for (int q = 0; q < 4; q += 2) {
    float o[8];
#pragma unroll
    for (int e = 0; e < (GLU ? 4 : 8); ++e) o[e] = GLU ? gated<ES == 2, SHORT>(v[4 * q + 2 * e], v[4 * q + 2 * e + 1], epi) : v[4 * q + e];
    if constexpr (ES == 4) {
      constexpr int W = GLU ? 2 : 4;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int c = 2 * W * (q + h) + W * half;
        uint32_t w[W];
#pragma unroll
        for (int e = 0; e < W; ++e) w[e] = __builtin_bit_cast(uint32_t, o[W * h + e]);
        if (have) store_words<WHOLE, 4, W>(row + c * 4, w, left_cols - c);
      }
    } else if constexpr (GLU) {
      uint32_t w[2] = {two<O>(o[0], o[1]), two<O>(o[2], o[3])};
      exchange_halves(w[0], w[1]);
      const int c = 4 * (q + half);
      if (have) store_words<WHOLE, 2, 2>(row + c * 2, w, left_cols - c);
    } else {
      uint32_t w[4] = {two<O>(o[0], o[1]), two<O>(o[2], o[3]), two<O>(o[4], o[5]), two<O>(o[6], o[7])};
      exchange_halves(w[0], w[2]);
      exchange_halves(w[1], w[3]);
      const int c = 8 * (q + half);
      if (have) store_words<WHOLE, 2, 4>(row + c * 2, w, left_cols - c);
    }
  }
}

// PARTS: blockIdx.y is a part of k, whose sums go to a matrix of their own in 32 bits; join_kernel adds them up.
template <class C, bool EXPERTS, class O, bool GLU, bool PARTS>
__global__ __launch_bounds__(C::THREADS, C::OCC < 2 ? C::OCC : 2) void mx_tile_kernel(MxParams p) {
  constexpr int BN = C::BN, BM = C::BM, NW = C::NW, S = C::S;
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
    swizzle2d(id / p.tiles_n, id % p.tiles_n, p.tiles_m, p.tiles_n, 4, &tm, &tn);
    rt.expert = 0;
    rt.row0 = tm * BM;
    rt.rows = p.m - rt.row0 < BM ? p.m - rt.row0 : BM;
  }
  const int n0 = tn * BN, ncols = p.n - n0 < BN ? p.n - n0 : BN;
  if (EXPERTS && rt.expert == p.experts) {               // rows of no expert
    const int c0 = p.epi != EPI_NONE ? n0 / 2 : n0, nc = p.epi != EPI_NONE ? ncols / 2 : ncols;
    for (int i = tid; i < rt.rows * nc; i += C::THREADS) store_out<float>(p.out, (int64_t)(rt.row0 + i / nc) * p.ldo + c0 + i % nc, 0.0f, p.out_dtype);
    return;
  }
  const int slab0 = PARTS ? (int)blockIdx.y * p.part_slabs : 0, slabs = PARTS && p.slabs - slab0 > p.part_slabs ? p.part_slabs : p.slabs - slab0;
  const uint8_t* b = uniform_ptr(p.b + (int64_t)rt.expert * p.b_expert + ((int64_t)n0 * p.slabs + slab0) * MX_ROWB);
  const uint8_t* bs = uniform_ptr(p.bs + (int64_t)rt.expert * p.bs_expert + (int64_t)(n0 >> 5) * ((p.slabs + 1) >> 1) * 512);

  // Direct loads.  Instruction q of wave w fills rows 8 (NW q + w) .. + 7 of a side, lane l the 16-byte place l % 8 of row l / 8,
  // which holds the chunk place ^ (row / 2 % 8): a fragment read (16 lanes a cycle, rows {0-3, 12-15, 20-27} or the others, one chunk)
  // then falls on 16 different places of 256 bytes.  Rows past the end are the last row again; nobody stores what they give.
  uint32_t b_off[C::B_OPS];
#pragma unroll
  for (int q = 0; q < C::B_OPS; ++q) {
    const int row = 8 * (NW * q + wave) + (lane >> 3), chunk = (lane & 7) ^ ((row >> 1) & 7);
    b_off[q] = (uint32_t)(row < ncols ? row : ncols - 1) * (uint32_t)(p.slabs * MX_ROWB) + chunk * 16;
  }
  uint32_t a_off[C::A_OPS];
  const uint8_t* a_at[EXPERTS ? C::A_OPS : 1];
  const uint8_t* a = nullptr;
  if (EXPERTS) {
#pragma unroll
    for (int q = 0; q < C::A_OPS; ++q) {
      const int row = 8 * (NW * q + wave) + (lane >> 3), chunk = (lane & 7) ^ ((row >> 1) & 7);
      a_at[q] = p.a + (int64_t)source_row(p, rt.row0 + (row < rt.rows ? row : rt.rows - 1)) * p.slabs * MX_ROWB + chunk * 16;
    }
  } else {
    a = uniform_ptr(p.a + ((int64_t)rt.row0 * p.slabs + slab0) * MX_ROWB);
#pragma unroll
    for (int q = 0; q < C::A_OPS; ++q) {
      const int row = 8 * (NW * q + wave) + (lane >> 3), chunk = (lane & 7) ^ ((row >> 1) & 7);
      a_off[q] = (uint32_t)(row < rt.rows ? row : rt.rows - 1) * (uint32_t)(p.slabs * MX_ROWB) + chunk * 16;
    }
  }
  // Scales: 16 bytes a row, for two slabs; wave w brings those of 64 rows, of the weights' first, then of a's
  constexpr int S_WAVES = C::S_WAVES;
  static_assert(S_WAVES <= NW && BN % 64 == 0, "a wave has one load of scales");
  const uint8_t* s_at;
  {
    const int row = 64 * wave + lane, ar = row - BN;
    if (64 * wave < BN) s_at = bs + mx_scale_at(row < ncols ? row : ncols - 1, slab0, p.slabs);
    else {
      const int r = rt.row0 + (ar < rt.rows ? ar : rt.rows - 1);
      s_at = p.as + mx_scale_at(EXPERTS ? source_row(p, r) : r, slab0, p.slabs);
    }
  }

  // one slab is OPS loads of a wave: op q of them (a constant after unrolling) into the slab's buffer
  constexpr int OPS = C::B_OPS + C::A_OPS + 1;
  auto fetch_op = [&](int slab, int q) __attribute__((always_inline)) {
    const uint32_t slot = lds0 + (slab & (S - 1)) * C::SLOT;
    if (q < C::B_OPS) {
      if (BM <= 128 && p.stream_b) dma16_nt(b + (int64_t)slab * MX_ROWB, b_off[q], __builtin_amdgcn_readfirstlane(slot + (NW * q + wave) * 1024));
      else dma16_from(b + (int64_t)slab * MX_ROWB, b_off[q], slot + (NW * q + wave) * 1024);
    }
    if (q >= C::B_OPS && q < C::B_OPS + C::A_OPS) {
      const int i = q - C::B_OPS;
      const uint32_t to = slot + C::B_BYTES + (NW * i + wave) * 1024;
      if (EXPERTS) dma16_at(a_at[i] + (int64_t)slab * MX_ROWB, to);
      else dma16_from(a + (int64_t)slab * MX_ROWB, a_off[i], to);
    } else if (q == C::B_OPS + C::A_OPS && (slab & 1) == 0 && wave < S_WAVES) {
      dma16_at(s_at + (int64_t)(slab >> 1) * 512, lds0 + S * C::SLOT + (slab >> 1 & (S - 1)) * C::S_BYTES + wave * 1024);
    }
  };

  const int wn = wave % C::WAVES_N * C::WTN, wm = wave / C::WAVES_N * C::WTM, half = lane >> 5, r32 = lane & 31;
  // place of chunk 4 half + step in this lane's row; the weights' and a's products further on are constants from here
  const uint32_t place = (uint32_t)r32 * MX_ROWB + (((4 * half) ^ ((r32 >> 1) & 7)) << 4);
  const uint32_t place_b = lds0 + place + wn * MX_ROWB, place_a = lds0 + place + C::B_BYTES + wm * MX_ROWB;
  const uint32_t place_s = lds0 + S * C::SLOT + r32 * 2 * MX_SCALEB + half * 4;
  constexpr int NM = C::TN * C::TM;
  f32x16 acc[C::TN][C::TM];
#pragma unroll
  for (int i = 0; i < C::TN; ++i)
#pragma unroll
    for (int j = 0; j < C::TM; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;
  // Fragments and scales.  A slab is four steps (blocks 4 half + step); a step goes through the products column by column of a's
  // fragments.  So a's fragment j is free once column j is done and takes the next step's at once; the weights' are in use to
  // a step's end and have two sets.
  i32x4 fb[2][C::TN], fa[C::TM];
  int sb[2][C::TN], sa[C::TM];
  auto read_b = [&](uint32_t slot, int step, int i) __attribute__((always_inline)) {
    fb[step & 1][i] = *TNX_LDS(i32x4, (place_b ^ (step << 4)) + slot + i * 32 * MX_ROWB);
  };
  auto read_a = [&](uint32_t slot, int step, int j) __attribute__((always_inline)) {
    fa[j] = *TNX_LDS(i32x4, (place_a ^ (step << 4)) + slot + j * 32 * MX_ROWB);
  };
  // (at: of the slab, in the scales' buffers)
  auto read_sb = [&](uint32_t at, int set, int i) __attribute__((always_inline)) { sb[set][i] = *TNX_LDS(int, place_s + at + (wn + 32 * i) * 2 * MX_SCALEB); };
  auto read_sa = [&](uint32_t at, int j) __attribute__((always_inline)) { sa[j] = *TNX_LDS(int, place_s + at + (BN + wm + 32 * j) * 2 * MX_SCALEB); };
  // A slab's products, in the order written: the compiler, left to itself, moves each fragment's read in front of its use and waits for it.
  // After the last step's first column comes the barrier; from there on the reads are the next slab's.  From there on, too, and far into the next
  // slab, one direct load every STRIDE products: a load of a wave takes the address unit 16 cycles, and a wave whose
  // load has to queue for it issues no products meanwhile.
  constexpr int BAR = C::TM > 1 ? C::TN : 0, EARLY = NM - BAR, ROOM = EARLY + 2 * NM;
  constexpr int STRIDE = ROOM / OPS > 0 ? ROOM / OPS : 1, DPER = (OPS * STRIDE + ROOM - 1) / ROOM;
  constexpr int FIRST_OPS = (EARLY + STRIDE - 1) / STRIDE * DPER < C::B_OPS + C::A_OPS ? (EARLY + STRIDE - 1) / STRIDE * DPER : C::B_OPS + C::A_OPS;
  constexpr int PER = (C::TN + EARLY - 1) / EARLY;
  // NEXT: there is a slab s + 1.  LATE: slab s + S - 1 is there, and the rest of its loads go out; FETCH: slab s + S is, and its first do.
  auto products = [&](int s, auto next_tag, auto late_tag, auto fetch_tag) __attribute__((always_inline)) {
    constexpr bool NEXT = decltype(next_tag)::value, LATE = decltype(late_tag)::value, FETCH = decltype(fetch_tag)::value;
    const uint32_t slot = (s & (S - 1)) * C::SLOT, other = ((s + 1) & (S - 1)) * C::SLOT;
    const uint32_t scales = ((s + 1) >> 1 & (S - 1)) * C::S_BYTES + ((s + 1) & 1) * MX_SCALEB;
#pragma unroll
    for (int step = 0; step < 4; ++step) {
#pragma unroll
      for (int e = 0; e < NM; ++e) {
        if (NEXT && step == 3 && e == BAR) {
          // The fragments of this slab are in registers and the loads of the next one have landed, in every wave.  (Younger are at least the code
          // loads of the S - 2 slabs after it, where those exist.)
          if (FETCH) TNX_WAIT_VM((S - 2) * (OPS - 1));
          else TNX_WAIT_VM(0);
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          __builtin_amdgcn_s_barrier();
          asm volatile("" ::: "memory");
          __builtin_amdgcn_sched_barrier(0);
        }
        const int j = e / C::TN, i = (j & 1) ? C::TN - 1 - e % C::TN : e % C::TN;
        acc[i][j] = mfma32(fb[step & 1][i], fa[j], acc[i][j], sb[0][i], sa[j], step);
        if (step < 3) {
          if (e < C::TN) read_b(slot, step + 1, e);
          if (e % C::TN == C::TN - 1) read_a(slot, step + 1, j);
        } else if (NEXT && e >= BAR) {
#pragma unroll
          for (int r = (e - BAR) * PER; r < (e - BAR) * PER + PER && r < C::TN; ++r) {
            read_b(other, 0, r);
            read_sb(scales, 1, r);
          }
          if (BAR > 0 && e == BAR) { read_a(other, 0, 0); read_sa(scales, 0); }
          if (e % C::TN == C::TN - 1) { read_a(other, 0, j); read_sa(scales, j); }
        }
        if (step == 3 ? FETCH && e >= BAR : LATE) {
          const int at = step == 3 ? e - BAR : EARLY + step * NM + e;
          if (at % STRIDE == 0) {
#pragma unroll
            for (int q = at / STRIDE * DPER; q < at / STRIDE * DPER + DPER; ++q)
              if (step == 3 ? q < FIRST_OPS : q >= FIRST_OPS && q < OPS) fetch_op(step == 3 ? s + S : s + S - 1, q);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if (NEXT) {
#pragma unroll
      for (int i = 0; i < C::TN; ++i) sb[0][i] = sb[1][i];
    }
  };

  static_assert((S - 2) * (OPS - 1) + FIRST_OPS < 64, "the counter of loads in flight");
#pragma unroll
  for (int t = 0; t < S - 1; ++t)
    if (t < slabs) {
#pragma unroll
      for (int q = 0; q < OPS; ++q) fetch_op(t, q);
    }
  if (slabs >= S) {
#pragma unroll
    for (int q = 0; q < FIRST_OPS; ++q) fetch_op(S - 1, q);
    TNX_WAIT_VM((S - 2) * (OPS - 1) + FIRST_OPS);          // (these go out in every wave: what is older has landed)
  } else {
    TNX_WAIT_VM(0);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < C::TN; ++i) { read_b(0, 0, i); read_sb(0, 0, i); }
#pragma unroll
  for (int j = 0; j < C::TM; ++j) { read_a(0, 0, j); read_sa(0, j); }
  if (wm >= rt.rows) {
    // A wave without rows (an expert's last tile, mostly) does its share of the loads and keeps the barriers; the wave of the other half on
    // its SIMD has the matrix unit to itself.
    for (int s = 0; s < slabs - 1; ++s) {
      if (s + S - 1 < slabs) {
#pragma unroll
        for (int q = FIRST_OPS; q < OPS; ++q) fetch_op(s + S - 1, q);
      }
      if (s + S < slabs) TNX_WAIT_VM((S - 2) * (OPS - 1));
      else TNX_WAIT_VM(0);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      if (s + S < slabs) {
#pragma unroll
        for (int q = 0; q < FIRST_OPS; ++q) fetch_op(s + S, q);
      }
    }
    return;
  }
  int s = 0;
  for (; s < slabs - S; ++s) products(s, BoolTag<true>(), BoolTag<true>(), BoolTag<true>());
  if (s == slabs - S) products(s++, BoolTag<true>(), BoolTag<true>(), BoolTag<false>());
  if (S > 2)
    for (; s < slabs - 1; ++s) products(s, BoolTag<true>(), BoolTag<false>(), BoolTag<false>());
  products(s, BoolTag<false>(), BoolTag<false>(), BoolTag<false>());

  // Epilogue, from the registers (LDS is not touched: nothing waits for the other waves).  The sums stay where the matrix instructions
  // left them until their turn: without the empty asm all 256 are copied out at once, to scratch memory for the most part.
  constexpr int ES = sizeof(typename O::raw), W = GLU ? 16 : 32;          // output columns of a product
  const int left_cols = GLU ? (ncols - wn) >> 1 : ncols - wn;
  uint8_t* out = p.out + ((PARTS ? (int64_t)blockIdx.y * p.m * p.ldo : 0) + (int64_t)(rt.row0 + wm) * p.ldo + (GLU ? (n0 + wn) >> 1 : n0 + wn)) * ES;
  const bool whole = rt.rows - wm >= C::WTM && ncols - wn >= C::WTN;
#pragma unroll
  for (int j = 0; j < C::TM; ++j)
#pragma unroll
    for (int i = 0; i < C::TN; ++i) {
      f32x16 v = acc[i][j];
      asm volatile("" : "+a"(v));
      uint8_t* at = out + ((int64_t)(32 * j) * p.ldo + W * i) * ES;
      if (whole) store_product<true, O, GLU>(v, at, p.ldo, r32, half, 32, W, p.epi);
      else store_product<false, O, GLU>(v, at, p.ldo, r32, half, rt.rows - wm - 32 * j, left_cols - W * i, p.epi);
      __builtin_amdgcn_sched_barrier(0);
    }
}

// ------------------------------------------------------------------------------------------------------------------
// Few rows: bound by streaming the weights, so nothing of them goes through LDS.  A wave has 16 rows of the weights and up to 16 rows of a; a
// workgroup's eight waves are wk parts of k (slabs kpart, kpart + wk, ...) times 8 / wk groups of weight rows, and the parts meet in LDS.  All of
// a turn's loads are in flight together.  16x16x128 instructions: lane group g (lane / 16) takes the blocks 2 g and 2 g + 1 of a slab, 32 neighbouring
// bytes and two neighbouring scales.
//
// RAW: the rows of a as 16- or 32-bit floats: every workgroup quantises them into LDS, 4096 elements in about 0.5 us, which saves a launch of 3 us and its
// gap.  (They are asked for after the first turn's weights and arrive behind them: loads come back in order.)  In one launch and in two: 4096 x 4096 of 1, 4 and 8 rows 5.1, 6.7 and 8.6 us, 10.1 to 10.2;
// 14336 x 4096 8.8, 11.1 and 14.2, 11.8 to 11.1; 4096 x 7000 6.9, 9.4 and 12.9, 8.9 to 9.3: up to 16384 elements, or one row.
constexpr int FEW_WAVES = 8, FEW_RAW_ROWS = 16, FEW_RAW_K = 30720, FEW_RAW_ELEMENTS = 16384;
// bytes of such a row: 16 more than its codes, so that the rows' chunks fall on different banks, and its scales
__host__ __device__ inline uint32_t raw_pitch(int64_t slabs) { return (uint32_t)slabs * MX_ROWB + 16; }
__host__ __device__ inline size_t raw_bytes(int64_t rows, int64_t slabs) { return (size_t)rows * (raw_pitch(slabs) + slabs * MX_SCALEB); }

template <class T> __device__ __forceinline__ void quantize_to_lds(const MxParams& p, uint32_t codes, uint32_t scales, int tid) {
  typedef typename Elem<T>::raw raw;
  const int per_row = p.slabs * 32, items = p.a_rows * per_row;
  for (int i0 = 0; i0 < items; i0 += FEW_WAVES * 64) {                    // (whole blocks of four lanes take each turn)
    const int i = i0 + tid, row = (int)((uint32_t)i / (uint32_t)per_row), at = i - row * per_row;
    if (i >= items) continue;
    const int left = p.k - at * 8;
    const raw* src = (const raw*)p.a + (int64_t)row * p.lda + (int64_t)at * 8;
    Run8<T> x;
    if (left >= 8) x = *(const Run8<T>*)src;
    else {
#pragma unroll
      for (int e = 0; e < 8; ++e) x.v[e] = e < left ? src[e] : (raw)0;
    }
    float v[8], factor;
    raw top = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const raw b = magnitude(x.v[e]);
      top = top > b ? top : b;
    }
    const uint32_t s = scale_byte(top_bits<T>((raw)quad_max(top)), &factor);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = scaled(Elem<T>::get(x.v[e]), factor);
    *TNX_LDS(uint32_t, codes + row * raw_pitch(p.slabs) + at * 4) = codes8(v);
    if ((at & 3) == 0) *TNX_LDS(uint8_t, scales + (i >> 2)) = (uint8_t)s;      // (a block of padding: codes 0, any finite scale)
  }
}

template <bool EXPERTS, bool RAW>
__global__ __launch_bounds__(FEW_WAVES * 64) void mx_few_kernel(MxParams p) {
  extern __shared__ __attribute__((aligned(16))) uint8_t mx_smem[];
  const uint32_t lds0 = (uint32_t)(uintptr_t)(uint8_t __attribute__((address_space(3)))*)mx_smem;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wk = 1 << p.wk_log, kpart = wave & (wk - 1);
  const int n0 = (blockIdx.x * (FEW_WAVES >> p.wk_log) + (wave >> p.wk_log)) * 16;
  RowTile rt;
  if (EXPERTS) {
    if (!find_rows<16>(p, blockIdx.y, lane, &rt)) return;                 // (the same answer in every wave)
  } else {
    rt.expert = 0;
    rt.row0 = blockIdx.y * 16;
    rt.rows = p.m - rt.row0 < 16 ? p.m - rt.row0 : 16;
  }
  const int row = lane & 15, g = lane >> 4;
  const bool empty = EXPERTS && rt.expert == p.experts;
  const uint32_t raw_scales = lds0 + p.a_rows * raw_pitch(p.slabs);
  f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};

  constexpr int DEPTH = 8;                               // slabs of a turn
  const uint8_t *b_at = nullptr, *bs_at = nullptr;
  i32x4 fb[DEPTH][2];
  int sb[DEPTH];
  auto load_weights = [&](int s0) __attribute__((always_inline)) {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      const int64_t s = s0 + d * wk;
      if (s < p.slabs) {
        fb[d][0] = *(const i32x4*)(b_at + s * MX_ROWB);
        fb[d][1] = *(const i32x4*)(b_at + s * MX_ROWB + 16);
        sb[d] = *(const uint16_t*)(bs_at + (s >> 1) * 512 + (s & 1) * 8);
      }
    }
  };
  if (!empty) {
    const int n = n0 + row < p.n ? n0 + row : p.n - 1;
    b_at = p.b + (int64_t)rt.expert * p.b_expert + (int64_t)n * p.slabs * MX_ROWB + 32 * g;
    bs_at = p.bs + (int64_t)rt.expert * p.bs_expert + mx_scale_at(n, 0, p.slabs) + 2 * g;
    load_weights(kpart);
  }
  if (RAW) {
    if (p.a_dtype == DT_BF16) quantize_to_lds<__bf16>(p, lds0, raw_scales, tid);
    else if (p.a_dtype == DT_F16) quantize_to_lds<_Float16>(p, lds0, raw_scales, tid);
    else quantize_to_lds<float>(p, lds0, raw_scales, tid);
    __syncthreads();
  }
  if (!empty) {
    const bool have = row < rt.rows;
    const int r = rt.row0 + (have ? row : 0), src = EXPERTS ? source_row(p, r) : r;
    const uint8_t* a_at = RAW ? nullptr : p.a + (int64_t)src * p.slabs * MX_ROWB + 32 * g;
    const uint8_t* as_at = RAW ? nullptr : p.as + mx_scale_at(src, 0, p.slabs) + 2 * g;
    for (int s0 = kpart;;) {
#pragma unroll
      for (int d = 0; d < DEPTH; ++d) {
        const int64_t s = s0 + d * wk;
        if (s < p.slabs) {
          i32x4 fa0 = {0, 0, 0, 0}, fa1 = {0, 0, 0, 0};
          int sa = 0x7f7f;
          if (have) {
            if (RAW) {
              const uint32_t at = lds0 + src * raw_pitch(p.slabs) + (uint32_t)s * MX_ROWB + 32 * g;
              fa0 = *TNX_LDS(i32x4, at);
              fa1 = *TNX_LDS(i32x4, at + 16);
              sa = *TNX_LDS(uint16_t, raw_scales + (uint32_t)(src * p.slabs + s) * MX_SCALEB + 2 * g);
            } else {
              fa0 = *(const i32x4*)(a_at + s * MX_ROWB);
              fa1 = *(const i32x4*)(a_at + s * MX_ROWB + 16);
              sa = *(const uint16_t*)(as_at + (s >> 1) * 512 + (s & 1) * 8);
            }
          }
          acc = mfma16<0>(fb[d][0], fa0, acc, sb[d], sa);
          acc = mfma16<1>(fb[d][1], fa1, acc, sb[d], sa);
        }
      }
      s0 += wk * DEPTH;
      if (s0 >= p.slabs) break;
      load_weights(s0);
    }
  }
  if (wk > 1) {
    // a part's sums beside the others', and the first part adds them up in order
    if (RAW) __syncthreads();                            // (the rows of a lie there)
    *TNX_LDS(f32x4, lds0 + (wave * 64 + lane) * 16) = acc;
    __syncthreads();
    if (kpart > 0) return;
    for (int w = 1; w < wk; ++w) acc += *TNX_LDS(f32x4, lds0 + ((wave + w) * 64 + lane) * 16);
  }
  const int c = n0 + 4 * g;
  if (row < rt.rows && c < p.n) store_columns(p, rt.row0 + row, c, p.n, acc);
}

// ------------------------------------------------------------------------------------------------------------------
int parts_pitch(int64_t n) { return (int)((n + 3) & ~(int64_t)3); }
// slabs of a part: even, since two slabs' scales lie together
int parts_slabs(int slabs, int parts) { return ((slabs + parts - 1) / parts + 1) & ~1; }
constexpr size_t MAX_PARTS_BYTES = (size_t)64 << 20;
size_t parts_bytes(int64_t m, int64_t n, int parts) { return parts > 1 ? (size_t)parts * m * parts_pitch(n) * 4 : 0; }

// The parts' sums, in their order, through the epilogue: four columns a thread.  sums: [parts][m][pitch]
__global__ __launch_bounds__(256) void join_kernel(MxParams p, const float* sums, int parts, int pitch) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = i / (pitch >> 2);
  if (row >= p.m) return;
  const int col = (int)(i - row * (pitch >> 2)) * 4;
  const f32x4* at = (const f32x4*)(sums + row * pitch + col);
  const int64_t next = (int64_t)p.m * pitch >> 2;
  f32x4 v = *at;
  for (int s = 1; s < parts; ++s) v += at[s * next];
  store_columns(p, row, col, p.n, v);
}

template <class C, bool EXPERTS> int launch_tile(MxParams p, int64_t row_tiles, hipStream_t stream, int parts = 1, void* sums = nullptr) {
  p.tiles_n = (p.n + C::BN - 1) / C::BN;
  p.tiles_m = (p.m + C::BM - 1) / C::BM;
  // 64 tokens through 64 experts' up-projections, weights not in the caches: 62 us, so 55; with 1024 tokens, two tiles an expert, 99 and 104
  p.stream_b = EXPERTS ? (int64_t)p.m * 2 <= (int64_t)p.experts * C::BM : p.tiles_m == 1;
  const int64_t grid = row_tiles * p.tiles_n;
  if (grid > 0x7fffffff) return TNX_E_UNSUPPORTED;
  if constexpr (!EXPERTS && C::S == 4) {
    if (parts > 1) {
      const int pitch = parts_pitch(p.n);
      MxParams q = p;
      q.out = (uint8_t*)sums;
      q.ldo = pitch;
      q.part_slabs = parts_slabs(p.slabs, parts);
      parts = (p.slabs + q.part_slabs - 1) / q.part_slabs;                  // (rounded up to even, fewer may do)
      hipLaunchKernelGGL((mx_tile_kernel<C, false, OutF32, false, true>), dim3((unsigned)grid, (unsigned)parts), dim3(C::THREADS), C::LDS, stream, q);
      const int status = mx_launched();
      if (status != TNX_OK) return status;
      const int64_t items = (int64_t)p.m * (pitch >> 2);
      hipLaunchKernelGGL(join_kernel, dim3((unsigned)((items + 255) / 256)), dim3(256), 0, stream, p, (const float*)sums, parts, pitch);
      return mx_launched();
    }
  }
  auto go = [&](auto out_tag, auto glu_tag) {
    typedef typename decltype(out_tag)::type O;
    hipLaunchKernelGGL((mx_tile_kernel<C, EXPERTS, O, decltype(glu_tag)::value, false>), dim3((unsigned)grid), dim3(C::THREADS), C::LDS, stream, p);
    return mx_launched();
  };
  auto gated = [&](auto out_tag) { return p.epi != EPI_NONE ? go(out_tag, BoolTag<true>()) : go(out_tag, BoolTag<false>()); };
  if (p.out_dtype == DT_BF16) return gated(TypeTag<OutBF16>());
  return p.out_dtype == DT_F16 ? gated(TypeTag<OutF16>()) : gated(TypeTag<OutF32>());
}

// as few parts of k (log2) as give every SIMD two waves: a part less is a sum less, and its wave has more loads in flight
int few_parts(int64_t outputs, int64_t slabs) {
  int log = 0;
  while (log < 3 && (2 << log) <= slabs && (outputs << log) < 2048) ++log;
  return log;
}

template <bool EXPERTS, bool RAW> int launch_few(MxParams p, int64_t row_tiles, hipStream_t stream) {
  const int64_t groups = (p.n + 15) / 16;
  p.wk_log = few_parts(groups * row_tiles, p.slabs);
  const int64_t per = FEW_WAVES >> p.wk_log;
  size_t lds = p.wk_log ? (size_t)FEW_WAVES * 1024 : 0;
  const size_t raw = RAW ? raw_bytes(p.a_rows, p.slabs) : 0;
  if (raw > lds) lds = raw;
  hipLaunchKernelGGL((mx_few_kernel<EXPERTS, RAW>), dim3((unsigned)((groups + per - 1) / per), (unsigned)row_tiles), dim3(FEW_WAVES * 64), lds, stream, p);
  return mx_launched();
}

// Microseconds of `tiles` tiles, `slots` of them on the card at a time: a slab costs t, less (t_few) where at most half of the slots are taken, a
// tile o beside its slabs.
double tiles_us(int64_t tiles, int slots, double t, double t_few, double o, int64_t slabs) {
  const int64_t rounds = tiles / slots, rest = tiles % slots;
  return rounds * (slabs * t + o) + (rest ? slabs * (2 * rest <= slots ? t_few : t) + o : 0.0);
}

enum Kind { FEW, TILE_32, TILE_64, TILE_128, TILE_128_DEEP, TILE_256 };
struct Choice {
  Kind kind;
  int parts;
};

// The tile with the lowest estimate.  Fitted to products of 8 to 4096 rows with 256 x 1024 to 14336 x 14336 weights, and of 4 to 4096 tokens with 8 to
// 128 experts.  What it decides, measured in us: 1024 x 4096 x 4096 tiles of 64 18.5, of 128 15.1 (one on a CU, four buffers, eight waves; 15.6 with four) and 16.0 (two on a
// CU, two buffers), of 256 25.6; 2048 x 14336 x 4096 117, 88, 73 and 66; 512 x 4096 x 14336 27, 30, 46 and 69; 64 tokens through
// the up-projections of 64 experts (4096 -> 1024) 49, 56, 49 and 56, through the down-projections 44, 55, 37 and 44, with tiles of 32 30.6.
template <bool EXPERTS> struct Shape {
  int64_t m, n, slabs, experts;
  // tiles of BM rows: how many there are at most, and how many to expect (an expert's last is half full)
  int64_t most(int bm) const { return EXPERTS ? m / bm + 1 + (experts < m ? experts : m) : (m + bm - 1) / bm; }
  int64_t expect(int bm) const {
    if (!EXPERTS) return most(bm);
    const int64_t some = experts < m ? experts : m, some_tiles = m / bm + some / 2;
    return some_tiles > some ? some_tiles : some;
  }
  int64_t cols(int bn) const { return (n + bn - 1) / bn; }

  double us64(int parts = 1) const { return tiles_us(expect(64) * cols(64) * parts, 512, 0.5, 0.35, EXPERTS ? 3.8 : 1.5, (slabs + parts - 1) / parts); }
  double us128_deep(int parts = 1) const { return tiles_us(expect(128) * cols(128) * parts, 256, 0.5, 0.45, 6.0, (slabs + parts - 1) / parts); }

  Choice choose(size_t room) const {
    Choice best{TILE_64, 1};
    double us = us64();
    auto offer = [&](Kind kind, int parts, double t) {
      if (t < us) { us = t; best = {kind, parts}; }
    };
    offer(TILE_128_DEEP, 1, us128_deep());
    offer(TILE_128, 1, tiles_us(expect(128) * cols(128), 512, 1.1, 0.76, 4.5, slabs));
    offer(TILE_256, 1, tiles_us(expect(256) * cols(256), 256, 1.77, 1.15, 9.0, slabs));
    if constexpr (EXPERTS) {
      // Experts of a dozen rows: a tile of 32 brings 4 kB of rows with 16 of weights where one of 128 brings 16, most of it the last row over again, and three
      // are on a CU.  64 tokens, 8 of 128 experts, 2048 to 768, up 53 us on tiles of 128 and 35, down 37 and 30; 16 of 64 experts, 4096 to 1024, up 57 and 35; 512 of
      // them 84 and 92.
      offer(TILE_32, 1, tiles_us(expect(32) * cols(128), 768, 1.2, 1.2, 2.5, slabs));
    } else {
      // The streaming kernel: a slab of a workgroup's eight waves is 35 kB of weights and rows, which it brings in 1 us, however few CUs are
      // busy (a turn waits for all of its loads; a ring, which has some ahead, brings as much in half of that).  So it is for few rows, or few columns, and it shares
      // k out.  40 x 64 x 9630: 7.6 us, tiles of 64 13.7; 8 x 4096 x 4096 4.5 and 7.4; 64 x 1024 x 4096 4.9 and 7.8, 128 rows 7.0 and 7.4; 256 x 256 x
      // 16384 11.2 and 23; 48 x 4096 x 4096 11.6 and 7.2.
      const int64_t outputs = cols(16) * most(16);
      const int log = few_parts(outputs, slabs);
      if (most(16) <= 65535) offer(FEW, 1, 2.7 + (double)(((outputs << log) + 256 * FEW_WAVES - 1) / (256 * FEW_WAVES) * ((slabs + (1 << log) - 1) >> log)));
      // Few tiles of many slabs: k in parts, a workgroup each, and a second launch that adds them up.  100 x 4096 x 14336 20.7 us, in 4 parts 14.5; 128 x 1024 x
      // 16384 19.7, in 8 10.8; 64 x 64 x 30000 18.4 and 10.9; 64 x 4096 x 8192 12.4, in 4 10.1, 128 rows 12.7, in 2 13.5.
      for (int parts = 2; parts <= 8; ++parts) {
        if (slabs < 4 * parts || parts_bytes(m, n, parts) > room) break;
        const double join = 5.0 + (double)parts_bytes(m, n, parts) / 2e6;
        offer(TILE_64, parts, us64(parts) + join);
        offer(TILE_128_DEEP, parts, us128_deep(parts) + join);
      }
    }
    return best;
  }
};

typedef MxTile<256, 256, 4, 2, 2> Tile256;
typedef MxTile<64, 64, 2, 2, 4> Tile64;
typedef MxTile<128, 128, 4, 2, 4> Tile128Deep;
typedef MxTile<128, 128, 2, 2, 2> Tile128;
typedef MxTile<128, 32, 4, 1, 2> Tile32;                 // (experts only)

template <bool EXPERTS> int launch(const MxParams& p, bool raw, void* sums, size_t room, hipStream_t stream) {
  const Shape<EXPERTS> shape{p.m, p.n, p.slabs, p.experts};
  if (raw) return shape.most(16) <= 65535 ? launch_few<EXPERTS, true>(p, shape.most(16), stream) : TNX_E_UNSUPPORTED;
  const Choice c = shape.choose(sums ? room : 0);
  switch (c.kind) {
    case TILE_256: return launch_tile<Tile256, EXPERTS>(p, shape.most(256), stream);
    case TILE_64: return launch_tile<Tile64, EXPERTS>(p, shape.most(64), stream, c.parts, sums);
    case TILE_128_DEEP: return launch_tile<Tile128Deep, EXPERTS>(p, shape.most(128), stream, c.parts, sums);
    case TILE_128: return launch_tile<Tile128, EXPERTS>(p, shape.most(128), stream);
    default: break;
  }
  if constexpr (EXPERTS) return launch_tile<Tile32, true>(p, shape.most(32), stream);
  else return launch_few<false, false>(p, shape.most(16), stream);
}

// what launch() does, and tnx_mx_gemm_route's answer
template <bool EXPERTS> int route(const MxParams& p, bool raw, void* sums, size_t room, int32_t info[4]) {
  const Shape<EXPERTS> shape{p.m, p.n, p.slabs, p.experts};
  const Choice c = raw ? Choice{FEW, 1} : shape.choose(sums ? room : 0);
  auto tile = [&](auto t) {
    typedef typename decltype(t)::type C;
    const int per = parts_slabs(p.slabs, c.parts);
    info[0] = C::BN; info[1] = C::BM; info[2] = C::S;
    info[3] = c.parts > 1 ? (p.slabs + per - 1) / per : 1;
    return TNX_MX_ROUTE_TILES;
  };
  switch (c.kind) {
    case TILE_256: return tile(TypeTag<Tile256>());
    case TILE_64: return tile(TypeTag<Tile64>());
    case TILE_128_DEEP: return tile(TypeTag<Tile128Deep>());
    case TILE_128: return tile(TypeTag<Tile128>());
    case TILE_32: return tile(TypeTag<Tile32>());
    default: break;
  }
  info[0] = info[1] = 16; info[2] = 0; info[3] = 1;
  return shape.most(16) <= 65535 ? TNX_MX_ROUTE_STREAM : 0;
}

bool takes_rows(int64_t a_rows, int64_t k) {
  return a_rows == 1 ? k <= FEW_RAW_K : a_rows <= FEW_RAW_ROWS && a_rows * k <= FEW_RAW_ELEMENTS;
}

}  // namespace

extern "C" int tnx_mx_gemm_takes_rows(int64_t a_rows, int64_t k) { return a_rows > 0 && k > 0 && takes_rows(a_rows, k); }

extern "C" size_t tnx_mx_gemm_workspace_bytes(const tnx_mx_gemm_args* a) {
  if (!a || a->m <= 0 || a->n <= 0 || a->k <= 0 || a->experts != 0 || a->a_data || a->k > TNX_MX_MAX_K || a->m > 0x3fffffff || a->n > 0x3fffffff) return 0;
  const Shape<false> shape{a->m, a->n, mx_slabs(a->k), 0};
  return parts_bytes(a->m, a->n, shape.choose(MAX_PARTS_BYTES).parts);
}

namespace {

// the arguments' checks and the kernels' parameters
int prepare(const tnx_mx_gemm_args* a, MxParams* params) {
  if (!a || a->m < 0 || a->n < 0 || a->k < 0 || a->experts < 0 || a->epilogue < TNX_EPI_NONE || a->epilogue > TNX_EPI_GLU_IDENTITY) return TNX_E_INVALID;
  if (a->m == 0 || a->n == 0) return TNX_OK;
  if (a->out_dtype != TNX_BF16 && a->out_dtype != TNX_F16 && a->out_dtype != TNX_F32) return TNX_E_UNSUPPORTED;
  if (a->epilogue != TNX_EPI_NONE && a->n % 2) return TNX_E_UNSUPPORTED;
  const int64_t cols = a->epilogue != TNX_EPI_NONE ? a->n / 2 : a->n;
  if (!a->out || a->stride_out < cols || ((uintptr_t)a->out & (a->out_dtype == TNX_F32 ? 3 : 1))) return TNX_E_INVALID;
  if (a->k == 0 || a->k > TNX_MX_MAX_K || a->m > 0x3fffffff || a->n > 0x3fffffff || a->a_rows > 0x3fffffff) return TNX_E_UNSUPPORTED;
  const bool raw = a->a_data != nullptr;
  if (!a->b_codes || !a->b_scales || (((uintptr_t)a->b_codes | (uintptr_t)a->b_scales) & 15)) return TNX_E_INVALID;
  if (raw) {
    if (a->a_codes || a->a_scales) return TNX_E_INVALID;
    if (a->a_dtype != TNX_BF16 && a->a_dtype != TNX_F16 && a->a_dtype != TNX_F32) return TNX_E_UNSUPPORTED;
    if ((uintptr_t)a->a_data & (a->a_dtype == TNX_F32 ? 3 : 1)) return TNX_E_INVALID;
    if (!takes_rows(a->a_rows, a->k)) return TNX_E_UNSUPPORTED;
  } else if (!a->a_codes || !a->a_scales || (((uintptr_t)a->a_codes | (uintptr_t)a->a_scales) & 15)) return TNX_E_INVALID;
  if (a->experts > 0 ? (!a->offsets || a->experts > TNX_MOE_MAX_EXPERTS) : (a->offsets || a->order)) return TNX_E_INVALID;
  if (a->order ? (a->top_k < 1 || a->a_rows < 1) : a->a_rows != a->m) return TNX_E_INVALID;
  MxParams& p = *params;
  p.a = (const uint8_t*)(raw ? a->a_data : a->a_codes); p.as = (const uint8_t*)a->a_scales;
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
  p.a_dtype = a->a_dtype; p.lda = a->stride_a; p.k = (int)a->k; p.wk_log = 0; p.part_slabs = p.slabs; p.stream_b = false;
  if (a->workspace && ((uintptr_t)a->workspace & 15)) return TNX_E_INVALID;
  return TNX_OK;
}

size_t room_of(const tnx_mx_gemm_args* a) { return a->workspace_bytes < MAX_PARTS_BYTES ? a->workspace_bytes : MAX_PARTS_BYTES; }

}  // namespace

extern "C" int tnx_mx_gemm(const tnx_mx_gemm_args* a) {
  MxParams p;
  const int status = prepare(a, &p);
  if (status != TNX_OK || a->m == 0 || a->n == 0) return status;
  const bool raw = a->a_data != nullptr;
  const hipStream_t stream = (hipStream_t)a->stream;
  return a->experts > 0 ? launch<true>(p, raw, nullptr, 0, stream) : launch<false>(p, raw, a->workspace, room_of(a), stream);
}

extern "C" int tnx_mx_gemm_route(const tnx_mx_gemm_args* a, int32_t info[4]) {
  MxParams p;
  int32_t unused[4];
  if (prepare(a, &p) != TNX_OK || a->m == 0 || a->n == 0) return 0;
  const bool raw = a->a_data != nullptr;
  return a->experts > 0 ? route<true>(p, raw, nullptr, 0, info ? info : unused) : route<false>(p, raw, a->workspace, room_of(a), info ? info : unused);
}
