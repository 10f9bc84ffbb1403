// The tile kernels over groups of rows: rows sorted by group, a weight per group, the groups' bounds in device memory.
//
//   rows x weights      y[r, n] = a[r, k] b[g][k, n]            for offsets[g] <= r < offsets[g + 1]
//   weights' gradient   c[g][m, n] = a[rows of g, m]^T b[rows of g, n]      (AT: k is the group's rows)
//
// The grid is the most tiles that the rows can make, ceil(rows / BM) + one per group and per stretch without a group; each workgroup
// finds its tile in the bounds, 64 groups at a time by a scan over the wave, then the tile kernel runs on the group as if it were the
// whole problem.  Nothing waits for the host, nothing is launched ahead.
//
// Few tiles of a long k: PARTS workgroups to a tile, each over a part of k (of the group's rows), 32-bit sums in a workspace, and a launch that
// adds the parts up in order (grouped.hip).
//
// The bounds are data: taken into [0, rows] and to a sequence that does not decrease, so that whatever they hold every row belongs to
// one group or to none, is written once, and nothing outside the tensors is touched.  Rows of no group, ahead of the first and behind the
// last, are written as zeros: a tile whose k is 0.
#pragma once
#include "gemm_tile.h"

namespace tnx {

struct GroupedParams {
  const uint8_t* a;
  const uint8_t* b;
  uint8_t* c;
  const int32_t* offsets;    // [groups + 1]
  int64_t lda, ldb;          // of a's rows, of b's rows (BT: of its n)
  int64_t group_stride;      // elements from a group's matrix to the next: of b, AT: of c
  int32_t rows, n, k;        // AT: k is the number of a's columns, the rows of c
  int32_t groups, group_m;
  int32_t parts, per_part;   // PARTS: workgroups to a tile, slabs of k of each (rows times weights)
  int64_t part_stride;       // PARTS: elements from a part of c to the next
  uint32_t flags;            // PF_TAIL
};
static_assert(sizeof(GroupedParams) <= 112, "a longer argument list costs every launch 0.7 us");

// inclusive scans of a wave's 64 lanes, non-negative integers: rows of 16 lanes, then their last lanes
template <class F> __device__ __forceinline__ int wave_scan(int x, F f) {
  x = f(x, __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false));      // row_shr:1, 2, 4, 8
  x = f(x, __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false));
  x = f(x, __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false));
  x = f(x, __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false));
  x = f(x, __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false));      // row_bcast:15 into rows 1 and 3
  x = f(x, __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false));      // row_bcast:31 into rows 2 and 3
  return x;
}
__device__ __forceinline__ int scan_add(int x) {
  return wave_scan(x, [](int a, int b) __attribute__((always_inline)) { return a + b; });
}
__device__ __forceinline__ int scan_max(int x) {
  return wave_scan(x, [](int a, int b) __attribute__((always_inline)) { return a > b ? a : b; });
}
__device__ __forceinline__ int clamp_to(int v, int most) { return v < 0 ? 0 : v > most ? most : v; }

// Workgroups are dealt to the 8 XCDs in turn.  In windows of W of them each XCD takes W / 8 neighbouring tiles, which share rows or weights through
// its L2, and all XCDs are in the same few groups: with a run of the whole list for each XCD instead, the XCD of the longest groups is
// the last one (weights' gradient, 16384 rows in 8 uneven groups, 4096 x 4096: 786 us, in windows of 64 451; 32768 in 32, 2048 x 2048: 395, 291).
template <int W> __device__ __forceinline__ int windowed(int bid, int total) {
  const int first = bid - bid % W, size = total - first < W ? total - first : W;
  return first + xcd_remap(bid - first, size, 8);
}

template <bool PARTS> struct GroupedFamily {
  static constexpr bool LINEAR = false, GROUPED = true, SUMS = PARTS;
  template <bool> using params = GroupedParams;

  template <class C, bool BT, bool AT> static __device__ __forceinline__ GemmParams expand(const GroupedParams& q) {
    GemmParams p;
    p.a = q.a; p.b = q.b; p.c = q.c; p.ws = nullptr;
    p.sam = AT ? 1 : q.lda; p.sak = AT ? q.lda : 1;
    p.sbk = BT ? 1 : q.ldb; p.sbn = BT ? q.ldb : 1;
    p.scm = q.n; p.scn = 1;
    p.m = AT ? q.k : q.rows; p.n = q.n; p.k = AT ? 0 : q.k;
    p.tiles_m = (int)(((uint32_t)p.m + C::BM - 1) / C::BM); p.tiles_n = (int)(((uint32_t)q.n + C::BN - 1) / C::BN);
    p.group_m = q.group_m; p.split_k = 1; p.split_tile0 = 0; p.ktiles_per_split = 0;
    p.epilogue = EPI_NONE; p.out_dtype = 0;
    p.c_vec_ok = false; p.c_row_ok = true;
    p.tail_slab = (q.flags & PF_TAIL) != 0; p.b_once = false;
    p.tile_order = 0; p.atomic_reduce = 0; p.batch = 1;
    p.m_load = p.m; p.n_load = p.n;
    p.cv.bias = nullptr; p.cv.bias_dtype = 0;
    return p;
  }

  // one stretch of rows and what it takes: number (0: ahead of the first group, groups + 1: behind the last), first row, rows, tiles before it
  struct Stretch {
    int number, first, rows, before;
  };

  // The stretch that holds tile row `want` (of BM rows each), or with want < 0 only the number of tile rows, in *total.
  template <int BM> static __device__ __forceinline__ Stretch stretch_of(const GroupedParams& q, int lane, int want, int* total) {
    Stretch s = {-1, 0, 0, 0};
    int carry = 0, tiles = 0;
    for (int base = 0; base < q.groups + 2; base += 64) {
      const int i = base + lane;
      const int own = i <= q.groups ? clamp_to(q.offsets[i], q.rows) : q.rows;
      const int scanned = scan_max(own), end = scanned > carry ? scanned : carry;
      const int shifted = __shfl_up(end, 1), first = lane == 0 ? carry : shifted;
      const int mine = (int)(((uint32_t)(end - first) + BM - 1) / BM), sum = scan_add(mine);
      if (want >= 0) {
        const bool here = want >= tiles + sum - mine && want < tiles + sum;
        const uint64_t hit = __builtin_amdgcn_ballot_w64(here);
        if (hit) {
          const int l = (int)__builtin_ctzll(hit);
          s.number = base + l;
          s.first = __builtin_amdgcn_readlane(first, l);
          s.rows = __builtin_amdgcn_readlane(end - first, l);
          s.before = __builtin_amdgcn_readfirstlane(tiles) + __builtin_amdgcn_readlane(sum - mine, l);
          return s;
        }
      }
      carry = __builtin_amdgcn_readlane(end, 63);
      tiles += __builtin_amdgcn_readlane(sum, 63);
    }
    *total = tiles;
    return s;
  }

  template <class C, bool AT>
  static __device__ __forceinline__ bool find(const GroupedParams& q, GemmParams& p, int bid, int grid, int lane, int* pid_m, int* pid_n) {
    constexpr int OUT = PARTS ? 4 : C::ES;
    int part = 0;
    if constexpr (PARTS) {
      // (part after part, each over all tiles)
      grid /= q.parts;
      const int tile = bid % grid;
      part = bid / grid;
      bid = tile;
      p.c += (int64_t)part * q.part_stride * 4;
    }
    if constexpr (AT) {
      const int per = p.tiles_m * p.tiles_n;
      const int id = windowed<64>(bid, grid), g = id / per, r = id - g * per;
      swizzle2d(r / p.tiles_n, r % p.tiles_n, p.tiles_m, p.tiles_n, p.group_m, pid_m, pid_n);
      int first = 0;
      for (int base = 0; base <= g; base += 64) {
        const int i = base + lane;
        const int top = __builtin_amdgcn_readlane(scan_max(i <= g ? clamp_to(q.offsets[i], q.rows) : 0), 63);
        first = top > first ? top : first;
      }
      const int next = clamp_to(q.offsets[g + 1], q.rows);
      int end = __builtin_amdgcn_readfirstlane(next > first ? next : first);
      if constexpr (PARTS) {
        const int slabs = (int)((uint32_t)(end - first + C::BK - 1) / C::BK), span = (int)((uint32_t)(slabs + q.parts - 1) / (uint32_t)q.parts) * C::BK;
        first = first + part * span < end ? first + part * span : end;
        end = first + span < end ? first + span : end;
      }
      p.k = end - first;
      p.a += (int64_t)first * q.lda * C::ES;
      p.b += (int64_t)first * q.ldb * C::ES;
      p.c += (int64_t)g * q.group_stride * OUT;
      p.tail_slab = p.tail_slab || p.k % C::BK != 0;
      return true;
    } else {
      int total = 0;
      stretch_of<C::BM>(q, lane, -1, &total);
      const int tiles = total * p.tiles_n;
      if (bid >= tiles) return false;
      const int id = windowed<128>(bid, tiles);
      const Stretch s = stretch_of<C::BM>(q, lane, id / p.tiles_n, &total);
      const int r = id - s.before * p.tiles_n;
      p.tiles_m = (int)(((uint32_t)s.rows + C::BM - 1) / C::BM);
      swizzle2d(r / p.tiles_n, r % p.tiles_n, p.tiles_m, p.tiles_n, p.group_m, pid_m, pid_n);
      const bool none = s.number == 0 || s.number == q.groups + 1;
      p.m = p.m_load = s.rows;
      p.a += (int64_t)s.first * q.lda * C::ES;
      p.b += none ? 0 : (int64_t)(s.number - 1) * q.group_stride * C::ES;
      if constexpr (PARTS) {
        const int64_t start = (int64_t)part * q.per_part * C::BK, span = (int64_t)q.per_part * C::BK;
        p.a += start * C::ES;
        p.b += start * (p.sbk == 1 ? 1 : p.sbk) * C::ES;
        p.k = p.k - start < span ? p.k - start : span;
      }
      p.k = none ? 0 : p.k;
      p.c += (int64_t)s.first * q.n * OUT;
      p.b_once = p.tiles_m == 1;
      return true;
    }
  }
};

typedef hipError_t (*grouped_fn)(const GroupedParams& p, unsigned grid, hipStream_t stream);
struct GroupedEntry {
  int dtype, bm, bn, nw, stages;
  grouped_fn nn, bt, at;      // row-major and k-contiguous weights; the weights' gradient
  grouped_fn parts[3];        // the same in parts; may be null
};
struct GroupedGroup {
  GroupedEntry* entries;
  int count;
};

template <class T, class C, bool BT, bool AT, bool PARTS = false> hipError_t launch_grouped(const GroupedParams& p, unsigned grid, hipStream_t stream) {
  GroupedParams q = p;
  return launch_kernel((const void*)&gemm_tile_kernel<T, C, true, false, BT, false, false, AT, false, GroupedFamily<PARTS>>, grid, C::THREADS, 0, stream, &q);
}
template <class T, class C, bool PARTS, bool OK = C::VALID_AT> struct GroupedAt {
  static constexpr grouped_fn fn = nullptr;
};
template <class T, class C, bool PARTS> struct GroupedAt<T, C, PARTS, true> {
  static constexpr grouped_fn fn = &launch_grouped<T, C, false, true, PARTS>;
};
template <class T, class C, bool OK = (C::BM * C::BN <= 128 * 128)> struct GroupedParts {
  static constexpr grouped_fn nn = nullptr, bt = nullptr, at = nullptr;
};
template <class T, class C> struct GroupedParts<T, C, true> {
  static constexpr grouped_fn nn = &launch_grouped<T, C, false, false, true>, bt = &launch_grouped<T, C, true, false, true>, at = GroupedAt<T, C, true>::fn;
};

#define TNX_GROUPED_ENTRY(TAG, BM, BN, NW, ST)                                                                     \
  {TAG::ID, BM, BN, NW, ST, &launch_grouped<TAG, TileCfg<TAG, BM, BN, 128 / TAG::ES, NW, ST>, false, false>,       \
   &launch_grouped<TAG, TileCfg<TAG, BM, BN, 128 / TAG::ES, NW, ST>, true, false>,                                 \
   GroupedAt<TAG, TileCfg<TAG, BM, BN, 128 / TAG::ES, NW, ST>, false>::fn,                                         \
   {GroupedParts<TAG, TileCfg<TAG, BM, BN, 128 / TAG::ES, NW, ST>>::nn, GroupedParts<TAG, TileCfg<TAG, BM, BN, 128 / TAG::ES, NW, ST>>::bt, \
    GroupedParts<TAG, TileCfg<TAG, BM, BN, 128 / TAG::ES, NW, ST>>::at}}

}  // namespace tnx
