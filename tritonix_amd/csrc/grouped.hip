// Products grouped by ragged runs of rows (gemm_grouped.h): argument checks, the choice of tile, launch.
#include <hip/hip_runtime.h>

#include <cmath>
#include <string.h>
#include <unordered_map>

#include "../../include/tritonix_hip.h"
#include "registry.h"
#include "gemm_linear.h"
#include "gemm_grouped.h"
#include "gemm_stream.h"

using namespace tnx;

extern "C" const GroupedGroup* const* tnx_grouped_groups(int* ngroups);  // generated

namespace {

bool gradient(const tnx_grouped_args* a) { return a->form == TNX_GROUPED_WEIGHT_GRADIENT; }

int check(const tnx_grouped_args* a) {
  if (!a || a->rows < 0 || a->n < 0 || a->k < 0 || a->groups < 1 || a->parts < 0) return TNX_E_INVALID;
  if (a->form != TNX_GROUPED_ROWS && a->form != TNX_GROUPED_WEIGHT_GRADIENT) return TNX_E_INVALID;
  if (a->dtype != TNX_F16 && a->dtype != TNX_BF16 && a->dtype != TNX_F32) return TNX_E_UNSUPPORTED;
  if (a->rows > 0x3fffffff || a->n > 0x3fffffff || a->k > 0x3fffffff || a->groups > TNX_GROUPED_MAX_GROUPS) return TNX_E_UNSUPPORTED;
  return TNX_OK;
}

// Which kernel of a tile the operands take and whether the last slab of k is left out of its ring: the conditions of the tile kernels'
// DMA loader (dma_layout in capi.hip), for every group at once.  false: none takes them.
struct Layout {
  bool bt, tail;
};
bool layout_of(const tnx_grouped_args* a, int bm, int bn, Layout* l) {
  const int es = a->dtype == TNX_F32 ? 4 : 2, vec = 16 / es, bk = 128 / es;
  const bool at = gradient(a);
  if (a->stride_ak != 1 || a->stride_ar < a->k) return false;
  if (at && (a->stride_bn != 1 || a->stride_bk < a->n)) return false;
  l->bt = !at && !(a->stride_bn == 1 && a->stride_bk >= a->n);
  if (l->bt && !(a->stride_bk == 1 && a->stride_bn >= a->k)) return false;
  const int64_t ldb = l->bt ? a->stride_bn : a->stride_bk;
  // a lane's offsets within a tile are of 32 bits
  const int64_t reach_a = (int64_t)(at ? bk : bm) * a->stride_ar * es + (int64_t)bm * es, reach_b = (int64_t)(l->bt ? bn : bk) * ldb * es + (int64_t)bn * es;
  if (reach_a >= (1ll << 32) || reach_b >= (1ll << 32)) return false;
  const bool pointers = !(((uintptr_t)a->a | (uintptr_t)a->b) & 15);
  bool aligned = pointers && a->stride_ar * es % 16 == 0 && ldb * es % 16 == 0;
  if (at) aligned = aligned && a->k % vec == 0 && a->n % vec == 0;
  else aligned = aligned && a->stride_group * es % 16 == 0 && a->k % bk == 0 && (l->bt || a->n % vec == 0);
  l->tail = !aligned;
  if (aligned) return true;
  if (at) return ring_chunks_inside(1, a->n, ldb, vec) && ring_chunks_inside(1, a->k, a->stride_ar, vec);
  return l->bt || ring_chunks_inside((a->k - 1) % bk + 1, a->n, ldb, vec);
}

// Modelled microseconds of a tile, as capi.hip has them (TileCost), and what streaming the weights with it costs against the best, row-major and
// k-contiguous; four of the constants moved by up to 5 percent (one by a third) towards what 108 grouped problems measured, on which the choice
// then takes 1.011x the best tile's time in the mean, 1.24x at most.  burst: of a short k the results are the time, and tiles of long rows write them
// faster once they are more than a few MB (32768 rows, 32 groups, 128 x 2048 bf16: 256x256 44.7 us, 128x256 54, 128x128 79; 30000 rows, 4 groups, 64 x 3584 54, 65,
// 95), by what each takes of the results' bytes at 5.05 TB/s beyond the fastest.
struct Cost {
  int bm, bn, nw, stages;
  double start, turn, slab, shared, crowd, tail, stream_nn, stream_nt, burst;
};
const Cost COST16[] = {{256, 256, 8, 2, 4.16, 0.001, 1.12, 1.89, 0.278, 2.8, 1.35, 1.45, 0.0},    {256, 128, 8, 3, 4.24, 0.735, 0.575, 5.24, 0.439, 2.3, 1.2, 1.25, 0.27},
                       {128, 256, 8, 3, 4.5, 1.7, 0.545, 17.8, 0.442, 2.08, 1.1, 1.2, 0.3},       {128, 128, 8, 3, 3.91, 0.51, 0.374, 2.18, 0.439, 1.32, 1.12, 1.15, 0.95},
                       {64, 128, 8, 3, 3.63, 1.11, 0.328, 0.975, 0.0551, 0.653, 1.0, 1.08, 0.95},  {64, 64, 4, 4, 3.62, 0.794, 0.203, 0.656, 0.308, 0.896, 1.06, 1.03, 1.9},
                       {32, 128, 4, 3, 3.81, 0.918, 0.259, 0.495, 0.171, 0.983, 1.05, 1.1, 2.3},  {32, 64, 4, 4, 3.48, 0.431, 0.143, 1.1, 0.276, 0.682, 1.1, 1.05, 2.6}};
const Cost COST32[] = {{64, 64, 4, 4, 3.78, 0.0015, 0.508, 0.815, 0.006, 0.611, 1.0, 1.0, 0.0}, {32, 128, 4, 3, 4.29, 1.2, 0.535, 0.695, 0.151, 0.782, 1.0, 1.0, 0.0},
                       {32, 64, 4, 4, 3.68, 0.034, 0.279, 1.48, 0.133, 0.498, 1.0, 1.0, 0.0}};

constexpr double CUS = 256;

double compute_time(const Cost& t, double tiles, double kt, bool tail, bool at) {
  const int lds = (t.bm + t.bn) * 128 * t.stages, fit = TNX_LDS_LIMIT_BYTES / lds, most = t.nw == 8 ? 2 : 3;
  const double c = fit < 1 ? 1 : fit < most ? fit : most, fill = tiles < CUS ? tiles / CUS : 1.0, crowd = 1.0 + t.crowd * fill * fill;
  const double full = std::floor(tiles / (CUS * c)), rem = tiles - full * CUS * c, n = std::ceil(rem / CUS);
  // (a workgroup alone on its CU has its last slab, its first and its stores to itself; every group of a gradient has a last slab)
  const double own = (tail ? t.tail : 0.0) * (at ? 1.0 : 0.5) + (at ? 2.0 * t.bm * t.bn / 65536.0 : 0.0);
  double us = t.start + (tail ? t.tail : 0.0) + full * (t.slab * kt * (c > 1 ? 1.0 + t.shared : 1.0) * crowd + c * t.turn + own * c / (c > 1 ? 1.6 : 1.0));
  if (rem > 0) us += t.slab * kt * (c > 1 ? 1.0 + t.shared * (n - 1) / (c - 1) : 1.0) * crowd + (n - 1) * t.turn;
  return us;
}

struct Choice {
  const GroupedEntry* entry;
  int parts;
};

const GroupedEntry* entry_of(int dtype, int bm, int bn) {
  int ng = 0;
  const GroupedGroup* const* g = tnx_grouped_groups(&ng);
  for (int i = 0; i < ng; ++i)
    for (int j = 0; j < g[i]->count; ++j)
      if (g[i]->entries[j].dtype == dtype && g[i]->entries[j].bm == bm && g[i]->entries[j].bn == bn) return &g[i]->entries[j];
  return nullptr;
}

// The most tiles that the rows can make.
int64_t tiles_of(const tnx_grouped_args* a, int bm, int bn) {
  const int64_t down = gradient(a) ? a->groups * ((a->k + bm - 1) / bm) : a->rows / bm + (a->groups + 2 < a->rows ? a->groups + 2 : a->rows);
  return down * ((a->n + bn - 1) / bn);
}
// Parts of k, and slabs of each: none without a slab of its own.
int parts_of(const tnx_grouped_args* a, int asked, int64_t* per) {
  const int bk = a->dtype == TNX_F32 ? 32 : 64;
  const int64_t slabs = gradient(a) ? a->rows / bk + 1 : a->k > 0 ? (a->k + bk - 1) / bk : 1;
  const int parts = asked > slabs ? (int)slabs : asked;
  *per = parts > 1 ? (slabs + parts - 1) / parts : slabs;
  return parts > 1 && !gradient(a) ? (int)((slabs + *per - 1) / *per) : parts;
}
// A grid's threads are counted in 32 bits: what makes more is refused.
bool launchable(const tnx_grouped_args* a, const GroupedEntry* e, int parts) { return (double)tiles_of(a, e->bm, e->bn) * parts * e->nw * 64 < 4294967296.0; }

int64_t sums_of(const tnx_grouped_args* a) { return gradient(a) ? (int64_t)a->groups * a->k * a->n : a->rows * a->n; }
constexpr int64_t MOST_PART_BYTES = 64 << 20;

// The tile, and the parts of k, of the smallest modelled time.  What the groups are is not known here: rows are taken as spread evenly, half a tile of each group
// as empty.
Choice make_choice(const tnx_grouped_args* a) {
  const bool at = gradient(a);
  if (a->block_m > 0) return {entry_of(a->dtype, a->block_m, a->block_n), a->parts > 0 ? a->parts : 1};
  const bool f32 = a->dtype == TNX_F32;
  const Cost* table = f32 ? COST32 : COST16;
  const int count = f32 ? 3 : 8, es = f32 ? 4 : 2, bk = 128 / es;
  const double rows = (double)a->rows, groups = (double)a->groups, used = a->rows < a->groups ? rows : groups;
  const double active = groups * (1.0 - std::pow(1.0 - 1.0 / groups, rows));
  const double bytes = at ? (rows * (a->k + a->n) + groups * a->k * a->n) * es : (rows * (a->k + a->n) + active * a->k * a->n) * es;
  const double written = rows * (double)a->n * es;
  const bool bt = !at && a->stride_bn != 1, tail = at || a->k % bk != 0 || a->n % 8 != 0;
  static const int cuts[] = {1, 2, 3, 4, 6, 8, 12, 16};
  double best = 1e300;
  Choice pick = {nullptr, 1};
  for (int i = 0; i < count; ++i) {
    const Cost& t = table[i];
    const GroupedEntry* e = entry_of(a->dtype, t.bm, t.bn);
    if (!e || (at ? !e->at : false)) continue;
    const double each = rows / (used > 0 ? used : 1), across = std::ceil((double)a->n / t.bn);
    const double spare = each > t.bm / 2 ? 0.5 * used : used * (each < t.bm ? 1.0 - each / t.bm : 0.0);
    const double tiles = at ? groups * std::ceil((double)a->k / t.bm) * across : (rows / t.bm + spare) * across;
    const double kt = at ? std::ceil(each / bk) : std::ceil((double)a->k / bk);
    for (int s : cuts) {
      if (s > 1 && (!e->parts[at ? 2 : bt ? 1 : 0] || kt / s < 2 || tiles * s > 3 * CUS || (double)s * sums_of(a) * 4 > MOST_PART_BYTES)) break;
      if (!launchable(a, e, s)) break;
      double us = compute_time(t, tiles * s, std::ceil(kt / s), tail, at);
      const double stream = bytes / 5.1e6 * (at ? 1.1 : bt ? t.stream_nt : t.stream_nn) + 2.5;
      const double p = at ? 2.0 : 4.0;
      us = std::pow(std::pow(us, p) + std::pow(stream, p), 1.0 / p);
      if (!at) us += t.burst * (written > 3e6 ? written - 3e6 : 0.0) / 5.05e6 * (kt < 8 ? 1.0 : 8.0 / kt);
      if (s > 1) us += 3.0 + (2.0 * s * 4 + es) * sums_of(a) / 8e6;
      if (us < best * (s > 1 ? 0.95 : 1.0)) { best = us; pick = {e, s}; }
    }
  }
  return pick;
}

struct Key {
  int64_t v[8];
  bool operator==(const Key& o) const { return memcmp(this, &o, sizeof *this) == 0; }
};
struct KeyHash {
  size_t operator()(const Key& k) const {
    uint64_t h = 0x9e3779b97f4a7c15ull;
    for (int64_t w : k.v) h = ((h ^ (uint64_t)w) * 0xff51afd7ed558ccdull) ^ (h >> 29);
    return (size_t)h;
  }
};
// kept by thread: it takes longer than a launch
Choice choose(const tnx_grouped_args* a) {
  static thread_local std::unordered_map<Key, Choice, KeyHash> kept;
  const Key k = {{a->rows, a->n, a->k, a->groups, a->dtype, a->form * 2 + (a->stride_bn != 1), (int64_t)a->block_m << 32 | a->block_n, a->parts}};
  const auto hit = kept.find(k);
  if (hit != kept.end()) return hit->second;
  if (kept.size() >= 512) kept.clear();
  return kept[k] = make_choice(a);
}

// out[i] = the sum of the parts' i-th elements in order, four a thread
template <class O> __global__ __launch_bounds__(256) void join_kernel(const float* parts, int count, int64_t stride, int64_t total, uint8_t* out) {
  typedef typename O::raw raw;
  const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (at >= total) return;
  if (at + 4 <= total) {
    f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int i = 0; i < count; ++i) {
      f32x4 v;
      __builtin_memcpy(&v, parts + i * stride + at, 16);
      s += v;
    }
    raw r[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = O::cvt(s[e]);
    __builtin_memcpy((raw*)out + at, r, sizeof r);
  } else {
    for (int64_t j = at; j < total; ++j) {
      float s = 0.0f;
      for (int i = 0; i < count; ++i) s += parts[i * stride + j];
      ((raw*)out)[j] = O::cvt(s);
    }
  }
}

// Few rows by k-contiguous weights, which gemm_stream.h reads once a group for up to 8 rows: 8 rows in all, or 4 to a group on average (us,
// against the tile kernels': 32 rows, 8 groups, 14336 x 4096 144 and 164, 64 rows 212 and 164; 128 rows, 32 groups, 4096 x 4096 153 and 173), but not many workgroups of a short k (256 rows, 64 groups, 1024 x 4096
// 88 and 82; 4 rows 8.2 and 8.5, 64 rows, 16 groups, 700 x 1000 7.4 and 8.8).  float32 gains more: 8 rows, 128 groups, 2048 x 768 12.5 and 18.6, 128 rows,
// 32 groups, 4096 x 4096 318 and 339.  Rows off whole words, whose loads take twice the time, while there is little of them (1 row, 64 groups, 4097 x 2048 10.9 and
// 14.3, 4 rows 33 and 24).
bool takes_stream(const tnx_grouped_args* a) {
  if (gradient(a) || a->block_m > 0 || a->k == 0 || a->stride_ak != 1 || a->stride_ar < a->k) return false;
  if (a->stride_bn == 1 || a->stride_bk != 1 || a->stride_bn < a->k) return false;
  const int64_t columns = (a->rows < a->groups ? a->rows : a->groups) * a->n;
  if (a->k < 2048 && columns > 16384) return false;
  const bool words = a->dtype == TNX_F32 || (!(((uintptr_t)a->a | (uintptr_t)a->b) & 3) && a->stride_ar % 2 == 0 && a->stride_bn % 2 == 0 && a->stride_group % 2 == 0);
  if (!words && columns * a->k > 8 << 20) return false;
  // (a grid's threads are counted in 32 bits)
  return (a->rows <= 8 || a->rows <= 4 * (int64_t)a->groups) && stream_runs(a->rows, a->groups) * ((a->n + 7) / 8) < (1 << 23) - 1;
}

// Up to 8 rows by row-major weights, while blocks of 64 columns times groups leave half of the CUs without a workgroup and k has parts for them: those
// parts, a workgroup to a CU, or 0: not taken (us, against the tile kernels': 1 row, 64 groups, 4096 x 2048 9.5 and 15.7, 4 rows 17.4 and 21.2, 2 rows, 128
// groups, 2048 x 768 7.4 and 14.2; a workgroup to every block without parts, 8 rows, 64 groups, 4096 x 2048: 26.4 and 24.9).  float32 has blocks of 32 columns
// and as many parts for each, two workgroups to a CU: 4 rows, 64 groups, 4096 x 2048 27.4 and 32.2, 2 rows, 128 groups, 2048 x 768 9.3 and 15.9.
int stream_rows_parts(const tnx_grouped_args* a) {
  if (gradient(a) || a->block_m > 0 || a->stride_ak != 1 || a->stride_ar < a->k) return 0;
  if (a->stride_bn != 1 || a->stride_bk < a->n || a->n < 8 || a->rows > 8) return 0;
  const int64_t blocks = (a->rows < a->groups ? a->rows : a->groups) * ((a->n + 63) / 64), most = a->k / (64 * STREAM_ROWS_WAVES);
  int64_t parts = blocks > 0 ? 256 / blocks : 0;
  if (parts > most) parts = most;
  return parts >= 2 ? (int)parts : 0;
}

hipError_t join(const tnx_grouped_args* a, int parts, int64_t sums) {
  const dim3 grid((unsigned)((sums + 1023) / 1024));
  const float* from = (const float*)a->workspace;
  const hipStream_t stream = (hipStream_t)a->stream;
  if (a->dtype == TNX_BF16) hipLaunchKernelGGL(join_kernel<OutBF16>, grid, dim3(256), 0, stream, from, parts, sums, sums, (uint8_t*)a->c);
  else if (a->dtype == TNX_F16) hipLaunchKernelGGL(join_kernel<OutF16>, grid, dim3(256), 0, stream, from, parts, sums, sums, (uint8_t*)a->c);
  else hipLaunchKernelGGL(join_kernel<OutF32>, grid, dim3(256), 0, stream, from, parts, sums, sums, (uint8_t*)a->c);
  return hipGetLastError();
}

}  // namespace

extern "C" size_t tnx_grouped_workspace_bytes(const tnx_grouped_args* a) {
  if (check(a) != TNX_OK || a->n == 0 || (gradient(a) ? a->k == 0 : a->rows == 0)) return 0;
  if (takes_stream(a)) return 0;
  if (const int parts = stream_rows_parts(a)) return (size_t)parts * sums_of(a) * 4;
  const Choice c = choose(a);
  return c.entry && c.parts > 1 ? (size_t)c.parts * sums_of(a) * 4 : 0;
}

extern "C" int tnx_grouped(const tnx_grouped_args* a) {
  const int st = check(a);
  if (st != TNX_OK) return st;
  const bool at = gradient(a);
  if (a->n == 0 || (at ? a->k == 0 : a->rows == 0)) return TNX_OK;
  if (!a->offsets || !a->c || (a->rows > 0 && a->k > 0 && (!a->a || !a->b))) return TNX_E_INVALID;
  if (takes_stream(a)) {
    GroupedParams p = {};
    p.a = (const uint8_t*)a->a; p.b = (const uint8_t*)a->b; p.c = (uint8_t*)a->c;
    p.offsets = a->offsets;
    p.lda = a->stride_ar; p.ldb = a->stride_bn;
    p.group_stride = a->stride_group;
    p.rows = (int32_t)a->rows; p.n = (int32_t)a->n; p.k = (int32_t)a->k;
    p.groups = a->groups;
    const hipStream_t s = (hipStream_t)a->stream;
    const hipError_t err = a->dtype == TNX_F32 ? grouped_stream<TagF32>(p, s) : a->dtype == TNX_BF16 ? grouped_stream<TagBF16>(p, s) : grouped_stream<TagF16>(p, s);
    if (err != hipSuccess) { note_hip_error((int)err); return TNX_E_HIP; }
    return TNX_OK;
  }
  if (const int parts = a->workspace && a->k > 0 ? stream_rows_parts(a) : 0) {
    const int64_t sums = sums_of(a);
    if (a->workspace_bytes < (size_t)parts * sums * 4 || ((uintptr_t)a->workspace & 15)) return TNX_E_WORKSPACE;
    GroupedParams p = {};
    p.a = (const uint8_t*)a->a; p.b = (const uint8_t*)a->b; p.c = (uint8_t*)a->workspace;
    p.offsets = a->offsets;
    p.lda = a->stride_ar; p.ldb = a->stride_bk;
    p.group_stride = a->stride_group;
    p.rows = (int32_t)a->rows; p.n = (int32_t)a->n; p.k = (int32_t)a->k;
    p.groups = a->groups;
    p.parts = parts; p.part_stride = sums;
    const hipStream_t s = (hipStream_t)a->stream;
    hipError_t err = a->dtype == TNX_F32 ? grouped_stream_rows<TagF32>(p, s) : a->dtype == TNX_BF16 ? grouped_stream_rows<TagBF16>(p, s) : grouped_stream_rows<TagF16>(p, s);
    if (err == hipSuccess) err = join(a, parts, sums);
    if (err != hipSuccess) { note_hip_error((int)err); return TNX_E_HIP; }
    return TNX_OK;
  }
  Choice c = choose(a);
  const GroupedEntry* e = c.entry;
  if (!e) return TNX_E_UNSUPPORTED;
  Layout l;
  if (!layout_of(a, e->bm, e->bn, &l)) return TNX_E_UNSUPPORTED;
  const int which = at ? 2 : l.bt ? 1 : 0;
  const int64_t sums = sums_of(a);
  int64_t per;
  c.parts = parts_of(a, a->workspace ? c.parts : 1, &per);                    // (without a workspace no parts)
  const size_t need = c.parts > 1 ? (size_t)c.parts * sums * 4 : 0;
  if (c.parts > 1 && (a->workspace_bytes < need || ((uintptr_t)a->workspace & 15))) return TNX_E_WORKSPACE;
  const bool cut = c.parts > 1;
  const grouped_fn fn = cut ? e->parts[which] : which == 2 ? e->at : which == 1 ? e->bt : e->nn;
  if (!fn) return TNX_E_UNSUPPORTED;
  if (!launchable(a, e, c.parts) || (cut && (sums + 1023) / 1024 > 0xffffffffll / 256)) return TNX_E_UNSUPPORTED;
  GroupedParams p;
  p.a = (const uint8_t*)a->a; p.b = (const uint8_t*)a->b; p.c = cut ? (uint8_t*)a->workspace : (uint8_t*)a->c;
  p.offsets = a->offsets;
  p.lda = a->stride_ar; p.ldb = l.bt ? a->stride_bn : a->stride_bk;
  p.group_stride = a->stride_group;
  p.rows = (int32_t)a->rows; p.n = (int32_t)a->n; p.k = (int32_t)a->k;
  p.groups = a->groups; p.group_m = 8;
  p.parts = c.parts; p.per_part = (int32_t)per; p.part_stride = sums;
  p.flags = l.tail ? PF_TAIL : 0u;
  const hipError_t err = fn(p, (unsigned)(tiles_of(a, e->bm, e->bn) * c.parts), (hipStream_t)a->stream);
  if (err != hipSuccess) { note_hip_error((int)err); return TNX_E_HIP; }
  if (!cut) return TNX_OK;
  const hipError_t joined = join(a, c.parts, sums);
  if (joined != hipSuccess) { note_hip_error((int)joined); return TNX_E_HIP; }
  return TNX_OK;
}

extern "C" int tnx_grouped_route(const tnx_grouped_args* a, int32_t info[5]) {
  if (check(a) != TNX_OK) return 0;
  const int parts = a->k > 0 ? stream_rows_parts(a) : 0;
  if (parts || takes_stream(a)) {
    if (info) {
      memset(info, 0, 5 * sizeof *info);
      info[4] = parts;
    }
    return 2;
  }
  const Choice c = choose(a);
  const GroupedEntry* e = c.entry;
  Layout l;
  int64_t per;
  if (!e || !layout_of(a, e->bm, e->bn, &l) || !(gradient(a) ? e->at : l.bt ? e->bt : e->nn) || !launchable(a, e, parts_of(a, c.parts, &per))) return 0;
  if (info) { info[0] = e->bm; info[1] = e->bn; info[2] = e->nw; info[3] = l.tail; info[4] = c.parts; }
  return 1;
}
