// Products grouped by ragged runs of rows (gemm_grouped.h): argument checks, the choice of tile, launch.
#include <hip/hip_runtime.h>

#include "../../include/tritonix_hip.h"
#include "registry.h"
#include "gemm_grouped.h"

using namespace tnx;

extern "C" const GroupedGroup* const* tnx_grouped_groups(int* ngroups);  // generated

namespace {

bool gradient(const tnx_grouped_args* a) { return a->form == TNX_GROUPED_WEIGHT_GRADIENT; }

int check(const tnx_grouped_args* a) {
  if (!a || a->rows < 0 || a->n < 0 || a->k < 0 || a->groups < 1) return TNX_E_INVALID;
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

const GroupedEntry* entry_of(int dtype, int bm, int bn) {
  int ng = 0;
  const GroupedGroup* const* g = tnx_grouped_groups(&ng);
  for (int i = 0; i < ng; ++i)
    for (int j = 0; j < g[i]->count; ++j)
      if (g[i]->entries[j].dtype == dtype && (bm <= 0 || (g[i]->entries[j].bm == bm && g[i]->entries[j].bn == bn))) return &g[i]->entries[j];
  return nullptr;
}

const GroupedEntry* choose(const tnx_grouped_args* a) {
  if (a->block_m > 0) return entry_of(a->dtype, a->block_m, a->block_n);
  if (a->dtype == TNX_F32) return entry_of(a->dtype, 64, 64);
  if (gradient(a)) return (int64_t)a->groups * ((a->k + 127) / 128) * ((a->n + 127) / 128) >= 256 ? entry_of(a->dtype, 128, 128) : entry_of(a->dtype, 64, 64);
  const int64_t each = a->rows / a->groups;
  return each >= 256 ? entry_of(a->dtype, 256, 256) : each >= 64 ? entry_of(a->dtype, 128, 128) : entry_of(a->dtype, 64, 64);
}

}  // namespace

extern "C" int tnx_grouped(const tnx_grouped_args* a) {
  const int st = check(a);
  if (st != TNX_OK) return st;
  const bool at = gradient(a);
  if (a->n == 0 || (at ? a->k == 0 : a->rows == 0)) return TNX_OK;
  if (!a->offsets || !a->c || (a->rows > 0 && a->k > 0 && (!a->a || !a->b))) return TNX_E_INVALID;
  const GroupedEntry* e = choose(a);
  if (!e) return TNX_E_UNSUPPORTED;
  Layout l;
  if (!layout_of(a, e->bm, e->bn, &l)) return TNX_E_UNSUPPORTED;
  const grouped_fn fn = at ? e->at : l.bt ? e->bt : e->nn;
  if (!fn) return TNX_E_UNSUPPORTED;
  const int64_t tiles_n = (a->n + e->bn - 1) / e->bn;
  const int64_t tiles_m = at ? a->groups * ((a->k + e->bm - 1) / e->bm) : a->rows / e->bm + (a->groups + 2 < a->rows ? a->groups + 2 : a->rows);
  if (tiles_m * tiles_n > 0x7fffffff) return TNX_E_UNSUPPORTED;
  GroupedParams p;
  p.a = (const uint8_t*)a->a; p.b = (const uint8_t*)a->b; p.c = (uint8_t*)a->c;
  p.offsets = a->offsets;
  p.lda = a->stride_ar; p.ldb = l.bt ? a->stride_bn : a->stride_bk;
  p.group_stride = a->stride_group;
  p.rows = (int32_t)a->rows; p.n = (int32_t)a->n; p.k = (int32_t)a->k;
  p.groups = a->groups; p.group_m = 8;
  p.flags = l.tail ? PF_TAIL : 0u;
  const hipError_t err = fn(p, (unsigned)(tiles_m * tiles_n), (hipStream_t)a->stream);
  if (err != hipSuccess) { note_hip_error((int)err); return TNX_E_HIP; }
  return TNX_OK;
}

extern "C" int tnx_grouped_route(const tnx_grouped_args* a, int32_t info[4]) {
  if (check(a) != TNX_OK) return 0;
  const GroupedEntry* e = choose(a);
  Layout l;
  if (!e || !layout_of(a, e->bm, e->bn, &l) || !(gradient(a) ? e->at : l.bt ? e->bt : e->nn)) return 0;
  if (info) { info[0] = e->bm; info[1] = e->bn; info[2] = e->nw; info[3] = l.tail; }
  return 1;
}
