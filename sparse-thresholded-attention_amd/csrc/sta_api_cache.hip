// sta_api_cache.hip -- the C ABI of the paged cache and its operators (include/sta.h: sta_rotary,
// sta_cache_append, sta_paged_attention, sta_cache_evict).
#include <limits.h>
#include <math.h>

#include "../../include/sta.h"
#include "sta_api_util.h"
#include "sta_cache.h"

using namespace sta;
using namespace sta_api;

namespace {

bool dtype_ok(int dtype) {
  return dtype == STA_DTYPE_F32 || dtype == STA_DTYPE_BF16 || dtype == STA_DTYPE_F16;
}

// rows of 16-byte units at p: NULL, the pointer's and the strides' alignment
int check_rows(const char* name, const void* p, int dtype, int64_t s0, int64_t s1, int64_t s2 = 0) {
  if (!p) return fail(STA_ERR_INVALID_ARG, "%s is NULL", name);
  if (!aligned16(p)) return fail(STA_ERR_UNSUPPORTED, "%s is not 16-byte aligned", name);
  const int64_t s[3] = {s0, s1, s2};
  for (int i = 0; i < 3; ++i)
    if (s[i] < 0 || s[i] > (INT64_MAX >> 20) || (s[i] * esize(dtype)) % 16 != 0)
      return fail(STA_ERR_UNSUPPORTED, "%s stride %lld is negative, too large or not 16-byte aligned", name,
                  (long long)s[i]);
  return STA_OK;
}

// the shapes, all that the workspace sizes take
int check_cache_shape(const sta_cache& c) {
  if (!dtype_ok(c.dtype)) return fail(STA_ERR_INVALID_ARG, "dtype %d is not one of STA_DTYPE_F32/BF16/F16", c.dtype);
  if (c.D != 64 && c.D != 128) return fail(STA_ERR_UNSUPPORTED, "head_dim %d not in {64, 128}", c.D);
  if (c.Hkv < 1 || c.Hkv > 65535) return fail(STA_ERR_INVALID_ARG, "Hkv=%d outside [1, 65535]", c.Hkv);
  if (c.B < 1 || c.B > 65535) return fail(STA_ERR_INVALID_ARG, "B=%d outside [1, 65535]", c.B);
  if (c.pages < 1) return fail(STA_ERR_INVALID_ARG, "pages=%d must be >= 1", c.pages);
  if (c.page_size < 1 || c.page_size > 65536 || (c.page_size & (c.page_size - 1)) != 0)
    return fail(STA_ERR_UNSUPPORTED, "page_size %d is not a power of two up to 65536", c.page_size);
  if (c.table_width < 1 || c.table_stride < 0)
    return fail(STA_ERR_INVALID_ARG, "table_width %d must be >= 1 and table_stride %lld not negative", c.table_width,
                (long long)c.table_stride);
  return STA_OK;
}

int check_state(const char* name, const void* p, int64_t page_stride, int64_t head_stride) {
  if (p && (((uintptr_t)p & 3u) != 0 || page_stride < 0 || head_stride < 0))
    return fail(STA_ERR_UNSUPPORTED, "%s is not 4-byte aligned or has a negative stride", name);
  return STA_OK;
}

int check_cache(const sta_cache& c) {
  int rc = check_rows("cache.k", c.k, c.dtype, c.k_page_stride, c.k_head_stride, c.k_slot_stride);
  if (rc != STA_OK) return rc;
  if ((rc = check_rows("cache.v", c.v, c.dtype, c.v_page_stride, c.v_head_stride, c.v_slot_stride)) != STA_OK)
    return rc;
  if ((rc = check_state("cache.weight", c.weight, c.weight_page_stride, c.weight_head_stride)) != STA_OK) return rc;
  if ((rc = check_state("cache.pos", c.pos, c.pos_page_stride, c.pos_head_stride)) != STA_OK) return rc;
  if (!c.table || !c.lens) return fail(STA_ERR_INVALID_ARG, "cache.table and cache.lens must be non-NULL");
  return STA_OK;
}

CacheView view_of(const sta_cache& c, int max_len) {
  const int64_t es = esize(c.dtype);
  CacheView v{};
  v.k = (char*)c.k;
  v.v = (char*)c.v;
  v.k_ps = c.k_page_stride * es;
  v.k_hs = c.k_head_stride * es;
  v.k_ss = c.k_slot_stride * es;
  v.v_ps = c.v_page_stride * es;
  v.v_hs = c.v_head_stride * es;
  v.v_ss = c.v_slot_stride * es;
  v.weight = c.weight;
  v.w_ps = c.weight_page_stride;
  v.w_hs = c.weight_head_stride;
  v.pos = c.pos;
  v.p_ps = c.pos_page_stride;
  v.p_hs = c.pos_head_stride;
  v.table = c.table;
  v.t_stride = c.table_stride;
  v.lens = c.lens;
  v.pages = c.pages;
  while ((1 << v.shift) < c.page_size) ++v.shift;
  v.Hkv = c.Hkv;
  v.B = c.B;
  const int64_t cap = (int64_t)c.table_width * c.page_size;
  v.cap = (int)(cap < max_len ? cap : max_len);
  return v;
}

int check_ws(const void* ws, size_t bytes, size_t need) {
  if (!ws || bytes < need)
    return fail(STA_ERR_WORKSPACE, "workspace of %zu bytes at %p is smaller than the %zu needed", bytes, ws, need);
  if (((uintptr_t)ws & 255u) != 0) return fail(STA_ERR_WORKSPACE, "workspace must be 256-byte aligned");
  return STA_OK;
}

// -------------------------------------------------------------------------------- attention
int paged_check(const sta_paged_args* a) {
  if (!a) return fail(STA_ERR_INVALID_ARG, "args is NULL");
  int rc = check_cache_shape(a->cache);
  if (rc != STA_OK) return rc;
  if (a->H < 1 || a->H % a->cache.Hkv != 0)
    return fail(STA_ERR_INVALID_ARG, "H=%d must be a positive multiple of Hkv=%d", a->H, a->cache.Hkv);
  if (a->Q < 1 || (int64_t)a->H * a->Q > (1 << 20) || (int64_t)a->H * a->Q * a->cache.B > (1 << 26))
    return fail(STA_ERR_INVALID_ARG, "Q=%d must be >= 1, H * Q <= 2^20 and B * H * Q <= 2^26", a->Q);
  if (a->max_len < 1 || a->max_len >= (1 << 28))
    return fail(STA_ERR_INVALID_ARG, "max_len=%d outside [1, 2^28)", a->max_len);
  if (!isfinite(a->sm_scale)) return fail(STA_ERR_INVALID_ARG, "sm_scale must be finite");
  return STA_OK;
}

struct PagedLayout {
  PagedCut cut;
  size_t part_off, ml_off, stats_off, scores_off, total;
  int64_t score_stride;
};

int paged_cap(const sta_paged_args* a) {
  const int64_t cap = (int64_t)a->cache.table_width * a->cache.page_size;
  return (int)(cap < a->max_len ? cap : a->max_len);
}

PagedLayout paged_layout(const sta_paged_args* a) {
  PagedLayout L{};
  const size_t rows = (size_t)a->cache.B * a->H * a->Q;
  L.cut = paged_cut(a->cache.dtype, a->cache.D, a->H, a->cache.Hkv, a->Q, a->cache.B, paged_cap(a),
                    a->cache.page_size);
  L.score_stride = ((int64_t)paged_cap(a) + 255) / 256 * 256;   // whole units, and 256 keys of the weights
  const size_t part_rows = (size_t)L.cut.records * L.cut.rows;
  size_t off = 0;
  L.part_off = off;                                   // unfinished row tiles, fp32
  off = align256(off + part_rows * a->cache.D * 4);
  L.ml_off = off;                                     // their maxima and sums
  off = align256(off + part_rows * 8);
  // the rows' maxima and sums for the weights: several queries leave them in the whole kv heads' records, which the
  // join has read by then
  L.stats_off = a->Q > 1 ? L.ml_off + (size_t)2 * L.cut.runs * L.cut.tiles * L.cut.rows * 8 : off;
  if (a->accumulate && !L.cut.small && a->Q == 1) off = align256(off + rows * 8);
  L.scores_off = off;                                 // (B, H, Q, score_stride)
  if (a->accumulate && !L.cut.reform) off = align256(off + rows * L.score_stride * 4);
  L.total = off;
  return L;
}

// -------------------------------------------------------------------------------- eviction
int evict_check(const sta_evict_args* a) {
  if (!a) return fail(STA_ERR_INVALID_ARG, "args is NULL");
  int rc = check_cache_shape(a->cache);
  if (rc != STA_OK) return rc;
  // the kernel numbers the pairs in an int
  if ((int64_t)a->cache.B * a->cache.Hkv > INT_MAX)
    return fail(STA_ERR_INVALID_ARG, "B=%d times Hkv=%d must be below 2^31", a->cache.B, a->cache.Hkv);
  if (a->budget < 1) return fail(STA_ERR_INVALID_ARG, "budget=%d must be >= 1", a->budget);
  if (a->n_global < 0 || a->n_local < 0)
    return fail(STA_ERR_INVALID_ARG, "n_global=%d / n_local=%d must be >= 0", a->n_global, a->n_local);
  if (a->max_len < 1 || a->max_len >= (1 << 28))
    return fail(STA_ERR_INVALID_ARG, "max_len=%d outside [1, 2^28)", a->max_len);
  if (a->dst_table) {
    const int64_t keep = a->budget < a->max_len ? a->budget : a->max_len;
    if (a->dst_width < 1 || a->dst_stride < 0 || (int64_t)a->dst_width * a->cache.page_size < keep)
      return fail(STA_ERR_INVALID_ARG, "dst_table of %d pages a sequence does not hold the %lld keys that stay",
                  a->dst_width, (long long)keep);
  }
  return STA_OK;
}

struct EvictLayout {
  int moves;
  size_t counts_off, from_off, to_off, total;
};

EvictLayout evict_layout(const sta_evict_args* a) {
  EvictLayout L{};
  const int behind = a->max_len > a->budget ? a->max_len - a->budget : 0;
  // in place: at most the dropped slots in front of the budget, and at most the keys behind it
  L.moves = a->dst_table ? (a->budget < a->max_len ? a->budget : a->max_len)
                         : (a->budget < behind ? a->budget : behind);
  const size_t segs = (size_t)a->cache.B * a->cache.Hkv;
  size_t off = 0;
  L.counts_off = off;
  off = align256(off + segs * 4);
  L.from_off = off;
  off = align256(off + segs * L.moves * 4);
  L.to_off = off;
  off = align256(off + (a->dst_table ? 0 : segs * L.moves * 4));
  L.total = off;
  return L;
}

}  // namespace

extern "C" {

int sta_rotary(const sta_rotary_args* a, void* stream) {
  if (!a) return fail(STA_ERR_INVALID_ARG, "args is NULL");
  if (!dtype_ok(a->dtype)) return fail(STA_ERR_INVALID_ARG, "dtype %d is not one of STA_DTYPE_F32/BF16/F16", a->dtype);
  if (a->T < 0 || a->H < 0 || a->Hkv < 0 || a->H + (int64_t)a->Hkv < 1 || a->H + (int64_t)a->Hkv > (1 << 20))
    return fail(STA_ERR_INVALID_ARG, "T=%d, H=%d, Hkv=%d: need T >= 0 and 1 to 2^20 heads", a->T, a->H, a->Hkv);
  if (a->D < 8 || a->D > 512 || a->D % 8 != 0)
    return fail(STA_ERR_UNSUPPORTED, "head_dim %d is not a multiple of 8 up to 512", a->D);
  if (a->axes < 1 || a->axes > STA_ROTARY_MAX_AXES)
    return fail(STA_ERR_INVALID_ARG, "axes=%d outside [1, %d]", a->axes, STA_ROTARY_MAX_AXES);
  int64_t half = 0;
  for (int i = 0; i < a->axes; ++i) {
    if (a->section[i] < 0) return fail(STA_ERR_INVALID_ARG, "section[%d]=%d is negative", i, a->section[i]);
    half += a->section[i];
  }
  if (half < 1 || 2 * half > a->D || half % 8 != 0)
    return fail(STA_ERR_UNSUPPORTED, "the sections sum to %lld: need a multiple of 8 up to head_dim / 2 = %d",
                (long long)half, a->D / 2);
  if (a->pos_type < STA_POS_I32 || a->pos_type > STA_POS_F32)
    return fail(STA_ERR_INVALID_ARG, "pos_type %d is not one of STA_POS_*", a->pos_type);
  if (a->T == 0) return STA_OK;
  if (!a->positions || !a->inv_freq) return fail(STA_ERR_INVALID_ARG, "positions and inv_freq must be non-NULL");
  int rc;
  if (a->H) {
    if ((rc = check_rows("q", a->q, a->dtype, a->q_tok_stride, a->q_head_stride)) != STA_OK) return rc;
    if ((rc = check_rows("q_out", a->q_out, a->dtype, a->q_out_tok_stride, a->q_out_head_stride)) != STA_OK) return rc;
  }
  if (a->Hkv) {
    if ((rc = check_rows("k", a->k, a->dtype, a->k_tok_stride, a->k_head_stride)) != STA_OK) return rc;
    if ((rc = check_rows("k_out", a->k_out, a->dtype, a->k_out_tok_stride, a->k_out_head_stride)) != STA_OK) return rc;
  }
  hipError_t e = launch_rotary(*a, (hipStream_t)stream);
  return e == hipSuccess ? STA_OK : hip_fail(e, "rotary");
}

int sta_cache_append(const sta_append_args* a, void* stream) {
  if (!a) return fail(STA_ERR_INVALID_ARG, "args is NULL");
  int rc = check_cache_shape(a->cache);
  if (rc != STA_OK) return rc;
  if (a->T < 0) return fail(STA_ERR_INVALID_ARG, "T=%d must be >= 0", a->T);
  // four tokens a workgroup of 256 threads, below 2^32 threads
  if ((int64_t)a->T * a->cache.Hkv >= ((int64_t)1 << 31) || a->T > (1 << 26) - 4)
    return fail(STA_ERR_UNSUPPORTED, "T=%d must be at most 2^26 - 4, and times Hkv=%d below 2^31", a->T, a->cache.Hkv);
  if (!a->starts && a->T != a->cache.B)
    return fail(STA_ERR_INVALID_ARG, "without starts T=%d must be B=%d", a->T, a->cache.B);
  if ((rc = check_cache(a->cache)) != STA_OK) return rc;
  if (a->T) {
    if ((rc = check_rows("k", a->k, a->cache.dtype, a->k_tok_stride, a->k_head_stride)) != STA_OK) return rc;
    if ((rc = check_rows("v", a->v, a->cache.dtype, a->v_tok_stride, a->v_head_stride)) != STA_OK) return rc;
  }
  if (!a->new_lens) return fail(STA_ERR_INVALID_ARG, "new_lens must be non-NULL");
  if (a->new_lens == a->cache.lens) return fail(STA_ERR_INVALID_ARG, "new_lens must not be cache.lens");
  const int64_t es = esize(a->cache.dtype);
  AppendArgs d{};
  d.c = view_of(a->cache, INT_MAX);
  d.k = (const char*)a->k;
  d.v = (const char*)a->v;
  d.k_ts = a->k_tok_stride * es;
  d.k_hs = a->k_head_stride * es;
  d.v_ts = a->v_tok_stride * es;
  d.v_hs = a->v_head_stride * es;
  d.T = a->T;
  while ((16 << d.row_shift) < a->cache.D * es) ++d.row_shift;
  d.starts = a->starts;
  d.seen = a->seen;
  d.new_lens = a->new_lens;
  hipError_t e = launch_append(d, (hipStream_t)stream);
  return e == hipSuccess ? STA_OK : hip_fail(e, "cache append");
}

size_t sta_paged_workspace_size(const sta_paged_args* a) {
  if (paged_check(a) != STA_OK) return 0;
  const size_t total = paged_layout(a).total;
  return total ? total : 1;
}

int sta_paged_attention(const sta_paged_args* a, void* stream) {
  int rc = paged_check(a);
  if (rc != STA_OK) return rc;
  if ((rc = check_cache(a->cache)) != STA_OK) return rc;
  if ((rc = check_rows("q", a->q, a->cache.dtype, a->q_batch_stride, a->q_head_stride, a->q_tok_stride)) != STA_OK)
    return rc;
  if (!a->out || !aligned16(a->out)) return fail(STA_ERR_INVALID_ARG, "out must be non-NULL and 16-byte aligned");
  if (a->accumulate && !a->cache.weight) return fail(STA_ERR_INVALID_ARG, "accumulate needs cache.weight");
  const PagedLayout L = paged_layout(a);
  if (L.total && (rc = check_ws(a->workspace, a->workspace_bytes, L.total)) != STA_OK) return rc;
  char* ws = (char*)a->workspace;
  PagedArgs d{};
  d.c = view_of(a->cache, a->max_len);
  d.q = a->q;
  d.q_bs = a->q_batch_stride;
  d.q_hs = a->q_head_stride;
  d.q_ts = a->q_tok_stride;
  d.H = a->H;
  d.Q = a->Q;
  d.sm_scale = a->sm_scale;
  d.accumulate = a->accumulate != 0;
  d.out = a->out;
  d.lse = a->lse;
  d.stats = a->accumulate && !L.cut.small ? (float2*)(ws + L.stats_off) : nullptr;
  d.stat_stride = a->Q > 1 ? (int64_t)L.cut.tiles * L.cut.rows : a->H / a->cache.Hkv;
  d.scores = a->accumulate && !L.cut.reform ? (float*)(ws + L.scores_off) : nullptr;
  d.score_stride = L.score_stride;
  d.part_o = (float*)(ws + L.part_off);
  d.part_ml = (float2*)(ws + L.ml_off);
  d.runs = L.cut.runs;
  hipError_t e = launch_paged(a->cache.dtype, a->cache.D, d, (hipStream_t)stream);
  return e == hipSuccess ? STA_OK : hip_fail(e, "paged attention");
}

size_t sta_evict_workspace_size(const sta_evict_args* a) {
  if (evict_check(a) != STA_OK) return 0;
  return evict_layout(a).total;
}

int sta_cache_evict(const sta_evict_args* a, void* stream) {
  int rc = evict_check(a);
  if (rc != STA_OK) return rc;
  if ((rc = check_cache(a->cache)) != STA_OK) return rc;
  if (!a->cache.weight || !a->cache.pos)
    return fail(STA_ERR_INVALID_ARG, "eviction needs cache.weight and cache.pos");
  if (!a->new_lens) return fail(STA_ERR_INVALID_ARG, "new_lens must be non-NULL");
  if (a->new_lens == a->cache.lens) return fail(STA_ERR_INVALID_ARG, "new_lens must not be cache.lens");
  const EvictLayout L = evict_layout(a);
  if ((rc = check_ws(a->workspace, a->workspace_bytes, L.total)) != STA_OK) return rc;
  char* ws = (char*)a->workspace;
  EvictArgs d{};
  d.c = view_of(a->cache, a->max_len);
  d.budget = a->budget;
  d.n_global = a->n_global;
  d.n_local = a->n_local;
  d.row_bytes = a->cache.D * esize(a->cache.dtype);
  d.dst_table = a->dst_table;
  d.dst_stride = a->dst_stride;
  const int64_t dst_cap = (int64_t)a->dst_width * a->cache.page_size;
  d.dst_cap = (int)(dst_cap < INT_MAX ? dst_cap : INT_MAX);
  d.new_lens = a->new_lens;
  d.counts = (int32_t*)(ws + L.counts_off);
  d.from = (int32_t*)(ws + L.from_off);
  d.to = (int32_t*)(ws + L.to_off);
  d.moves = L.moves;
  hipError_t e = launch_evict(d, (hipStream_t)stream);
  return e == hipSuccess ? STA_OK : hip_fail(e, "cache eviction");
}

}  // extern "C"
