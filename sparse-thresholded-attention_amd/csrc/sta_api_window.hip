// sta_api_window.hip -- the C ABI of attention over packed sequences with a sliding window and sinks
// (include/sta.h: sta_window_attention, sta_window_attention_grad).
#include <float.h>
#include <limits.h>
#include <math.h>

#include "../../include/sta.h"
#include "sta_api_util.h"
#include "sta_window.h"

using namespace sta;
using namespace sta_api;

namespace {

// a copy's rows are 32-bit offsets from its first one, up to 7 token strides
int check_rows(const char* name, const void* p, int dtype, int rows, int64_t s0, int64_t s1) {
  if (!p) return fail(STA_ERR_INVALID_ARG, "%s is NULL", name);
  if (!aligned16(p)) return fail(STA_ERR_UNSUPPORTED, "%s is not 16-byte aligned", name);
  const int64_t s[2] = {s0, s1};
  for (int i = 0; i < 2; ++i)
    if (s[i] < 0 || s[i] > (INT64_MAX >> 20) || (s[i] * esize(dtype)) % 16 != 0)
      return fail(STA_ERR_UNSUPPORTED, "%s stride %lld is negative, too large or not 16-byte aligned", name,
                  (long long)s[i]);
  if (rows > 1 && s0 * esize(dtype) > (1 << 29))
    return fail(STA_ERR_UNSUPPORTED, "%s token stride %lld is above 2^29 bytes", name, (long long)s0);
  return STA_OK;
}

int check_out(const char* name, const void* p) {
  if (!p || !aligned16(p)) return fail(STA_ERR_INVALID_ARG, "%s must be non-NULL and 16-byte aligned", name);
  return STA_OK;
}

// keys of a window and sinks as the kernels take them: a window that with the sinks reaches every key is none
int window_of(const sta_window_args* a) {
  return a->window == 0 || (int64_t)a->window + a->sinks >= a->S ? INT_MAX : a->window;
}
int sinks_of(const sta_window_args* a) { return a->sinks < a->S ? a->sinks : a->S; }

WindowCut cut_of(const sta_window_args* a) {
  return window_cut(a->dtype, a->D, a->T, a->S, a->H, a->Hkv, a->B, a->starts != nullptr, a->k_starts != nullptr,
                    window_of(a), sinks_of(a));
}

// the shapes, all that the workspace size takes
int check_shape(const sta_window_args* a) {
  if (!a) return fail(STA_ERR_INVALID_ARG, "args is NULL");
  if (a->dtype != STA_DTYPE_F32 && a->dtype != STA_DTYPE_BF16 && a->dtype != STA_DTYPE_F16)
    return fail(STA_ERR_INVALID_ARG, "dtype %d is not one of STA_DTYPE_F32/BF16/F16", a->dtype);
  if (a->D != 64 && a->D != 128) return fail(STA_ERR_UNSUPPORTED, "head_dim %d not in {64, 128}", a->D);
  if (a->T < 0 || a->S < 0 || a->T > (1 << 28) || a->S > (1 << 28))
    return fail(STA_ERR_INVALID_ARG, "T=%d and S=%d must lie in [0, 2^28]", a->T, a->S);
  if (a->Hkv < 1 || a->H < 1 || a->H > 65535 || a->H % a->Hkv != 0)
    return fail(STA_ERR_INVALID_ARG, "H=%d must be a multiple of Hkv=%d up to 65535", a->H, a->Hkv);
  if (a->B < 1 || a->B > 65535) return fail(STA_ERR_INVALID_ARG, "B=%d outside [1, 65535]", a->B);
  if ((!a->starts || !a->k_starts) && a->B != 1)
    return fail(STA_ERR_INVALID_ARG, "B=%d sequences need starts and k_starts", a->B);
  if (a->window < 0 || a->sinks < 0)
    return fail(STA_ERR_INVALID_ARG, "window=%d and sinks=%d must not be negative", a->window, a->sinks);
  if (!isfinite(a->sm_scale)) return fail(STA_ERR_INVALID_ARG, "sm_scale must be finite");
  const WindowCut cut = cut_of(a);
  // a dimension of a grid holds below 2^32 threads
  const int64_t most = (1 << 24) - 8;
  if ((int64_t)cut.q_tiles * a->H > most || (int64_t)cut.items * a->Hkv > most || (int64_t)cut.k_tiles * 16 > most)
    return fail(STA_ERR_UNSUPPORTED, "T=%d, S=%d, H=%d and B=%d need more workgroups than a grid holds", a->T, a->S, a->H,
                a->B);
  return STA_OK;
}

int check_call(const sta_window_args* a) {
  int rc = check_shape(a);
  if (rc != STA_OK) return rc;
  if (a->T) {
    if ((rc = check_rows("q", a->q, a->dtype, a->T, a->q_tok_stride, a->q_head_stride)) != STA_OK) return rc;
    if ((rc = check_out("out", a->out)) != STA_OK) return rc;
    if (a->rest && !aligned16(a->rest)) return fail(STA_ERR_UNSUPPORTED, "rest is not 16-byte aligned");
    if (!a->lse) return fail(STA_ERR_INVALID_ARG, "lse must be non-NULL");
  }
  if (a->S) {
    if ((rc = check_rows("k", a->k, a->dtype, a->S, a->k_tok_stride, a->k_head_stride)) != STA_OK) return rc;
    if ((rc = check_rows("v", a->v, a->dtype, a->S, a->v_tok_stride, a->v_head_stride)) != STA_OK) return rc;
  }
  return STA_OK;
}

WindowArgs args_of(const sta_window_args* a) {
  const int64_t es = esize(a->dtype);
  WindowArgs d{};
  d.q = (const char*)a->q;
  d.k = (const char*)a->k;
  d.v = (const char*)a->v;
  d.q_ts = a->q_tok_stride * es;
  d.q_hs = a->q_head_stride * es;
  d.k_ts = a->k_tok_stride * es;
  d.k_hs = a->k_head_stride * es;
  d.v_ts = a->v_tok_stride * es;
  d.v_hs = a->v_head_stride * es;
  d.starts = a->starts;
  d.k_starts = a->k_starts;
  d.T = a->T;
  d.S = a->S;
  d.H = a->H;
  d.Hkv = a->Hkv;
  d.B = a->B;
  d.window = window_of(a);
  d.sinks = sinks_of(a);
  d.scale = a->sm_scale;
  const float c = fabsf(a->sm_scale) * 1.44269504088896340736f;
  // scores of a scale that is none are 0, as 0 times the keys; a product that passes the type's largest stays below it
  const bool none = !(c >= FLT_MIN);
  d.c = none ? 1.f : isfinite(c) ? c : FLT_MAX;
  d.keep = none ? 0u : ~0u;
  d.flip = a->sm_scale < 0.f ? (a->dtype == STA_DTYPE_F32 ? 0x80000000u : 0x80008000u) : 0u;
  d.out = (char*)a->out;
  d.rest = (char*)a->rest;
  d.lse = a->lse;
  const WindowCut cut = cut_of(a);
  d.q_tiles = cut.q_tiles;
  d.k_tiles = cut.k_tiles;
  d.items = cut.items;
  d.q_waves = cut.q_waves;
  d.k_waves = cut.k_waves;
  d.steps = cut.steps;
  d.far_steps = cut.far_steps;
  d.near_steps = cut.near_steps;
  d.delta_blocks = cut.delta_blocks;
  return d;
}

struct GradLayout {
  size_t lse_off, delta_off, row_norm_off, key_norm_off, record_off, total;
};
GradLayout layout_of(const sta_window_args* a) {
  const WindowCut cut = cut_of(a);
  const size_t rows = (size_t)a->T * a->H;
  GradLayout l{};
  size_t off = 0;
  l.lse_off = off;
  off = align256(off + rows * 4);
  l.delta_off = off;
  off = align256(off + rows * 4);
  l.row_norm_off = off;
  off = align256(off + (a->dtype == STA_DTYPE_F16 ? rows * 4 : 0));
  l.key_norm_off = off;
  off = align256(off + (a->dtype == STA_DTYPE_F16 ? (size_t)a->S * a->Hkv * 4 : 0));
  l.record_off = off;
  off = align256(off + (size_t)a->Hkv * cut.records * 2 * (32 * cut.k_waves) * a->D * 4);
  l.total = off ? off : 1;
  return l;
}

}  // namespace

extern "C" {

int sta_window_attention(const sta_window_args* a, void* stream) {
  const int rc = check_call(a);
  if (rc != STA_OK || a->T == 0) return rc;
  hipError_t e = launch_window(a->dtype, a->D, args_of(a), (hipStream_t)stream);
  return e == hipSuccess ? STA_OK : hip_fail(e, "window attention");
}

size_t sta_window_grad_workspace_size(const sta_window_grad_args* a) {
  if (!a || check_shape(&a->fwd) != STA_OK) return 0;
  return layout_of(&a->fwd).total;
}

int sta_window_attention_grad(const sta_window_grad_args* a, void* stream) {
  if (!a) return fail(STA_ERR_INVALID_ARG, "args is NULL");
  int rc = check_call(&a->fwd);
  if (rc != STA_OK) return rc;
  const sta_window_args& f = a->fwd;
  if (f.T) {
    if ((rc = check_rows("dout", a->dout, f.dtype, f.T, a->dout_tok_stride, a->dout_head_stride)) != STA_OK) return rc;
    if ((rc = check_out("dq", a->dq)) != STA_OK) return rc;
  }
  if (f.S && ((rc = check_out("dk", a->dk)) != STA_OK || (rc = check_out("dv", a->dv)) != STA_OK)) return rc;
  const GradLayout l = layout_of(&f);
  if (!a->workspace || a->workspace_bytes < l.total)
    return fail(STA_ERR_WORKSPACE, "workspace of %zu bytes at %p is smaller than the %zu needed", a->workspace_bytes,
                a->workspace, l.total);
  if (((uintptr_t)a->workspace & 255u) != 0) return fail(STA_ERR_WORKSPACE, "workspace must be 256-byte aligned");
  char* ws = (char*)a->workspace;
  WindowArgs d = args_of(&f);
  d.dout = (const char*)a->dout;
  d.do_ts = a->dout_tok_stride * esize(f.dtype);
  d.do_hs = a->dout_head_stride * esize(f.dtype);
  d.lse_in = f.lse;
  d.dq = (char*)a->dq;
  d.dk = (char*)a->dk;
  d.dv = (char*)a->dv;
  d.row_lse = (float*)(ws + l.lse_off);
  d.row_delta = (float*)(ws + l.delta_off);
  d.row_norm = (float*)(ws + l.row_norm_off);
  d.key_norm = (float*)(ws + l.key_norm_off);
  d.record = (float*)(ws + l.record_off);
  hipError_t e = launch_window_grad(f.dtype, f.D, d, cut_of(&f).records, (hipStream_t)stream);
  return e == hipSuccess ? STA_OK : hip_fail(e, "window attention gradient");
}

}  // extern "C"
