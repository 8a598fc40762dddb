// The C ABI of include/webgllm_paged.h: argument checks and launches.
#include <cuda_runtime.h>

#include <climits>
#include <cstdarg>
#include <cstdio>

#include "../../include/webgllm_paged.h"
#include "capi_internal.cuh"
#include "paged.cuh"

namespace {

int pfail(wg_ctx *ctx, int status, const char *fmt, ...) {
  if (ctx) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    try {
      ctx->last_error = buf;
    } catch (...) {  // no memory for the text: the status still says what happened
    }
  }
  return status;
}

int finish(wg_ctx *ctx, cudaError_t e, const char *what) {
  if (e == cudaSuccess) return WG_OK;
  return pfail(ctx, wg::status_of(e), "%s: %s", what, cudaGetErrorString(e));
}

bool aligned(const void *p, size_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

// The checks that both calls share.
int check(wg_ctx *ctx, const char *what, int rows, int batch, const int32_t *row_start, int H, int Hkv, int Dh,
          const wg_paged_kv *kv) {
  if (rows < 0 || batch <= 0) return pfail(ctx, WG_INVALID_SHAPE, "%s: %d rows of %d sequences", what, rows, batch);
  if (!row_start && rows % batch)
    return pfail(ctx, WG_INVALID_SHAPE, "%s: rows (%d) must be a multiple of batch (%d) without row_start", what, rows,
                 batch);
  if (H <= 0 || Hkv <= 0 || H % Hkv || !(Dh == 64 || Dh == 128 || Dh == 256))
    return pfail(ctx, WG_INVALID_SHAPE, "%s: bad heads (H %d, Hkv %d, Dh %d)", what, H, Hkv, Dh);
  if (!kv) return pfail(ctx, WG_INVALID_ARGUMENT, "%s: null cache", what);
  if (kv->dtype != WG_F16 && kv->dtype != WG_BF16)
    return pfail(ctx, WG_INVALID_ARGUMENT, "%s: the cache's dtype must be WG_F16 or WG_BF16", what);
  if (kv->num_pages <= 0 || kv->max_pages <= 0 || kv->page_size <= 0 || kv->page_size % 16 ||
      kv->page_size > (1 << 20) || (long long)kv->max_pages * kv->page_size > INT_MAX)
    return pfail(ctx, WG_INVALID_SHAPE, "%s: bad cache (%d pages of %d positions, %d a sequence)", what, kv->num_pages,
                 kv->page_size, kv->max_pages);
  if (!kv->k || !kv->v || !kv->table || !aligned(kv->k, 16) || !aligned(kv->v, 16) || !aligned(kv->table, 4))
    return pfail(ctx, WG_INVALID_ARGUMENT, "%s: null or misaligned cache", what);
  for (int64_t s : {kv->page_stride, kv->head_stride, kv->row_stride})
    if (s < 0 || s % 8 || s >= (1LL << 38))
      return pfail(ctx, WG_INVALID_SHAPE, "%s: strides must be multiples of 8 elements below 2^38", what);
  if (kv->row_stride && kv->row_stride < Dh)
    return pfail(ctx, WG_INVALID_SHAPE, "%s: row_stride %lld below Dh", what, (long long)kv->row_stride);
  return WG_OK;
}

}  // namespace

#define WG_PAGED_BEGIN(ctx)                                            \
  do {                                                                 \
    if (!ctx) return WG_INVALID_ARGUMENT;                              \
    if (cudaError_t e_ = cudaSetDevice(ctx->device); e_ != cudaSuccess) \
      return finish(ctx, e_, "cudaSetDevice");                         \
  } while (0)

extern "C" {

int wg_paged_rope_kv(wg_ctx *ctx, const float *qkv, int rows, int batch, const int32_t *row_start, int H, int Hkv,
                     int Dh, const int32_t *pos, double theta, const float *q_norm, const float *k_norm, float eps,
                     void *q_out, const wg_paged_kv *kv) {
  WG_PAGED_BEGIN(ctx);
  if (int st = check(ctx, "wg_paged_rope_kv", rows, batch, row_start, H, Hkv, Dh, kv)) return st;
  if (!(theta > 0.0)) return pfail(ctx, WG_INVALID_ARGUMENT, "wg_paged_rope_kv: theta must be positive");
  if (!rows) return WG_OK;
  if ((long long)rows * (H + 2LL * Hkv) > INT_MAX)
    return pfail(ctx, WG_UNSUPPORTED, "wg_paged_rope_kv: %d rows of %d heads", rows, H + 2 * Hkv);
  if (!qkv || !pos || !q_out) return pfail(ctx, WG_INVALID_ARGUMENT, "wg_paged_rope_kv: null");
  if (!aligned(qkv, 16) || !aligned(q_out, 16) || !aligned(pos, 4) || !aligned(row_start, 4) || !aligned(q_norm, 4) ||
      !aligned(k_norm, 4))
    return pfail(ctx, WG_INVALID_ARGUMENT, "wg_paged_rope_kv: misaligned tensor");
  const size_t elems = (size_t)rows * H * Dh;
  if (wg::overlap(qkv, (size_t)rows * (H + 2 * (size_t)Hkv) * Dh * 4, q_out, elems * 2))
    return pfail(ctx, WG_INVALID_ARGUMENT, "wg_paged_rope_kv: qkv and q_out overlap");
  return finish(ctx,
                wg::launch_paged_rope_kv(qkv, wg::PagedRows{row_start, pos, rows, batch}, H, Hkv, Dh, theta, q_norm,
                                         k_norm, eps, q_out, *kv, ctx->d_flags, ctx->num_sms, ctx->stream, ctx->pdl),
                "wg_paged_rope_kv");
}

int wg_paged_attention(wg_ctx *ctx, const void *q, int rows, int batch, const int32_t *row_start, int H, int Hkv,
                       int Dh, const int32_t *pos, const wg_paged_kv *kv, int window, int sinks, void *out,
                       void *workspace, size_t workspace_bytes) {
  WG_PAGED_BEGIN(ctx);
  if (int st = check(ctx, "wg_paged_attention", rows, batch, row_start, H, Hkv, Dh, kv)) return st;
  if (window < 0 || sinks < 0)
    return pfail(ctx, WG_INVALID_ARGUMENT, "wg_paged_attention: window %d, sinks %d", window, sinks);
  if (!rows) return WG_OK;
  // the device counts key tiles of all sequences and heads in 31 bits
  const long long row_tiles = ((long long)rows * (H / Hkv) + 15) / 16 + batch;
  const long long key_tiles = ((long long)kv->max_pages * kv->page_size + 63) / 64 + 1;
  if (row_tiles >= INT_MAX / Hkv || row_tiles * Hkv >= INT_MAX / key_tiles)
    return pfail(ctx, WG_UNSUPPORTED, "wg_paged_attention: %d rows over %lld positions are too many for one call", rows,
                 key_tiles * 64);
  if (!q || !pos || !out || !workspace) return pfail(ctx, WG_INVALID_ARGUMENT, "wg_paged_attention: null");
  if (!aligned(q, 16) || !aligned(out, 16) || !aligned(workspace, 16) || !aligned(pos, 4) || !aligned(row_start, 4))
    return pfail(ctx, WG_INVALID_ARGUMENT, "wg_paged_attention: misaligned tensor");
  const size_t bytes = (size_t)rows * H * Dh * 2;
  if (wg::overlap(q, bytes, out, bytes))
    return pfail(ctx, WG_INVALID_ARGUMENT, "wg_paged_attention: q and out overlap");
  const size_t need = wg::paged_attention_workspace(Dh, ctx->num_sms);
  if (workspace_bytes < need)
    return pfail(ctx, WG_INVALID_ARGUMENT, "wg_paged_attention: a workspace of %zu bytes, %zu needed", workspace_bytes,
                 need);
  if (wg::overlap(workspace, need, q, bytes) || wg::overlap(workspace, need, out, bytes))
    return pfail(ctx, WG_INVALID_ARGUMENT, "wg_paged_attention: the workspace overlaps q or out");
  return finish(ctx,
                wg::launch_paged_attention(q, wg::PagedRows{row_start, pos, rows, batch}, H, Hkv, Dh, *kv, window,
                                           sinks, out, workspace, ctx->d_flags, ctx->num_sms, ctx->stream, ctx->pdl),
                "wg_paged_attention");
}

int wg_paged_attention_workspace(wg_ctx *ctx, int Dh, size_t *bytes) {
  if (!ctx || !bytes) return WG_INVALID_ARGUMENT;
  *bytes = 0;
  if (!(Dh == 64 || Dh == 128 || Dh == 256))
    return pfail(ctx, WG_INVALID_SHAPE, "wg_paged_attention_workspace: Dh %d", Dh);
  *bytes = wg::paged_attention_workspace(Dh, ctx->num_sms);
  return WG_OK;
}

}  // extern "C"
