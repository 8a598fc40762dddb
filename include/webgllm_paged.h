/*
 * webgllm_paged.h: a key-value cache in pages, and attention over it
 * (libwebgllm_b200.so). The reference keeps one cache texture per sequence
 * as long as its context (headPrep / attend, src/gpu/kernels.ts:2196-2579);
 * these calls stand beside wg_rope_kv and wg_attention (webgllm_decoder.h)
 * for hosts that serve sequences of different length from one pool of
 * pages. Conventions as webgllm_q4.h.
 *
 * The cache. A page holds page_size consecutive positions of one sequence
 * for every KV head. table int32 [batch][max_pages] (device memory) names
 * the page of positions i page_size .. (i + 1) page_size - 1 of sequence b
 * at table[b][i]; an entry outside [0, num_pages) names no page. Pages may
 * be shared by sequences (a common prefix) as long as nothing is appended to
 * them, and may be taken out of the table (-1) once no row sees them.
 *
 * Rows. `rows` rows belong to `batch` sequences, in order: rows / batch each
 * (row_start NULL), or sequence b's rows are row_start[b] ..
 * row_start[b + 1] - 1 (int32 [batch + 1] on the device, ascending; rows
 * outside [row_start[0], row_start[batch]) belong to nobody: what they hold
 * changes nothing and their outputs stay as they were). pos int32 [batch] (device) is
 * the position of each sequence's first row. A row at a negative position is
 * padding: it appends nothing, sees nothing and its outputs are zeros.
 */
#ifndef WEBGLLM_PAGED_H
#define WEBGLLM_PAGED_H

#include <stddef.h>
#include <stdint.h>

#include "webgllm_q4.h"

#ifdef __cplusplus
extern "C" {
#endif

/* One layer's pages. Element (page, KV head, row, d) of k and of v is at
 * page * page_stride + head * head_stride + row * row_stride + d, in elements
 * (three zeros: [num_pages][Hkv][page_size][Dh] without gaps). Strides are
 * multiples of 8 elements, k and v 16-byte aligned. */
typedef struct wg_paged_kv {
  void *k, *v;
  const int32_t *table;  /* [batch][max_pages] */
  int dtype;             /* WG_F16 or WG_BF16 */
  int num_pages;
  int page_size;         /* a multiple of 16 */
  int max_pages;
  int64_t page_stride, head_stride, row_stride;
} wg_paged_kv;

/* wg_rope_kv into pages: qkv fp32 [rows][(H + 2 Hkv) Dh] (q | k | v); per head
 * an optional RMS norm over Dh (q_norm / k_norm fp32 [Dh], NULL: none), then
 * rotate-half RoPE of the pairs (j, j + Dh/2) by p theta^(-2j/Dh) (the angle
 * reduced in 64 bits: exact to fp32 at any position). q_out [rows][H][Dh]
 * in the cache's dtype, scaled by 1/sqrt(Dh), not overlapping qkv; k (rotated) and v
 * go to the row's page.
 * Dh in {64, 128, 256}. A row past the table, or whose page entry names no
 * page, is not appended and reported by wg_sync. */
int wg_paged_rope_kv(wg_ctx *ctx, const float *qkv, int rows, int batch, const int32_t *row_start, int H, int Hkv,
                     int Dh, const int32_t *pos, double theta, const float *q_norm, const float *k_norm, float eps,
                     void *q_out, const wg_paged_kv *kv);

/* Attention of every row over its sequence's pages: a row at position p of
 * query head h sees the keys j <= p of KV head h / (H / Hkv); with
 * window > 0 only those with j > p - window or j < sinks (a sliding window
 * and the first `sinks` positions, which stay visible). out = softmax(q . k)
 * v, a row that sees nothing gets zeros. q (scaled) and out [rows][H][Dh] in
 * the cache's dtype, not overlapping. Dh in {64, 128, 256}, H a multiple of
 * Hkv, any rows per sequence (one for a decode step, k + 1 to verify drafts, a
 * prompt's chunk). One kernel serves a call, chosen by its sequences' rows on
 * average: prompt chunks and single rows over long contexts are faster in two
 * calls. Scores (q . k) are below 2^24 in size. What a row does not see may
 * hold anything, NaN included. A visible position whose page entry names no
 * page is left out and reported by wg_sync; positions past the table are left
 * out.
 * `workspace` (16-byte aligned device memory of at least
 * wg_paged_attention_workspace bytes, any content) holds the partial sums of
 * sequences that several CTAs share: calls that may overlap on the GPU need
 * one each, which overlaps neither q nor out. */
int wg_paged_attention(wg_ctx *ctx, const void *q, int rows, int batch, const int32_t *row_start, int H, int Hkv,
                       int Dh, const int32_t *pos, const wg_paged_kv *kv, int window, int sinks, void *out,
                       void *workspace, size_t workspace_bytes);

/* The workspace of any wg_paged_attention of this head size on this context. */
int wg_paged_attention_workspace(wg_ctx *ctx, int Dh, size_t *bytes);

#ifdef __cplusplus
}
#endif

#endif /* WEBGLLM_PAGED_H */
