// The paged cache's kernels (paged.cu): arguments and launchers; internal.
#pragma once
#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

#include "../../include/webgllm_paged.h"

namespace wg {

// Rows and sequences of a call, on the device (webgllm_paged.h).
struct PagedRows {
  const int32_t *row_start;  // or null: rows / batch each
  const int32_t *pos;
  int rows, batch;
};

struct PagedTable {
  const int32_t *table;
  int max_pages, num_pages, page_size;
};

cudaError_t launch_paged_rope_kv(const float *qkv, const PagedRows &rows, int H, int Hkv, int Dh, double theta,
                                 const float *q_norm, const float *k_norm, float eps, void *q_out,
                                 const wg_paged_kv &kv, unsigned *flags, int num_sms, cudaStream_t s, bool pdl);

// Bytes of workspace that launch_paged_attention may use.
size_t paged_attention_workspace(int Dh, int num_sms);
cudaError_t launch_paged_attention(const void *q, const PagedRows &rows, int H, int Hkv, int Dh,
                                   const wg_paged_kv &kv, int window, int sinks, void *out, void *workspace,
                                   unsigned *flags, int num_sms, cudaStream_t s, bool pdl);

// Many rows a sequence (paged_prompt_sm100.cu): launch_paged_attention sends the
// shapes there for which this says so.
bool paged_prompt_wins(const PagedRows &rows, int H, int Hkv, int Dh, int num_sms);
cudaError_t launch_paged_prompt(const void *q, const PagedRows &rows, int H, int Hkv, int Dh, const wg_paged_kv &kv,
                                int window, int sinks, void *out, unsigned *flags, int num_sms, cudaStream_t s,
                                bool pdl);

}  // namespace wg
