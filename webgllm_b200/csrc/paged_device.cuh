// Device helpers shared by the paged-cache kernels: 16-bit types, the rows of
// a sequence, page boxes by TMA.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "device_utils.cuh"
#include "paged.cuh"
#include "tma.cuh"

namespace wg {

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}

template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t u);
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t u) {
  return __half22float2(*reinterpret_cast<const __half2 *>(&u));
}
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t u) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&u));
}

// Exponent bits of an infinity or NaN.
template <typename T>
constexpr uint32_t kNonfinite = std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;

// Whether a packed pair holds an infinity or NaN.
template <typename T>
__device__ __forceinline__ bool nonfinite2(uint32_t u) {
  constexpr uint32_t e = kNonfinite<T>;
  return (u & e) == e || (u >> 16 & e) == e;
}

// Rows of sequence b: [r0, r0 + n), clamped to the buffers.
__device__ __forceinline__ void seq_rows(const PagedRows &a, int b, int &r0, int &n) {
  if (a.row_start) {
    r0 = min(max(a.row_start[b], 0), a.rows);
    n = max(min(a.row_start[b + 1], a.rows) - r0, 0);
  } else {
    n = a.rows / a.batch;
    r0 = b * n;
  }
}

// The keys that rows at positions p .. p + n - 1 see, in tiles of `tile` keys:
// [0, se) and [ws, hi) in tiles [0, a) and [c, c + nt - a).
struct KeySpan {
  int hi, ws, se;
  int a, c, nt;
};

__device__ __forceinline__ KeySpan key_span(long long p, int n, int window, int sinks, const PagedTable &pt, int tile) {
  KeySpan k;
  const long long cap = (long long)pt.max_pages * pt.page_size;
  k.hi = (int)max(0LL, min(p + n, cap));
  k.ws = window > 0 ? (int)min((long long)k.hi, max(0LL, p - window + 1)) : 0;
  k.se = min(sinks, k.ws);
  k.a = (k.se + tile - 1) / tile;
  k.c = max(k.ws / tile, k.a);
  k.nt = k.a + max(0, (k.hi + tile - 1) / tile - k.c);
  if (k.nt == 0) k.nt = 1;  // rows that see nothing still get their zeros
  return k;
}

__device__ __forceinline__ bool sees_key(int p, int key, int window, int sinks) {
  return key <= p && (window == 0 || key > p - window || key < sinks);
}

__device__ __forceinline__ void tma_load_4d(void *dst, const CUtensorMap *map, int c0, int c1, int c2, int c3,
                                            uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], "
      "[%2];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}

// The pages as a tensor of (dim, row in page, head, page), read in boxes of 64
// dims x box_rows rows of one head of one page (128-byte swizzle).
inline bool page_map(CUtensorMap *m, void *base, const wg_paged_kv &kv, int Hkv, int Dh, int box_rows) {
  EncodeTiled enc = encode_fn();
  if (!enc) return false;
  auto bytes = [](int64_t s, int64_t dense) { return (cuuint64_t)(s ? s : dense) * 2; };
  const cuuint64_t dims[4] = {(cuuint64_t)Dh, (cuuint64_t)kv.page_size, (cuuint64_t)Hkv, (cuuint64_t)kv.num_pages};
  const cuuint64_t strides[3] = {bytes(kv.row_stride, Dh), bytes(kv.head_stride, (int64_t)kv.page_size * Dh),
                                 bytes(kv.page_stride, (int64_t)Hkv * kv.page_size * Dh)};
  const cuuint32_t box[4] = {64, (cuuint32_t)box_rows, 1, 1};
  const cuuint32_t one[4] = {1, 1, 1, 1};
  return enc(m, kv.dtype == WG_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, base, dims,
             strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename... KArgs, typename... Args>
cudaError_t launch_pdl(void (*kern)(KArgs...), dim3 grid, int threads, size_t smem, cudaStream_t s, bool pdl,
                       const Args &...args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  if (pdl) {
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
  }
  return cudaLaunchKernelEx(&cfg, kern, static_cast<KArgs>(args)...);
}

}  // namespace wg
