// Sampled speculative decoding: the verification of drafted tokens against the
// target's probabilities (wg_spec_sample, webgllm_decoder.h).
//
//   p_j = softmax(target_j / T), q_j = softmax(draft_j / T); draft token d_j is
//   kept iff u_j q_j(d_j) < p_j(d_j); at the first j = n that is not, the token
//   is drawn from max(p_n - q_n, 0) by inverse CDF with u_k; if all are kept,
//   from p_k. Together the kept tokens and the drawn one are distributed as
//   samples of the target.
//
// A thread-block cluster serves a sequence: each CTA takes a slice of the
// vocabulary of every row, and the CTAs exchange sums through distributed
// shared memory, so one launch does everything and nothing is kept in global
// memory.
// The answer is a whole number, so it must not hang on rounding. The
// statistics that decide acceptance are fp32 exponentials (their sum is good
// to kSlack), and a decision closer than that is taken again from sums of
// 64-bit exponentials. The one row that is drawn from is computed in 64 bits
// throughout: p - q cancels where draft and target agree, and its running sum
// is compared with u at a resolution of one token in V.
// Bound: the (2k + 1) V logits of a sequence, read once (HBM), plus the 64-bit
// exponentials of the drawn rows (2 V a sequence).
#include <cooperative_groups.h>

#include "common.cuh"
#include "decoder_kernels.cuh"
#include "device_utils.cuh"

namespace wg {

namespace cg = cooperative_groups;

namespace {

constexpr int kSampleThreads = 512;
constexpr int kSampleWarps = kSampleThreads / 32;
constexpr int kSampleCluster = 16;  // largest cluster
constexpr int kMaxRows = 2 * kSampleMaxDrafts + 1;
// Relative error bound of u q(d) / p(d) when the two normalising sums come from
// fp32 exponentials. A term exp(-a) is off by at most a 2^-22 + 2^-21 of
// itself, and terms that matter have a <= ln V (15 at the largest vocabulary);
// a thread adds at most V / (16 x 512) = 256 of them, each addition off by at
// most 2^-24. Both sums: below 2 (4e-6 + 1.6e-5) = 4e-5.
constexpr double kSlack = 4e-5;

struct SampleArgs {
  const float *target;    // [k + 1][batch][V]
  const float *draft;     // [k][batch][V]
  const int32_t *drafts;  // [batch][k]
  const float *u;         // [batch][k + 1]
  int32_t *picks;         // [k + 1][batch]
  int batch, k, V;
  int slice;              // vocabulary entries per CTA
  double temperature;
  unsigned *flags;
};

struct MaxSum {
  float m, s;
};

__device__ __forceinline__ MaxSum join(MaxSum a, MaxSum b, float c) {
  const float m = fmaxf(a.m, b.m);
  if (m == -INFINITY) return MaxSum{m, 0.0f};
  return MaxSum{m, a.s * exp2f((a.m - m) * c) + b.s * exp2f((b.m - m) * c)};
}

__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The sum of one double per thread over the whole cluster, the same bits in
// every thread of every CTA (summed in rank order).
struct ClusterSum {
  double warp[kSampleWarps];
  double cta;
};

__device__ double cta_sum(double v, ClusterSum &sh) {
  v = warp_sum_f64(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh.warp[threadIdx.x >> 5] = v;
  __syncthreads();
  double t = 0.0;
#pragma unroll
  for (int i = 0; i < kSampleWarps; i++) t += sh.warp[i];
  return t;
}

__device__ double cluster_sum(double v, ClusterSum &sh, double *before = nullptr, double *own = nullptr) {
  cg::cluster_group cl = cg::this_cluster();
  const double mine = cta_sum(v, sh);
  if (threadIdx.x == 0) sh.cta = mine;
  if (own) *own = mine;
  cl.sync();
  double t = 0.0;
  const int me = (int)cl.block_rank(), n = (int)cl.num_blocks();
  for (int i = 0; i < n; i++) {
    if (before && i == me) *before = t;
    t += *cl.map_shared_rank(&sh.cta, i);
  }
  cl.sync();  // sh.cta may be written again
  return t;
}

__global__ void __launch_bounds__(kSampleThreads) spec_sample_kernel(const SampleArgs a) {
  pdl_trigger();
  pdl_wait();
  cg::cluster_group cl = cg::this_cluster();
  const int rank = (int)cl.block_rank(), CL = (int)cl.num_blocks();
  const int b = blockIdx.x / CL;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int k = a.k, R = 2 * k + 1, V = a.V;
  const int v0 = min((long long)V, (long long)rank * a.slice), v1 = min((long long)V, (long long)v0 + a.slice);
  __shared__ MaxSum warp_ms[kMaxRows][kSampleWarps];
  __shared__ MaxSum cta_ms[kMaxRows];
  __shared__ float row_m[kMaxRows];
  __shared__ double row_z[kMaxRows];
  __shared__ ClusterSum csum;
  __shared__ double groups[kSampleWarps];
  __shared__ int found;

  // rows 0 .. k: the target's; k + 1 .. 2k: the draft's
  auto row = [&](int r) {
    return r <= k ? a.target + ((size_t)r * a.batch + b) * V : a.draft + ((size_t)(r - k - 1) * a.batch + b) * V;
  };
  const float c = (float)(1.4426950408889634 / a.temperature);

  // ---- maximum and sum of every row
  for (int r = 0; r < R; r++) {
    const float *x = row(r);
    MaxSum ms{-INFINITY, 0.0f};
    auto one = [&](float v) {
      if (v > ms.m) {
        ms.s *= exp2f((ms.m - v) * c);
        ms.m = v;
      }
      if (ms.m > -INFINITY) ms.s += exp2f((v - ms.m) * c);
    };
    // the 16-byte aligned middle of the slice four at a time
    const int lead = min((int)((4 - (((uintptr_t)(x + v0) >> 2) & 3)) & 3), v1 - v0);
    const int quads = (v1 - v0 - lead) / 4;
    if (tid < lead) one(x[v0 + tid]);
    const float4 *x4 = reinterpret_cast<const float4 *>(x + v0 + lead);
#pragma unroll 4
    for (int i = tid; i < quads; i += kSampleThreads) {
      const float4 v = x4[i];
      const float m = fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w));
      if (m > ms.m) {
        ms.s *= exp2f((ms.m - m) * c);
        ms.m = m;
      }
      if (ms.m > -INFINITY)
        ms.s += (exp2f((v.x - ms.m) * c) + exp2f((v.y - ms.m) * c)) +
                (exp2f((v.z - ms.m) * c) + exp2f((v.w - ms.m) * c));
    }
    const int tail = v0 + lead + 4 * quads + tid;
    if (tail < v1) one(x[tail]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
      ms = join(ms, MaxSum{__shfl_xor_sync(0xffffffffu, ms.m, o), __shfl_xor_sync(0xffffffffu, ms.s, o)}, c);
    if (lane == 0) warp_ms[r][warp] = ms;
  }
  __syncthreads();
  for (int r = tid; r < R; r += kSampleThreads) {
    MaxSum ms = warp_ms[r][0];
    for (int i = 1; i < kSampleWarps; i++) ms = join(ms, warp_ms[r][i], c);
    cta_ms[r] = ms;
  }
  cl.sync();
  for (int r = tid; r < R; r += kSampleThreads) {
    float m = -INFINITY;
    for (int i = 0; i < CL; i++) m = fmaxf(m, cl.map_shared_rank(&cta_ms[r], i)->m);
    double z = 0.0;
    for (int i = 0; i < CL; i++) {
      const MaxSum ms = *cl.map_shared_rank(&cta_ms[r], i);
      if (ms.m > -INFINITY) z += (double)ms.s * (double)exp2f((ms.m - m) * c);
    }
    row_m[r] = m;
    row_z[r] = z;
  }
  __syncthreads();
  // (a peer's cta_ms is not written again: no barrier is owed for it until exit)

  // exp((x - max) / T) in 64 bits
  auto weight = [&](float x, float m) { return exp(((double)x - (double)m) / a.temperature); };
  auto exact_sum = [&](int r) {
    const float *x = row(r);
    const float m = row_m[r];
    double s = 0.0;
    for (int i = v0 + tid; i < v1; i += kSampleThreads) s += weight(x[i], m);
    return cluster_sum(s, csum);
  };

  // ---- acceptance: the same in every thread of the cluster
  int n = 0;
  for (; n < k; n++) {
    const int d = a.drafts[(size_t)b * k + n];
    double u = (double)a.u[(size_t)b * (k + 1) + n];
    if (u >= 1.0) u = 1.0 - 0x1p-24;
    double pe = 0.0, qe = 0.0;
    if (d >= 0 && d < V) {
      pe = weight(row(n)[d], row_m[n]);
      qe = weight(row(k + 1 + n)[d], row_m[k + 1 + n]);
    }
    double lhs = u * (qe / row_z[k + 1 + n]), rhs = pe / row_z[n];
    if (fabs(lhs - rhs) <= kSlack * rhs && rhs > 0.0) {
      const double zq = exact_sum(k + 1 + n), zp = exact_sum(n);
      lhs = u * (qe / zq);
      rhs = pe / zp;
    }
    if (!(lhs < rhs)) break;
  }

  // rows without probabilities (NaN, +inf, -inf throughout): a token all the
  // same, never the rejected one, and a report
  const int dn = n < k ? a.drafts[(size_t)b * k + n] : -1;
  auto is_row = [&](int r) { return row_z[r] > 0.0 && row_z[r] < INFINITY; };
  auto report = [&]() {
    if (rank == 0 && tid == 0) {
      a.picks[(size_t)n * a.batch + b] = dn == 0 && V > 1 ? 1 : 0;
      raise_flag(a.flags, kFlagBadArgument);
    }
  };
  if (rank == 0 && tid == 0) {
    for (int j = 0; j < n; j++) a.picks[(size_t)j * a.batch + b] = a.drafts[(size_t)b * k + j];
    for (int j = n + 1; j <= k; j++) a.picks[(size_t)j * a.batch + b] = -1;
  }
  if (!is_row(n) || (n < k && !is_row(k + 1 + n))) {
    report();
    cl.sync();  // peers may still read this CTA's shared memory
    return;
  }

  // ---- the draw: from max(p - q, 0) of row n, or from p of row k
  const float *xp = row(n), *xq = n < k ? row(k + 1 + n) : nullptr;
  const float mp = row_m[n], mq = n < k ? row_m[k + 1 + n] : 0.0f;
  double ip = 1.0, iq = 0.0;
  if (n < k) {
    ip = 1.0 / exact_sum(n);
    iq = 1.0 / exact_sum(k + 1 + n);
  }
  int mode = n < k ? 0 : 1;  // 0: p - q; 1: p; 2: p without the rejected token
  auto mass = [&](int i) {
    const double p = weight(xp[i], mp);
    if (mode == 0) return fmax(p * ip - weight(xq[i], mq) * iq, 0.0);
    return mode == 2 && i == dn ? 0.0 : fmax(p, 0.0);
  };
  double total, before, mine;
  for (;;) {
    double s = 0.0;
    for (int i = v0 + tid; i < v1; i += kSampleThreads) s += mass(i);
    total = cluster_sum(s, csum, &before, &mine);
    // p and q may agree to the last bit everywhere: then the rejected token's
    // place goes to another token of p
    if (mode != 0 || total > 0.0) break;
    mode = 2;
  }
  double u = (double)a.u[(size_t)b * (k + 1) + k];
  if (!(u < 1.0)) u = 1.0 - 0x1p-24;
  if (!(u > 0.0)) u = 0.0;
  const double goal = u * total;  // the token is the first whose running sum exceeds it
  if (!(total > 0.0)) {  // all of p on a token that was rejected: q cannot have been a distribution
    report();
    return;
  }
  // the CTA whose slice holds the goal finds the token: runs of 512 entries,
  // a running sum over warps and lanes
  const bool owner = before <= goal && goal < before + mine;  // before + mine is the next CTA's before, to the bit
  if (owner) {
    double run = before;
    int last = -1;  // the last entry with mass: where rounding left the goal behind the slice's sum
    if (tid == 0) found = 0x7fffffff;
    __syncthreads();
    for (int i0 = v0; i0 < v1; i0 += kSampleThreads) {
      const int i = i0 + tid;
      const double m = i < v1 ? mass(i) : 0.0;
      if (m > 0.0) last = i;
      double s = m;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double t = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += t;
      }
      if (lane == 31) groups[warp] = s;
      __syncthreads();
      double head = run, all = 0.0;
      for (int w = 0; w < kSampleWarps; w++) {
        if (w < warp) head += groups[w];
        all += groups[w];
      }
      if (m > 0.0 && head + s > goal) atomicMin(&found, i);
      __syncthreads();
      if (found != 0x7fffffff) break;
      run += all;
    }
    if (found == 0x7fffffff) {
      __syncthreads();
      if (tid == 0) found = -1;
      __syncthreads();
      if (last >= 0) atomicMax(&found, last);
      __syncthreads();
    }
    if (tid == 0) a.picks[(size_t)n * a.batch + b] = found;
  }
}

}  // namespace

cudaError_t launch_spec_sample(const float *target, const float *draft, const int32_t *drafts, int batch, int k, int V,
                               double temperature, const float *u, int32_t *picks, unsigned *flags, cudaStream_t s,
                               bool pdl) {
  // CTAs per sequence: slices of at least 2048 entries, up to the largest cluster
  int CL = 1;
  while (CL < kSampleCluster && (long long)CL * 2048 < V) CL *= 2;
  SampleArgs a{target, draft, drafts, u, picks, batch, k, V, 0, temperature, flags};
  a.slice = ((V + CL - 1) / CL + 3) / 4 * 4;
  cudaError_t e =
      cudaFuncSetAttribute(spec_sample_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(batch * CL));
  cfg.blockDim = dim3(kSampleThreads);
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)CL;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = pdl ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, spec_sample_kernel, a);
}

}  // namespace wg
