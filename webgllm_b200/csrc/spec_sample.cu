// Sampled speculative decoding: the verification of drafted tokens against the
// target's probabilities (wg_spec_sample, webgllm_decoder.h).
//
//   p_j = softmax(target_j / T), q_j = softmax(draft_j / T); draft token d_j is
//   kept iff u_j q_j(d_j) < p_j(d_j); at the first j = n that is not, the token
//   is drawn from max(p_n - q_n, 0) by inverse CDF with u_k; if all are kept,
//   from p_k. Together the kept tokens and the drawn one are distributed as
//   samples of the target.
//
// Two launches (one for k = 0 where the clusters have room). sample_stats_kernel streams every row once over the whole machine
// (pieces of 8192 logits a CTA, all of its loads in flight at once) and leaves
// (max, sum) of each piece in the workspace. spec_sample_kernel, a thread-block
// cluster a sequence, (1) combines them, (2) decides acceptance, a lane a draft,
// (3) makes the drawn row's weights in 64 bits, a slice of the vocabulary a CTA,
// the CTAs' sums exchanged through distributed shared memory, and (4) finds the
// token by the running sum over CTAs, warps, rounds of 256 and runs of 32. (In
// one launch, the clusters doing the streaming too, 61 sequences of 11 rows of
// 65543 took 144 us: their phases run in step, and the memory idles through the
// later ones.) Those 61 sequences take 66 us: 28 us of streaming (6.2 TB/s) and
// the 64-bit passes; 8 of k = 4 over 128256 tokens 22 us.
// The answer is a whole number, so it must not hang on rounding. The
// statistics that decide acceptance are fp32 exponentials (their sum is good
// to kSlack), and a decision closer than that is taken again from sums of
// 64-bit exponentials. The one row that is drawn from is computed in 64 bits
// throughout: p - q cancels where draft and target agree, and its running sum
// is compared with u at a resolution of one token in V.
// Bound: the (2k + 1) V logits of a sequence, read once (HBM), plus the 64-bit
// exponentials of the drawn rows (V to 4 V a sequence, 10 operations each).
#include <cooperative_groups.h>

#include "common.cuh"
#include "decoder_kernels.cuh"
#include "device_utils.cuh"

namespace wg {

namespace cg = cooperative_groups;

namespace {

constexpr int kSampleCluster = 16;  // largest cluster
constexpr int kSlots = 64;
constexpr size_t kKeepBytes = 200 * 1024;  // of shared memory for the drawn rows' weights
constexpr int kMaxRows = 2 * kSampleMaxDrafts + 1;
// Relative error bound of u q(d) / p(d) when the two normalising sums come from
// fp32 exponentials. A term exp(-a) is off by at most a 2^-22 + 2^-21 of
// itself, and terms that matter have a <= ln V (15 at the largest vocabulary):
// 4e-6; a thread adds 36 of them and the CTA's threads 13 levels deep, each
// addition off by at most 2^-24: 3e-6. Both sums: below 2e-5.
constexpr double kSlack = 2e-5;

struct SampleArgs {
  const float *target;    // [k + 1][batch][V]
  const float *draft;     // [k][batch][V]
  const int32_t *drafts;  // [batch][k]
  const float *u;         // [batch][k + 1]
  int32_t *picks;         // [k + 1][batch]
  int batch, k, V;
  float2 *stats;          // [2k + 1][batch][chunks]: (max, sum) of a row's pieces
  int chunks;
  int slice;              // vocabulary entries per CTA
  int own_max;            // k = 0 and no statistics: the cluster finds the row's maximum
  int keep;               // whether both rows' weights of the slice are kept in shared memory
  float log2_scale;       // log2 e / T
  double scale, span;     // 16 log2 e / T; 990 octaves as a difference of logits
  unsigned *flags;
};

__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Running sum of the 16 lanes' values (lanes 16 .. 31 as 0 .. 15), inclusive.
__device__ __forceinline__ double scan16(double v, int lane) {
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) {
    const double t = __shfl_up_sync(0xffffffffu, v, o, 16);
    if ((lane & 15) >= o) v += t;
  }
  return v;
}

__device__ __forceinline__ double last16(double scanned) { return __shfl_sync(0xffffffffu, scanned, 15); }

// The sum of one double per thread over the CTA, the same bits in every thread;
// `warp_part` afterwards holds the warps' sums.
template <int kWarps>
__device__ __forceinline__ double cta_sum(double v, double *warp_part) {
  v = warp_sum_f64(v);
  __syncthreads();
  const int lane = threadIdx.x & 31;
  if (lane == 0) warp_part[threadIdx.x >> 5] = v;
  __syncthreads();
  return last16(scan16((lane & 15) < kWarps ? warp_part[lane & 15] : 0.0, lane));
}

// The cluster's CTAs' values (their *mine) in lanes 0 .. 15 and again in 16 .. 31,
// and their running sums, the same bits in every CTA. The sums of neighbouring
// lanes are added in different orders: next to a CTA without weight they may fall
// or rise by their last bit, so they order no shares. Needs a cluster barrier
// between the writes and the call.
__device__ __forceinline__ double rank_value(const double *mine, int lane, int CL) {
  const int i = lane & 15;
  return i < CL ? *cg::this_cluster().map_shared_rank(mine, i) : 0.0;
}
__device__ __forceinline__ double ranks_scan(const double *mine, int lane, int CL) {
  return scan16(rank_value(mine, lane, CL), lane);
}
// exp((x - ref) / T) in 64 bits, off by less than 2^-47: with y = 16 log2 e x / T
// - whole, 2^(n / 16) from a table (16 doubles in shared memory: one bank row, no
// conflicts whatever the lanes pick), n the nearest to y, times the polynomial of
// degree 5 through 2^(f / 16) at the six Chebyshev points of |f| <= 1/2 (off by
// 4.6e-15). `whole` is the whole number at or below 16 log2 e max / T, so ref is
// at most 1/16 octave below the maximum and weights reach 2^(1/16). It has to be
// whole: next to the rounding constant a fraction would be lost, and |f| with it
// reach 1, where the polynomial is off by 6e-12. Ten 64-bit operations and no
// branch: the 64-bit pipe (a warp's operation every 2.8 cycles) bounds these
// passes. Below 2^-990 and at -inf: 0.
__constant__ double kRoots[16] = {
    1.0, 1.0442737824274138, 1.0905077326652577, 1.1387886347566916,
    1.189207115002721, 1.241857812073484, 1.2968395546510096, 1.3542555469368927,
    1.4142135623730951, 1.4768261459394993, 1.5422108254079407, 1.6104903319492543,
    1.681792830507429, 1.7562521603732995, 1.8340080864093424, 1.9152065613971474};
struct Exp64 {
  double scale, shift;  // 16 log2 e / T, and -whole
  float low, max;       // logits at or below `low` have weight 0
  const double *table;
  __device__ __forceinline__ double operator()(float x) const {
    // (a hidden logit as the maximum, whose n is 0 or 1, times the table's 17th
    // entry, 0: its exponent must not be lowered)
    const bool some = x > low;
    const double xd = (double)(some ? x : max);
    const double t = fma(xd, scale, shift + 6755399441055744.0);  // n in the low bits
    const int n = __double2loint(t);
    const double f = fma(xd, scale, shift - (t - 6755399441055744.0));
    double p = 0x1.5d897e525c216p-30;
    p = fma(p, f, 0x1.3b2c9b8a6caeap-23);
    p = fma(p, f, 0x1.c6b08d6f2a289p-17);
    p = fma(p, f, 0x1.ebfbdff555824p-11);
    p = fma(p, f, 0x1.62e42fefa39f3p-5);
    p = fma(p, f, 0x1.0000000000014p+0);
    const double r = p * table[some ? n & 15 : 16];
    return __hiloint2double(__double2hiint(r) + (n & ~15) * 65536, __double2loint(r));
  }
};

constexpr int kChunk = 8192;        // logits of a piece
constexpr int kStatsThreads = 256;  // 8 float4 a thread, and the row's unaligned ends

// (max, sum of exp((x - max) / T)) of piece blockIdx.x of row blockIdx.y (rows in
// memory order: the target's, then the draft's).
__global__ void __launch_bounds__(kStatsThreads) sample_stats_kernel(const SampleArgs a) {
  pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, V = a.V;
  const int rows_t = (a.k + 1) * a.batch, r = blockIdx.y;
  const float *p = r < rows_t ? a.target + (size_t)r * V : a.draft + (size_t)(r - rows_t) * V;
  const float c = a.log2_scale;
  // the piece's aligned float4s; the row's ends (fewer than 4 logits each) go to
  // its first and its last piece
  const int lead = min((int)((4 - ((uintptr_t)p >> 2 & 3)) & 3), V), quads = (V - lead) / 4;
  const int q0 = blockIdx.x * (kChunk / 4);
  const float4 *x = reinterpret_cast<const float4 *>(p + lead);
  float4 v[8];
#pragma unroll
  for (int e = 0; e < 8; e++) {
    const int i = q0 + tid + e * kStatsThreads;
    v[e] = i < quads ? __ldg(x + i) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
  }
  float end = -INFINITY;
  const int tail = lead + 4 * quads + tid - 4;
  if (blockIdx.x == 0 && tid < lead) end = p[tid];
  if (blockIdx.x == gridDim.x - 1 && tid >= 4 && tail < V) end = p[tail];
  float m = end;
#pragma unroll
  for (int e = 0; e < 8; e++) m = fmaxf(fmaxf(m, fmaxf(v[e].x, v[e].y)), fmaxf(v[e].z, v[e].w));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  __shared__ float sm[kStatsThreads / 32], ss[kStatsThreads / 32];
  if (lane == 0) sm[tid >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kStatsThreads / 32; i++) m = fmaxf(m, sm[i]);
  const float sub = m > -INFINITY ? m : 0.0f;  // (-inf throughout: every term 0; NaN: NaN)
  float s = ex2((end - sub) * c);
#pragma unroll
  for (int e = 0; e < 8; e++)
    s += (ex2((v[e].x - sub) * c) + ex2((v[e].y - sub) * c)) + (ex2((v[e].z - sub) * c) + ex2((v[e].w - sub) * c));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0) ss[tid >> 5] = s;
  __syncthreads();
  if (tid == 0) {
#pragma unroll
    for (int i = 1; i < kStatsThreads / 32; i++) s += ss[i];
    a.stats[(size_t)r * a.chunks + blockIdx.x] = make_float2(m, s);
  }
}

template <int kWarps, int kCtasPerSm>
__global__ void __launch_bounds__(kWarps * 32, kCtasPerSm) spec_sample_kernel(const SampleArgs a) {
  cg::cluster_group cl = cg::this_cluster();
  const int rank = (int)cl.block_rank(), CL = (int)cl.num_blocks();
  const int b = blockIdx.x / CL;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int k = a.k, R = 2 * k + 1, V = a.V;
  extern __shared__ __align__(16) double kept[];  // weights of the drawn row: p's, then q's (a.keep)
  __shared__ float row_m[kMaxRows];
  __shared__ double row_z[kMaxRows];
  __shared__ double table[17], warp_part[kWarps], cta_part[4];
  __shared__ float cta_max;
  __shared__ double slots[kWarps][kSlots];  // each warp's sums of the draw's weights, by rounds
  __shared__ int s_n, s_owner;
  static_assert(kWarps <= 16 && kSampleCluster == 16, "16 lanes scan");

  pdl_trigger();
  if (tid < 17) table[tid] = tid < 16 ? kRoots[tid] : 0.0;
  pdl_wait();

  // rows 0 .. k: the target's; k + 1 .. 2k: the draft's
  auto row = [&](int r) {
    return r <= k ? a.target + ((size_t)r * a.batch + b) * V : a.draft + ((size_t)(r - k - 1) * a.batch + b) * V;
  };
  const float c = a.log2_scale;

  // ---- (1) every row's maximum and sum, from its pieces'; meanwhile the last
  // warp fetches what acceptance needs (lane j: draft j)
  int d = -1;
  float xp_d = 0.0f, xq_d = 0.0f;
  double u_d = 0.0;
  if (warp == kWarps - 1 && lane < k) {
    d = a.drafts[(size_t)b * k + lane];
    u_d = (double)a.u[(size_t)b * (k + 1) + lane];
    if (u_d >= 1.0) u_d = 1.0 - 0x1p-24;
    if (d >= 0 && d < V) {
      xp_d = row(lane)[d];
      xq_d = row(k + 1 + lane)[d];
    }
  }
  for (int r = a.own_max ? R : warp; r < R; r += kWarps) {
    const float2 *st = a.stats + ((size_t)r * a.batch + b) * a.chunks;
    float2 v = lane < a.chunks ? __ldcg(st + lane) : make_float2(-INFINITY, 0.0f);
    float m = v.x;
    for (int i = lane + 32; i < a.chunks; i += 32) m = fmaxf(m, __ldcg(st + i).x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    // (a piece of nothing: -inf and 0, or a NaN on its way)
    auto share = [&](float2 w) { return (double)w.y * (w.x > -INFINITY ? (double)ex2((w.x - m) * c) : 1.0); };
    double z = share(v);
    for (int i = lane + 32; i < a.chunks; i += 32) z += share(__ldcg(st + i));
    z = warp_sum_f64(z);
    if (lane == 0) {
      row_m[r] = m;
      row_z[r] = z;
    }
  }
  __syncthreads();

  const int v0 = (int)min((long long)V, (long long)rank * a.slice), n_v = (int)min((long long)a.slice, (long long)V - v0);
  // this warp's run of the slice, in rounds of 256 (8 logits a lane, 32 apart)
  const int per_warp = (n_v + 256 * kWarps - 1) / (256 * kWarps) * 256;
  const int w0 = min(n_v, warp * per_warp), w1 = min(n_v, w0 + per_warp);
  auto weights = [&](int r) {
    const double m = (double)row_m[r], low = m - a.span;
    // A maximum so large that its neighbours in fp32 lie below 2^-990 (where the
    // product with the scale would lose its last bits): weights 1 and 0.
    if (fabs(m * a.scale) > 1e12) return Exp64{0.0, 0.0, nextafterf(row_m[r], -INFINITY), row_m[r], table};
    return Exp64{a.scale, -floor(m * a.scale), low > -3.4e38 ? (float)low : -3.4e38f, row_m[r], table};
  };
  // a row's sum from its pieces (over the maximum), as one of weights(r)
  auto sum_of = [&](int r, const Exp64 &w) { return row_z[r] * w(row_m[r]); };
  auto round_of = [&](const float *x, int i0, float v[8]) {
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = i0 + 32 * e < w1 ? __ldg(x + i0 + 32 * e) : -INFINITY;
  };
  // f(i, logit) over this warp's run of a row (-inf past its end)
  auto each = [&](const float *x, auto &&f) {
    for (int i0 = w0 + lane; i0 < w1 + lane; i0 += 256) {
      float v[8];
      round_of(x, i0, v);
#pragma unroll
      for (int e = 0; e < 8; e++) f(i0 + 32 * e, v[e]);
    }
  };
  if (a.own_max) {  // the row's maximum (+inf stands for a NaN too); its sum is made below
    float m = -INFINITY;
    bool nan = false;
    each(row(0) + v0, [&](int, float x) {
      m = fmaxf(m, x);
      nan |= isnan(x);
    });
    if (nan) m = INFINITY;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) warp_part[warp] = (double)m;
    __syncthreads();
    if (tid == 0) {
      for (int i = 1; i < kWarps; i++) m = fmaxf(m, (float)warp_part[i]);
      cta_max = m;
    }
    cl.sync();
    m = (lane & 15) < CL ? *cl.map_shared_rank(&cta_max, lane & 15) : -INFINITY;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (tid == 0) {
      row_m[0] = m;
      row_z[0] = fabsf(m) < INFINITY ? 1.0 : 0.0;
    }
    __syncthreads();
  }
  // the sum of row r's weights over the whole vocabulary
  auto exact_sum = [&](int r) {
    const Exp64 w = weights(r);
    double s = 0.0;
    each(row(r) + v0, [&](int, float x) { s += w(x); });
    s = cta_sum<kWarps>(s, warp_part);
    if (tid == 0) cta_part[0] = s;
    cl.sync();
    s = last16(ranks_scan(&cta_part[0], lane, CL));
    cl.sync();  // cta_part may be written again
    return s;
  };

  // ---- (2) acceptance: lane j decides draft j, the same in every CTA
  int n = 0;
  if (k > 0) {
    if (warp == kWarps - 1) {
      bool kept_it = false, close = false;
      if (lane < k && d >= 0 && d < V) {
        const Exp64 wp = weights(lane), wq = weights(k + 1 + lane);
        const double lhs = u_d * wq(xq_d) * sum_of(lane, wp), rhs = wp(xp_d) * sum_of(k + 1 + lane, wq);
        kept_it = lhs < rhs;
        close = fabs(lhs - rhs) <= kSlack * rhs && rhs > 0.0;
      }
      const unsigned stop = __ballot_sync(0xffffffffu, lane < k && (!kept_it || close));
      const unsigned near_ = __ballot_sync(0xffffffffu, close);
      // the first that is not clearly kept; negative: too close for the fp32 sums
      const int first = stop ? __ffs(stop) - 1 : k;
      if (lane == 0) s_n = first < k && (near_ >> first & 1) ? -1 - first : first;
    }
    __syncthreads();
    n = s_n;
    if (n < 0)  // from there on one by one
      for (n = -1 - n; n < k; n++) {
        const int dd = a.drafts[(size_t)b * k + n];
        double u = (double)a.u[(size_t)b * (k + 1) + n];
        if (u >= 1.0) u = 1.0 - 0x1p-24;
        if (dd < 0 || dd >= V) break;
        const Exp64 wp = weights(n), wq = weights(k + 1 + n);
        const double pe = wp(row(n)[dd]), qe = wq(row(k + 1 + n)[dd]);
        const double lhs = u * qe * sum_of(n, wp), rhs = pe * sum_of(k + 1 + n, wq);
        if (fabs(lhs - rhs) <= kSlack * rhs && rhs > 0.0) {
          const double zq = exact_sum(k + 1 + n), zp = exact_sum(n);
          if (!(u * (qe / zq) < pe / zp)) break;
        } else if (!(lhs < rhs)) {
          break;
        }
      }
  }

  // rows without probabilities (NaN, +inf, -inf throughout): a token all the
  // same, never the rejected one, and a report
  const int dn = n < k ? a.drafts[(size_t)b * k + n] : -1;  // (-1: no token is left out)
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

  // ---- (3) the weights of the draw: of max(p - q, 0) of row n, or of p of row k
  const bool diff = n < k;
  const float *xp = row(n) + v0, *xq = diff ? row(k + 1 + n) + v0 : nullptr;
  const Exp64 wp = weights(n), wq = weights(diff ? k + 1 + n : n);
  double ip = 1.0, iq = 0.0;
  double *const kept_q = kept + (a.slice + 255) / 256 * 256;
  if (diff) {
    double sp = 0.0, sq = 0.0;
    for (int i0 = w0 + lane; i0 < w1 + lane; i0 += 256) {
      float x[8], y[8];
      round_of(xp, i0, x);
      round_of(xq, i0, y);
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const double ep = wp(x[e]), eq = wq(y[e]);
        if (a.keep) {
          kept[i0 + 32 * e] = ep;
          kept_q[i0 + 32 * e] = eq;
        }
        sp += ep;
        sq += eq;
      }
    }
    sp = cta_sum<kWarps>(sp, warp_part);
    sq = cta_sum<kWarps>(sq, warp_part);
    if (tid == 0) {
      cta_part[1] = sp;
      cta_part[2] = sq;
    }
    cl.sync();
    const double rp = ranks_scan(&cta_part[1], lane, CL), rq = ranks_scan(&cta_part[2], lane, CL);
    ip = 1.0 / last16(rp);
    iq = 1.0 / last16(rq);
  }
  bool without = false;  // p without the rejected token instead
  // what each of a lane's 8 tokens i0, i0 + 32, ... of a round weighs
  auto masses = [&](int i0, double m[8]) {
    float v[8];
    if (diff && a.keep && !without) {
#pragma unroll
      for (int e = 0; e < 8; e++) m[e] = fmax(kept[i0 + 32 * e] * ip - kept_q[i0 + 32 * e] * iq, 0.0);
      return;
    }
    round_of(xp, i0, v);
    if (diff && !without) {
      float y[8];
      round_of(xq, i0, y);
#pragma unroll
      for (int e = 0; e < 8; e++) m[e] = fmax(wp(v[e]) * ip - wq(y[e]) * iq, 0.0);
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) m[e] = v0 + i0 + 32 * e == dn ? 0.0 : wp(v[e]);
    }
  };

  // ---- (4) the token: the first whose running sum exceeds u times the total
  double total, rank_head, warp_total, warp_head;  // (rank_head: lane i's of CTA i)
  const int per_slot = (per_warp / 256 + kSlots - 1) / kSlots * 256;  // rounds that share a slot
  for (;;) {
    warp_total = 0.0;
    for (int slot = 0, i0 = w0; i0 < w1; slot++) {
      double s = 0.0;
      for (const int i1 = min(w1, i0 + per_slot); i0 < i1; i0 += 256) {
        double m[8];
        masses(i0 + lane, m);
        s += ((m[0] + m[1]) + (m[2] + m[3])) + ((m[4] + m[5]) + (m[6] + m[7]));
      }
      s = warp_sum_f64(s);
      if (lane == 0) slots[warp][slot] = s;
      warp_total += s;
    }
    __syncthreads();
    if (lane == 0) warp_part[warp] = warp_total;
    if (tid == 0) s_owner = -1;
    __syncthreads();
    const double warps = scan16((lane & 15) < kWarps ? warp_part[lane & 15] : 0.0, lane);
    warp_head = warp > 0 ? __shfl_sync(0xffffffffu, warps, warp - 1) : 0.0;
    if (tid == 15) cta_part[3] = warps;
    cl.sync();
    const double mass = rank_value(&cta_part[3], lane, CL), ranks = scan16(mass, lane);
    total = last16(ranks);
    rank_head = __shfl_up_sync(0xffffffffu, ranks, 1, 16);
    if (!(lane & 15)) rank_head = 0.0;
    if (!(mass > 0.0)) rank_head = INFINITY;
    // p and q may agree to the last bit everywhere: then the rejected token's
    // place goes to another token of p
    if (!diff || without || total > 0.0) break;
    without = true;
    cl.sync();
  }
  double u = (double)a.u[(size_t)b * (k + 1) + k];
  if (!(u < 1.0)) u = 1.0 - 0x1p-24;
  if (!(u > 0.0)) u = 0.0;
  const double goal = u * total;
  if (!(total > 0.0)) report();  // all of p on the rejected token: q was no distribution
  // The last CTA that has weight and whose head is not past the goal (the first
  // that has weight has head 0, so there is always one, the same in every CTA),
  // in it the last such warp, there the last round, the last run of 32, and in
  // that the first token past the goal. (Where rounding leaves the goal past the
  // run's own sum: its last token with weight.)
  const unsigned ranks_at = __ballot_sync(0xffffffffu, lane < 16 && rank_head <= goal);
  if (total > 0.0 && 31 - __clz(ranks_at) == rank) {
    double head = __shfl_sync(0xffffffffu, rank_head, rank) + warp_head;
    if (lane == 0 && warp_total > 0.0 && head <= goal) atomicMax(&s_owner, warp);
    __syncthreads();
    if (warp == s_owner) {
      int at = w0;
      double at_head = head, m[8];
      for (int slot = 0, i0 = w0; i0 < w1; slot++, i0 += per_slot) {
        const double s = slots[warp][slot];
        if (s > 0.0 && head <= goal) {
          at = i0;
          at_head = head;
        }
        head += s;
      }
      if (per_slot > 256) {  // (a vocabulary a warp: the slot's rounds once more)
        head = at_head;
        for (int i0 = at, i1 = min(w1, at + per_slot); i0 < i1; i0 += 256) {
          masses(i0 + lane, m);
          const double s =
              warp_sum_f64(((m[0] + m[1]) + (m[2] + m[3])) + ((m[4] + m[5]) + (m[6] + m[7])));
          if (s > 0.0 && head <= goal) {
            at = i0;
            at_head = head;
          }
          head += s;
        }
      }
      masses(at + lane, m);
      double sums[8];
#pragma unroll
      for (int e = 0; e < 8; e++) sums[e] = warp_sum_f64(m[e]);
      head = at_head;
      double run = 0.0, run_head = head;
      int run_at = at;
#pragma unroll
      for (int e = 0; e < 8; e++) {
        if (sums[e] > 0.0 && head <= goal) {
          run = m[e];
          run_head = head;
          run_at = at + 32 * e;
        }
        head += sums[e];
      }
      double s = run;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double t = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += t;
      }
      const unsigned past = __ballot_sync(0xffffffffu, run > 0.0 && run_head + s > goal);
      const unsigned some = __ballot_sync(0xffffffffu, run > 0.0);
      if (lane == 0)
        a.picks[(size_t)n * a.batch + b] = v0 + run_at + (past ? __ffs(past) - 1 : 31 - __clz(some));
    }
  }
  cl.sync();  // peers may still read this CTA's shared memory
}

}  // namespace

static int sample_chunks(int V) { return (V + kChunk - 1) / kChunk; }

size_t spec_sample_workspace(int batch, int k, int V) {
  return (size_t)batch * (2 * k + 1) * sample_chunks(V) * sizeof(float2);
}

cudaError_t launch_spec_sample(const float *target, const float *draft, const int32_t *drafts, int batch, int k, int V,
                               double temperature, const float *u, int32_t *picks, void *workspace, unsigned *flags,
                               int num_sms, cudaStream_t s, bool pdl) {
  // CTAs per sequence: as many as leave slices of 4096 entries, and no more than
  // let all sequences run at once (61 sequences of 65543, k = 5: 8 CTAs each 66
  // us, 4 or 16 CTAs 82 and 79 us)
  int CL = 1;
  while (CL < kSampleCluster && (long long)CL * 4096 < V && (long long)batch * CL * 2 <= 4 * num_sms) CL *= 2;
  // 16 warps a CTA where it has an SM to itself and work for them (8 sequences of
  // 128256, k = 4: 22 us, with 8 warps 28 us), else 8
  const bool wide = batch * CL <= num_sms && (V + CL - 1) / CL >= 4096;
  SampleArgs a{};
  a.target = target;
  a.draft = draft;
  a.drafts = drafts;
  a.u = u;
  a.picks = picks;
  a.batch = batch;
  a.k = k;
  a.V = V;
  a.stats = reinterpret_cast<float2 *>(workspace);
  a.chunks = sample_chunks(V);
  a.slice = (V + CL - 1) / CL;
  a.log2_scale = (float)(1.4426950408889634 / temperature);
  a.scale = 16.0 * 1.4426950408889634074 / temperature;
  a.span = 15840.0 / a.scale;
  a.flags = flags;
  // Plain sampling needs the row's maximum alone: a cluster of slices up to 4096
  // finds it sooner than the other launch would end (8 rows of 32000: 9.1 us, with
  // the statistics 10.4, and half the launches on the host; 8 rows of 128256,
  // slices of 8016: 21.5 and 19.7 us)
  a.own_max = k == 0 && a.slice <= 4096;
  // A rejected sequence's weights are used twice: kept where that costs no other
  // CTA its place (each SM has one at most), made again otherwise
  const size_t weights = 2 * (size_t)((a.slice + 255) / 256 * 256) * sizeof(double);
  a.keep = k && weights <= kKeepBytes && wide;
  cudaLaunchConfig_t cfg = {};
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = (unsigned)CL;
  at[1].val.clusterDim.y = 1;
  at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = pdl ? 1 : 0;
  cfg.gridDim = dim3((unsigned)a.chunks, (unsigned)((2 * k + 1) * batch));
  cfg.blockDim = dim3(kStatsThreads);
  cudaError_t e = a.own_max ? cudaSuccess : cudaLaunchKernelEx(&cfg, sample_stats_kernel, a);
  auto kern = wide ? spec_sample_kernel<16, 1> : spec_sample_kernel<8, 4>;
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kKeepBytes);
  if (e != cudaSuccess) return e;
  cfg.attrs = pdl ? at : at + 1;
  cfg.numAttrs = pdl ? 2 : 1;
  cfg.gridDim = dim3((unsigned)(batch * CL));
  cfg.blockDim = dim3(wide ? 512 : 256);
  cfg.dynamicSmemBytes = a.keep ? weights : 0;
  return cudaLaunchKernelEx(&cfg, kern, a);
}

}  // namespace wg
