// The paged key-value cache (webgllm_paged.h): the append of new rows (qk-norm
// and RoPE on the way) and attention over the pages.
#include <cmath>

#include "common.cuh"
#include "paged_device.cuh"

namespace wg {

namespace {

template <typename T>
__device__ __forceinline__ void mma16816(float d[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t r[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t r[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}

// ---- rows and sequences ----------------------------------------------------

// The sequence of row r (by the whole warp), or -1 if it belongs to none:
// the last b with row_start[b] <= r, found 32 entries at a step.
__device__ __forceinline__ int row_seq(const PagedRows &a, int r, int lane) {
  if (!a.row_start) return r / (a.rows / a.batch);
  int lo = 0, hi = a.batch;  // row_start[lo] <= r (checked below), r < row_start[hi]
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32;
    const int i = lo + (lane + 1) * step;
    const unsigned m = __ballot_sync(0xffffffffu, i < hi && a.row_start[i] <= r);
    const int c = __popc(m);  // ascending: the lanes that hold are the first c
    lo += c * step;
    hi = min(hi, lo + step);
  }
  return a.row_start[lo] <= r && r < a.row_start[lo + 1] ? lo : -1;
}

// ---- append ----------------------------------------------------------------
// A warp takes one row and up to `heads_per_warp` of its H + 2 Hkv heads: lane
// l holds the rotate-half pairs (j, j + Dh/2) of a few neighbouring j, so that
// a head is two coalesced loads and two coalesced stores, and the angles'
// sines are made once for all the warp's heads. The angle of pair j at
// position p, in turns, is p theta^(-2j/Dh) / 2 pi: its factor comes from the
// host in 64 bits and the whole turns are taken off in 64 bits (one product,
// one rounding, one difference), so that the fp32 sine sees an argument in
// [-1, 1] half turns, exact at any position. Bound by its bytes for prompts
// and by launch latency for decode rows.

struct RopeTurns {
  double t[128];  // theta^(-2j/Dh) / (2 pi)
};

template <typename T, int Dh>
__global__ void __launch_bounds__(256)
    paged_rope_kernel(const float *qkv, const PagedRows pr, int H, int Hkv, const RopeTurns turns,
                      const float *q_norm, const float *k_norm, float eps, T *q_out, T *k_pages, T *v_pages,
                      int64_t page_stride, int64_t head_stride, int64_t row_stride, const PagedTable pt,
                      int heads_per_warp, int warps_per_row, unsigned *flags) {
  pdl_trigger();
  pdl_wait();
  constexpr int kVec = Dh == 256 ? 4 : 2;          // neighbouring j a lane holds
  constexpr int kLanes = Dh / 2 / kVec;            // lanes of a head (16 for Dh = 64: two heads at once)
  constexpr int kHeads = 32 / kLanes;
  const int lane = threadIdx.x & 31;
  const long long w = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int r = (int)(w / warps_per_row);
  if (r >= pr.rows) return;
  const int b = row_seq(pr, r, lane);
  if (b < 0) return;
  int r0, n;
  seq_rows(pr, b, r0, n);
  const long long p = (long long)pr.pos[b] + (r - r0);
  const int j0 = (lane % kLanes) * kVec, sub = lane / kLanes;
  float cs[kVec], sn[kVec];
#pragma unroll
  for (int i = 0; i < kVec; i++) {
    const double t = (double)p * turns.t[j0 + i];
    sincospif((float)(2.0 * (t - rint(t))), &sn[i], &cs[i]);
  }
  // the row's place in the cache
  const long long cap = (long long)pt.max_pages * pt.page_size;
  long long place = -1;
  if (p >= 0) {
    int page = -1;
    if (p < cap) page = pt.table[(size_t)b * pt.max_pages + p / pt.page_size];
    if (page >= 0 && page < pt.num_pages)
      place = page * (long long)page_stride + (p % pt.page_size) * (long long)row_stride;
    else if (lane == 0)
      raise_flag(flags, kFlagBadArgument);
  }
  const int NH = H + 2 * Hkv;
  const int h0 = (int)(w - (long long)r * warps_per_row) * heads_per_warp;
  const float scale = rsqrtf((float)Dh);
  for (int hh = h0; hh < min(h0 + heads_per_warp, NH); hh += kHeads) {
    const int h = hh + sub;
    const bool on = h < min(h0 + heads_per_warp, NH);
    float x[kVec], y[kVec];  // dims j0 + i and j0 + i + Dh / 2
    if (on) {
      const float *src = qkv + ((size_t)r * NH + h) * Dh + j0;
      if constexpr (kVec == 4) {
        const float4 u = *reinterpret_cast<const float4 *>(src), v = *reinterpret_cast<const float4 *>(src + Dh / 2);
        x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w;
        y[0] = v.x, y[1] = v.y, y[2] = v.z, y[3] = v.w;
      } else {
        const float2 u = *reinterpret_cast<const float2 *>(src), v = *reinterpret_cast<const float2 *>(src + Dh / 2);
        x[0] = u.x, x[1] = u.y;
        y[0] = v.x, y[1] = v.y;
      }
    } else {
#pragma unroll
      for (int i = 0; i < kVec; i++) x[i] = y[i] = 0.0f;
    }
    const bool is_q = h < H, is_v = h >= H + Hkv;
    if (q_norm || k_norm) {  // the whole warp: a head's lanes sum its squares
      float ss = 0.0f;
#pragma unroll
      for (int i = 0; i < kVec; i++) ss += x[i] * x[i] + y[i] * y[i];
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float *nw = is_q ? q_norm : is_v ? nullptr : k_norm;
      if (nw && on) {
        const float inv = rsqrtf(ss / (float)Dh + eps);
#pragma unroll
        for (int i = 0; i < kVec; i++) {
          x[i] *= inv * nw[j0 + i];
          y[i] *= inv * nw[j0 + Dh / 2 + i];
        }
      }
    }
    if (!on) continue;
    if (!is_v) {
      const float sc = is_q ? scale : 1.0f;
#pragma unroll
      for (int i = 0; i < kVec; i++) {
        const float a = x[i], c = y[i];
        x[i] = (a * cs[i] - c * sn[i]) * sc;
        y[i] = (c * cs[i] + a * sn[i]) * sc;
      }
    }
    T *dst;
    if (is_q) {
      dst = q_out + ((size_t)r * H + h) * Dh;
      if (p < 0) {
#pragma unroll
        for (int i = 0; i < kVec; i++) x[i] = y[i] = 0.0f;
      }
    } else {
      if (place < 0) continue;
      const int hk = is_v ? h - H - Hkv : h - H;
      dst = (is_v ? v_pages : k_pages) + place + hk * head_stride;
    }
    dst += j0;
#pragma unroll
    for (int i = 0; i < kVec; i += 2) {
      *reinterpret_cast<uint32_t *>(dst + i) = pack2<T>(x[i], x[i + 1]);
      *reinterpret_cast<uint32_t *>(dst + Dh / 2 + i) = pack2<T>(y[i], y[i + 1]);
    }
  }
}

// ---- attention, split over the keys ---------------------------------------
// o = softmax(q k^T) v per (sequence, KV head, 16 MT rows of queries), where
// the sequence's rows times the G query heads of the KV head are the rows of
// one small matrix product: a K / V tile is read once for all of them. Decode
// is bound by those reads, so the work is counted in tiles of 64 keys over
// all sequences and heads and each of P resident CTAs takes an equal run of
// tiles, wherever sequences begin and end in it: short and long sequences
// share the machine evenly whatever their lengths, which only the device
// knows. Per CTA:
//   warp 4      the producer: page entries, then one TMA copy per box of a
//               page's rows x 64 dims (128-byte swizzle) into a ring of
//               stages (K and V of 64 keys each);
//   warps 0-3   16 keys of a tile each, for all its query rows: S = Q K^T and
//               O += P V on mma.m16n8k16 with fp32 sums, a running maximum
//               and sum per row in registers (log2 domain). The warps meet
//               only at the end of a run of tiles.
// P stays at fp32 precision: hi + lo 16-bit halves, two products (the tensor
// pipe idles under the loads).
// A (sequence, head, rows) unit that one CTA finishes alone is written by it;
// else each CTA leaves (max, sum, O) in the workspace and paged_join_kernel
// adds them in order: no atomics, the same bits every time.

constexpr int kKeys = 64;          // keys per tile
constexpr int kSplitWarps = 4;     // consumer warps (16 keys each)
constexpr int kSplitThreads = (kSplitWarps + 1) * 32;
constexpr int kMaxStages = 8;

struct SplitArgs {
  PagedRows pr;
  PagedTable pt;
  const void *q;
  void *out;
  int H, Hkv, G;
  int window, sinks;
  int box_rows;  // keys of one TMA box: divides page_size and 64
  int stages;
  int *rec;      // workspace: [P][8]
  float *part;   // workspace: [2 P][rows * (Dh + 2)]
  unsigned *flags;
};

// One sequence's share of the work: row tiles (per KV head) times key tiles.
struct SeqWork : KeySpan {
  int r0, n;  // rows
  int p;      // position of its first row
  int mt;     // row tiles
};

__device__ __forceinline__ SeqWork seq_work(const SplitArgs &A, int b, int rows_per_tile) {
  SeqWork w;
  seq_rows(A.pr, b, w.r0, w.n);
  w.p = A.pr.pos[b];
  w.mt = (int)(((long long)w.n * A.G + rows_per_tile - 1) / rows_per_tile);
  static_cast<KeySpan &>(w) = key_span(w.p, w.n, A.window, A.sinks, A.pt, kKeys);
  return w;
}

__device__ __forceinline__ int block_scan_incl(int v, int *red, int &total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += t;
  }
  __syncthreads();
  if (lane == 31) red[warp] = v;
  __syncthreads();
  int before = 0;
  total = 0;
  for (int i = 0; i < nw; i++) {
    if (i < warp) before += red[i];
    total += red[i];
  }
  return v + before;
}

template <typename T, int Dh, int MT>
struct SplitSmem {
  static constexpr int kRows = 16 * MT;
  static constexpr int kTileBytes = kKeys * Dh * 2;  // K or V of a stage
  static constexpr int kStageBytes = 2 * kTileBytes;
  static constexpr int kRedBytes = 2 * kRows * Dh * 4;  // the warps' merge
  static constexpr int kFixed = 1024 /* alignment */ + kRedBytes + 4 * kSplitWarps * kRows * 2 + 256;
};

template <typename T, int Dh, int MT>
__global__ void __launch_bounds__(kSplitThreads, MT == 1 && Dh <= 128 ? 2 : 1)
    paged_split_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                       const SplitArgs A) {
  using S = SplitSmem<T, Dh, MT>;
  constexpr int kBlk = Dh / 64;                    // 64-dim blocks of a row
  constexpr int kBlkBytes = kKeys * 128;           // one block of a stage's K or V
  constexpr float kLog2e = 1.4426950408889634f;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  uint8_t *smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  float *red = reinterpret_cast<float *>(smem + (size_t)A.stages * S::kStageBytes);  // [2][kRows][Dh]
  float *sm_m = red + 2 * S::kRows * Dh;           // [warps][kRows]
  float *sm_l = sm_m + kSplitWarps * S::kRows;
  __shared__ uint64_t full[kMaxStages], empty[kMaxStages];
  __shared__ int held[kMaxStages];                 // which of a stage's boxes were loaded
  __shared__ int scan_red[kSplitThreads / 32];
  __shared__ int s_b, s_base, aborted;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int P = (int)gridDim.x, cta = (int)blockIdx.x;

  if (tid == 0) {
    for (int i = 0; i < A.stages; i++) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], kSplitWarps);
    }
    fence_mbar_init();
    aborted = 0;
    s_b = A.pr.batch;
    s_base = 0;
  }
  if (warp == kSplitWarps && lane == 0) {
    prefetch_tensormap(&tm_k);
    prefetch_tensormap(&tm_v);
  }
  pdl_trigger();
  pdl_wait();  // rows, positions, pages and queries come from earlier kernels
  __syncthreads();

  // the total work, then where this CTA's run begins
  int total = 0;
  for (int b0 = 0; b0 < A.pr.batch; b0 += kSplitThreads) {
    int v = 0, t;
    if (b0 + tid < A.pr.batch) {
      const SeqWork w = seq_work(A, b0 + tid, S::kRows);
      v = A.Hkv * w.mt * w.nt;
    }
    block_scan_incl(v, scan_red, t);
    total += t;
  }
  const int per = (total + P - 1) / P;
  const int start = min((long long)total, (long long)cta * per), end = min((long long)total, (long long)start + per);
  for (int b0 = 0, run = 0; b0 < A.pr.batch && run <= start; b0 += kSplitThreads) {
    int v = 0, t;
    if (b0 + tid < A.pr.batch) {
      const SeqWork w = seq_work(A, b0 + tid, S::kRows);
      v = A.Hkv * w.mt * w.nt;
    }
    const int incl = run + block_scan_incl(v, scan_red, t);
    if (incl - v <= start && start < incl) {
      s_b = b0 + tid;
      s_base = incl - v;
    }
    run += t;
  }
  __syncthreads();
  int b = s_b, base = s_base;

  auto wait = [&](uint64_t *bar, uint32_t parity) {
    if (*(volatile int *)&aborted) return;
    if (!mbar_wait_bounded(bar, parity, A.flags)) *(volatile int *)&aborted = 1;
  };
  int stage = 0, phase = 0;
  auto advance = [&]() {
    if (++stage == A.stages) {
      stage = 0;
      phase ^= 1;
    }
  };

  if (warp == kSplitWarps) {
    // ---- producer ----
    const int nb = kKeys / A.box_rows;  // boxes per tile
    const int nops = nb * kBlk * 2;
    const int box = lane % nb, blk = (lane / nb) % kBlk, is_v = lane / (nb * kBlk);
    const uint32_t box_bytes = (uint32_t)A.box_rows * 128;
    for (int pos = start; pos < end;) {
      const SeqWork w = seq_work(A, b, S::kRows);
      const int work = A.Hkv * w.mt * w.nt;
      if (pos >= base + work) {
        base += work;
        b++;
        continue;
      }
      const int unit = (pos - base) / w.nt, t0 = (pos - base) - unit * w.nt;
      const int t1 = min(w.nt, t0 + (end - pos));
      const int hk = unit / w.mt;
      const int32_t *row = A.pt.table + (size_t)b * A.pt.max_pages;
      // the box's page entry and whether any row sees a key of it
      auto entry = [&](int t, int &key, bool &seen) {
        key = (t < w.a ? t : t - w.a + w.c) * kKeys + box * A.box_rows;
        seen = lane < nops && key < w.hi && (key < w.se || key + A.box_rows > w.ws);
        return seen ? row[key / A.pt.page_size] : -1;
      };
      int key, key_next;
      bool seen, seen_next;
      int page = entry(t0, key, seen), page_next = -1;
      for (int t = t0; t < t1; t++) {
        if (t + 1 < t1) page_next = entry(t + 1, key_next, seen_next);
        wait(&empty[stage], phase ^ 1);
        const bool ok = seen && page >= 0 && page < A.pt.num_pages;
        if (seen && !ok) raise_flag(A.flags, kFlagBadArgument);
        const unsigned loaded = __ballot_sync(0xffffffffu, ok && lane < nb);
        if (lane == 0) {
          held[stage] = (int)loaded;
          mbar_expect_tx(&full[stage], (uint32_t)__popc(loaded) * box_bytes * kBlk * 2);
        }
        __syncwarp();
        if (ok) {
          uint8_t *dst = smem + (size_t)stage * S::kStageBytes + is_v * S::kTileBytes + blk * kBlkBytes +
                         box * box_bytes;
          const CUtensorMap *tm = is_v ? &tm_v : &tm_k;
          tma_load_4d(dst, tm, blk * 64, key % A.pt.page_size, hk, page, &full[stage]);
        }
        page = page_next;
        key = key_next;
        seen = seen_next;
        advance();
      }
      pos += t1 - t0;
    }
    // after a wait that ran out, no copy may still be on its way into this
    // CTA's memory when it exits
    __syncwarp();
    if (*(volatile int *)&aborted && lane == 0)
      for (int i = 0; i < A.stages; i++) {
        mbar_wait_bounded(&full[stage], phase ^ 1, A.flags);
        advance();
      }
  } else {
    // ---- consumers ----
    const int g = lane >> 2, t4 = lane & 3;
    const int jm = lane >> 3, jr = lane & 7;  // ldmatrix: this lane addresses row jr of matrix jm
    int rec_parts = 0;
    int rec[6] = {0, 0, 0, 0, 0, 0};
    for (int pos = start; pos < end;) {
      const SeqWork w = seq_work(A, b, S::kRows);
      const int work = A.Hkv * w.mt * w.nt;
      if (pos >= base + work) {
        base += work;
        b++;
        continue;
      }
      const int unit = (pos - base) / w.nt, t0 = (pos - base) - unit * w.nt;
      const int t1 = min(w.nt, t0 + (end - pos));
      const int hk = unit / w.mt, m0 = (unit - hk * w.mt) * S::kRows;

      // queries as A fragments; the position of each of this thread's rows
      uint32_t qa[MT][Dh / 16][4];
      int rp[MT][2];
#pragma unroll
      for (int mt = 0; mt < MT; mt++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const int m = m0 + mt * 16 + g + 8 * e, i = m / A.G;
          const bool valid = i < w.n;
          const long long rpos = valid ? (long long)w.p + i : -1;
          rp[mt][e] = (int)max(-1LL, min(rpos, 0x7ffffffeLL));
          const T *src = reinterpret_cast<const T *>(A.q) +
                         ((size_t)(w.r0 + (valid ? i : 0)) * A.H + hk * A.G + (valid ? m - i * A.G : 0)) * Dh + 2 * t4;
#pragma unroll
          for (int kk = 0; kk < Dh / 16; kk++) {
            qa[mt][kk][e] = valid ? *reinterpret_cast<const uint32_t *>(src + 16 * kk) : 0u;
            qa[mt][kk][e + 2] = valid ? *reinterpret_cast<const uint32_t *>(src + 16 * kk + 8) : 0u;
          }
        }
      float o[MT][Dh / 8][4];
      float mx[MT][2], ls[MT][2];
#pragma unroll
      for (int mt = 0; mt < MT; mt++) {
        mx[mt][0] = mx[mt][1] = -INFINITY;
        ls[mt][0] = ls[mt][1] = 0.0f;
#pragma unroll
        for (int d = 0; d < Dh / 8; d++) o[mt][d][0] = o[mt][d][1] = o[mt][d][2] = o[mt][d][3] = 0.0f;
      }
      const long long p_last = (long long)w.p + w.n - 1;

      for (int t = t0; t < t1; t++) {
        wait(&full[stage], phase);
        const int key0 = (t < w.a ? t : t - w.a + w.c) * kKeys + warp * 16;  // this warp's 16 keys
        const bool have = held[stage] >> (warp * 16 / A.box_rows) & 1;
        if (have) {
          const uint32_t kaddr = smem_u32(smem) + (uint32_t)stage * S::kStageBytes;
          const uint32_t vaddr = kaddr + S::kTileBytes;
          // every row sees every one of the 16 keys
          const bool open = key0 + 15 <= w.p &&
                            (A.window == 0 || key0 + 15 < A.sinks || (long long)key0 > p_last - A.window);
          bool odd = false;  // some V row that not every row sees holds an infinity or NaN
          if (!open) {
            // V rows that no row of the sequence sees: zeros (their P is 0,
            // and 0 times whatever the page holds there would not be)
            for (int i = lane; i < 16 * (Dh / 8); i += 32) {
              const int kr = i / (Dh / 8), ch = i - kr * (Dh / 8), key = key0 + kr, row = warp * 16 + kr;
              uint8_t *at = smem + (size_t)stage * S::kStageBytes + S::kTileBytes + (ch >> 3) * kBlkBytes +
                            row * 128 + (((ch & 7) ^ (row & 7)) << 4);
              uint4 *v = reinterpret_cast<uint4 *>(at);
              if (key >= w.hi || (key >= w.se && key < w.ws)) {
                *v = make_uint4(0, 0, 0, 0);
              } else {
                const uint4 u = *v;
                odd |= nonfinite2<T>(u.x) || nonfinite2<T>(u.y) || nonfinite2<T>(u.z) || nonfinite2<T>(u.w);
              }
            }
            odd = __any_sync(0xffffffffu, odd);
            __syncwarp();  // the zeros, before the reads below
          }
          // S = Q K^T
          float s[MT][2][4];
#pragma unroll
          for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int nt = 0; nt < 2; nt++) s[mt][nt][0] = s[mt][nt][1] = s[mt][nt][2] = s[mt][nt][3] = 0.0f;
          {
            const int row = warp * 16 + 8 * (jm >> 1) + jr;
#pragma unroll
            for (int kk = 0; kk < Dh / 16; kk++) {
              const int ch = 2 * kk + (jm & 1);
              uint32_t bf[4];
              ldsm4(kaddr + (ch >> 3) * kBlkBytes + row * 128 + (((ch & 7) ^ (row & 7)) << 4), bf);
#pragma unroll
              for (int mt = 0; mt < MT; mt++) {
                mma16816<T>(s[mt][0], qa[mt][kk], bf[0], bf[1]);
                mma16816<T>(s[mt][1], qa[mt][kk], bf[2], bf[3]);
              }
            }
          }
          if (!open) {
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
              for (int nt = 0; nt < 2; nt++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                  const int key = key0 + nt * 8 + 2 * t4 + (e & 1), p = rp[mt][e >> 1];
                  if (key >= w.hi || !sees_key(p, key, A.window, A.sinks)) s[mt][nt][e] = -INFINITY;
                }
          }
          // online softmax; the probabilities as hi + lo halves
          uint32_t ph[MT][4], pl[MT][4];
#pragma unroll
          for (int mt = 0; mt < MT; mt++) {
            float f[2];
#pragma unroll
            for (int e = 0; e < 2; e++) {
              float m = fmaxf(fmaxf(s[mt][0][2 * e], s[mt][0][2 * e + 1]), fmaxf(s[mt][1][2 * e], s[mt][1][2 * e + 1]));
              m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
              m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
              const float mn = fmaxf(mx[mt][e], m * kLog2e);
              f[e] = mn == -INFINITY ? 1.0f : ex2(mx[mt][e] - mn);
              const float sub = mn == -INFINITY ? 0.0f : mn;
              mx[mt][e] = mn;
              float sum = 0.0f;
#pragma unroll
              for (int nt = 0; nt < 2; nt++)
#pragma unroll
                for (int c = 0; c < 2; c++) {
                  const float v = ex2(s[mt][nt][2 * e + c] * kLog2e - sub);
                  s[mt][nt][2 * e + c] = v;
                  sum += v;
                }
              ls[mt][e] = ls[mt][e] * f[e] + sum;
            }
            if (f[0] != 1.0f || f[1] != 1.0f) {
#pragma unroll
              for (int d = 0; d < Dh / 8; d++) {
                o[mt][d][0] *= f[0];
                o[mt][d][1] *= f[0];
                o[mt][d][2] *= f[1];
                o[mt][d][3] *= f[1];
              }
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
              const float v0 = s[mt][i >> 1][2 * (i & 1)], v1 = s[mt][i >> 1][2 * (i & 1) + 1];
              ph[mt][i] = pack2<T>(v0, v1);
              const float2 h = unpack2<T>(ph[mt][i]);
              pl[mt][i] = pack2<T>(v0 - h.x, v1 - h.y);
            }
          }
          // O += P V
          if (!odd) {
            const int row = warp * 16 + 8 * (jm & 1) + jr;
#pragma unroll
            for (int dp = 0; dp < Dh / 16; dp++) {
              const int ch = 2 * dp + (jm >> 1);
              uint32_t bf[4];
              ldsm4_t(vaddr + (ch >> 3) * kBlkBytes + row * 128 + (((ch & 7) ^ (row & 7)) << 4), bf);
#pragma unroll
              for (int mt = 0; mt < MT; mt++) {
                mma16816<T>(o[mt][2 * dp], ph[mt], bf[0], bf[1]);
                mma16816<T>(o[mt][2 * dp], pl[mt], bf[0], bf[1]);
                mma16816<T>(o[mt][2 * dp + 1], ph[mt], bf[2], bf[3]);
                mma16816<T>(o[mt][2 * dp + 1], pl[mt], bf[2], bf[3]);
              }
            }
          } else {
            // one key at a time, for the rows that see it
            for (int kr = 0; kr < 16; kr++) {
              const int key = key0 + kr, row = warp * 16 + kr, src = (lane & ~3) | ((kr & 7) >> 1);
#pragma unroll
              for (int mt = 0; mt < MT; mt++) {
                float pv[2];
                bool see[2];
#pragma unroll
                for (int e = 0; e < 2; e++) {
                  const float lo = kr < 8 ? s[mt][0][2 * e] : s[mt][1][2 * e];
                  const float hi = kr < 8 ? s[mt][0][2 * e + 1] : s[mt][1][2 * e + 1];
                  pv[e] = __shfl_sync(0xffffffffu, kr & 1 ? hi : lo, src);
                  const int p = rp[mt][e];
                  see[e] = key < w.hi && sees_key(p, key, A.window, A.sinks);
                }
#pragma unroll
                for (int d = 0; d < Dh / 8; d++) {
                  const uint32_t u = *reinterpret_cast<const uint32_t *>(
                      smem + (size_t)stage * S::kStageBytes + S::kTileBytes + (d >> 3) * kBlkBytes + row * 128 +
                      (((d & 7) ^ (row & 7)) << 4) + 4 * t4);
                  const float2 v = unpack2<T>(u);
                  if (see[0]) {
                    o[mt][d][0] += pv[0] * v.x;
                    o[mt][d][1] += pv[0] * v.y;
                  }
                  if (see[1]) {
                    o[mt][d][2] += pv[1] * v.x;
                    o[mt][d][3] += pv[1] * v.y;
                  }
                }
              }
            }
          }
          if (!open) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the zeros, before the next copy
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[stage]);
        advance();
      }

      // ---- the warps' shares together ----
      auto sync = [&]() { asm volatile("bar.sync 1, %0;" ::"n"(kSplitWarps * 32) : "memory"); };
#pragma unroll
      for (int mt = 0; mt < MT; mt++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          float l = ls[mt][e];
          l += __shfl_xor_sync(0xffffffffu, l, 1);
          l += __shfl_xor_sync(0xffffffffu, l, 2);
          if (t4 == 0) {
            sm_m[warp * S::kRows + mt * 16 + g + 8 * e] = mx[mt][e];
            sm_l[warp * S::kRows + mt * 16 + g + 8 * e] = l;
          }
        }
      sync();
#pragma unroll
      for (int mt = 0; mt < MT; mt++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const int row = mt * 16 + g + 8 * e;
          float m = -INFINITY;
#pragma unroll
          for (int i = 0; i < kSplitWarps; i++) m = fmaxf(m, sm_m[i * S::kRows + row]);
          const float f = m == -INFINITY ? 0.0f : ex2(mx[mt][e] - m);
#pragma unroll
          for (int d = 0; d < Dh / 8; d++) {
            o[mt][d][2 * e] *= f;
            o[mt][d][2 * e + 1] *= f;
          }
        }
      auto put = [&](float *dst) {
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
          for (int d = 0; d < Dh / 8; d++)
#pragma unroll
            for (int e = 0; e < 2; e++)
              *reinterpret_cast<float2 *>(dst + (mt * 16 + g + 8 * e) * Dh + d * 8 + 2 * t4) =
                  make_float2(o[mt][d][2 * e], o[mt][d][2 * e + 1]);
      };
      if (warp >= 2) put(red + (warp - 2) * S::kRows * Dh);
      sync();
      if (warp < 2) {
        float *mine = red + warp * S::kRows * Dh;
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
          for (int d = 0; d < Dh / 8; d++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
              float2 *at = reinterpret_cast<float2 *>(mine + (mt * 16 + g + 8 * e) * Dh + d * 8 + 2 * t4);
              float2 v = *at;
              v.x += o[mt][d][2 * e];
              v.y += o[mt][d][2 * e + 1];
              *at = v;
            }
      }
      sync();
      const bool whole = t0 == 0 && t1 == w.nt;
      const int slot = 2 * cta + (pos == start ? 0 : 1);
      float *part = A.part + (size_t)slot * S::kRows * (Dh + 2);
      for (int i = tid; i < S::kRows * (Dh / 4); i += kSplitWarps * 32) {
        const int row = i / (Dh / 4), d = (i - row * (Dh / 4)) * 4, m = m0 + row, qi = m / A.G;
        if (qi >= w.n) continue;
        float mm = -INFINITY, l = 0.0f;
#pragma unroll
        for (int k = 0; k < kSplitWarps; k++) mm = fmaxf(mm, sm_m[k * S::kRows + row]);
#pragma unroll
        for (int k = 0; k < kSplitWarps; k++)
          l += mm == -INFINITY ? 0.0f : sm_l[k * S::kRows + row] * ex2(sm_m[k * S::kRows + row] - mm);
        const float4 x = *reinterpret_cast<const float4 *>(red + row * Dh + d);
        const float4 y = *reinterpret_cast<const float4 *>(red + (S::kRows + row) * Dh + d);
        float4 v = make_float4(x.x + y.x, x.y + y.y, x.z + y.z, x.w + y.w);
        if (whole) {
          const float inv = mm == -INFINITY ? 0.0f : 1.0f / l;
          uint2 u;
          u.x = pack2<T>(v.x * inv, v.y * inv);
          u.y = pack2<T>(v.z * inv, v.w * inv);
          *reinterpret_cast<uint2 *>(reinterpret_cast<T *>(A.out) +
                                     ((size_t)(w.r0 + qi) * A.H + hk * A.G + (m - qi * A.G)) * Dh + d) = u;
        } else {
          *reinterpret_cast<float4 *>(part + 2 * S::kRows + row * Dh + d) = v;
          if (d == 0) {
            part[row] = mm;
            part[S::kRows + row] = l;
          }
        }
      }
      if (t0 == 0 && !whole) {  // this CTA begins a unit that others finish
        const int last_cta = (base + (unit + 1) * w.nt - 1) / per;
        rec_parts = last_cta - cta + 1;
        rec[0] = slot;
        rec[1] = w.r0;
        rec[2] = w.n;
        rec[3] = hk;
        rec[4] = m0;
      }
      sync();  // red and sm_m / sm_l are free again
      pos += t1 - t0;
    }
    if (tid == 0) {
      int *r = A.rec + cta * 8;
      r[0] = rec_parts;
#pragma unroll
      for (int i = 0; i < 5; i++) r[1 + i] = rec[i];
    }
  }
}

// The sums of a unit that several CTAs share: block (c, row) joins row `row` of
// the unit that begins in CTA c, its parts in CTA order. 512 threads: groups of
// Dh / 4 threads take every n-th part.
constexpr int kJoinThreads = 512;

template <typename T, int Dh>
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(const int *recs, const float *parts, int unit_rows,
                                                                  int H, int G, T *out) {
  constexpr int kLanes = Dh / 4, kGroups = kJoinThreads / kLanes;
  __shared__ float4 acc[kGroups][kLanes];
  __shared__ float warp_m[kJoinThreads / 32], lsum[kGroups];
  pdl_trigger();
  pdl_wait();
  const int *rec = recs + blockIdx.x * 8;
  const int np = rec[0];
  if (np == 0) return;
  const int slot = rec[1], r0 = rec[2], n = rec[3], hk = rec[4], m0 = rec[5], row = (int)blockIdx.y;
  const int m = m0 + row, qi = m / G;
  if (qi >= n) return;
  const int tid = threadIdx.x, lane = tid % kLanes, grp = tid / kLanes;
  const size_t stride = (size_t)unit_rows * (Dh + 2);
  // part j: the first in `slot`, then the first slots of the CTAs that follow
  auto part = [&](int j) { return parts + (j == 0 ? (size_t)slot : (size_t)2 * (blockIdx.x + j)) * stride; };
  float mm = -INFINITY;
  for (int j = tid; j < np; j += kJoinThreads) mm = fmaxf(mm, part(j)[row]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, o));
  if ((tid & 31) == 0) warp_m[tid >> 5] = mm;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kJoinThreads / 32; i++) mm = fmaxf(mm, warp_m[i]);
  float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float l = 0.0f;
#pragma unroll 4
  for (int j = grp; j < np; j += kGroups) {
    const float *p = part(j);
    const float f = mm == -INFINITY ? 0.0f : ex2(p[row] - mm);
    const float4 v = *reinterpret_cast<const float4 *>(p + 2 * unit_rows + (size_t)row * Dh + lane * 4);
    a.x += v.x * f;
    a.y += v.y * f;
    a.z += v.z * f;
    a.w += v.w * f;
    l += p[unit_rows + row] * f;
  }
  acc[grp][lane] = a;
  if (lane == 0) lsum[grp] = l;
  __syncthreads();
  if (grp == 0) {
#pragma unroll
    for (int i = 1; i < kGroups; i++) {
      const float4 v = acc[i][lane];
      a.x += v.x;
      a.y += v.y;
      a.z += v.z;
      a.w += v.w;
      l += lsum[i];
    }
    const float inv = mm == -INFINITY ? 0.0f : 1.0f / l;
    uint2 u;
    u.x = pack2<T>(a.x * inv, a.y * inv);
    u.y = pack2<T>(a.z * inv, a.w * inv);
    *reinterpret_cast<uint2 *>(out + ((size_t)(r0 + qi) * H + hk * G + (m - qi * G)) * Dh + lane * 4) = u;
  }
}

int64_t stride_or(int64_t s, int64_t dense) { return s ? s : dense; }

template <typename T, int Dh>
cudaError_t rope_t(const float *qkv, const PagedRows &pr, int H, int Hkv, const RopeTurns &turns, const float *q_norm,
                   const float *k_norm, float eps, void *q_out, const wg_paged_kv &kv, unsigned *flags, int num_sms,
                   cudaStream_t s, bool pdl) {
  const int NH = H + 2 * Hkv;
  // heads a warp takes: few rows, one (or the two that share a warp) for the
  // shortest path; many, up to 8, which share the row's sines
  const int least = Dh == 64 ? 2 : 1;
  int hpw = least;
  while (hpw < 8 && (long long)pr.rows * ((NH + hpw - 1) / hpw) > (long long)num_sms * 64) hpw *= 2;
  const int wpr = (NH + hpw - 1) / hpw;
  const long long warps = (long long)pr.rows * wpr;
  const PagedTable pt{kv.table, kv.max_pages, kv.num_pages, kv.page_size};
  const int64_t rs = stride_or(kv.row_stride, Dh), hs = stride_or(kv.head_stride, (int64_t)kv.page_size * Dh),
                ps = stride_or(kv.page_stride, (int64_t)Hkv * kv.page_size * Dh);
  const int threads = warps <= num_sms * 4 ? 64 : 256;
  const unsigned blocks = (unsigned)((warps * 32 + threads - 1) / threads);
  return launch_pdl(paged_rope_kernel<T, Dh>, dim3(blocks), threads, 0, s, pdl, qkv, pr, H, Hkv, turns, q_norm, k_norm, eps,
                reinterpret_cast<T *>(q_out), reinterpret_cast<T *>(kv.k), reinterpret_cast<T *>(kv.v), ps, hs, rs, pt,
                hpw, wpr, flags);
}

constexpr int split_ctas_per_sm(int Dh, int MT) { return MT == 1 && Dh <= 128 ? 2 : 1; }
constexpr int kSplitSmemPerSm = 224 * 1024;

template <typename T, int Dh, int MT>
cudaError_t split_t(SplitArgs A, const wg_paged_kv &kv, void *workspace, int num_sms, cudaStream_t s, bool pdl) {
  using S = SplitSmem<T, Dh, MT>;
  const int occ = split_ctas_per_sm(Dh, MT);
  const int budget = kSplitSmemPerSm / occ - 1024;
  A.stages = (budget - S::kFixed) / S::kStageBytes;
  if (A.stages > kMaxStages) A.stages = kMaxStages;
  static_assert((kSplitSmemPerSm / split_ctas_per_sm(Dh, MT) - 1024 - S::kFixed) / S::kStageBytes >= 2, "two stages");
  const size_t smem = (size_t)A.stages * S::kStageBytes + S::kFixed;
  auto kern = paged_split_kernel<T, Dh, MT>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  CUtensorMap tk, tv;
  if (!page_map(&tk, kv.k, kv, A.Hkv, Dh, A.box_rows) || !page_map(&tv, kv.v, kv, A.Hkv, Dh, A.box_rows))
    return cudaErrorInvalidValue;
  const int P = num_sms * occ;
  A.rec = reinterpret_cast<int *>(workspace);
  A.part = reinterpret_cast<float *>(A.rec + (size_t)P * 8);
  e = launch_pdl(kern, dim3((unsigned)P), kSplitThreads, smem, s, pdl, tk, tv, A);
  if (e != cudaSuccess) return e;
  // rows of a unit that can exist: none past the longest sequence's
  const long long most = A.pr.row_start ? A.pr.rows : A.pr.rows / A.pr.batch;
  const unsigned rows = (unsigned)(most * A.G < S::kRows ? most * A.G : S::kRows);
  return launch_pdl(paged_join_kernel<T, Dh>, dim3((unsigned)P, rows), kJoinThreads, 0, s, pdl, A.rec, A.part, S::kRows,
                A.H, A.G, reinterpret_cast<T *>(A.out));
}

template <typename T>
cudaError_t split_d(const SplitArgs &A, int Dh, const wg_paged_kv &kv, void *ws, int num_sms, cudaStream_t s,
                    bool pdl) {
  // 32 query rows a CTA where the sequences have more than 16 (their keys
  // are then read once instead of twice)
  const long long m = (long long)A.pr.rows / A.pr.batch * A.G;
  if (Dh == 64)
    return m > 16 ? split_t<T, 64, 2>(A, kv, ws, num_sms, s, pdl) : split_t<T, 64, 1>(A, kv, ws, num_sms, s, pdl);
  if (Dh == 128)
    return m > 16 ? split_t<T, 128, 2>(A, kv, ws, num_sms, s, pdl) : split_t<T, 128, 1>(A, kv, ws, num_sms, s, pdl);
  return split_t<T, 256, 1>(A, kv, ws, num_sms, s, pdl);
}

}  // namespace

cudaError_t launch_paged_rope_kv(const float *qkv, const PagedRows &rows, int H, int Hkv, int Dh, double theta,
                                 const float *q_norm, const float *k_norm, float eps, void *q_out,
                                 const wg_paged_kv &kv, unsigned *flags, int num_sms, cudaStream_t s, bool pdl) {
  // theta^(-2j/Dh) / 2 pi by repeated products in extended precision (at
  // most 127 roundings of 2^-64 each)
  RopeTurns t;
  const long double step = powl((long double)theta, -2.0L / Dh);
  long double f = 0.159154943091895335768883763372514362L;
  for (int j = 0; j < Dh / 2; j++) {
    t.t[j] = (double)f;
    f *= step;
  }
  for (int j = Dh / 2; j < 128; j++) t.t[j] = 0.0;
#define WG_ROPE(T, D) \
  return rope_t<T, D>(qkv, rows, H, Hkv, t, q_norm, k_norm, eps, q_out, kv, flags, num_sms, s, pdl)
  if (kv.dtype == WG_F16) {
    if (Dh == 64) WG_ROPE(__half, 64);
    if (Dh == 128) WG_ROPE(__half, 128);
    WG_ROPE(__half, 256);
  }
  if (Dh == 64) WG_ROPE(__nv_bfloat16, 64);
  if (Dh == 128) WG_ROPE(__nv_bfloat16, 128);
  WG_ROPE(__nv_bfloat16, 256);
#undef WG_ROPE
}

size_t paged_attention_workspace(int Dh, int num_sms) {
  // the larger of the 16-row and the 32-row kernels' needs
  size_t most = 0;
  for (int mt = 1; mt <= 2; mt++) {
    const size_t P = (size_t)num_sms * split_ctas_per_sm(Dh, mt);
    const size_t need = P * 8 * sizeof(int) + 2 * P * (16 * mt) * (size_t)(Dh + 2) * sizeof(float);
    if (need > most) most = need;
  }
  return most;
}

cudaError_t launch_paged_attention(const void *q, const PagedRows &rows, int H, int Hkv, int Dh,
                                   const wg_paged_kv &kv, int window, int sinks, void *out, void *workspace,
                                   unsigned *flags, int num_sms, cudaStream_t s, bool pdl) {
  if (paged_prompt_supported(rows, H, Hkv, num_sms))
    return launch_paged_prompt(q, rows, H, Hkv, Dh, kv, window, sinks, out, flags, num_sms, s, pdl);
  SplitArgs A{};
  A.pr = rows;
  A.pt = PagedTable{kv.table, kv.max_pages, kv.num_pages, kv.page_size};
  A.q = q;
  A.out = out;
  A.H = H;
  A.Hkv = Hkv;
  A.G = H / Hkv;
  A.window = window;
  A.sinks = sinks;
  A.box_rows = kv.page_size % 64 == 0 ? 64 : kv.page_size % 32 == 0 ? 32 : 16;
  A.flags = flags;
  return kv.dtype == WG_F16 ? split_d<__half>(A, Dh, kv, workspace, num_sms, s, pdl)
                            : split_d<__nv_bfloat16>(A, Dh, kv, workspace, num_sms, s, pdl);
}

}  // namespace wg
