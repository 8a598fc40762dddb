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
// A warp takes one row and up to `heads_per_warp` (16) of its H + 2 Hkv heads: lane
// l holds the rotate-half pairs (j, j + Dh/2) of four neighbouring j, so that a
// head is two 16-byte loads and two 8-byte stores of Dh / 8 lanes, 1 to 4 heads
// share a warp, 4 to 8 heads are in flight, and the row's sequence, page and
// sines are found once for all the warp's heads, behind the first loads. The
// angle of pair j at position p, in turns, is p theta^(-2j/Dh) / 2 pi: its
// factor comes from the host in 64 bits and the whole turns are taken off in 64
// bits (one product, one rounding, one difference), so that the fp32 sine sees
// an argument in [-1, 1] half turns, exact at any position. Bound by its bytes
// for prompts and by launch latency for decode rows: 16 sequences of up to 512
// rows of 40 heads of 64 take 14.9 us from HBM, 4.1 TB/s with the ramps of one
// launch in it (17.5 in blocks of 256 threads, 32 heads a warp and with loads that
// stay in L2, 15.7 with 8 heads a warp); 8 decode rows 2.5 us.

struct RopeTurns {
  double t[128];  // theta^(-2j/Dh) / (2 pi)
};

template <typename T, int Dh>
__global__ void __launch_bounds__(64)
    paged_rope_kernel(const float *qkv, const PagedRows pr, int H, int Hkv, const RopeTurns turns,
                      const float *q_norm, const float *k_norm, float eps, T *q_out, T *k_pages, T *v_pages,
                      int64_t page_stride, int64_t head_stride, int64_t row_stride, const PagedTable pt,
                      int heads_per_warp, int warps_per_row, unsigned *flags) {
  pdl_trigger();
  pdl_wait();
  constexpr int kLanes = Dh / 8, kHeads = 32 / kLanes;  // lanes of a head, heads at once
  constexpr int kSets = Dh == 64 ? 2 : 4;                // times kHeads heads in flight
  const int lane = threadIdx.x & 31;
  const unsigned w = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);  // (the launcher keeps it in 32 bits)
  const int r = (int)(w / (unsigned)warps_per_row);
  if (r >= pr.rows) return;
  const int j0 = (lane % kLanes) * 4, sub = lane / kLanes;
  const int NH = H + 2 * Hkv;
  const int h0 = (int)(w - (unsigned)r * warps_per_row) * heads_per_warp, h1 = min(h0 + heads_per_warp, NH);
  float x[kSets][4], y[kSets][4];  // dims j0 + i and j0 + i + Dh / 2
  auto load = [&](int hh) {
#pragma unroll
    for (int e = 0; e < kSets; e++) {
      const int h = hh + e * kHeads + sub;
      float4 u = make_float4(0.0f, 0.0f, 0.0f, 0.0f), v = u;
      if (h < h1) {
        const float *src = qkv + ((size_t)r * NH + h) * Dh + j0;
        u = __ldcs(reinterpret_cast<const float4 *>(src));  // read once
        v = __ldcs(reinterpret_cast<const float4 *>(src + Dh / 2));
      }
      x[e][0] = u.x, x[e][1] = u.y, x[e][2] = u.z, x[e][3] = u.w;
      y[e][0] = v.x, y[e][1] = v.y, y[e][2] = v.z, y[e][3] = v.w;
    }
  };
  load(h0);  // on its way while the row finds its sequence, page and angles
  const int b = row_seq(pr, r, lane);
  if (b < 0) return;
  int r0, n;
  seq_rows(pr, b, r0, n);
  const long long p = (long long)pr.pos[b] + (r - r0);
  float cs[4], sn[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const double t = (double)p * turns.t[j0 + i];
    sincospif((float)(2.0 * (t - rint(t))), &sn[i], &cs[i]);
  }
  // the row's place in the cache
  const long long cap = (long long)pt.max_pages * pt.page_size;
  long long place = -1;
  if (p >= 0) {
    int page = -1;
    const unsigned slot = p < cap ? (unsigned)p / (unsigned)pt.page_size : 0;  // (cap fits an int)
    if (p < cap) page = pt.table[(size_t)b * pt.max_pages + slot];
    if (page >= 0 && page < pt.num_pages)
      place = page * (long long)page_stride + (int)((unsigned)p - slot * pt.page_size) * (long long)row_stride;
    else if (lane == 0)
      raise_flag(flags, kFlagBadArgument);
  }
  const float scale = rsqrtf((float)Dh);
  for (int hh = h0; hh < h1; hh += kSets * kHeads) {
    if (hh > h0) load(hh);
#pragma unroll
    for (int e = 0; e < kSets; e++) {
      const int h = hh + e * kHeads + sub;
      if (hh + e * kHeads >= h1) break;
      const bool is_q = h < H, is_v = h >= H + Hkv;
      if (q_norm || k_norm) {  // the whole warp: a head's lanes sum its squares
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; i++) ss += x[e][i] * x[e][i] + y[e][i] * y[e][i];
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float *nw = is_q ? q_norm : is_v ? nullptr : k_norm;
        if (nw) {
          const float inv = rsqrtf(ss / (float)Dh + eps);
#pragma unroll
          for (int i = 0; i < 4; i++) {
            x[e][i] *= inv * nw[j0 + i];
            y[e][i] *= inv * nw[j0 + Dh / 2 + i];
          }
        }
      }
      if (h >= h1) continue;
      if (!is_v) {
        const float sc = is_q ? scale : 1.0f;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float a = x[e][i], c = y[e][i];
          x[e][i] = (a * cs[i] - c * sn[i]) * sc;
          y[e][i] = (c * cs[i] + a * sn[i]) * sc;
        }
      }
      T *dst;
      if (is_q) {
        dst = q_out + ((size_t)r * H + h) * Dh;
        if (p < 0) {
#pragma unroll
          for (int i = 0; i < 4; i++) x[e][i] = y[e][i] = 0.0f;
        }
      } else {
        if (place < 0) continue;
        const int hk = is_v ? h - H - Hkv : h - H;
        dst = (is_v ? v_pages : k_pages) + place + hk * head_stride;
      }
      dst += j0;
      *reinterpret_cast<uint2 *>(dst) = make_uint2(pack2<T>(x[e][0], x[e][1]), pack2<T>(x[e][2], x[e][3]));
      *reinterpret_cast<uint2 *>(dst + Dh / 2) = make_uint2(pack2<T>(y[e][0], y[e][1]), pack2<T>(y[e][2], y[e][3]));
    }
  }
}

// ---- attention, split over the keys ---------------------------------------
// o = softmax(q k^T) v per (sequence, KV head, 16 MT rows of queries), where
// the sequence's rows times the G query heads of the KV head are the rows of
// one small matrix product: a K / V tile is read once for all of them. Decode
// is bound by those reads, so the work is counted in tiles of 4 KW keys over
// all sequences and heads and each of P resident CTAs takes an equal run of
// tiles, wherever sequences begin and end in it: short and long sequences
// share the machine evenly whatever their lengths, which only the device
// knows. Per CTA:
//   the last warp   the producer: page entries, then one TMA copy per box of a
//                   page's rows x 64 dims (128-byte swizzle) into a ring of
//                   stages (K and V of a tile each);
//   4 MT warps      KW keys of a tile and 16 of the query rows each: S = Q K^T
//                   and O += P V on mma.m16n8k16 with fp32 sums, a running
//                   maximum and sum per row in registers (log2 domain). The
//                   warps meet only at the end of a run of tiles. A tile's chain
//                   (wait, scores, maximum, exponentials, P V) takes a warp
//                   about 2000 cycles whatever KW is, so small heads take 32
//                   keys at a time (Dh = 64, 32 sequences with a window of 4096:
//                   59 us with 16 keys, 53 with 32), and 32 query rows
//                   take eight warps (five rows of 4 heads, 8 sequences of 4k:
//                   52 us with four warps of both row tiles, 39 with eight).
// P is hi + lo 16-bit halves, two products (the tensor pipe idles under the
// loads): off by up to 2^-17 of itself in bf16. In fp16 by 2^-23, down to 2^-2;
// below that what is rounded off is 2^-25, so P is lifted by 2^14 against keys far
// below the maximum (a first token with a high score above thousands of others):
// 2^-39 of the largest. The sums carry the same factor, the quotient does not.
// 2^14 leaves two octaves below 65504 for a reference that is rounded (scores up
// to 2^24).
// A (sequence, head, rows) unit that one CTA finishes alone is written by it;
// else each CTA leaves (max, sum, O) in the workspace and paged_join_kernel
// adds them in order: no atomics, the same bits every time.

constexpr int kMaxStages = 8;
// A CTA takes at least this many keys, or one tile.
constexpr int kMinKeys = 64;

struct SplitArgs {
  PagedRows pr;
  PagedTable pt;
  const void *q;
  void *out;
  int H, Hkv, G;
  int window, sinks;
  int box_rows;  // keys of one TMA box: divides page_size and the tile
  int stages;
  int whole;     // units are not split: a CTA takes whole ones
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

__device__ __forceinline__ SeqWork seq_work(const SplitArgs &A, int b, int rows_per_tile, int tile_keys) {
  SeqWork w;
  seq_rows(A.pr, b, w.r0, w.n);
  w.p = A.pr.pos[b];
  w.mt = (int)(((long long)w.n * A.G + rows_per_tile - 1) / rows_per_tile);
  static_cast<KeySpan &>(w) = key_span(w.p, w.n, A.window, A.sinks, A.pt, tile_keys);
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

template <int Dh_, int MT>
struct SplitCfg {
  static constexpr int Dh = Dh_;
  static constexpr int KW = Dh == 64 ? 32 : 16;    // keys of a warp
  static constexpr int kKeys = 4 * KW;             // of a tile
  static constexpr int kRows = 16 * MT;
  static constexpr int kWhole = Dh == 256 ? 3 : 4;  // tiles up to which a unit is not split
  static constexpr int kWarps = 4 * MT;            // consumers
  static constexpr int kThreads = (kWarps + 1) * 32;
  static constexpr int kCtas = MT == 1 && Dh <= 128 ? 2 : 1;  // per SM
  // With eight consumer warps the queries' fragments are read from shared memory
  // with each tile: in registers too they spill (verify rows: 39 us, so 36).
  static constexpr bool kQSmem = MT == 2;
  static constexpr int kQRow = Dh + 8;
  static constexpr int kQBytes = kQSmem ? kRows * kQRow * 2 : 0;
  static constexpr int kTileBytes = kKeys * Dh * 2;  // K or V of a stage
  static constexpr int kStageBytes = 2 * kTileBytes;
  // The warps' merge: two sets of the rows' sums, 8 floats between rows (the 8
  // rows a warp writes at once then meet in 2 bank rounds instead of 8). The
  // same memory stages the queries, and P where a V row is odd.
  static constexpr int kRedRow = Dh + 8;
  static constexpr int kRedBytes = 2 * kRows * kRedRow * 4;
  static constexpr int kFixed = 1024 /* alignment */ + kRedBytes + kQBytes + 4 * 4 * kRows * 2 + 256;
  static constexpr int kBudget = 224 * 1024 / kCtas - 1024;
  static constexpr int kFit = (kBudget - kFixed) / kStageBytes;
  static constexpr int kStages = kFit > kMaxStages ? kMaxStages : kFit;
  static constexpr int kSmem = kStages * kStageBytes + kFixed;
  static_assert(kStages >= 2, "two stages");
  static_assert(kRedBytes >= kWarps * 16 * KW * 4 && kRedBytes >= kRows * (Dh + 8) * 2, "the merge buffer's other uses");
};

template <typename T, int Dh, int MT>
__global__ void __launch_bounds__(SplitCfg<Dh, MT>::kThreads, SplitCfg<Dh, MT>::kCtas)
    paged_split_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                       const SplitArgs A) {
  using C = SplitCfg<Dh, MT>;
  constexpr int KW = C::KW, kKeys = C::kKeys, S = C::kStages;
  constexpr int kBlk = Dh / 64;                    // 64-dim blocks of a row
  constexpr int kBlkBytes = kKeys * 128;           // one block of a stage's K or V
  constexpr float kLog2e = 1.4426950408889634f;
  constexpr float kLift = std::is_same<T, __half>::value ? 14.0f : 0.0f;  // P is 2^kLift at the maximum
  extern __shared__ __align__(16) uint8_t smem_raw[];
  uint8_t *smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  float *red = reinterpret_cast<float *>(smem + (size_t)S * C::kStageBytes);  // [2][kRows][kRedRow]
  float *sm_m = red + 2 * C::kRows * C::kRedRow;           // [4 key groups][kRows]
  float *sm_l = sm_m + 4 * C::kRows;
  T *sq = reinterpret_cast<T *>(C::kQSmem ? sm_l + 4 * C::kRows : red);  // [kRows][kQRow]
  __shared__ uint64_t full[S], empty[S];
  __shared__ int held[S];                          // which 16-key groups of a stage's pages were loaded
  __shared__ int scan_red[C::kThreads / 32];
  __shared__ int s_b, s_base, aborted;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int P = (int)gridDim.x, cta = (int)blockIdx.x;

  if (tid == 0) {
    for (int i = 0; i < S; i++) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], C::kWarps);
    }
    fence_mbar_init();
    aborted = 0;
    s_b = A.pr.batch;
    s_base = 0;
  }
  if (warp == C::kWarps && lane == 0) {
    prefetch_tensormap(&tm_k);
    prefetch_tensormap(&tm_v);
  }
  pdl_trigger();
  pdl_wait();  // rows, positions, pages and queries come from earlier kernels
  __syncthreads();

  // the total work, then where this CTA's run begins: by every warp itself for
  // up to 32 sequences, else by the CTA, in passes of a thread a sequence
  int total = 0, b = A.pr.batch, base = 0, per, start, end;
  auto share = [&]() {
    per = max((total + P - 1) / P, A.whole ? 1 : max(1, kMinKeys / kKeys));
    start = (int)min((long long)total, (long long)cta * per);
    end = (int)min((long long)total, (long long)start + per);
  };
  auto work_of = [&](int i) {
    if (i >= A.pr.batch) return 0;
    const SeqWork w = seq_work(A, i, C::kRows, kKeys);
    return A.Hkv * w.mt * (A.whole ? 1 : w.nt);
  };
  if (A.pr.batch <= 32) {
    const int v = work_of(lane);
    int incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += t;
    }
    total = __shfl_sync(0xffffffffu, incl, 31);
    share();
    const unsigned at = __ballot_sync(0xffffffffu, incl - v <= start && start < incl);
    if (at) {
      b = __ffs(at) - 1;
      base = __shfl_sync(0xffffffffu, incl - v, b);
    }
  } else {
    int v = 0, incl = 0, t;
    for (int b0 = 0; b0 < A.pr.batch; b0 += C::kThreads) {
      v = work_of(b0 + tid);
      incl = block_scan_incl(v, scan_red, t);
      total += t;
    }
    share();
    for (int b0 = 0, run = 0; b0 < A.pr.batch && run <= start; b0 += C::kThreads) {
      if (A.pr.batch > C::kThreads) {
        v = work_of(b0 + tid);
        incl = run + block_scan_incl(v, scan_red, t);
      }
      if (incl - v <= start && start < incl) {
        s_b = b0 + tid;
        s_base = incl - v;
      }
      run += t;
    }
    __syncthreads();
    b = s_b;
    base = s_base;
  }

  auto wait = [&](uint64_t *bar, uint32_t parity) {
    if (mbar_try_wait(bar, parity) || *(volatile int *)&aborted) return;
    if (!mbar_wait_bounded(bar, parity, A.flags)) *(volatile int *)&aborted = 1;
  };
  int stage = 0, phase = 0;
  auto advance = [&]() {
    if (++stage == S) {
      stage = 0;
      phase ^= 1;
    }
  };

  if (warp == C::kWarps) {
    // ---- producer ----
    const int nb = kKeys / A.box_rows;  // boxes per tile
    const int nops = nb * kBlk * 2;
    const int box = lane % nb, blk = (lane / nb) % kBlk, is_v = lane / (nb * kBlk);
    const uint32_t box_bytes = (uint32_t)A.box_rows * 128;
    const int groups = A.box_rows / 16, gmask = (1 << groups) - 1;
    for (int pos = start; pos < end;) {
      const SeqWork w = seq_work(A, b, C::kRows, kKeys);
      const int steps = A.whole ? 1 : w.nt, work = A.Hkv * w.mt * steps;
      if (pos >= base + work) {
        base += work;
        b++;
        continue;
      }
      const int unit = (pos - base) / steps, t0 = (pos - base) - unit * steps;
      const int t1 = A.whole ? w.nt : min(w.nt, t0 + (end - pos));
      const int hk = unit / w.mt;
      const int32_t *row = A.pt.table + (size_t)b * A.pt.max_pages;
      // the box's page entry and whether any row sees a key of it
      auto entry = [&](int t, int &key, bool &seen) {
        key = (t < w.a ? t : t - w.a + w.c) * kKeys + box * A.box_rows;
        seen = lane < nops && key < w.hi && (key < w.se || key + A.box_rows > w.ws);
        return seen ? row[key / A.pt.page_size] : -1;
      };
      int key, key_next = 0;
      bool seen, seen_next = false;
      int page = entry(t0, key, seen), page_next = -1;
      for (int t = t0; t < t1; t++) {
        if (t + 1 < t1) page_next = entry(t + 1, key_next, seen_next);
        wait(&empty[stage], phase ^ 1);
        const bool ok = seen && page >= 0 && page < A.pt.num_pages;
        if (seen && !ok) raise_flag(A.flags, kFlagBadArgument);
        const unsigned loaded = __ballot_sync(0xffffffffu, ok && lane < nb);
        if (lane == 0) {
          int m = 0;
          for (int i = 0; i < nb; i++)
            if (loaded >> i & 1) m |= gmask << (i * groups);
          held[stage] = m;
          mbar_expect_tx(&full[stage], (uint32_t)__popc(loaded) * box_bytes * kBlk * 2);
        }
        __syncwarp();
        if (ok)
          tma_load_4d(smem + (size_t)stage * C::kStageBytes + is_v * C::kTileBytes + blk * kBlkBytes + box * box_bytes,
                      is_v ? &tm_v : &tm_k, blk * 64, key % A.pt.page_size, hk, page, &full[stage]);
        page = page_next;
        key = key_next;
        seen = seen_next;
        advance();
      }
      pos += A.whole ? 1 : t1 - t0;
    }
    // after a wait that ran out, no copy may still be on its way into this
    // CTA's memory when it exits
    __syncwarp();
    if (*(volatile int *)&aborted && lane == 0)
      for (int i = 0; i < S; i++) {
        mbar_wait_bounded(&full[stage], phase ^ 1, A.flags);
        advance();
      }
  } else {
    // ---- consumers ----
    const int wk = warp & 3, wr = warp >> 2;  // this warp's keys and rows
    const int g = lane >> 2, t4 = lane & 3;
    const int jm = lane >> 3, jr = lane & 7;  // ldmatrix: this lane addresses row jr of matrix jm
    int rec_parts = 0;
    int rec[5] = {0, 0, 0, 0, 0};
    for (int pos = start; pos < end;) {
      const SeqWork w = seq_work(A, b, C::kRows, kKeys);
      const int steps = A.whole ? 1 : w.nt, work = A.Hkv * w.mt * steps;
      if (pos >= base + work) {
        base += work;
        b++;
        continue;
      }
      const int unit = (pos - base) / steps, t0 = (pos - base) - unit * steps;
      const int t1 = A.whole ? w.nt : min(w.nt, t0 + (end - pos));
      const int hk = unit / w.mt, m0 = (unit - hk * w.mt) * C::kRows;

      // queries, 16 bytes a load, through the merge buffer into A fragments; the
      // position of each of this thread's rows
      auto sync = [&]() { asm volatile("bar.sync 1, %0;" ::"n"(C::kWarps * 32) : "memory"); };
      for (int i = tid; i < C::kRows * (Dh / 8); i += C::kWarps * 32) {
        const int row = i / (Dh / 8), ch = i - row * (Dh / 8), m = m0 + row, qi = m / A.G;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (qi < w.n)
          v = __ldg(reinterpret_cast<const uint4 *>(reinterpret_cast<const T *>(A.q) +
                                                    ((size_t)(w.r0 + qi) * A.H + hk * A.G + (m - qi * A.G)) * Dh) +
                    ch);
        *reinterpret_cast<uint4 *>(sq + row * C::kQRow + ch * 8) = v;
      }
      int rp[2];
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const int i = (m0 + wr * 16 + g + 8 * e) / A.G;
        rp[e] = (int)max(-1LL, min(i < w.n ? (long long)w.p + i : -1LL, 0x7ffffffeLL));
      }
      sync();
      const uint32_t q_at = smem_u32(sq + (wr * 16 + (jm & 1) * 8 + jr) * C::kQRow + (jm >> 1) * 8);
      uint32_t qa[C::kQSmem ? 1 : Dh / 16][4];
      if constexpr (!C::kQSmem) {
#pragma unroll
        for (int kk = 0; kk < Dh / 16; kk++) ldsm4(q_at + kk * 32, qa[kk]);
        sync();  // the buffer is free again
      }
      float o[Dh / 8][4];
      float mx[2] = {-INFINITY, -INFINITY}, ls[2] = {0.0f, 0.0f};
#pragma unroll
      for (int d = 0; d < Dh / 8; d++) o[d][0] = o[d][1] = o[d][2] = o[d][3] = 0.0f;
      // keys that every row sees: up to open_to, and from open_from on or sinks
      const int open_to = (int)max(-1LL, (long long)w.p - (KW - 1));
      const int open_from = A.window > 0 ? (int)min(max(0LL, (long long)w.p + w.n - A.window), 0x7fffffffLL) : 0;
      const int open_sinks = A.sinks - (KW - 1);

      for (int t = t0; t < t1; t++) {
        wait(&full[stage], phase);
        const int key0 = (t < w.a ? t : t - w.a + w.c) * kKeys + wk * KW;  // this warp's keys
        constexpr int kAll = (1 << (KW / 16)) - 1;
        const int have = held[stage] >> (wk * KW / 16) & kAll;
        if (have) {
          uint8_t *stage_v = smem + (size_t)stage * C::kStageBytes + C::kTileBytes;
          const uint32_t kaddr = smem_u32(smem) + (uint32_t)stage * C::kStageBytes;
          const uint32_t vaddr = kaddr + C::kTileBytes;
          const bool open = key0 <= open_to && have == kAll && (key0 >= open_from || key0 < open_sinks);
          // whether some row of the sequence sees key i of these
          auto seen = [&](int i) {
            const int key = key0 + i;
            return key < w.hi && (key < w.se || key >= w.ws) && (have >> (i >> 4) & 1);
          };
          bool odd = false;  // some V row that not every row sees holds an infinity or NaN
          if (!open) {
            // V rows that no row of the sequence sees: zeros (their P is 0,
            // and 0 times whatever the page holds there would not be)
            for (int i = lane; i < KW * (Dh / 8); i += 32) {
              const int kr = i / (Dh / 8), ch = i - kr * (Dh / 8), row = wk * KW + kr;
              uint4 *v = reinterpret_cast<uint4 *>(stage_v + (ch >> 3) * kBlkBytes + row * 128 +
                                                   (((ch & 7) ^ (row & 7)) << 4));
              if (!seen(kr)) {
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
          float s[KW / 8][4];
#pragma unroll
          for (int nt = 0; nt < KW / 8; nt++) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.0f;
#pragma unroll
          for (int kk = 0; kk < Dh / 16; kk++) {
            const int ch = 2 * kk + (jm & 1);
            if constexpr (C::kQSmem) ldsm4(q_at + kk * 32, qa[0]);
            const uint32_t(&qk)[4] = qa[C::kQSmem ? 0 : kk];
#pragma unroll
            for (int np = 0; np < KW / 16; np++) {
              const int row = wk * KW + np * 16 + 8 * (jm >> 1) + jr;
              uint32_t bf[4];
              ldsm4(kaddr + (ch >> 3) * kBlkBytes + row * 128 + (((ch & 7) ^ (row & 7)) << 4), bf);
              mma16816<T>(s[2 * np], qk, bf[0], bf[1]);
              mma16816<T>(s[2 * np + 1], qk, bf[2], bf[3]);
            }
          }
          if (!open) {
#pragma unroll
            for (int nt = 0; nt < KW / 8; nt++)
#pragma unroll
              for (int e = 0; e < 4; e++) {
                const int i = nt * 8 + 2 * t4 + (e & 1);
                if (!seen(i) || !sees_key(rp[e >> 1], key0 + i, A.window, A.sinks)) s[nt][e] = -INFINITY;
              }
          }
          // online softmax
          float f[2];
#pragma unroll
          for (int e = 0; e < 2; e++) {
            float m = fmaxf(s[0][2 * e], s[0][2 * e + 1]);
#pragma unroll
            for (int nt = 1; nt < KW / 8; nt++) m = fmaxf(m, fmaxf(s[nt][2 * e], s[nt][2 * e + 1]));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
            const float mn = fmaxf(mx[e], m * kLog2e - kLift);
            f[e] = mn == -INFINITY ? 1.0f : ex2(mx[e] - mn);
            const float sub = mn == -INFINITY ? 0.0f : mn;
            mx[e] = mn;
            float sum = 0.0f;
#pragma unroll
            for (int nt = 0; nt < KW / 8; nt++)
#pragma unroll
              for (int c = 0; c < 2; c++) {
                const float v = ex2(s[nt][2 * e + c] * kLog2e - sub);
                s[nt][2 * e + c] = v;
                sum += v;
              }
            ls[e] = ls[e] * f[e] + sum;
          }
          if (f[0] != 1.0f || f[1] != 1.0f) {
#pragma unroll
            for (int d = 0; d < Dh / 8; d++) {
              o[d][0] *= f[0];
              o[d][1] *= f[0];
              o[d][2] *= f[1];
              o[d][3] *= f[1];
            }
          }
          // O += P V
          if (!odd) {
#pragma unroll
            for (int kc = 0; kc < KW / 16; kc++) {
              uint32_t ph[4], pl[4];  // P of 16 keys as hi + lo halves
#pragma unroll
              for (int i = 0; i < 4; i++) {
                const float v0 = s[2 * kc + (i >> 1)][2 * (i & 1)], v1 = s[2 * kc + (i >> 1)][2 * (i & 1) + 1];
                ph[i] = pack2<T>(v0, v1);
                const float2 h = unpack2<T>(ph[i]);
                pl[i] = pack2<T>(v0 - h.x, v1 - h.y);
              }
              const int row = wk * KW + kc * 16 + 8 * (jm & 1) + jr;
#pragma unroll
              for (int dp = 0; dp < Dh / 16; dp++) {
                const int ch = 2 * dp + (jm >> 1);
                uint32_t bf[4];
                ldsm4_t(vaddr + (ch >> 3) * kBlkBytes + row * 128 + (((ch & 7) ^ (row & 7)) << 4), bf);
                mma16816<T>(o[2 * dp], ph, bf[0], bf[1]);
                mma16816<T>(o[2 * dp + 1], ph, bf[2], bf[3]);
                mma16816<T>(o[2 * dp], pl, bf[0], bf[1]);
                mma16816<T>(o[2 * dp + 1], pl, bf[2], bf[3]);
              }
            }
          } else {
            // one key at a time, for the rows that see it (rare: kept small)
            float *sp = red + warp * 16 * KW;
#pragma unroll
            for (int nt = 0; nt < KW / 8; nt++)
#pragma unroll
              for (int e = 0; e < 4; e++) sp[(g + 8 * (e >> 1)) * KW + nt * 8 + 2 * t4 + (e & 1)] = s[nt][e];
            __syncwarp();
#pragma unroll 1
            for (int kr = 0; kr < KW; kr++) {
              const int row = wk * KW + kr;
              float pv[2];
              bool see[2];
#pragma unroll
              for (int e = 0; e < 2; e++) {
                pv[e] = sp[(g + 8 * e) * KW + kr];
                see[e] = seen(kr) && sees_key(rp[e], key0 + kr, A.window, A.sinks);
              }
#pragma unroll
              for (int d = 0; d < Dh / 8; d++) {
                const float2 v = unpack2<T>(*reinterpret_cast<const uint32_t *>(
                    stage_v + (d >> 3) * kBlkBytes + row * 128 + (((d & 7) ^ (row & 7)) << 4) + 4 * t4));
                if (see[0]) {
                  o[d][0] += pv[0] * v.x;
                  o[d][1] += pv[0] * v.y;
                }
                if (see[1]) {
                  o[d][2] += pv[1] * v.x;
                  o[d][3] += pv[1] * v.y;
                }
              }
            }
            __syncwarp();
          }
          if (!open) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the zeros, before the next copy
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[stage]);
        advance();
      }

      // ---- the warps' shares together ----
#pragma unroll
      for (int e = 0; e < 2; e++) {
        float l = ls[e];
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        if (t4 == 0) {
          sm_m[wk * C::kRows + wr * 16 + g + 8 * e] = mx[e];
          sm_l[wk * C::kRows + wr * 16 + g + 8 * e] = l;
        }
      }
      sync();
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const int row = wr * 16 + g + 8 * e;
        float m = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4; i++) m = fmaxf(m, sm_m[i * C::kRows + row]);
        const float f = m == -INFINITY ? 0.0f : ex2(mx[e] - m);
#pragma unroll
        for (int d = 0; d < Dh / 8; d++) {
          o[d][2 * e] *= f;
          o[d][2 * e + 1] *= f;
        }
      }
      // key groups 2 and 3 leave their sums, 0 and 1 add theirs
      float *mine = red + ((wk & 1) * C::kRows + wr * 16) * C::kRedRow;
      if (wk >= 2) {
#pragma unroll
        for (int d = 0; d < Dh / 8; d++)
#pragma unroll
          for (int e = 0; e < 2; e++)
            *reinterpret_cast<float2 *>(mine + (g + 8 * e) * C::kRedRow + d * 8 + 2 * t4) =
                make_float2(o[d][2 * e], o[d][2 * e + 1]);
      }
      sync();
      if (wk < 2) {
#pragma unroll
        for (int d = 0; d < Dh / 8; d++)
#pragma unroll
          for (int e = 0; e < 2; e++) {
            float2 *at = reinterpret_cast<float2 *>(mine + (g + 8 * e) * C::kRedRow + d * 8 + 2 * t4);
            float2 v = *at;
            v.x += o[d][2 * e];
            v.y += o[d][2 * e + 1];
            *at = v;
          }
      }
      sync();
      const bool whole = t0 == 0 && t1 == w.nt;
      const int slot = 2 * cta + (pos == start ? 0 : 1);
      float *part = A.part + (size_t)slot * C::kRows * (Dh + 2);
      for (int i = tid; i < C::kRows * (Dh / 4); i += C::kWarps * 32) {
        const int row = i / (Dh / 4), d = (i - row * (Dh / 4)) * 4, m = m0 + row, qi = m / A.G;
        if (qi >= w.n) continue;
        float mm = -INFINITY, l = 0.0f;
#pragma unroll
        for (int k = 0; k < 4; k++) mm = fmaxf(mm, sm_m[k * C::kRows + row]);
#pragma unroll
        for (int k = 0; k < 4; k++)
          l += mm == -INFINITY ? 0.0f : sm_l[k * C::kRows + row] * ex2(sm_m[k * C::kRows + row] - mm);
        const float4 x = *reinterpret_cast<const float4 *>(red + row * C::kRedRow + d);
        const float4 y = *reinterpret_cast<const float4 *>(red + (C::kRows + row) * C::kRedRow + d);
        float4 v = make_float4(x.x + y.x, x.y + y.y, x.z + y.z, x.w + y.w);
        if (whole) {
          const float inv = mm == -INFINITY ? 0.0f : 1.0f / l;
          uint2 u;
          u.x = pack2<T>(v.x * inv, v.y * inv);
          u.y = pack2<T>(v.z * inv, v.w * inv);
          *reinterpret_cast<uint2 *>(reinterpret_cast<T *>(A.out) +
                                     ((size_t)(w.r0 + qi) * A.H + hk * A.G + (m - qi * A.G)) * Dh + d) = u;
        } else {
          *reinterpret_cast<float4 *>(part + 2 * C::kRows + row * Dh + d) = v;
          if (d == 0) {
            part[row] = mm;
            part[C::kRows + row] = l;
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
      pos += A.whole ? 1 : t1 - t0;
    }
    if (tid == 0) {
      int *r = A.rec + cta * 8;
      r[0] = rec_parts;
#pragma unroll
      for (int i = 0; i < 5; i++) r[1 + i] = rec[i];
    }
  }
}

// The sums of a unit that several CTAs share: the blocks (c, .) join the rows of
// the unit that begins in CTA c, each row's parts in CTA order. Dh / 4 threads
// hold a row's dims; a unit of few parts has a group of them for each row, one of
// many parts several groups a row, each of them every n-th part. Bound by the
// latency of two dependent reads.
constexpr int kJoinThreads = 512;

template <typename T, int Dh>
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(const int *recs, const float *parts, int unit_rows,
                                                                  int H, int G, T *out) {
  constexpr int kLanes = Dh / 4, kGroups = kJoinThreads / kLanes, kSpan = kLanes < 32 ? kLanes : 32;
  __shared__ float4 acc[kGroups][kLanes];
  __shared__ float lsum[kGroups];
  pdl_trigger();
  pdl_wait();
  const int *rec = recs + blockIdx.x * 8;
  const int np = rec[0];
  if (np == 0) return;
  const int slot = rec[1], r0 = rec[2], n = rec[3], hk = rec[4], m0 = rec[5];
  const int tid = threadIdx.x, lane = tid % kLanes, grp = tid / kLanes;
  int per_row = 1;  // groups of a row: two to four parts each
  while (per_row < kGroups && per_row * 4 < np) per_row *= 2;
  const int sub = grp % per_row, at_once = kGroups / per_row;
  const size_t stride = (size_t)unit_rows * (Dh + 2);
  // part j: the first in `slot`, then the first slots of the CTAs that follow
  auto part = [&](int j) { return parts + (j == 0 ? (size_t)slot : (size_t)2 * (blockIdx.x + j)) * stride; };
  const int rows = min((long long)unit_rows, (long long)n * G - m0);  // of the unit
  for (int first = blockIdx.y * at_once; first < rows; first += gridDim.y * at_once) {
    const int row = first + grp / per_row;
    const bool on = row < rows;
    float mm = -INFINITY, l = 0.0f;
    float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (on)
      for (int j = tid % kSpan; j < np; j += kSpan) mm = fmaxf(mm, part(j)[row]);
#pragma unroll
    for (int o = kSpan / 2; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, o));
    if (on) {
#pragma unroll 4
      for (int j = sub; j < np; j += per_row) {
        const float *p = part(j);
        const float f = mm == -INFINITY ? 0.0f : ex2(p[row] - mm);
        const float4 v = *reinterpret_cast<const float4 *>(p + 2 * unit_rows + (size_t)row * Dh + lane * 4);
        a.x += v.x * f;
        a.y += v.y * f;
        a.z += v.z * f;
        a.w += v.w * f;
        l += p[unit_rows + row] * f;
      }
    }
    if (per_row > 1) {
      acc[grp][lane] = a;
      if (lane == 0) lsum[grp] = l;
      __syncthreads();
      if (sub == 0)
        for (int i = 1; i < per_row; i++) {
          const float4 v = acc[grp + i][lane];
          a.x += v.x;
          a.y += v.y;
          a.z += v.z;
          a.w += v.w;
          l += lsum[grp + i];
        }
      __syncthreads();
    }
    if (on && sub == 0) {
      const int m = m0 + row, qi = m / G;
      const float inv = mm == -INFINITY ? 0.0f : 1.0f / l;
      uint2 u;
      u.x = pack2<T>(a.x * inv, a.y * inv);
      u.y = pack2<T>(a.z * inv, a.w * inv);
      *reinterpret_cast<uint2 *>(out + ((size_t)(r0 + qi) * H + hk * G + (m - qi * G)) * Dh + lane * 4) = u;
    }
  }
}

int64_t stride_or(int64_t s, int64_t dense) { return s ? s : dense; }

template <typename T, int Dh>
cudaError_t rope_t(const float *qkv, const PagedRows &pr, int H, int Hkv, const RopeTurns &turns, const float *q_norm,
                   const float *k_norm, float eps, void *q_out, const wg_paged_kv &kv, unsigned *flags, int num_sms,
                   cudaStream_t s, bool pdl) {
  const int NH = H + 2 * Hkv;
  // heads a warp takes: few rows, those that share it at Dh / 8 lanes each, for
  // the shortest path; many, up to 16, which share the row's sines
  const int least = 256 / Dh;
  int hpw = least;
  while (hpw < 16 && (long long)pr.rows * ((NH + hpw - 1) / hpw) > (long long)num_sms * 64) hpw *= 2;
  const int wpr = (NH + hpw - 1) / hpw;
  const long long warps = (long long)pr.rows * wpr;
  if (warps > 0xFFFFFF00LL) return cudaErrorInvalidValue;  // (a terabyte of heads)
  const PagedTable pt{kv.table, kv.max_pages, kv.num_pages, kv.page_size};
  const int64_t rs = stride_or(kv.row_stride, Dh), hs = stride_or(kv.head_stride, (int64_t)kv.page_size * Dh),
                ps = stride_or(kv.page_stride, (int64_t)Hkv * kv.page_size * Dh);
  constexpr int threads = 64;
  const unsigned blocks = (unsigned)((warps * 32 + threads - 1) / threads);
  return launch_pdl(paged_rope_kernel<T, Dh>, dim3(blocks), threads, 0, s, pdl, qkv, pr, H, Hkv, turns, q_norm, k_norm, eps,
                reinterpret_cast<T *>(q_out), reinterpret_cast<T *>(kv.k), reinterpret_cast<T *>(kv.v), ps, hs, rs, pt,
                hpw, wpr, flags);
}

template <typename T, int Dh, int MT>
cudaError_t split_t(SplitArgs A, const wg_paged_kv &kv, void *workspace, int num_sms, cudaStream_t s, bool pdl) {
  using C = SplitCfg<Dh, MT>;
  auto kern = paged_split_kernel<T, Dh, MT>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
  if (e != cudaSuccess) return e;
  // keys of a box: the largest power of two that divides the page, up to 64
  A.box_rows = kv.page_size % 64 == 0 ? 64 : kv.page_size % 32 == 0 ? 32 : 16;
  CUtensorMap tk, tv;
  if (!page_map(&tk, kv.k, kv, A.Hkv, Dh, A.box_rows) || !page_map(&tv, kv.v, kv, A.Hkv, Dh, A.box_rows))
    return cudaErrorInvalidValue;
  // CTAs: no more than there can be work for
  const long long units = (((long long)A.pr.rows * A.G + C::kRows - 1) / C::kRows + A.pr.batch) * A.Hkv;
  const long long keys = (long long)kv.max_pages * kv.page_size;
  // Few keys that a row can see (by the table's width and the window, what the
  // host knows): whole units, and no second launch to join their parts (one
  // sequence, Dh = 64, 4 KV heads: 256 keys 5.8 us for 7.6, 384 7.1 for 8.1, 512
  // 8.3 for 8.1; Dh = 128, 8 KV heads: 128 keys 6.8 for 8.6, 256 9.0 for 9.3; Dh =
  // 256: 128 keys 9.0 for 10.2, 192 10.8 for 10.7; and a launch less on the host)
  const long long rows_seq = A.pr.row_start ? A.pr.rows : A.pr.rows / A.pr.batch;
  const long long seen = A.window ? (long long)A.window + A.sinks + rows_seq + 2 * C::kKeys : keys;
  A.whole = (seen < keys ? seen : keys) <= C::kWhole * C::kKeys;
  const long long work = A.whole ? units : units * ((keys + kMinKeys - 1) / kMinKeys);
  const int P = (int)(work < num_sms * C::kCtas ? work : num_sms * C::kCtas);
  A.rec = reinterpret_cast<int *>(workspace);
  A.part = reinterpret_cast<float *>(A.rec + (size_t)P * 8);
  e = launch_pdl(kern, dim3((unsigned)P), C::kThreads, C::kSmem, s, pdl, tk, tv, A);
  if (e != cudaSuccess || A.whole) return e;
  // blocks of a unit: one pass over the rows that can exist (none past the
  // longest sequence's), with the groups a row that equal sequences would give
  const long long most = A.pr.row_start ? A.pr.rows : A.pr.rows / A.pr.batch;
  const long long rows = most * A.G < C::kRows ? most * A.G : C::kRows, groups = kJoinThreads / (Dh / 4);
  const long long parts = P / ((long long)A.pr.batch * A.Hkv) + 2;
  const long long share = parts / 4 < groups ? (parts + 3) / 4 : groups;
  const unsigned blocks = (unsigned)((rows * share + groups - 1) / groups);
  return launch_pdl(paged_join_kernel<T, Dh>, dim3((unsigned)P, blocks), kJoinThreads, 0, s, pdl, A.rec, A.part,
                    C::kRows, A.H, A.G, reinterpret_cast<T *>(A.out));
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
  // two CTAs an SM of 16 rows, or one of 32
  const size_t P = (size_t)num_sms * 2;
  return P * 8 * sizeof(int) + 2 * P * 16 * (size_t)(Dh + 2) * sizeof(float);
}

cudaError_t launch_paged_attention(const void *q, const PagedRows &rows, int H, int Hkv, int Dh,
                                   const wg_paged_kv &kv, int window, int sinks, void *out, void *workspace,
                                   unsigned *flags, int num_sms, cudaStream_t s, bool pdl) {
  if (paged_prompt_wins(rows, H, Hkv, Dh, num_sms))
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
  A.flags = flags;
  return kv.dtype == WG_F16 ? split_d<__half>(A, Dh, kv, workspace, num_sms, s, pdl)
                            : split_d<__nv_bfloat16>(A, Dh, kv, workspace, num_sms, s, pdl);
}

}  // namespace wg
