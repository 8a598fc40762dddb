// Attention of many rows over the paged cache (prompt chunks) on the Blackwell
// tensor cores: the same operator as paged.cu's split kernel, for shapes that
// are bound by the products instead of the reads.
//
// A unit is (sequence, KV head, NT tiles of 128 query rows); a tile's rows are
// RP = 128 / G consecutive rows of the sequence times the G query heads of the
// KV head, so that one K / V tile serves the whole group and a tile spans few
// positions (little of it is cut by the causal border). Persistent CTAs, one an
// SM, take units round robin, longest first. Per CTA:
//   warps 0 .. 4 NT - 1  softmax: a thread owns a row. tcgen05.ld of the row's
//                scores, mask, maximum, exp2, P as 16-bit pairs back into the
//                scores' tensor-memory columns (the A operand of P V), the row
//                sum in a register; at the end O from tensor memory to `out`.
//                The reference of the exponentials is the first 64 keys' maximum
//                and moves only when the P of 64 keys add up to too much for
//                their type or, in fp16, to so little that they would lose bits
//                (PRange): O is then rescaled in tensor memory, which almost
//                never happens after the first tiles;
//   one warp     MMA: one thread issues S_t = Q_t K^T (both operands in shared
//                memory) and O_t += P_t V (P from tensor memory, V as it lies,
//                [key][dim], the MN-major form). The two tiles alternate:
//                while one's softmax runs, the other's products do;
//   one warp     loads: Q by one 3-D TMA box a tile and 64 dims, K and V by the
//                boxes of pages into a ring of stages;
//   two warps    clean V tiles that not every row sees in full: rows that no
//                row sees become zeros (their P is 0, but 0 times what a page
//                holds there need not be), and infinities or NaN in the others
//                are set aside (P = 0 must not meet them) and added at the end
//                for the rows that do see them.
// Every MMA is issued by one thread, so they execute in order: S_t(j + 1) may
// overwrite P_t(j) after P V(j) was issued, and the commit that reports
// S_t(j) reports P_t(j - 1) V too.
// Waits are bounded, and tensor memory is freed on every path.
#include <cuda.h>

#include "common.cuh"
#include "paged_device.cuh"

namespace wg {

namespace {

// Entries by key tile (not by stage: a stage carries K of one round and V of
// another): which page boxes of the tile were loaded; whether its V is clean.
constexpr int kHeldRing = 16;
constexpr int kOddRing = 8, kOddMax = 14;

template <int Dh_>
struct PromptCfg {
  static constexpr int Dh = Dh_;
  static constexpr int NT = Dh == 256 ? 1 : 2;   // query tiles of a CTA
  static constexpr int KT = Dh == 128 ? 128 : 64;  // keys of a tile
  static constexpr int NB = Dh == 128 ? 1 : 2;     // score buffers of a query tile
  static constexpr int kQBytes = 128 * Dh * 2;     // one query tile
  static constexpr int kStageBytes = KT * Dh * 2;  // K or V of a key tile
  static constexpr int kFit = (224 * 1024 - NT * kQBytes) / kStageBytes;
  static constexpr int kStages = kFit > 12 ? 12 : kFit;
  static constexpr int NH = KT / 64;  // parts of a tile that softmax hands over on its own
  static constexpr int kSoftWarps = 4 * NT;
  static constexpr int kThreads = (kSoftWarps + 4) * 32;
  // Registers a thread: two softmax warpgroups and the four other warps share
  // what the launch got (384 x 168); with one tile 256 threads have 255.
  static constexpr bool kSplitRegs = NT == 2;
  static constexpr int kLaunchRegs = 168, kSoftRegs = 208, kHelpRegs = 88;
  static_assert(!kSplitRegs || 256 * kSoftRegs + 128 * kHelpRegs <= kThreads * kLaunchRegs, "register split");
  // score buffer of the np-th tile of a CTA, and its round's parity
  static __device__ int buffer(int np) { return NB == 2 ? np & 1 : 0; }
  static __device__ int parity(int np) { return NB == 2 ? (np >> 1) & 1 : np & 1; }
  static __device__ int score_col(int t, int x) { return (t * NB + x) * KT; }
  static constexpr int kSmem = 1024 + NT * kQBytes + kStages * kStageBytes;
  static constexpr int kOCol = 256;  // tensor memory: scores at [0, 256), O after them
};

// P = 2^(s log2 e - ref) as a 16-bit number, and where the reference follows.
// P of 64 keys are at most 64 times 2^lift where the reference is their maximum
// (ref = maximum - lift) and may grow to a sum of `most`: no P is larger.
// fp16 ends at 65504 and has all its bits down to 2^-14 only: a key 10 nats below
// the reference would be rounded by more than its share, one 17 nats below be
// lost (a first token with a high score above thousands of others), while the
// row sum counts it in full. So P is lifted by 2^7, and 64 keys whose P add up to
// less than `least` move the reference down to their own maximum. What is
// rounded off below 2^-14 is then at most 64 x 2^-25 of a sum of at least 2^-4
// (2^-15 of it), or of a sum that holds a key at the reference (2^-26). The row
// sum, O and P carry the same factor: the quotient does not. A reference is not
// lowered where the row sum would pass 2^80 (and O 2^96): such keys are below
// 2^-60 of it. The test stands behind those for rows of nobody and for rows that
// have seen nothing: in front of them it costs 16 bytes of spills and 2 % (8192
// rows as calls: 517 us, so 509, without any 504).
// bf16 has the range of fp32.
template <typename T>
struct PRange {
  static constexpr bool kNarrow = std::is_same<T, __half>::value;
  static constexpr float lift = kNarrow ? 7.0f : 0.0f;
  static constexpr float most = kNarrow ? 32768.0f : 256.0f;
  static constexpr float least = 0x1p-4f, span = 0x1p80f;
  static constexpr float drop = 11.0f;  // lift - log2(least): the maximum of 64 keys that add up to less is as far below
};

struct PromptArgs {
  PagedRows pr;
  PagedTable pt;
  void *out;
  const void *v;  // for values set aside
  int64_t page_stride, head_stride, row_stride;
  int H, Hkv, G, RP;
  int window, sinks;
  int box_rows;
  unsigned *flags;
};

__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// The issuing warp runs as one: every lane follows the same path and `lead`
// (one lane, elected once) guards only the instruction itself, so that its
// operands stay in uniform registers. Issued from a branch of a single lane
// each product cost 100 cycles of operand moves: more than it runs for.
__device__ __forceinline__ uint32_t elect_lane() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r;
}

__device__ __forceinline__ void tc_commit_to(uint32_t bar, uint32_t lead) {
  asm volatile(
      "{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %1, 0;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar),
      "r"(lead)
      : "memory");
}

// D (+)= A B with A and B in shared memory, or A in tensor memory.
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc,
                                       uint32_t lead) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 e, %5, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(lead)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc,
                                       uint32_t lead) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 e, %5, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc), "r"(lead)
      : "memory");
}

// Shared-memory descriptor, 128-byte swizzle: 8-row groups 1024 bytes apart
// (SBO), and for the MN-major form `lbo` bytes between 64-element blocks.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lbo) {
  return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)((lbo >> 4) & 0x3FFFu) << 16) |
         ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

// kind::f16, M = 128: A and B of type T (K-major, or B MN-major), fp32 sums.
template <typename T>
__host__ __device__ constexpr uint32_t instr_desc(int N, bool b_mn) {
  return (1u << 4) | (std::is_same<T, __half>::value ? 0u : (1u << 7) | (1u << 10)) | (b_mn ? 1u << 16 : 0u) |
         ((uint32_t)(N >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}

__device__ __forceinline__ void tmem_ld32(uint32_t addr, float *v) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr)
      : "memory");
#pragma unroll
  for (int i = 0; i < 32; i++) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t *r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, float *v) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr)
      : "memory");
#pragma unroll
  for (int i = 0; i < 16; i++) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t *r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// mbar_wait_bounded as one piece of code (the compiler sees no loop whose trips
// could differ between lanes): false after about `cycles`.
constexpr long long kWaitCycles = 2000000000LL;
__device__ __forceinline__ bool wait_one_path(uint64_t *bar, uint32_t parity, long long cycles) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .u64 t0, t1;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "@p bra DONE;\n\t"
      "mov.u64 t0, %%clock64;\n\t"
      "AGAIN:\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "@p bra DONE;\n\t"
      "mov.u64 t1, %%clock64;\n\t"
      "sub.u64 t1, t1, t0;\n\t"
      "setp.lt.u64 q, t1, %3;\n\t"
      "@q bra AGAIN;\n\t"
      "DONE:\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity), "l"(cycles)
      : "memory");
  return ok != 0;
}

// Two fp32 operations in one instruction.
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Bits [a, b) of a 32-bit word (a, b clamped to 0 .. 32).
__device__ __forceinline__ uint32_t bit_range(int a, int b) {
  a = max(0, min(a, 32));
  b = max(0, min(b, 32));
  const uint32_t below_b = b >= 32 ? 0xFFFFFFFFu : (1u << b) - 1;
  const uint32_t below_a = a >= 32 ? 0xFFFFFFFFu : (1u << a) - 1;
  return below_b & ~below_a;
}

struct Unit : KeySpan {
  int b, hk, r0, n, p;
  int i0;  // first row of its NT tiles
};

// The units in order: sequence, then the rows from the last to the first, then
// the KV head; dealt to the CTAs in rounds, every other round backwards (the
// units of a sequence get shorter, so a fixed order would give the first CTA
// the longest of every round: 1.3x the mean). Each role of a CTA walks the
// same ones.
struct UnitWalk {
  int b = 0, round = 0;
  long long base = 0;
  __device__ long long next() {
    const long long item = (long long)round * gridDim.x + (round & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
    round++;
    return item;
  }
  __device__ bool get(const PromptArgs &A, long long item, int rows_per_unit, int KT, Unit &u) {
    for (; b < A.pr.batch; b++) {
      seq_rows(A.pr, b, u.r0, u.n);
      const int chunks = (u.n + rows_per_unit - 1) / rows_per_unit;
      const long long cnt = (long long)chunks * A.Hkv;
      if (item < base + cnt) {
        const long long local = item - base;
        u.b = b;
        u.p = A.pr.pos[b];
        u.i0 = (chunks - 1 - (int)(local / A.Hkv)) * rows_per_unit;
        u.hk = (int)(local % A.Hkv);
        static_cast<KeySpan &>(u) =
            key_span((long long)u.p + u.i0, min(u.n - u.i0, rows_per_unit), A.window, A.sinks, A.pt, KT);
        return true;
      }
      base += cnt;
    }
    return false;
  }
};

template <typename T, int Dh>
__global__ void __launch_bounds__(PromptCfg<Dh>::kThreads, 1)
    paged_prompt_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                        const __grid_constant__ CUtensorMap tm_v, const PromptArgs A) {
  using C = PromptCfg<Dh>;
  constexpr int NT = C::NT, KT = C::KT, S = C::kStages;
  constexpr int kBlk = Dh / 64, kBlkBytes = KT * 128;
  constexpr float kLog2e = 1.4426950408889634f;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  uint8_t *smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  uint8_t *ring = smem + NT * C::kQBytes;
  __shared__ uint64_t q_full, q_empty, kv_full[S], kv_empty[S], v_ready[kHeldRing], s_full[2][2], p_full[2][2], o_full[2],
      o_empty[2], pv_done[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int held[kHeldRing];
  __shared__ int odd[kOddRing][2][kOddMax + 2];  // of each half: how many, then the tiles
  __shared__ int aborted;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int w_mma = C::kSoftWarps, w_load = w_mma + 1;
  const int rows_per_unit = NT * A.RP;
  constexpr int kAll = (1 << (KT / 16)) - 1;

  if (tid == 0) {
    mbar_init(&q_full, 1);
    mbar_init(&q_empty, 1);
    for (int i = 0; i < S; i++) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], 1);
    }
    for (int i = 0; i < kHeldRing; i++) mbar_init(&v_ready[i], 2);
    for (int i = 0; i < 2; i++) {
      for (int x = 0; x < 2; x++) {
        mbar_init(&s_full[i][x], 1);
        mbar_init(&p_full[i][x], 4);
      }
      mbar_init(&o_full[i], 1);
      mbar_init(&o_empty[i], 4);
      mbar_init(&pv_done[i], 1);
    }
    fence_mbar_init();
    aborted = 0;
  }
  if (warp == w_mma) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&tmem_slot))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (warp == w_load && lane == 0) {
    prefetch_tensormap(&tm_q);
    prefetch_tensormap(&tm_k);
    prefetch_tensormap(&tm_v);
  }
  pdl_trigger();
  pdl_wait();
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = tmem_slot;

  auto wait = [&](uint64_t *bar, uint32_t parity) {
    if (mbar_try_wait(bar, parity)) return;
    if (!wait_one_path(bar, parity, *(volatile int *)&aborted ? 0 : kWaitCycles)) {
      raise_flag(A.flags, kFlagTimeout);
      *(volatile int *)&aborted = 1;
    }
  };
  // whether every row of the unit sees every key of tile t
  auto open_tile = [&](const Unit &u, int key0) {
    const long long first = (long long)u.p + u.i0, last = (long long)u.p + min(u.n, u.i0 + rows_per_unit) - 1;
    return key0 + KT - 1 <= first &&
           (A.window == 0 || key0 + KT - 1 < A.sinks || (long long)key0 > last - A.window);
  };
  auto tile_key = [&](const Unit &u, int t) { return (t < u.a ? t : t - u.a + u.c) * KT; };

  UnitWalk walk;
  Unit u;
  if (warp >= C::kSoftWarps) {
    if constexpr (C::kSplitRegs) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kHelpRegs));
    if (warp == w_load) {
      // ---- loads ----
      const int nb = KT / A.box_rows, nops = nb * kBlk;
      const int box = lane % nb, blk = lane / nb;
      const uint32_t box_bytes = (uint32_t)A.box_rows * 128;
      const int groups = A.box_rows / 16, gmask = (1 << groups) - 1;
      int stage = 0, phase = 0, nu = 0, nt = 0;
      for (; walk.get(A, walk.next(), rows_per_unit, KT, u); nu++) {
        wait(&q_empty, (nu & 1) ^ 1);
        if (lane == 0) {
          mbar_expect_tx(&q_full, (uint32_t)(NT * kBlk * A.G * A.RP * 128));
          for (int t = 0; t < NT; t++)
            for (int i = 0; i < kBlk; i++)
              tma_load_3d(smem + t * C::kQBytes + i * 16384, &tm_q, i * 64, u.hk * A.G, u.r0 + u.i0 + t * A.RP, &q_full);
        }
        const int32_t *row = A.pt.table + (size_t)u.b * A.pt.max_pages;
        auto entry = [&](int t, int &key, bool &seen) {
          key = tile_key(u, t) + box * A.box_rows;
          seen = lane < nops && key < u.hi && (key < u.se || key + A.box_rows > u.ws);
          return seen ? row[key / A.pt.page_size] : -1;
        };
        int key, key_next = 0;
        bool seen, seen_next = false;
        int page = entry(0, key, seen), page_next = -1;
        for (int t = 0; t < u.nt; t++, nt++) {
          if (t + 1 < u.nt) page_next = entry(t + 1, key_next, seen_next);
          const bool ok = seen && page >= 0 && page < A.pt.num_pages;
          if (seen && !ok) raise_flag(A.flags, kFlagBadArgument);
          const unsigned loaded = __ballot_sync(0xffffffffu, ok && lane < nb);
#pragma unroll
          for (int kv = 0; kv < 2; kv++) {  // K, then V
            wait(&kv_empty[stage], phase ^ 1);
            if (lane == 0) {
              if (kv == 0) {
                int m = 0;
                for (int i = 0; i < nb; i++)
                  if (loaded >> i & 1) m |= gmask << (i * groups);
                held[nt % kHeldRing] = m;
              }
              mbar_expect_tx(&kv_full[stage], (uint32_t)__popc(loaded) * box_bytes * kBlk);
            }
            __syncwarp();
            if (ok)
              tma_load_4d(ring + (size_t)stage * C::kStageBytes + blk * kBlkBytes + box * box_bytes, kv ? &tm_v : &tm_k,
                          blk * 64, key % A.pt.page_size, u.hk, page, &kv_full[stage]);
            if (++stage == S) stage = 0, phase ^= 1;
          }
          page = page_next;
          key = key_next;
          seen = seen_next;
        }
      }
      // after a wait that ran out, no copy may still be on its way when the CTA exits
      __syncwarp();
      if (*(volatile int *)&aborted && lane == 0) {
        for (int i = 0; i < S; i++) {
          mbar_wait_bounded(&kv_full[stage], phase ^ 1, A.flags);
          if (++stage == S) stage = 0, phase ^= 1;
        }
        if (nu) mbar_wait_bounded(&q_full, (nu - 1) & 1, A.flags);
      }
    } else if (warp == w_mma) {
      // ---- products ----
      {
        const uint32_t lead = elect_lane();
        const uint32_t smem0 = __shfl_sync(0xffffffffu, smem_u32(smem), 0), ring0 = smem0 + NT * C::kQBytes;
        const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
        auto commit = [&](uint64_t *bar) { tc_commit_to(smem_u32(bar), lead); };
        auto wait1 = [&](uint64_t *bar, uint32_t parity) {
          wait(bar, parity);
          __syncwarp();
        };
        constexpr uint32_t qk_desc = instr_desc<T>(KT, false), pv_desc = instr_desc<T>(Dh, true);
        int stage = 0, phase = 0, nu = 0, np = 0;
        auto step = [&](int &s, int &ph) {
          if (++s == S) s = 0, ph ^= 1;
        };
        // S_t = Q_t K^T into score buffer x of tile t; O_t += P_t V
        auto qk = [&](int t, int x, int st) {
          const uint32_t q = smem0 + t * C::kQBytes, k = ring0 + st * C::kStageBytes;
#pragma unroll
          for (int kk = 0; kk < Dh / 16; kk++)
            mma_ss(tm + C::score_col(t, x), smem_desc(q + (kk >> 2) * 16384 + (kk & 3) * 32, 16),
                   smem_desc(k + (kk >> 2) * kBlkBytes + (kk & 3) * 32, 16), qk_desc, kk > 0, lead);
          commit(&s_full[t][x]);
          if (t == NT - 1) commit(&kv_empty[st]);
        };
        auto pv = [&](int t, int x, int part, int st, bool first) {
          const uint32_t v = ring0 + st * C::kStageBytes;
#pragma unroll
          for (int kk = 4 * part; kk < 4 * part + 4; kk++)
            mma_ts(tm + C::kOCol + t * Dh, tm + C::score_col(t, x) + kk * 8, smem_desc(v + kk * 2048, kBlkBytes),
                   pv_desc, !(first && kk == 0), lead);
          if (t == NT - 1 && part == C::NH - 1) commit(&kv_empty[st]);
          if (part < C::NH - 1 || C::NB == 2) commit(&pv_done[t]);
        };
        for (; __shfl_sync(0xffffffffu, walk.get(A, walk.next(), rows_per_unit, KT, u), 0); nu++) {
          u.nt = __shfl_sync(0xffffffffu, u.nt, 0);
          wait1(&q_full, nu & 1);
          wait1(&kv_full[stage], phase);  // K of tile 0
          tc_after();
#pragma unroll
          for (int t = 0; t < NT; t++) qk(t, C::buffer(np), stage);
          step(stage, phase);
          for (int j = 0; j < u.nt; j++, np++) {
            const int vs = stage, x = C::buffer(np);
            step(stage, phase);
            const bool more = j + 1 < u.nt;
            if (more)
              wait1(&kv_full[stage], phase);  // K of tile j + 1
            else
              commit(&q_empty);
            if (C::NB == 1) wait1(&v_ready[np % kHeldRing], (np / kHeldRing) & 1);
            tc_after();
#pragma unroll
            for (int t = 0; t < NT; t++) {
              if (C::NB == 2 && more) qk(t, x ^ 1, stage);
              if (C::NB == 2 && t == 0) wait1(&v_ready[np % kHeldRing], (np / kHeldRing) & 1);
              if (j == 0) wait1(&o_empty[t], (nu & 1) ^ 1);
#pragma unroll
              for (int part = 0; part < C::NH; part++) {
                wait1(&p_full[t][C::NH == 1 ? x : part], C::parity(np));
                tc_after();
                pv(t, x, part, vs, j == 0 && part == 0);
              }
              if (!more) commit(&o_full[t]);
              if (C::NB == 1 && more) qk(t, x, stage);
            }
            if (more) step(stage, phase);
          }
        }
      }
    } else {
      // ---- V tiles that some rows do not see in full: two warps, half a tile each ----
      const int half = warp - w_load - 1;
      int stage = 0, phase = 0, nu = 0, nt = 0;
      for (; walk.get(A, walk.next(), rows_per_unit, KT, u); nu++) {
        int *list = odd[nu % kOddRing][half];
        int nodd = 0;
        for (int t = 0; t < u.nt; t++, nt++) {
          if (++stage == S) stage = 0, phase ^= 1;  // past K
          wait(&kv_full[stage], phase);
          const int key0 = tile_key(u, t), m = held[nt % kHeldRing];
          if (!open_tile(u, key0) || m != kAll) {
            bool found = false;
            uint8_t *v = ring + (size_t)stage * C::kStageBytes;
            // 16-byte pieces, eight a lane in flight
            constexpr int kPieces = KT / 2 * (Dh / 8), kPer = 8;
            for (int i0 = lane; i0 < kPieces; i0 += 32 * kPer) {
              uint4 x[kPer];
              uint4 *at[kPer];
              bool none[kPer];
#pragma unroll
              for (int e = 0; e < kPer; e++) {
                const int i = i0 + 32 * e, kr = half * (KT / 2) + i / (Dh / 8), ch = i % (Dh / 8),
                          key = key0 + kr;
                at[e] = reinterpret_cast<uint4 *>(v + (ch >> 3) * kBlkBytes + kr * 128 + (((ch & 7) ^ (kr & 7)) << 4));
                none[e] = key >= u.hi || (key >= u.se && key < u.ws) || !(m >> (kr >> 4) & 1);
                x[e] = *at[e];
              }
#pragma unroll
              for (int e = 0; e < kPer; e++) {
                if (none[e]) {
                  *at[e] = make_uint4(0, 0, 0, 0);
                } else if (nonfinite2<T>(x[e].x) || nonfinite2<T>(x[e].y) || nonfinite2<T>(x[e].z) ||
                           nonfinite2<T>(x[e].w)) {
                  uint32_t w[4] = {x[e].x, x[e].y, x[e].z, x[e].w};
#pragma unroll
                  for (int k = 0; k < 4; k++) {
                    constexpr uint32_t ex = kNonfinite<T>;
                    if ((w[k] & ex) == ex) w[k] &= 0xFFFF0000u;
                    if ((w[k] >> 16 & ex) == ex) w[k] &= 0xFFFFu;
                  }
                  *at[e] = make_uint4(w[0], w[1], w[2], w[3]);
                  found = true;
                }
              }
            }
            static_assert(kPieces % (32 * kPer) == 0, "whole rounds");
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            if (__any_sync(0xffffffffu, found) && nodd < kOddMax) {
              if (lane == 0) list[1 + nodd] = t;
              nodd++;
            }
          }
          if (t + 1 == u.nt && lane == 0) list[0] = nodd;
          __syncwarp();
          if (lane == 0) mbar_arrive(&v_ready[nt % kHeldRing]);
          if (++stage == S) stage = 0, phase ^= 1;
        }
      }
    }
  } else {
    // ---- softmax: one row a thread ----
    if constexpr (C::kSplitRegs) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kSoftRegs));
    const int t = warp >> 2, m = tid & 127;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t o_addr = tmem + lanes + C::kOCol + t * Dh;
    const int i_in = m / A.G, g = m - i_in * A.G;
    int nu = 0, np = 0;
    for (; walk.get(A, walk.next(), rows_per_unit, KT, u); nu++) {
      const int i = u.i0 + t * A.RP + i_in;
      const bool valid = i_in < A.RP && i < u.n;
      const int p = valid ? (int)max(-1LL, min((long long)u.p + i, 0x7ffffffeLL)) : -1;
      // tiles whose keys every row of the unit sees: key0 <= open_to, and past the
      // last row's window start or all sinks
      const long long first = (long long)u.p + u.i0, last = (long long)u.p + min(u.n, u.i0 + rows_per_unit) - 1;
      const int open_to = (int)max(-1LL, min(first, 0x7ffffffeLL) - (KT - 1));
      const int open_from = A.window > 0 ? (int)max(0LL, min(last, 0x7ffffffeLL) - A.window + 1) : 0;
      const int open_sinks = A.sinks - (KT - 1);
      float ref = -INFINITY, l = 0.0f;  // the reference maximum (log2 units) and the row sum over it
      for (int j = 0; j < u.nt; j++, np++) {
        const int x = C::buffer(np);
        const uint32_t s_addr = tmem + lanes + C::score_col(t, x);
        const int key0 = tile_key(u, j);
        wait(&s_full[t][x], C::parity(np));
        tc_after();
        float s[KT];
#pragma unroll
        for (int c = 0; c < KT / 32; c++) tmem_ld32(s_addr + c * 32, s + c * 32);
        tmem_wait_ld();
        const int hm = held[np % kHeldRing];
        if (key0 > open_to || (key0 < open_from && key0 >= open_sinks) || hm != kAll) {
          // the row's keys of this tile: below its position and the sequence's
          // end, inside the window or among the sinks, on a page that exists
          const int end = min(p + 1, u.hi) - key0;
          const int from = A.window > 0 ? (int)max(0LL, (long long)p - A.window + 1 - key0) : 0;
#pragma unroll
          for (int w = 0; w < KT / 32; w++) {
            uint32_t see = bit_range(from - 32 * w, end - 32 * w) |
                           bit_range(0, min(end, min(A.sinks, 1 << 30) - key0) - 32 * w);
            if (!(hm >> (2 * w) & 1)) see &= 0xFFFF0000u;
            if (!(hm >> (2 * w + 1) & 1)) see &= 0xFFFFu;
            if (see != 0xFFFFFFFFu) {  // (a border cuts few of a warp's words)
#pragma unroll
              for (int c = 0; c < 32; c++)
                if (!(see >> c & 1)) s[32 * w + c] = -INFINITY;
            }
          }
        }
#pragma unroll
        for (int part = 0; part < C::NH; part++) {
          const float *sp = s + 64 * part;
          // P = 2^(s log2 e - ref) of 64 keys, packed; their share of the sum
          uint32_t r[32];
          auto exps = [&]() {
            const float sub = ref == -INFINITY ? 0.0f : ref;
            const uint64_t scale2 = pair(kLog2e, kLog2e), sub2 = pair(-sub, -sub);
            uint64_t sum[4] = {0, 0, 0, 0};
#pragma unroll
            for (int e = 0; e < 32; e++) {
              float2 v = unpair(fma2(pair(sp[2 * e], sp[2 * e + 1]), scale2, sub2));
              v = make_float2(ex2(v.x), ex2(v.y));
              sum[e & 3] = add2(sum[e & 3], pair(v.x, v.y));
              r[e] = pack2<T>(v.x, v.y);
            }
            const float2 v = unpair(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])));
            return v.x + v.y;
          };
          // The reference of the keys before nearly always still holds, so P is
          // made with it and its sum tells (PRange). (No maximum is taken on this
          // path.)
          using R = PRange<T>;
          float sum = 0.0f;
          bool holds = false;
          if (j > 0 || part > 0) {
            sum = exps();
            if (p < 0) {
              holds = true;  // (rows of nobody hold anything: they decide nothing for their warp)
            } else if (ref == -INFINITY) {  // nothing seen so far: still so?
              float top = -INFINITY;
#pragma unroll
              for (int c = 0; c < 64; c += 2) top = max3(top, sp[c], sp[c + 1]);
              holds = !(top > -INFINITY) && !isnan(sum);
            } else {
              holds = sum <= R::most && !(R::kNarrow && sum < R::least && sum > 0.0f);
            }
          }
          if (!__all_sync(0xffffffffu, holds)) {
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int c = 0; c < 64; c += 2) mx[(c >> 1) & 3] = max3(mx[(c >> 1) & 3], sp[c], sp[c + 1]);
            const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * kLog2e - R::lift;
            float f = ref > -INFINITY ? ex2(ref - top) : 0.0f;
            const bool move = top > ref || (R::kNarrow && top < ref - R::drop && l * f < R::span);
            if (!move) f = 1.0f;
            if (move) ref = top;
            l *= f;
            if (j > 0 || part > 0) {
              // O must hold all keys before these: the scores' commit says so
              // for the tile before (with one score buffer), pv_done else
              if (C::NB == 2 || part > 0) wait(&pv_done[t], (C::NB == 2 ? np - 1 : np) & 1);
              tc_after();
#pragma unroll 1
              for (int c = 0; c < Dh / 16; c++) {
                float o[16];
                tmem_ld16(o_addr + c * 16, o);
                tmem_wait_ld();
                uint32_t w[16];
#pragma unroll
                for (int e = 0; e < 16; e++) w[e] = __float_as_uint(o[e] * f);
                tmem_st16(o_addr + c * 16, w);
              }
            }
            sum = exps();
          }
          l += sum;
          tmem_st32(s_addr + part * 32, r);
          tmem_wait_st();
          tc_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[t][C::NH == 1 ? x : part]);
        }
      }
      // ---- the rows' results
      wait(&o_full[t], nu & 1);
      tc_after();
      const int nodd[2] = {odd[nu % kOddRing][0][0], odd[nu % kOddRing][1][0]};
      const float inv = ref == -INFINITY ? 0.0f : 1.0f / l;
      T *dst = reinterpret_cast<T *>(A.out) + ((size_t)(u.r0 + i) * A.H + u.hk * A.G + g) * Dh;
#pragma unroll 1
      for (int c = 0; c < Dh / 32; c++) {
        float o[32];
        tmem_ld32(o_addr + c * 32, o);
        tmem_wait_ld();
        if ((nodd[0] | nodd[1]) && valid) {
          // infinities and NaN of V that this row does see
          for (int k = 0; k < nodd[0] + nodd[1]; k++) {
            const int h = k >= nodd[0];
            const int k0 = tile_key(u, odd[nu % kOddRing][h][1 + k - (h ? nodd[0] : 0)]) + h * (KT / 2);
            for (int key = k0; key < k0 + KT / 2; key++) {
              if (key >= u.hi || !sees_key(p, key, A.window, A.sinks)) continue;
              const int page = A.pt.table[(size_t)u.b * A.pt.max_pages + key / A.pt.page_size];
              if (page < 0 || page >= A.pt.num_pages) continue;
              const uint32_t *v = reinterpret_cast<const uint32_t *>(
                  reinterpret_cast<const T *>(A.v) + page * A.page_stride + u.hk * A.head_stride +
                  (key % A.pt.page_size) * A.row_stride + c * 32);
#pragma unroll
              for (int e = 0; e < 16; e++) {
                const uint32_t w = v[e];
                const float2 f = unpack2<T>(w);
                if ((w & kNonfinite<T>) == kNonfinite<T>) o[2 * e] += f.x;
                if ((w >> 16 & kNonfinite<T>) == kNonfinite<T>) o[2 * e + 1] += f.y;
              }
            }
          }
        }
        if (valid) {
          // a row that saw nothing: O may hold anything, its result is zeros
#pragma unroll
          for (int e = 0; e < 4; e++) {
            uint4 w = make_uint4(0, 0, 0, 0);
            if (ref > -INFINITY || isnan(l)) {
              w.x = pack2<T>(o[8 * e] * inv, o[8 * e + 1] * inv);
              w.y = pack2<T>(o[8 * e + 2] * inv, o[8 * e + 3] * inv);
              w.z = pack2<T>(o[8 * e + 4] * inv, o[8 * e + 5] * inv);
              w.w = pack2<T>(o[8 * e + 6] * inv, o[8 * e + 7] * inv);
            }
            *reinterpret_cast<uint4 *>(dst + c * 32 + 8 * e) = w;
          }
        }
      }
      tc_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&o_empty[t]);
    }
  }

  tc_before();
  __syncthreads();
  if (warp == w_mma) {
    tc_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

template <typename T, int Dh>
cudaError_t prompt_t(const void *q, PromptArgs A, const wg_paged_kv &kv, int num_sms, cudaStream_t s, bool pdl) {
  using C = PromptCfg<Dh>;
  auto kern = paged_prompt_kernel<T, Dh>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
  if (e != cudaSuccess) return e;
  if constexpr (C::kSplitRegs) {
    // the split needs what it was counted against
    static const bool enough = [&] {
      cudaFuncAttributes at;
      return cudaFuncGetAttributes(&at, kern) == cudaSuccess && at.numRegs >= C::kLaunchRegs;
    }();
    if (!enough) return cudaErrorInvalidConfiguration;
  }
  A.box_rows = kv.page_size % 128 == 0 && C::KT == 128 ? 128 : kv.page_size % 64 == 0 ? 64 : kv.page_size % 32 == 0 ? 32 : 16;
  CUtensorMap tq, tk, tv;
  EncodeTiled enc = encode_fn();
  if (!enc || !page_map(&tk, kv.k, kv, A.Hkv, Dh, A.box_rows) || !page_map(&tv, kv.v, kv, A.Hkv, Dh, A.box_rows))
    return cudaErrorInvalidValue;
  // queries as (dim, head, row): a box is 64 dims x the group's heads x RP rows
  const cuuint64_t dims[3] = {(cuuint64_t)Dh, (cuuint64_t)A.H, (cuuint64_t)A.pr.rows};
  const cuuint64_t strides[2] = {(cuuint64_t)Dh * 2, (cuuint64_t)A.H * Dh * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)A.G, (cuuint32_t)A.RP}, one[3] = {1, 1, 1};
  if (enc(&tq, kv.dtype == WG_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
          const_cast<void *>(q), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
          CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return cudaErrorInvalidValue;
  const long long rpu = (long long)C::NT * A.RP;
  const long long most = ((A.pr.rows + rpu - 1) / rpu + A.pr.batch) * A.Hkv;  // units there can be
  const unsigned grid = (unsigned)(most < num_sms ? most : num_sms);
  return launch_pdl(kern, dim3(grid), C::kThreads, C::kSmem, s, pdl, tq, tk, tv, A);
}

}  // namespace

// Which of the two kernels, from the rows a sequence has on average (lengths are
// on the device). For sequences of about as many rows both times are proportional
// to the keys; in a call of a chunk and single rows they are not, since only the
// split kernel spreads one row's keys over the machine (H 32, Hkv 8, Dh 128: 512
// rows and a row of 131k keys 1709 us, in two calls 17 and 93; 2048 rows and 63
// single ones of up to 16k keys 817, in two calls 51 and 404). This one
// takes rounds of num_sms units of 256 rows (128 at Dh = 256), a CTA for all keys
// of a unit; the split kernel spreads row tiles of 32 (16 at Dh = 256) over the
// machine. Per 64 keys, a round here costs what kSplitWorth row tiles an SM cost
// there (8 sequences x 4096 keys, Dh = 128, 8 KV heads of 4: 16 rows 65 us here and
// 88 us there, 8 rows 65 and 54; one sequence of 128 rows 63 and 88 us, of 64 rows
// 62 and 53; Dh = 64, 8 sequences: 32 rows 68 and 89 us, 16 rows 67 and 59).
bool paged_prompt_wins(const PagedRows &rows, int H, int Hkv, int Dh, int num_sms) {
  const int G = H / Hkv;
  if (G > 128) return false;  // a tile of 128 rows holds no whole row of such a group
  const long long n = (rows.rows + rows.batch - 1) / rows.batch, heads = (long long)rows.batch * Hkv;
  if (n * G <= 16) return false;  // one 16-row tile: K and V are read once, at the memory's rate
  const double kSplitWorth = Dh == 64 ? 1.46 : Dh == 128 ? 0.79 : 0.82;
  const long long unit = (Dh == 256 ? 1 : 2) * (128 / G), tile = Dh == 256 ? 16 : 32;
  const long long units = heads * ((n + unit - 1) / unit), tiles = heads * ((n * G + tile - 1) / tile);
  return (double)((units + num_sms - 1) / num_sms) * num_sms * kSplitWorth < (double)tiles;
}

cudaError_t launch_paged_prompt(const void *q, const PagedRows &rows, int H, int Hkv, int Dh, const wg_paged_kv &kv,
                                int window, int sinks, void *out, unsigned *flags, int num_sms, cudaStream_t s,
                                bool pdl) {
  PromptArgs A{};
  A.pr = rows;
  A.pt = PagedTable{kv.table, kv.max_pages, kv.num_pages, kv.page_size};
  A.out = out;
  A.v = kv.v;
  A.row_stride = kv.row_stride ? kv.row_stride : Dh;
  A.head_stride = kv.head_stride ? kv.head_stride : (int64_t)kv.page_size * Dh;
  A.page_stride = kv.page_stride ? kv.page_stride : (int64_t)Hkv * kv.page_size * Dh;
  A.H = H;
  A.Hkv = Hkv;
  A.G = H / Hkv;
  A.RP = 128 / A.G;
  A.window = window;
  A.sinks = sinks;
  A.flags = flags;
#define WG_PROMPT(T)                                                       \
  if (Dh == 64) return prompt_t<T, 64>(q, A, kv, num_sms, s, pdl);   \
  if (Dh == 128) return prompt_t<T, 128>(q, A, kv, num_sms, s, pdl); \
  return prompt_t<T, 256>(q, A, kv, num_sms, s, pdl)
  if (kv.dtype == WG_F16) {
    WG_PROMPT(__half);
  }
  WG_PROMPT(__nv_bfloat16);
#undef WG_PROMPT
}

}  // namespace wg
