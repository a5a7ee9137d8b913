// Prefix-aware (chunked) causal prefill over the 4-bit KV pool on the
// 5th-generation tensor cores: bf16/f16, head_dim 64, any block_size, up to
// 128 q heads per kv head.
//
// Mathematics.  A row's values are mid + step (c - 7.5).  K goes to the tensor
// cores as two operands of type T: each value rounded to T and what that
// leaves out, rounded again (together 2^-17 of the value or less), so that S
// needs nothing but the softmax's own scale.  V is an f16 operand next to f16
// probabilities, each rounded by 2^-12 at most: for bf16 step (c - 7.5), scaled
// by a power of two; for f16, whose results show a second rounding of that
// size (1.8 times the error of the attention over decoded rows), the bare
// codes, which are exact, with the steps on the probabilities before their
// rounding.  The mids, which no cancellation with the codes may touch, are
// summed in fp32 beside the denominator.  K's codes could stay bare as well,
// with step and mid applied to S: that reads four factors per key from shared
// memory in every softmax thread (57% of the shared-memory cycles) and was no
// faster.
//
// Tiles.  The q heads of a kv head read the same keys, so a tile's 128 rows
// are TQ = 128 / group consecutive tokens times the group's heads (one TMA box
// of [TQ, group, 64]): a short chunk of few tokens still fills a tile.  Two
// consecutive tiles of a sequence make a pair and share each step's 64 decoded
// keys.  The steps of all pairs, in (kv head, pair, step) order, are dealt
// evenly over a persistent grid of two CTAs per SM; a pair cut by a CTA
// boundary leaves fp32 partials that int4_prefill_combine_kernel joins (a single
// chunk on a long prefix has fewer pairs than the GPU has SMs).
//
// CTA: eight warps.  Warps 0-3 are the softmax (thread r = TMEM lane r = row r
// of a tile), which takes the two tiles of a step in turn: half-steps.  In
// warps 4-7 one lane issues the Q loads and the products - S = Q K^T (eight
// tcgen05.mma M 128 N 64 K 16) two half-steps ahead of O += P V (P read from TMEM
// over the S it came from; two S buffers in turn, one O per tile) - and three
// warps decode: 32 keys each for K, all 64 for V, into rings of shared-memory
// stages (128-byte swizzle).  The four roles are turned by one warp in the
// second half of the grid, which spreads the decoding of an SM's two CTAs over
// its schedulers.  The softmax half has 160 registers, the other 96 (setmaxnreg;
// 256 x 128 at launch).
//
// Four roles share an SM's instruction caches, so every loop has one body:
// the same kernel with its loops unrolled and peeled (121 KB of code) spent
// more issue slots waiting for instructions than on anything else.
//
// What bounds it: the chain of a half-step, 2300 cycles: the softmax (TMEM,
// maximum, exponentials, TMEM: 1750, at two warps a scheduler) and the issuing
// lane (1700: twelve products and their commits), each waiting for the other's
// last; V's decoding is busy 3000 of the 4600 of a step, half of the issue slots
// are used, the exponentials take a third of their pipe.  With one tile a step, V's decoding bounded it and
// 512 tokens on 32 K took 200 us where this takes 150.  512 tokens on 8 K: 54.7
// us (paged_prefill over a 16-bit pool: 152 us), of which 18 us do not depend on
// the context (plan, first look-ups, join); six chunks of 1 K: 118 us (181 us);
// 32 requests of 5 tokens: 18.3 us (61 us).  Tried without gain: twelve warps (two
// threads per row, or twice the decoding warps), a third S buffer, one issuing
// warp per kind of product; P through shared memory, which frees S's buffer as
// soon as it is read, cost more than it parted (172 against 150 us on 32 K).
//
// Every mbarrier wait is bounded; no barrier can run two phases ahead of a
// waiter: a stage's next phase needs its own release, the half-steps' barriers
// alternate, and a half-step's buffer is written again only after its products.
#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>

#include "common.cuh"
#include "host_util.h"
#include "int4_attention.h"
#include "int4_cache.cuh"

namespace psb {
namespace {

constexpr int kThreads = 256;
constexpr int kRows = 128;          // rows of a tile
constexpr int kBN = 64;             // keys per step
constexpr int kDim = 64;
constexpr int kKStages = 2, kVStages = 3;
constexpr uint32_t kQTile = kRows * kDim * 2;
constexpr uint32_t kKvTile = kBN * kDim * 2;
constexpr uint32_t kTmemCols = 256;
constexpr uint32_t kSCol = 0, kOCol = 128;
constexpr float kGrowth = 4.f;      // log2 of how far a score may exceed the exponents' reference
constexpr int kPBits = 11;          // probabilities are 2^kPBits p, at most 2^(kPBits + kGrowth)
constexpr float kPUnit = 1.f / (1 << kPBits);
constexpr int kVBits = 9;           // V's codes are (c - 7.5) 2^-kVBits
// Where V's steps go, scaled to below 2^kStepBits: bf16, into V's operand;
// f16, onto the probabilities (below 1, so that those stay below 2^15).
template <typename T>
constexpr bool kStepInV = Elem<T>::code == PSB_BF16;
template <typename T>
constexpr int kStepBits = kStepInV<T> ? 15 : 0;
constexpr int kMaxCtas = 320;       // grid limit
constexpr int kPartFloats = kRows * (kDim + 2);
constexpr int kMaxSeqs = 2048, kMaxPairs = 4096;

// What a V stage's 64 tokens need besides their codes and steps.
struct Extra {
  float mid[kBN];   // mid 2^-kPBits (next to 2^kPBits p); 0 where it is not finite
  float step[kBN];  // scaled; f16 only
  uint32_t bad[2];  // bit t: token t's block is outside the pool
  uint32_t nan[2];  // bit t: token t's mid is not finite
  int vexp;         // steps were scaled by 2^(kStepBits<T> - vexp)
  int pad[3];
};

// dynamic shared memory (1024-byte aligned): Q0 | Q1 | K ring (high, low parts) | V ring | extras | barriers | tables
constexpr uint32_t kOffK = 2 * kQTile, kOffV = kOffK + kKStages * 2 * kKvTile;
constexpr uint32_t kOffX = kOffV + kVStages * kKvTile;
constexpr uint32_t kOffBars = kOffX + kVStages * sizeof(Extra);
constexpr uint32_t kOffTab = kOffBars + 256;

// A pair that several CTAs have a piece of: its kv head, first row of q and
// tokens, and the first and last of the CTAs (first | last << 16; the same: it
// is not cut).  One entry per pair of every kv head where those are fewer than
// the CTAs, else one per CTA, for the pair it leaves unfinished.
struct Cut {
  int32_t kvh, row0, ctas, tokens;
};

struct TcParams {
  Int4PrefillParams a;
  int32_t group, tq;      // q heads per kv head, tokens per tile
  int32_t max_pairs;      // room for the pair table
  int32_t by_pair;        // cuts are kept per pair
  int32_t block_shift;    // block_size is 2^block_shift, or -1
  uint32_t block_div;     // else 2^32 / block_size, rounded up
  int64_t block_rows;     // pool rows from a block to the next
  // scale log2 e as k_sign * scale: K carries the sign (0: a scale of 0), so that
  // the largest S has the largest score
  float k_sign, scale;
  float* part;            // workspace: cuts, then per CTA two pieces of a pair, two tiles each
};

template <int N>
__device__ __forceinline__ void reg_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void reg_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

__device__ __forceinline__ void st_shared_v4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ float4 ld_shared_f4(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float fmax3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}

__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
// Two fp32 values rounded to T, finite ones to the largest finite value at most.
template <typename T>
__device__ __forceinline__ uint32_t pack2_sat(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2_sat<__nv_bfloat16>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <>
__device__ __forceinline__ uint32_t pack2_sat<__half>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// 16 columns of a warp's TMEM lanes.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// mbar_wait with one copy of the instruction.
__device__ __forceinline__ bool wait_at(uint32_t addr, uint32_t parity) {
  uint64_t t0 = 0;
#pragma unroll 1
  while (!mbar_try_wait_sleep(addr, parity, 100000u)) {
    const uint64_t t = globaltimer_ns();
    if (t0 == 0) t0 = t;
    if (t - t0 > kWaitLimitNs) return false;
  }
  return true;
}
// The issuing lane keeps shared addresses and the descriptors' low words (their
// high ones are constant) in 32 bits: it is as busy as the softmax.
__device__ __forceinline__ void commit_at(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ uint64_t desc_of(uint32_t lo, uint32_t hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "r"(hi));
  return d;
}

__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity) { return wait_at(smem_u32(bar), parity); }
// The same for a whole warp: its lanes give up together or not at all.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) {
  return __all_sync(0xffffffffu, wait(bar, parity));
}

// What every role knows of the batch (in shared memory).
struct Plan {
  const int32_t* len;    // [num_seqs] query rows
  const int32_t* ctx;    // [num_seqs] tokens in the pool
  const int32_t* q0;     // [num_seqs] first row
  const int32_t* pfirst; // [num_seqs + 1] pairs before a sequence
  const int32_t* sfirst; // [pairs + 1] steps before a pair, of one kv head
  const int32_t* pseq;   // [pairs] a pair's sequence
  int32_t pairs, tq;
};

__device__ __forceinline__ int last_le(const int32_t* v, int n, int x) {  // last i < n with v[i] <= x
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (v[mid] <= x) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// A run of steps of one pair of tiles.
struct Run {
  int kvh, pair, seq, tok0;  // tok0: the pair's first token in its sequence
  int j0, n;                 // its steps j0 .. j0 + n - 1 of n_kv
  int n_kv;
  bool two;                  // there is a second tile
};

// Walks a CTA's steps pair by pair.
struct Cursor {
  int kvh, pair, j0, left;
  __device__ Run take(const Plan& pl) {  // the next run (left > 0)
    Run s;
    s.kvh = kvh;
    s.pair = pair;
    s.seq = pl.pseq[pair];
    s.tok0 = (pair - pl.pfirst[s.seq]) * 2 * pl.tq;
    s.two = s.tok0 + pl.tq < pl.len[s.seq];
    s.n_kv = pl.sfirst[pair + 1] - pl.sfirst[pair];
    s.j0 = j0;
    s.n = min(s.n_kv - j0, left);
    left -= s.n;
    j0 = 0;
    if (++pair == pl.pairs) {
      pair = 0;
      ++kvh;
    }
    return s;
  }
};

template <typename T>
__global__ void __launch_bounds__(kThreads, 2)
    int4_prefill_tc_kernel(const TcParams tp, const __grid_constant__ CUtensorMap tm_q) {
  extern __shared__ uint8_t smem_raw[];
  // (an offset, so that the compiler still knows it for shared memory)
  uint8_t* const smem = smem_raw + ((0u - smem_u32(smem_raw)) & 1023u);
  const Int4PrefillParams& p = tp.a;
  Extra* const ext = reinterpret_cast<Extra*>(smem + kOffX);
  uint64_t* const bar_q = reinterpret_cast<uint64_t*>(smem + kOffBars);  // a run's Q loaded
  uint64_t* const bar_k = bar_q + 1;          // [kKStages] K decoded (two warps)
  uint64_t* const bar_kfree = bar_k + kKStages;  // [kKStages] Q K^T done
  uint64_t* const bar_v = bar_kfree + kKStages;  // [kVStages] V decoded
  uint64_t* const bar_vfree = bar_v + kVStages;  // [kVStages] P V done
  uint64_t* const bar_s = bar_vfree + kVStages;  // [2]
  uint64_t* const bar_p = bar_s + 2;          // [2]
  uint64_t* const bar_pv = bar_p + 2;         // [2]
  uint64_t* const bar_drain = bar_pv + 2;     // after a failed wait: every product issued so far is done
  uint32_t* const s_tmem = reinterpret_cast<uint32_t*>(bar_drain + 1);
  static_assert((1 + 2 * kKStages + 2 * kVStages + 7) * 8 + 4 <= 256, "barriers fit their area");
  int32_t* const s_len = reinterpret_cast<int32_t*>(smem + kOffTab);
  int32_t* const s_ctx = s_len + p.num_seqs;
  int32_t* const s_q0 = s_ctx + p.num_seqs;
  int32_t* const s_pfirst = s_q0 + p.num_seqs;
  int32_t* const s_sfirst = s_pfirst + p.num_seqs + 1;
  int32_t* const s_pseq = s_sfirst + tp.max_pairs + 1;
  __shared__ int32_t warp_sums[kThreads / 32];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int TQ = tp.tq, group = tp.group, PQ = 2 * TQ;  // tokens of a tile, of a pair
  if (tid == 0) {
    mbar_init(bar_q, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar_s + i, 1);
      mbar_init(bar_p + i, 128);
      mbar_init(bar_pv + i, 1);
    }
    for (int i = 0; i < kKStages; ++i) {
      mbar_init(bar_k + i, 2);
      mbar_init(bar_kfree + i, 1);
    }
    for (int i = 0; i < kVStages; ++i) {
      mbar_init(bar_v + i, 1);
      mbar_init(bar_vfree + i, 1);
    }
    mbar_init(bar_drain, 1);
    fence_barrier_init();
  }
  if (warp == 0) {
    tmem_alloc(s_tmem, kTmemCols);
    tmem_relinquish();
  }
  pdl_wait();  // cu_seqlens, lengths and q may come from the stream predecessor

  // ---- the plan: every CTA builds the same tables ------------------------------
  auto scan = [&](int v, int& total) -> int {  // exclusive over the CTA
    int incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += x;
    }
    if (lane == 31) warp_sums[warp] = incl;
    __syncthreads();
    int run = incl - v;
    total = 0;
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) run += warp_sums[w];
      total += warp_sums[w];
    }
    __syncthreads();
    return run;
  };
  int n_pairs = 0, n_steps = 0;
  {
    const int per = (p.num_seqs + kThreads - 1) / kThreads;
    const int s0 = min(tid * per, p.num_seqs), s1 = min(s0 + per, p.num_seqs);
    int pairs = 0;
    for (int s = s0; s < s1; ++s) {
      const int a = p.cu[s], b = p.cu[s + 1];
      // a malformed batch is reported by the caller's check and read nowhere
      int len = a < 0 || b < a || b > p.total ? 0 : min(b - a, p.max_seqlen);
      int ctx = p.ctx[s];
      if (len > 0 && (ctx < len || ctx > p.max_context)) {
        if (blockIdx.x == 0) flag_error(p.err, PSB_DEVERR_CONTEXT);
        ctx = min(max(ctx, len), p.max_context);
        len = min(len, ctx);
      }
      s_len[s] = len;
      s_ctx[s] = ctx;
      s_q0[s] = a;
      pairs += (len + PQ - 1) / PQ;
    }
    int run = scan(pairs, n_pairs);
    for (int s = s0; s < s1; ++s) {
      s_pfirst[s] = run;
      run += (s_len[s] + PQ - 1) / PQ;
    }
    if (tid == 0) s_pfirst[p.num_seqs] = n_pairs;
    __syncthreads();
    if (n_pairs > tp.max_pairs) {  // rows named by two sequences: a malformed batch
      if (tid == 0) flag_error(p.err, PSB_DEVERR_SEQLENS);
      n_pairs = 0;
    }
    const int tper = (n_pairs + kThreads - 1) / kThreads;
    const int t0 = min(tid * tper, n_pairs), t1 = min(t0 + tper, n_pairs);
    int steps = 0;
    for (int t = t0; t < t1; ++t) {
      const int s = last_le(s_pfirst, p.num_seqs, t), qt = t - s_pfirst[s];
      // keys 0 .. position of the pair's last row
      const int n = (s_ctx[s] - s_len[s] + min(s_len[s], (qt + 1) * PQ) + kBN - 1) / kBN;
      s_sfirst[t] = n;
      s_pseq[t] = s;
      steps += n;
    }
    run = scan(steps, n_steps);
    for (int t = t0; t < t1; ++t) {
      const int n = s_sfirst[t];
      s_sfirst[t] = run;
      run += n;
    }
    if (tid == 0) s_sfirst[n_pairs] = n_steps;
    __syncthreads();
  }
  const Plan plan{s_len, s_ctx, s_q0, s_pfirst, s_sfirst, s_pseq, n_pairs, TQ};
  const uint32_t total_steps = static_cast<uint32_t>(n_steps) * p.hkv;  // below 2^31
  const uint32_t act = min(gridDim.x, total_steps);
  Cut* const cuts = reinterpret_cast<Cut*>(tp.part);
  float* const part = tp.part + kMaxCtas * (sizeof(Cut) / sizeof(float));
  const uint32_t cta = blockIdx.x;
  if (tp.by_pair && cta == 0) {  // entries of pairs there is room for but that do not exist
    const int spare = tp.max_pairs - n_pairs;
    for (int i = tid; i < spare * p.hkv; i += kThreads)
      cuts[(i / spare) * tp.max_pairs + n_pairs + i % spare] = Cut{0, 0, 0, 0};
  }
  if (cta >= act) {
    if (!tp.by_pair && tid == 0) cuts[cta] = Cut{0, 0, 0, 0};
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {  // nothing to do but to give the columns back
      tc_fence_after();
      tmem_dealloc(*s_tmem, kTmemCols);
    }
    return;
  }
  const uint32_t share = total_steps / act, extra = total_steps - share * act;
  auto cta_start = [&](uint32_t c) -> uint32_t { return share * c + min(c, extra); };
  const uint32_t my_a = cta_start(cta), my_e = cta_start(cta + 1);
  const int n_mine = static_cast<int>(my_e - my_a);
  Cursor first;
  first.kvh = static_cast<int>(my_a / n_steps);
  first.j0 = static_cast<int>(my_a - static_cast<uint32_t>(first.kvh) * n_steps);
  first.pair = last_le(s_sfirst, n_pairs, first.j0);
  first.j0 -= s_sfirst[first.pair];
  first.left = n_mine;
  const uint32_t s_base = smem_u32(smem);

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;
  pdl_launch_dependents();
  bool fail = false;

  if (warp >= 4) {
    reg_dec<96>();
    // roles of warps 4-7: issue, decode K rows 0-31, decode V, decode K rows 32-63
    const int role = (warp - 4 + (cta >= (gridDim.x + 1) / 2 ? 1 : 0)) & 3;
    if (role == 0) {
      if (lane == 0) {
        const uint32_t idesc_s = umma_idesc_f16(Elem<T>::code == PSB_BF16 ? 1 : 0, kRows, kBN, 0, 0);
        const uint32_t idesc_o = umma_idesc_f16(0, kRows, kDim, 0, 1);
        const uint64_t dq = umma_desc_sw128(s_base, 1024, 16);
        const uint64_t dk = umma_desc_sw128(s_base + kOffK, 1024, 16);
        const uint64_t dv = umma_desc_sw128(s_base + kOffV, 1024, 8192);
        prefetch_tmap(&tm_q);
        // Half-steps (a step of one tile), in order: a step's first tile, its
        // second.  Number i uses S buffer i & 1 (b8: 8 times that, ph: the
        // parity of its use, i >> 1).  S runs two half-steps ahead of O.
        const uint32_t a_q = smem_u32(bar_q), a_k = smem_u32(bar_k), a_kfree = smem_u32(bar_kfree), a_v = smem_u32(bar_v),
                       a_vfree = smem_u32(bar_vfree), a_s = smem_u32(bar_s), a_p = smem_u32(bar_p), a_pv = smem_u32(bar_pv);
        const uint32_t qlo = static_cast<uint32_t>(dq), klo = static_cast<uint32_t>(dk), vlo = static_cast<uint32_t>(dv);
        const uint32_t shi = static_cast<uint32_t>(dk >> 32), vhi = static_cast<uint32_t>(dv >> 32);  // (Q's and K's are alike)
        const uint32_t box = static_cast<uint32_t>(TQ * group) * kDim * 2;
        Cursor sc = first, oc = first;
        int s_left = 0, o_left = 0;     // steps left of the runs of S and O
        uint32_t s_two = 0, o_two = 0;  // whether they have a second tile
        uint32_t sh = 0, oh = 0;        // tile of the step
        uint32_t k_st = 0, k_ph = 0, v_st = 0, v_ph = 0, q_ph = 1, b8 = 0, ph = 1;
        bool begins = false, s_more = true, started = false;
        bool q_flight = false;          // a copy of Q is on its way
#pragma unroll 1
        for (int i = -2;; ++i) {
          if (i >= 0) {  // P V of half-step i
            if (oh == 0) {
              if (o_left == 0) {
                if (oc.left == 0) break;
                const Run r = oc.take(plan);
                o_left = r.n;
                o_two = r.two;
                begins = true;
              }
              if (!wait_at(a_v + 8 * v_st, v_ph)) {
                fail = true;
                break;
              }
            }
            if (!wait_at(a_p + b8, ph)) {
              fail = true;
              break;
            }
            tc_fence_after();
            const uint32_t pcol = tmem + kSCol + 8 * b8, ocol = tmem + kOCol + oh * kDim, vd = vlo + v_st * (kKvTile >> 4);
#pragma unroll
            for (int kk = 0; kk < kBN / 16; ++kk)
              umma_f16_ts(ocol, pcol + 8 * kk, desc_of(vd + 128 * kk, vhi), idesc_o, !begins || kk > 0);
            commit_at(a_pv + b8);
            if (oh == o_two) {
              commit_at(a_vfree + 8 * v_st);
              oh = 0;
              if (++v_st == kVStages) {
                v_st = 0;
                v_ph ^= 1;
              }
              --o_left;
              begins = false;
            } else {
              oh = 1;
            }
          }
          if (s_more) {  // S of half-step i + 2, whose buffer held S and then P of half-step i
            if (i >= 0 && !wait_at(a_pv + b8, ph)) {
              fail = true;
              break;
            }
            if (sh == 0) {
              if (s_left == 0) {  // a run begins: its Q, once the last S of the run before is done
                const Run r = sc.take(plan);
                s_left = r.n;
                s_two = r.two;
                if (started && !wait_at(a_s + (b8 ^ 8), b8 == 0 ? ph : ph ^ 1)) {
                  fail = true;
                  break;
                }
                started = true;
                mbar_arrive_expect_tx(bar_q, box << s_two);
                const int row0 = plan.q0[r.seq] + r.tok0;
                tma_load_3d(smem, &tm_q, 0, r.kvh * group, row0, bar_q);
                if (r.two) tma_load_3d(smem + kQTile, &tm_q, 0, r.kvh * group, row0 + TQ, bar_q);
                q_ph ^= 1;
                q_flight = true;
                if (!wait_at(a_q, q_ph)) {
                  fail = true;
                  break;
                }
                q_flight = false;
              }
              if (!wait_at(a_k + 8 * k_st, k_ph)) {
                fail = true;
                break;
              }
            }
            tc_fence_after();
            const uint32_t scol = tmem + kSCol + 8 * b8, qd = qlo + sh * (kQTile >> 4), kd = klo + k_st * (2 * kKvTile >> 4);
#pragma unroll
            for (int kk = 0; kk < 2 * kDim / 16; ++kk)  // the values rounded to T, then their rests
              umma_f16_ss(scol, desc_of(qd + 2 * (kk & 3), shi), desc_of(kd + (kk >> 2) * (kKvTile >> 4) + 2 * (kk & 3), shi),
                          idesc_s, kk > 0);
            commit_at(a_s + b8);
            if (sh == s_two) {
              commit_at(a_kfree + 8 * k_st);
              sh = 0;
              if (++k_st == kKStages) {
                k_st = 0;
                k_ph ^= 1;
              }
              --s_left;
              s_more = s_left > 0 || sc.left > 0;
            } else {
              sh = 1;
            }
          }
          b8 ^= 8;
          if (b8 == 0) ph ^= 1;
        }
        if (fail) {
          flag_error(p.err, PSB_DEVERR_TIMEOUT);
          // let the copies and products in flight land before shared memory and TMEM are released
          if (q_flight) (void)wait_at(a_q, q_ph);
          umma_commit(bar_drain);
          (void)wait(bar_drain, 0);
        }
      }
    } else {
      // ---- decode: lane l of a K warp takes one row of a step's 64 keys, of the V warp rows l and l + 32 ----
      // The block id of a row is looked up two steps, its codes are loaded one
      // step ahead of their decoding.
      Cursor cc = first;
      int left = 0, pos0 = 0, ctx = 0;  // of the run being looked up: steps left, first key of the next, tokens
      const int32_t* row = nullptr;
      int64_t row0 = 0;  // pool row of token 0 of block 0, K
      auto next_run = [&]() {
        const Run s = cc.take(plan);
        pos0 = s.j0 * kBN;
        left = s.n;
        row = p.tables + static_cast<int64_t>(s.seq) * p.table_stride;
        ctx = plan.ctx[s.seq];
        row0 = int4_row(p.layer_tiles + s.kvh, 0, 0, p.block_size);
      };
      // row r's place in the pool (-1: past the sequence, -2: its block is outside the pool)
      auto place = [&](int r, int kv) -> int64_t {
        const uint32_t pos = pos0 + r;
        if (static_cast<int>(pos) >= ctx) return -1;
        const uint32_t bi = tp.block_shift >= 0 ? pos >> tp.block_shift : __umulhi(pos, tp.block_div);
        const int blk = __ldg(row + bi);
        if (blk < 0 || blk >= p.num_blocks) return -2;
        return row0 + blk * tp.block_rows + (kv * p.block_size + pos - bi * p.block_size);
      };
      struct Row {
        uint4 c[2];
        uint32_t par;
      };
      auto load = [&](Row& r, int64_t at) {
        r.c[0] = r.c[1] = make_uint4(0, 0, 0, 0);
        r.par = 0;
        if (at >= 0) {
          const uint4* src = reinterpret_cast<const uint4*>(p.codes + at * (kDim / 2));
          r.c[0] = __ldg(src);
          r.c[1] = __ldg(src + 1);
          r.par = __ldg(reinterpret_cast<const uint32_t*>(p.params) + at);
        }
      };
      if (role != 2) {
        const int r = lane + (role == 3 ? 32 : 0);
        const uint32_t dst = s_base + kOffK + r * 128;
        Row cur, nxt{};
        int64_t at = -1;
#pragma unroll 1
        for (int i = 0; i < n_mine + 2; ++i) {
          cur = nxt;
          load(nxt, at);
          at = -1;
          if (i < n_mine) {
            if (left == 0) next_run();
            at = place(r, 0);
            pos0 += kBN;
            --left;
          }
          const int g = i - 2;
          if (g < 0) continue;
          const int st = g % kKStages;
          if (g >= kKStages && !warp_wait(bar_kfree + st, (g / kKStages - 1) & 1)) {
            fail = true;
            break;
          }
          // value = step (c - 8) + (mid + step / 2); its rounding to T and the rest
          const float2 pr = unpack2<T>(cur.par);
          const float base = fmaf(pr.x, 0.5f, pr.y) * tp.k_sign, step = pr.x * tp.k_sign;
          const uint64_t st2 = f2_pack(step, step), base2 = f2_pack(base, base), minus = f2_pack(-1.f, -1.f);
          const uint64_t off2 = f2_pack(-8388616.f, -8388616.f);  // - (2^23 + 8)
          const uint32_t tile = dst + st * 2 * kKvTile;
#pragma unroll 1
          for (int h = 0; h < 2; ++h) {
            const uint4 q = h == 0 ? cur.c[0] : cur.c[1];
            const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const uint32_t t = w[c] & 0x0f0f0f0fu, u = (w[c] >> 4) & 0x0f0f0f0fu;
              uint32_t hi[4], lo[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {  // elements 2 e and 2 e + 1 of the word: 2^23 + c
                const uint64_t cc2 = f2_pack(__uint_as_float(__byte_perm(t, 0x4b000000u, 0x7440 | e)),
                                             __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7440 | e)));
                const uint64_t v = f2_fma(f2_add(cc2, off2), st2, base2);
                const float2 vf = f2_unpack(v);
                hi[e] = pack2_sat<T>(vf.x, vf.y);
                const float2 hf = unpack2<T>(hi[e]);
                const float2 rest = f2_unpack(f2_fma(f2_pack(hf.x, hf.y), minus, v));
                lo[e] = pack2<T>(rest.x, rest.y);
              }
              const uint32_t to = tile + (((4 * h + c) ^ (r & 7)) << 4);
              st_shared_v4(to, hi[0], hi[1], hi[2], hi[3]);
              st_shared_v4(to + kKvTile, lo[0], lo[1], lo[2], lo[3]);
            }
          }
          fence_proxy_async_smem();  // visible to the tensor core
          __syncwarp();
          if (lane == 0) mbar_arrive(bar_k + st);
        }
      } else {
        Row cur0, cur1, nxt0{}, nxt1{};
        int64_t at0 = -1, at1 = -1;
        uint32_t f_cur = 0, f_nxt = 0, f_at = 0;  // bits 0, 1: the row's block is outside the pool; 2: a run's first step
        int vexp = 0;
        float vlim = 0.f, vscale = 1.f;
#pragma unroll 1
        for (int i = 0; i < n_mine + 2; ++i) {
          cur0 = nxt0;
          cur1 = nxt1;
          f_cur = f_nxt;
          load(nxt0, at0);
          load(nxt1, at1);
          f_nxt = f_at;
          at0 = at1 = -1;
          f_at = 0;
          if (i < n_mine) {
            if (left == 0) {
              next_run();
              f_at = 4;
            }
            at0 = place(lane, 1);
            at1 = place(lane + 32, 1);
            f_at |= (at0 == -2 ? 1u : 0u) | (at1 == -2 ? 2u : 0u);
            pos0 += kBN;
            --left;
          }
          const int g = i - 2;
          if (g < 0) continue;
          const int st = g % kVStages;
          if (g >= kVStages && !warp_wait(bar_vfree + st, (g / kVStages - 1) & 1)) {
            fail = true;
            break;
          }
          Extra& x = ext[st];
          const float2 p0 = unpack2<T>(cur0.par), p1 = unpack2<T>(cur1.par);
          if (f_cur & 4) {
            vlim = 0.f;
            vexp = 0;
            vscale = 1.f;
          }
          if (__any_sync(0xffffffffu, fmaxf(p0.x, p1.x) > vlim)) {
            float top = fmaxf(p0.x, p1.x);
#pragma unroll 1
            for (int d = 1; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            vexp = max(-100, ilogb_f32(top)) + 1;  // top < 2^vexp
            vlim = exp2_int(min(vexp, 127));
            vscale = exp2_int(max(-126, kStepBits<T> - vexp));
          }
          const bool fin0 = finite_f32(p0.y), fin1 = finite_f32(p1.y);
          x.mid[lane] = fin0 ? p0.y * kPUnit : 0.f;
          x.mid[lane + 32] = fin1 ? p1.y * kPUnit : 0.f;
          if constexpr (!kStepInV<T>) {
            x.step[lane] = p0.x * vscale;
            x.step[lane + 32] = p1.x * vscale;
          }
          const uint32_t bad0 = __ballot_sync(0xffffffffu, f_cur & 1), bad1 = __ballot_sync(0xffffffffu, f_cur & 2);
          const uint32_t nan0 = __ballot_sync(0xffffffffu, !fin0), nan1 = __ballot_sync(0xffffffffu, !fin1);
          if (lane == 0) {
            x.bad[0] = bad0;
            x.bad[1] = bad1;
            x.nan[0] = nan0;
            x.nan[1] = nan1;
            x.vexp = vexp;
            if (bad0 | bad1) flag_error(p.err, PSB_DEVERR_BLOCK_RANGE);
          }
          // codes in f16: the nibble pairs (i, i + 4) are the subnormals
          // c 2^-24 (even i) and c 2^-20 (odd i), which one exact fma turns into
          // (c - 7.5) 2^-9; element 8 w + i + 4 h of a row sits at 8 w + 2 i + h
          const uint32_t tile = s_base + kOffV + st * kKvTile + lane * 128;
#pragma unroll 1
          for (int h = 0; h < 4; ++h) {  // row h / 2, half h & 1
            const uint4 q = h == 0 ? cur0.c[0] : h == 1 ? cur0.c[1] : h == 2 ? cur1.c[0] : cur1.c[1];
            const float stf = (h < 2 ? p0.x : p1.x) * vscale;
            const uint32_t st2 = pack2<__half>(stf, stf);
            auto scaled = [&](uint32_t v) { return kStepInV<T> ? hmul2(v, st2) : v; };
            const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const uint32_t a = w[c], b = a >> 8;
              // 2^15, 2^11 and - 7.5 / 512 as f16 pairs
              st_shared_v4(tile + (h >> 1) * (32 * 128) + (((4 * (h & 1) + c) ^ (lane & 7)) << 4),
                           scaled(hfma2(a & 0x000f000fu, 0x78007800u, 0xa380a380u)),
                           scaled(hfma2(a & 0x00f000f0u, 0x68006800u, 0xa380a380u)),
                           scaled(hfma2(b & 0x000f000fu, 0x78007800u, 0xa380a380u)),
                           scaled(hfma2(b & 0x00f000f0u, 0x68006800u, 0xa380a380u)));
            }
          }
          fence_proxy_async_smem();  // visible to the tensor core
          __syncwarp();
          if (lane == 0) mbar_arrive(bar_v + st);
        }
      }
      if (fail && lane == 0) flag_error(p.err, PSB_DEVERR_TIMEOUT);
    }
  } else {
    reg_inc<160>();
    // ---- softmax warps ------------------------------------------------------
    const int row = warp * 32 + lane;
    const int rtok = row / group, rhead = row - rtok * group;
    const uint32_t t_lane = tmem + (static_cast<uint32_t>(warp * 32) << 16);
    const bool out16 = reinterpret_cast<uintptr_t>(p.out) % 16 == 0 && p.ost % 8 == 0 && p.osh % 8 == 0;
    // Per tile: the exponents' reference; sums of 2^kPBits p and p mid; the last
    // key of this row, from the step's first.  The tile at work is in the plain
    // names, the other in the rest; a step's end swaps them.
    float ref = 0.f, l = 0.f, z = 0.f, ref_o = 0.f, l_o = 0.f, z_o = 0.f;
    int last = 0, last_o = 0, vexp = 0, vexp_o = 0;
    bool fresh = true, fresh_o = true;
    auto swap_tiles = [&]() {
      auto sw = [](auto& a, auto& b) {
        auto c = a;
        a = b;
        b = c;
      };
      sw(ref, ref_o);
      sw(l, l_o);
      sw(z, z_o);
      sw(last, last_o);
      sw(vexp, vexp_o);
      sw(fresh, fresh_o);
    };
    Cursor cc = first;
    Run s{};
    int g = 0, i = 0;  // step, half-step
#pragma unroll 1
    while (cc.left > 0 && !fail) {
      s = cc.take(plan);
      const int tiles = s.two ? 2 : 1, len = plan.len[s.seq], start = plan.ctx[s.seq] - len - s.j0 * kBN;
      // rows past a tile's tokens are not written: they need no mask
      const int tok = s.tok0 + rtok;
      last = rtok < TQ && tok < len ? start + tok : INT_MAX;
      last_o = rtok < TQ && tok + TQ < len ? start + tok + TQ : INT_MAX;
      ref = l = z = ref_o = l_o = z_o = 0.f;
      fresh = fresh_o = true;
      vexp = vexp_o = 0;
#pragma unroll 1
      for (int hs = 0; hs < s.n * tiles; ++hs, ++i) {
        const int h = s.two ? hs & 1 : 0, st = g % kVStages;
        if (!warp_wait(bar_s + (i & 1), (i >> 1) & 1) || (h == 0 && !warp_wait(bar_v + st, (g / kVStages) & 1))) {
          fail = true;
          break;
        }
        tc_fence_after();
        const uint32_t t_s = t_lane + kSCol + (i & 1) * kBN, t_o = t_lane + kOCol + h * kDim;
        const Extra& f = ext[st];
        const uint4 odd = *reinterpret_cast<const uint4*>(f.bad);  // bad, nan
        const int ve = f.vexp;
        uint32_t sr[kBN];
        tmem_ld32(t_s, sr);
        tmem_ld32(t_s + 32, sr + 32);
        tmem_wait_ld();
        // bit c: the row sees key c of the step
        const uint32_t seen0 = last >= 31 ? ~0u : last < 0 ? 0u : (2u << last) - 1;
        const uint32_t seen1 = last >= 63 ? ~0u : last < 32 ? 0u : (2u << (last - 32)) - 1;
        const uint32_t ok0 = seen0 & ~odd.x, ok1 = seen1 & ~odd.y;
        if ((ok0 & ok1) != ~0u) {
#pragma unroll
          for (int c = 0; c < kBN; ++c)
            if (!((c < 32 ? ok0 : ok1) >> (c & 31) & 1)) sr[c] = __float_as_uint(-INFINITY);
        }
        float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
        for (int c = 0; c < kBN; c += 4) {
          mx0 = fmax3(mx0, __uint_as_float(sr[c]), __uint_as_float(sr[c + 1]));
          mx1 = fmax3(mx1, __uint_as_float(sr[c + 2]), __uint_as_float(sr[c + 3]));
        }
        // exponents are scores minus reference, plus kPBits
        const float mx = fmaf(fmaxf(mx0, mx1), tp.scale, kPBits - ref);
        // A row's reference moves when a score is above it by more than the
        // limit, or at its first score; O is rescaled then, or when the scale
        // of V's steps changed.  The warp's TMEM access is collective.
        const bool begins = hs < tiles;
        const bool grow = mx > (fresh ? -INFINITY : kGrowth + kPBits);
        if (__any_sync(0xffffffffu, grow) || (!begins && ve != vexp)) {
          const float up = grow ? fminf(fmaxf(mx - kPBits, -3e38f), 3e38f) : 0.f;
          const float al = grow ? (fresh ? 0.f : ex2_approx(-up)) : 1.f;
          if (!begins) {  // O holds P V of the earlier steps once the last of them is done
            const int before = i - tiles;  // the tile's last half-step
            if (!warp_wait(bar_pv + (before & 1), (before >> 1) & 1)) {
              fail = true;
              break;
            }
            tc_fence_after();
            const float ao = al * exp2_int(max(-126, vexp - ve));
#pragma unroll 1
            for (int h = 0; h < 4; ++h) {
              uint32_t ot[16];
              tmem_ld16(t_o + 16 * h, ot);
              tmem_wait_ld();
#pragma unroll
              for (int d = 0; d < 16; ++d) ot[d] = __float_as_uint(__uint_as_float(ot[d]) * ao);
              tmem_st16(t_o + 16 * h, ot);
            }
            tmem_wait_st();
          }
          l *= al;
          z *= al;
          ref += up;
          fresh = fresh && !grow;
        }
        vexp = ve;
        uint32_t pk[kBN / 2];
        uint64_t l2 = f2_pack(0.f, 0.f), z2 = f2_pack(0.f, 0.f);
        const uint64_t scale2 = f2_pack(tp.scale, tp.scale), nref2 = f2_pack(kPBits - ref, kPBits - ref);
#pragma unroll
        for (int c = 0; c < kBN; c += 4) {
          const float4 vm = ld_shared_f4(f.mid + c);
          const float2 xa = f2_unpack(f2_fma(f2_pack(__uint_as_float(sr[c]), __uint_as_float(sr[c + 1])), scale2, nref2));
          const float2 xb = f2_unpack(f2_fma(f2_pack(__uint_as_float(sr[c + 2]), __uint_as_float(sr[c + 3])), scale2, nref2));
          const float a0 = ex2_approx(xa.x), a1 = ex2_approx(xa.y), b0 = ex2_approx(xb.x), b1 = ex2_approx(xb.y);
          const uint64_t a = f2_pack(a0, a1), b = f2_pack(b0, b1);
          l2 = f2_add(l2, f2_add(a, b));
          z2 = f2_fma(a, f2_pack(vm.x, vm.y), z2);
          z2 = f2_fma(b, f2_pack(vm.z, vm.w), z2);
          if constexpr (kStepInV<T>) {
            pk[c / 2] = pack2<__half>(a0, a1);
            pk[c / 2 + 1] = pack2<__half>(b0, b1);
          } else {
            const float4 vs = ld_shared_f4(f.step + c);
            const float2 pa = f2_unpack(f2_mul(a, f2_pack(vs.x, vs.y))), pb = f2_unpack(f2_mul(b, f2_pack(vs.z, vs.w)));
            pk[c / 2] = pack2<__half>(pa.x, pa.y);
            pk[c / 2 + 1] = pack2<__half>(pb.x, pb.y);
          }
        }
        const float2 lf = f2_unpack(l2), zf = f2_unpack(z2);
        l += lf.x + lf.y;
        z += zf.x + zf.y;
        // a token that stands for NaN: for the rows that see it
        if (((odd.z & seen0) | (odd.w & seen1)) != 0) z = __int_as_float(0x7fffffff);
        tmem_st32(t_s, pk);
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(bar_p + (i & 1));
        last -= kBN;
        if (h == tiles - 1) ++g;
        if (s.two) swap_tiles();
      }
      // the run's output, a tile at a time
      const bool whole = s.n == s.n_kv;
#pragma unroll 1
      for (int h = 0; h < tiles && !fail; ++h) {
        const int at = i - tiles + h;  // the tile's last half-step
        if (!warp_wait(bar_pv + (at & 1), (at >> 1) & 1)) {
          fail = true;
          break;
        }
        tc_fence_after();
        const int tok_h = tok + h * TQ;
        const bool live = rtok < TQ && tok_h < len;
        const float back = exp2_int(max(-126, min(127, vexp - kStepBits<T> + kVBits - kPBits)));  // of one unit of O
        const float sum = l * kPUnit;
        const float inv = !whole ? 1.f : sum == 0.f ? 0.f : 1.f / sum;
        const float scale = back * inv, base = z * inv;
        float* const dst = part + static_cast<int64_t>(4 * cta + (s.j0 > 0 ? 0 : 2) + h) * kPartFloats;
        T* const out = reinterpret_cast<T*>(p.out) + static_cast<int64_t>(plan.q0[s.seq] + tok_h) * p.ost +
                       static_cast<int64_t>(s.kvh * group + rhead) * p.osh;
#pragma unroll 1
        for (int q = 0; q < 4; ++q) {
          uint32_t ot[16];
          tmem_ld16(t_lane + kOCol + h * kDim + 16 * q, ot);
          tmem_wait_ld();
          float o[16];
#pragma unroll
          for (int w = 0; w < 2; ++w) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {  // columns 2 e, 2 e + 1 of a word are its elements e, e + 4
              o[8 * w + e] = fmaf(__uint_as_float(ot[8 * w + 2 * e]), scale, base);
              o[8 * w + e + 4] = fmaf(__uint_as_float(ot[8 * w + 2 * e + 1]), scale, base);
            }
          }
          if (live && !whole) {
#pragma unroll
            for (int d = 0; d < 16; d += 4)
              *reinterpret_cast<float4*>(dst + row * kDim + 16 * q + d) = make_float4(o[d], o[d + 1], o[d + 2], o[d + 3]);
          } else if (live && out16) {
#pragma unroll
            for (int d = 0; d < 16; d += 8)
              *reinterpret_cast<uint4*>(out + 16 * q + d) = make_uint4(pack2<T>(o[d], o[d + 1]), pack2<T>(o[d + 2], o[d + 3]),
                                                                       pack2<T>(o[d + 4], o[d + 5]), pack2<T>(o[d + 6], o[d + 7]));
          } else if (live) {
#pragma unroll
            for (int d = 0; d < 16; ++d) out[16 * q + d] = Elem<T>::from_float(o[d]);
          }
          __syncwarp();  // the next read of TMEM is the whole warp's
        }
        if (!whole) *reinterpret_cast<float2*>(dst + kRows * kDim + 2 * row) = make_float2(fresh ? -INFINITY : ref, sum);
        if (s.two) swap_tiles();
      }
      tc_fence_before();  // the next run's first P V comes after its P
    }
    if (fail && lane == 0) flag_error(p.err, PSB_DEVERR_TIMEOUT);
    if (warp == 0) {
      // the pair that begins here and runs past the CTA's end, if any: the last run
      Cut c{0, 0, 0, 0};
      const uint32_t t_e = my_e - static_cast<uint32_t>(s.j0 + s.n) + static_cast<uint32_t>(s.n_kv);
      if (!fail && s.j0 == 0 && t_e > my_e) {
        uint32_t c1 = cta;
        for (uint32_t c0 = cta + 1; c0 < act; c0 += 32) {  // CTAs that start before its end
          const bool in = c0 + lane < act && cta_start(min(c0 + lane, act)) < t_e;
          const int n = __popc(__ballot_sync(0xffffffffu, in));
          c1 += n;
          if (n < 32) break;
        }
        c = Cut{s.kvh, s_q0[s.seq] + s.tok0, static_cast<int32_t>(cta | c1 << 16), min(PQ, s_len[s.seq] - s.tok0)};
      }
      if (lane == 0) {
        if (!tp.by_pair) {
          cuts[cta] = c;
        } else {  // the pairs that begin here: whole ones, and the last
          cc = first;
          while (cc.left > 0) {
            const Run r = cc.take(plan);
            if (r.j0 == 0) cuts[r.kvh * tp.max_pairs + r.pair] = cc.left > 0 ? Cut{0, 0, 0, 0} : c;
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// Joins the partials of the pair in entry blockIdx.x: kCombineRows of a tile's
// rows per CTA, kWarpRows rows per warp, two elements a lane, kBatch partials
// in flight (they come from L2: a round of loads costs more than their bytes).
constexpr int kCombineThreads = 256, kCombineRows = 16, kWarpRows = kCombineRows / (kCombineThreads / 32), kBatch = 8;

template <typename T>
__global__ void __launch_bounds__(kCombineThreads) int4_prefill_combine_kernel(const TcParams tp) {
  const Int4PrefillParams& p = tp.a;
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int4 cut = __ldcg(reinterpret_cast<const int4*>(tp.part) + blockIdx.x);
  const int c0 = cut.z & 0xffff, c1 = cut.z >> 16;
  const int tile = blockIdx.z, tokens = cut.w - tile * tp.tq;  // tokens from the tile's first on
  const int row0 = blockIdx.y * kCombineRows + (threadIdx.x >> 5) * kWarpRows;
  if (c1 <= c0 || row0 >= min(tokens, tp.tq) * tp.group) return;
  const float* const part = tp.part + kMaxCtas * (sizeof(Cut) / sizeof(float));
  auto piece_of = [&](int c) { return part + static_cast<int64_t>(4 * c + (c == c0 ? 2 : 0) + tile) * kPartFloats; };
  float m[kWarpRows], l[kWarpRows];
  float2 o[kWarpRows];
#pragma unroll
  for (int r = 0; r < kWarpRows; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
    o[r] = make_float2(0.f, 0.f);
  }
  for (int c = c0; c <= c1; c += kBatch) {
    float2 ml[kBatch][kWarpRows], v[kBatch][kWarpRows];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
#pragma unroll
      for (int r = 0; r < kWarpRows; ++r) {
        ml[j][r] = make_float2(-INFINITY, 0.f);
        v[j][r] = make_float2(0.f, 0.f);
        if (c + j <= c1) {
          const float* pc = piece_of(c + j);
          ml[j][r] = __ldcg(reinterpret_cast<const float2*>(pc + kRows * kDim + 2 * (row0 + r)));
          v[j][r] = __ldcg(reinterpret_cast<const float2*>(pc + (row0 + r) * kDim) + lane);
        }
      }
    }
#pragma unroll
    for (int r = 0; r < kWarpRows; ++r) {
      float mn = m[r];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) mn = fmaxf(mn, ml[j][r].x);
      const float mu = mn == -INFINITY ? 0.f : mn, a = ex2_approx(m[r] - mu);
      m[r] = mn;
      l[r] *= a;
      o[r].x *= a;
      o[r].y *= a;
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const float w = ex2_approx(ml[j][r].x - mu);
        l[r] = fmaf(ml[j][r].y, w, l[r]);
        o[r].x = fmaf(v[j][r].x, w, o[r].x);
        o[r].y = fmaf(v[j][r].y, w, o[r].y);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < kWarpRows; ++r) {
    const int rtok = (row0 + r) / tp.group, rhead = row0 + r - rtok * tp.group;
    if (rtok >= min(tokens, tp.tq)) continue;
    const float inv = l[r] == 0.f ? 0.f : 1.f / l[r];
    T* out = reinterpret_cast<T*>(p.out) + static_cast<int64_t>(cut.y + tile * tp.tq + rtok) * p.ost +
             static_cast<int64_t>(cut.x * tp.group + rhead) * p.osh + 2 * lane;
    out[0] = Elem<T>::from_float(o[r].x * inv);
    out[1] = Elem<T>::from_float(o[r].y * inv);
  }
}

size_t tc_smem(int num_seqs, int max_pairs) {
  return 1024 + kOffTab + sizeof(int32_t) * (4 * static_cast<size_t>(num_seqs) + 1 + 2 * static_cast<size_t>(max_pairs) + 1);
}

int64_t pairs_bound(int total, int num_seqs, int tq) { return static_cast<int64_t>(total) / (2 * tq) + num_seqs; }

// An upper bound of the CTAs: of the steps, or the grid's limit.
int64_t ctas_bound(int total, int num_seqs, int tq, int hkv, int max_context) {
  return std::min<int64_t>(std::max<int64_t>(1, pairs_bound(total, num_seqs, tq) * hkv * ((max_context + kBN - 1) / kBN)),
                           kMaxCtas);
}

}  // namespace

bool int4_prefill_tc_geometry(int dtype, int total, int num_seqs, int q_heads, int hkv, int head_dim, int block_size,
                              int max_context) {
  const int group = q_heads / hkv;
  if (!(dtype == PSB_BF16 || dtype == PSB_F16) || head_dim != kDim || group > kRows) return false;
  const int64_t pairs = pairs_bound(total, num_seqs, kRows / group);
  return num_seqs <= kMaxSeqs && pairs <= kMaxPairs &&
         static_cast<int64_t>(max_context + kBN) * block_size < (int64_t(1) << 32) &&
         pairs * (max_context / kBN + 1) < (int64_t(1) << 31) / hkv;
}

size_t int4_prefill_tc_workspace(int total, int num_seqs, int q_heads, int hkv, int max_context) {
  return sizeof(Cut) * kMaxCtas +
         sizeof(float) * 4 * kPartFloats * static_cast<size_t>(ctas_bound(total, num_seqs, kRows / (q_heads / hkv), hkv, max_context));
}

int int4_prefill_tc_launch(const Int4PrefillParams& p, int dtype, float* workspace, cudaStream_t s) {
  TcParams tp;
  tp.a = p;
  tp.group = p.hq / p.hkv;
  tp.tq = kRows / tp.group;
  tp.max_pairs = static_cast<int32_t>(pairs_bound(p.total, p.num_seqs, tp.tq));
  tp.block_shift = -1;
  if ((p.block_size & (p.block_size - 1)) == 0)
    for (tp.block_shift = 0; (1 << tp.block_shift) < p.block_size;) ++tp.block_shift;
  tp.block_div = tp.block_shift >= 0 ? 0 : static_cast<uint32_t>(((uint64_t(1) << 32) + p.block_size - 1) / p.block_size);
  tp.block_rows = static_cast<int64_t>(p.hkv) * 2 * p.block_size;
  tp.k_sign = p.scale_log2 > 0.f ? 1.f : p.scale_log2 < 0.f ? -1.f : p.scale_log2;  // (a NaN stays)
  tp.scale = p.scale_log2 == 0.f ? 1.f : std::fabs(p.scale_log2);
  tp.part = workspace;
  CUtensorMap tq;
  if (!encode_row_groups_map(&tq, p.q, p.total, p.hq, kDim, p.qst, p.qsh, tp.group, tp.tq,
                             dtype == PSB_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16))
    return PSB_ERR_CUDA;
  const int sms = device_sm_count();
  if (sms <= 0) return PSB_ERR_CUDA;
  const auto kern = dtype == PSB_BF16 ? int4_prefill_tc_kernel<__nv_bfloat16> : int4_prefill_tc_kernel<__half>;
  const auto comb = dtype == PSB_BF16 ? int4_prefill_combine_kernel<__nv_bfloat16> : int4_prefill_combine_kernel<__half>;
  const size_t smem = tc_smem(p.num_seqs, tp.max_pairs);
  // the register split draws on what the block was launched with
  static_assert(160 + 96 == 2 * 128, "two warpgroups' shares");
  static std::atomic<bool> checked[2];  // per element type
  if (!checked[dtype == PSB_BF16].load(std::memory_order_relaxed)) {
    cudaFuncAttributes fa;
    const cudaError_t fe = cudaFuncGetAttributes(&fa, reinterpret_cast<const void*>(kern));
    if (fe != cudaSuccess) return record_cuda_error(fe);
    if (fa.numRegs < 128) return PSB_ERR_UNSUPPORTED;
    checked[dtype == PSB_BF16].store(true, std::memory_order_relaxed);
  }
  int occ = 0;
  if (!kernel_occupancy(reinterpret_cast<const void*>(kern), kThreads, smem, &occ) || occ < 1) return PSB_ERR_CUDA;
  const int64_t grid = std::min<int64_t>(ctas_bound(p.total, p.num_seqs, tp.tq, p.hkv, p.max_context),
                                         static_cast<int64_t>(sms) * std::min(occ, 2));
  const int64_t entries = std::min<int64_t>(static_cast<int64_t>(tp.max_pairs) * p.hkv, grid - 1);
  tp.by_pair = entries < grid - 1;
  discard_stale_error();
  cudaError_t e = launch_pdl(kern, dim3(static_cast<unsigned>(grid)), dim3(kThreads), smem, s, tp, tq);
  if (e != cudaSuccess) return record_cuda_error(e);
  if (grid > 1 && p.max_seqlen > 0) {
    // only rows that a sequence of max_seqlen tokens has
    const int rows = std::min(p.max_seqlen, tp.tq) * tp.group;
    e = launch_pdl(comb, dim3(static_cast<unsigned>(entries), (rows + kCombineRows - 1) / kCombineRows, p.max_seqlen > tp.tq ? 2 : 1),
                   dim3(kCombineThreads), 0, s, tp);
    if (e != cudaSuccess) return record_cuda_error(e);
  }
  return check_launch();
}

}  // namespace psb
