// Prefix-aware (chunked) causal prefill over the 4-bit KV pool on the
// 5th-generation tensor cores: bf16/f16, head_dim 64, any block_size, up to
// 128 q heads per kv head.
//
// Mathematics.  As in int4_decode_fast.cu: with codes c, step and mid per
// (token, kv head), q . k_t = step_t (q . (c_t - 7.5)) + mid_t sum(q) and
// sum_t p_t v_t = sum_t (p_t step_t)(c_t - 7.5) + sum_t p_t mid_t.  The codes
// become exact 16-bit operands in shared memory; step and mid act on scores
// and probabilities in fp32.  K's operand is 128 + c (bf16) or 1024 + c (f16),
// a constant high byte over the code, and the offset goes with mid; V's is
// (c - 7.5) 2^-9 in f16 whatever T is, next to p step scaled by a power of two
// and rounded to f16 - the one rounding below fp32.
//
// Tiles.  The q heads of a kv head read the same keys, so a tile's 128 rows
// are TQ = 128 / group consecutive tokens times the group's heads (one TMA box
// of [TQ, group, 64]): a short chunk of few tokens still fills a tile, and
// each key tile is decoded once for all heads of the group.  A step is 64 keys.
// The steps of all tiles, in (kv head, tile, step) order, are dealt evenly over
// a persistent grid of two CTAs per SM; a tile cut by a CTA boundary leaves
// fp32 partials that int4_prefill_combine_kernel joins (a single chunk on a
// long prefix has fewer tiles than the GPU has SMs).
//
// CTA: eight warps.  Warps 0-3 are the softmax (thread r = TMEM lane r = row r
// of the tile).  In warps 4-7 one lane issues the Q loads and S = Q K^T (four
// tcgen05.mma M 128 N 64 K 16, one step ahead, two TMEM S buffers), one lane
// O += P V (P read from TMEM over the S it came from, two O buffers in turn),
// and two warps decode K and V into a ring of kStages shared-memory stages
// (128-byte swizzle), together with the 64 tokens' factors.  A warp pair's
// two roles are swapped in the second half of the grid, so that the decoding
// warps of an SM's two CTAs sit on different schedulers.  The softmax half has
// 168 registers, the other 88 (setmaxnreg; 256 x 128 at launch).
//
// Every mbarrier wait is bounded; no barrier can run two phases ahead of a
// waiter: a stage's next phase needs its own release, a step's barriers
// alternate and step g + 2 needs step g's products.
#include <algorithm>
#include <atomic>

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
constexpr int kStages = 3;
constexpr uint32_t kQTile = kRows * kDim * 2;
constexpr uint32_t kKvTile = kBN * kDim * 2;
constexpr uint32_t kTmemCols = 256;
constexpr uint32_t kSCol = 0, kOCol = 128;
constexpr float kGrowth = 4.f;      // log2 of how far a score may exceed the exponents' reference
constexpr int kPBits = 11;          // p step is scaled to at most 2^kGrowth 2^kPBits
constexpr float kVBack = 512.f;     // V's operand is (c - 7.5) / kVBack
constexpr int kMaxCtas = 320;       // grid limit
constexpr int kPartFloats = kRows * (kDim + 2);
constexpr int kMaxSeqs = 2048, kMaxTiles = 8192;

// factors of a stage's 64 tokens, and what is wrong with them
struct Factors {
  float ks[kBN], km[kBN], vs[kBN], vm[kBN];
  uint32_t bad[2];  // bit t: token t's block is outside the pool
  int vexp;         // p step was scaled by 2^(kPBits - vexp)
  int pad;
};

// dynamic shared memory (1024-byte aligned): Q0 | Q1 | K ring | V ring | factors | barriers | tables
constexpr uint32_t kOffK = 2 * kQTile, kOffV = kOffK + kStages * kKvTile;
constexpr uint32_t kOffF = kOffV + kStages * kKvTile;
constexpr uint32_t kOffBars = kOffF + kStages * sizeof(Factors);
constexpr uint32_t kOffTab = kOffBars + 256;

// A tile cut at a CTA's end that began in it: its kv head, first row of q and
// tokens, and the last CTA with a piece (0: none).
struct Cut {
  int32_t kvh, row0, c1, tokens;
};

struct TcParams {
  Int4PrefillParams a;
  int32_t group, tq;      // q heads per kv head, tokens per tile
  int32_t max_tiles;      // room for the tile table
  uint64_t block_div;     // 2^32 / block_size, rounded up
  float* part;            // workspace: cuts, then two partials per CTA
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

// A wait of a whole warp: its lanes give up together or not at all.
__device__ __forceinline__ bool warp_ok(bool ok) { return __all_sync(0xffffffffu, ok); }

// What every role knows of the batch: lengths per sequence, tiles, steps.
struct Plan {
  const int32_t* len;    // [num_seqs] query rows
  const int32_t* ctx;    // [num_seqs] tokens in the pool
  const int32_t* q0;     // [num_seqs] first row
  const int32_t* tfirst; // [num_seqs + 1] tiles before a sequence
  const int32_t* sfirst; // [tiles + 1] steps before a tile
  int32_t num_seqs, tiles, steps;  // of one kv head
};

__device__ __forceinline__ int last_le(const int32_t* v, int n, int x) {  // last i < n with v[i] <= x
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (v[mid] <= x) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// A run of steps of one tile.
struct Seg {
  int kvh, tile, seq, qt;  // qt: the tile's number in its sequence
  int j0, n;               // its steps j0 .. j0 + n - 1 of n_kv
  int n_kv;
};

// Walks a CTA's steps [pos, end) tile by tile.
struct Cursor {
  const Plan& pl;
  int64_t pos, end;
  int kvh, tile, seq;
  __device__ Cursor(const Plan& p, int64_t a, int64_t e) : pl(p), pos(a), end(e), kvh(0), tile(0), seq(0) {
    if (a >= e) return;
    kvh = static_cast<int>(a / p.steps);
    const int r = static_cast<int>(a - static_cast<int64_t>(kvh) * p.steps);
    tile = last_le(p.sfirst, p.tiles, r);
    seq = last_le(p.tfirst, p.num_seqs, tile);
  }
  __device__ bool more() const { return pos < end; }
  __device__ Seg take() {  // the next run
    Seg s;
    s.kvh = kvh;
    s.tile = tile;
    s.seq = seq;
    s.qt = tile - pl.tfirst[seq];
    s.n_kv = pl.sfirst[tile + 1] - pl.sfirst[tile];
    s.j0 = static_cast<int>(pos - (static_cast<int64_t>(kvh) * pl.steps + pl.sfirst[tile]));
    s.n = static_cast<int>(min(static_cast<int64_t>(s.n_kv - s.j0), end - pos));
    pos += s.n;
    if (pos < end && ++tile == pl.tiles) {
      tile = 0;
      ++kvh;
      seq = last_le(pl.tfirst, pl.num_seqs, 0);
    } else if (pos < end) {
      while (pl.tfirst[seq + 1] <= tile) ++seq;  // sequences without rows have no tiles
    }
    return s;
  }
};

template <typename T>
__global__ void __launch_bounds__(kThreads, 2)
    int4_prefill_tc_kernel(const TcParams tp, const __grid_constant__ CUtensorMap tm_q) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const Int4PrefillParams& p = tp.a;
  Factors* const fac = reinterpret_cast<Factors*>(smem + kOffF);
  uint64_t* const bar_q = reinterpret_cast<uint64_t*>(smem + kOffBars);  // [2] Q loaded
  uint64_t* const bar_qfree = bar_q + 2;      // [2] Q K^T of the run in the buffer done
  uint64_t* const bar_qread = bar_q + 4;      // [2] the softmax has its row sums
  uint64_t* const bar_k = bar_q + 6;          // [kStages] K decoded
  uint64_t* const bar_v = bar_k + kStages;    // [kStages] V decoded
  uint64_t* const bar_kfree = bar_v + kStages;  // [kStages] softmax of the step done (so is its Q K^T)
  uint64_t* const bar_vfree = bar_kfree + kStages;  // [kStages] P V done
  uint64_t* const bar_s = bar_vfree + kStages;  // [2]
  uint64_t* const bar_p = bar_s + 2;          // [2]
  uint64_t* const bar_pv = bar_p + 2;         // [2]
  uint32_t* const s_tmem = reinterpret_cast<uint32_t*>(bar_pv + 2);
  static_assert((6 + 4 * kStages + 6) * 8 + 4 <= 256, "barriers fit their area");
  int32_t* const s_len = reinterpret_cast<int32_t*>(smem + kOffTab);
  int32_t* const s_ctx = s_len + p.num_seqs;
  int32_t* const s_q0 = s_ctx + p.num_seqs;
  int32_t* const s_tfirst = s_q0 + p.num_seqs;
  int32_t* const s_sfirst = s_tfirst + p.num_seqs + 1;
  __shared__ int32_t warp_sums[kThreads / 32];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int TQ = tp.tq, group = tp.group;
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
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) run += warp_sums[w];
      total += warp_sums[w];
    }
    __syncthreads();
    return run;
  };
  int n_tiles = 0, n_steps = 0;
  {
    const int per = (p.num_seqs + kThreads - 1) / kThreads;
    const int s0 = min(tid * per, p.num_seqs), s1 = min(s0 + per, p.num_seqs);
    int tiles = 0;
    for (int s = s0; s < s1; ++s) {
      const int a = p.cu[s], b = p.cu[s + 1];
      // a malformed batch is reported by the caller's check and read nowhere
      int len = a < 0 || b < a || b > p.total ? 0 : b - a;
      int ctx = p.ctx[s];
      if (len > 0 && (ctx < len || ctx > p.max_context)) {
        if (blockIdx.x == 0) flag_error(p.err, PSB_DEVERR_CONTEXT);
        ctx = min(max(ctx, len), p.max_context);
        len = min(len, ctx);
      }
      s_len[s] = len;
      s_ctx[s] = ctx;
      s_q0[s] = a;
      tiles += (len + TQ - 1) / TQ;
    }
    int run = scan(tiles, n_tiles);
    for (int s = s0; s < s1; ++s) {
      s_tfirst[s] = run;
      run += (s_len[s] + TQ - 1) / TQ;
    }
    if (tid == 0) s_tfirst[p.num_seqs] = n_tiles;
    __syncthreads();
    if (n_tiles > tp.max_tiles) {  // rows named by two sequences: a malformed batch
      if (tid == 0) flag_error(p.err, PSB_DEVERR_SEQLENS);
      n_tiles = 0;
    }
    const int tper = (n_tiles + kThreads - 1) / kThreads;
    const int t0 = min(tid * tper, n_tiles), t1 = min(t0 + tper, n_tiles);
    int steps = 0;
    for (int t = t0; t < t1; ++t) {
      const int s = last_le(s_tfirst, p.num_seqs, t), qt = t - s_tfirst[s];
      // keys 0 .. position of the tile's last row
      const int n = (s_ctx[s] - s_len[s] + min(s_len[s], (qt + 1) * TQ) + kBN - 1) / kBN;
      s_sfirst[t] = n;
      steps += n;
    }
    run = scan(steps, n_steps);
    for (int t = t0; t < t1; ++t) {
      const int n = s_sfirst[t];
      s_sfirst[t] = run;
      run += n;
    }
    if (tid == 0) s_sfirst[n_tiles] = n_steps;
    __syncthreads();
  }
  const Plan plan{s_len, s_ctx, s_q0, s_tfirst, s_sfirst, p.num_seqs, n_tiles, n_steps};
  const int64_t total_steps = static_cast<int64_t>(n_steps) * p.hkv;
  const int act = static_cast<int>(min(static_cast<int64_t>(gridDim.x), total_steps));
  Cut* const cuts = reinterpret_cast<Cut*>(tp.part);
  float* const part = tp.part + kMaxCtas * (sizeof(Cut) / sizeof(float));
  const int cta = blockIdx.x;
  if (cta >= act) {
    if (tid == 0) cuts[cta] = Cut{0, 0, 0, 0};
    return;
  }
  auto cta_start = [&](int c) -> int64_t { return total_steps * c / act; };
  const int64_t my_a = cta_start(cta), my_e = cta_start(cta + 1);
  const uint32_t s_base = smem_u32(smem);

  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar_q + i, 1);
      mbar_init(bar_qfree + i, 1);
      mbar_init(bar_qread + i, 4);
      mbar_init(bar_s + i, 1);
      mbar_init(bar_p + i, 128);
      mbar_init(bar_pv + i, 1);
    }
    for (int i = 0; i < kStages; ++i) {
      mbar_init(bar_k + i, 1);
      mbar_init(bar_v + i, 1);
      mbar_init(bar_kfree + i, 4);
      mbar_init(bar_vfree + i, 1);
    }
    fence_barrier_init();
  }
  if (warp == 0) {
    tmem_alloc(s_tmem, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;
  pdl_launch_dependents();
  bool fail = false;

  if (warp >= 4) {
    reg_dec<88>();
    // roles of warps 4-7: Q loads + Q K^T, P V, decode K, decode V
    const int role = (warp - 4) ^ (cta >= (static_cast<int>(gridDim.x) + 1) / 2 ? 2 : 0);
    if (role == 0) {
      if (lane == 0) {
        const uint32_t idesc = umma_idesc_f16(Elem<T>::code == PSB_BF16 ? 1 : 0, kRows, kBN, 0, 0);
        const uint64_t dq = umma_desc_sw128(s_base, 1024, 16);
        const uint64_t dk = umma_desc_sw128(s_base + kOffK, 1024, 16);
        prefetch_tmap(&tm_q);
        Cursor qc(plan, my_a, my_e), cc(plan, my_a, my_e);
        int q_req = 0, q_seen = 0, g = 0;
        auto load_q = [&]() {  // the next run's rows into buffer q_req & 1
          const Seg s = qc.take();
          const int b = q_req & 1;
          mbar_arrive_expect_tx(bar_q + b, static_cast<uint32_t>(TQ * group) * kDim * 2);
          tma_load_3d(smem + b * kQTile, &tm_q, 0, s.kvh * group, plan.q0[s.seq] + s.qt * TQ, bar_q + b);
          ++q_req;
        };
        load_q();
        if (qc.more()) load_q();
        for (int k = 0; cc.more() && !fail; ++k) {
          const Seg s = cc.take();
          const int b = k & 1;
          if (!mbar_wait(bar_q + b, (k >> 1) & 1)) {
            fail = true;
            break;
          }
          ++q_seen;
          const uint64_t dqs = dq + static_cast<uint64_t>(b * (kQTile >> 4));
          for (int j = 0; j < s.n; ++j, ++g) {
            const int st = g % kStages;
            // S buffer g & 1 held S and then P of step g - 2
            if ((g >= 2 && !mbar_wait(bar_pv + (g & 1), ((g - 2) >> 1) & 1)) ||
                !mbar_wait(bar_k + st, (g / kStages) & 1)) {
              fail = true;
              break;
            }
            tc_fence_after();
            const uint64_t dks = dk + static_cast<uint64_t>(st * (kKvTile >> 4));
#pragma unroll
            for (int kk = 0; kk < kDim / 16; ++kk)
              umma_f16_ss(tmem + kSCol + (g & 1) * kBN, dqs + 2 * kk, dks + 2 * kk, idesc, kk > 0);
            umma_commit(bar_s + (g & 1));
          }
          if (fail) break;
          umma_commit(bar_qfree + b);
          if (qc.more()) {  // run k + 2 goes into this buffer
            if (!mbar_wait(bar_qfree + b, (k >> 1) & 1) || !mbar_wait(bar_qread + b, (k >> 1) & 1)) {
              fail = true;
              break;
            }
            load_q();
          }
        }
        if (fail) {
          flag_error(p.err, PSB_DEVERR_TIMEOUT);
          for (int t = q_seen; t < q_req; ++t) (void)mbar_wait(bar_q + (t & 1), (t >> 1) & 1);
        }
      }
    } else if (role == 1) {
      if (lane == 0) {
        const uint32_t idesc = umma_idesc_f16(0, kRows, kDim, 0, 1);
        const uint64_t dv = umma_desc_sw128(s_base + kOffV, 1024, 8192);
        Cursor cc(plan, my_a, my_e);
        int g = 0, issued = 0;
        for (int k = 0; cc.more() && !fail; ++k) {
          const Seg s = cc.take();
          const uint32_t obuf = tmem + kOCol + (k & 1) * kDim;
          for (int j = 0; j < s.n; ++j, ++g) {
            const int st = g % kStages;
            if (!mbar_wait(bar_p + (g & 1), (g >> 1) & 1) || !mbar_wait(bar_v + st, (g / kStages) & 1)) {
              fail = true;
              break;
            }
            tc_fence_after();
            const uint64_t dvs = dv + static_cast<uint64_t>(st * (kKvTile >> 4));
            const uint32_t pcol = tmem + kSCol + (g & 1) * kBN;
#pragma unroll
            for (int kk = 0; kk < kBN / 16; ++kk)
              umma_f16_ts(obuf, pcol + 8 * kk, dvs + 128 * kk, idesc, j > 0 || kk > 0);
            umma_commit(bar_pv + (g & 1));
            umma_commit(bar_vfree + st);
            ++issued;
          }
        }
        if (fail) {
          flag_error(p.err, PSB_DEVERR_TIMEOUT);
          // let the products in flight land before shared memory and TMEM are released
          if (issued > 0) (void)mbar_wait(bar_pv + ((issued - 1) & 1), ((issued - 1) >> 1) & 1);
        }
      }
    } else {
      // ---- decode: lane l of a warp takes rows l and l + 32 of a step's 64 keys ----
      const bool is_v = role == 3;
      const uint32_t ring = s_base + (is_v ? kOffV : kOffK);
      uint64_t* const bar_full = is_v ? bar_v : bar_k;
      uint64_t* const bar_free = is_v ? bar_vfree : bar_kfree;
      Cursor cc(plan, my_a, my_e);
      Seg seg{};
      int j = 0, left = 0;  // next step to look up: step j of seg, left of them
      const int32_t* row = nullptr;
      int ctx = 0;
      // The pipeline of a lane's two rows: block ids of one step ahead of the
      // codes' loads, those one step ahead of their decoding.
      struct Rows {
        uint4 c[2][2];
        uint32_t par[2];
        uint32_t flags;  // bits 0, 1: row's block is outside the pool; 2: first step of a run; 3: there is a step
      };
      int64_t at[2] = {-1, -1};  // pool rows of the step after next, -1: nothing to read
      uint32_t at_flags = 0;
      auto look = [&]() {
        at[0] = at[1] = -1;
        at_flags = 0;
        if (left == 0) {
          if (!cc.more()) return;
          seg = cc.take();
          j = seg.j0;
          left = seg.n;
          row = p.tables + static_cast<int64_t>(seg.seq) * p.table_stride;
          ctx = plan.ctx[seg.seq];
          at_flags = 4;
        }
        at_flags |= 8;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t pos = j * kBN + lane + 32 * i;
          if (static_cast<int>(pos) >= ctx) continue;
          const uint32_t bi = static_cast<uint32_t>((static_cast<uint64_t>(pos) * tp.block_div) >> 32);
          const int blk = __ldg(row + bi);
          if (blk < 0 || blk >= p.num_blocks) {
            at_flags |= 1u << i;
          } else {
            at[i] = int4_row(p.layer_tiles + static_cast<int64_t>(blk) * p.hkv + seg.kvh, is_v ? 1 : 0,
                             static_cast<int>(pos - bi * p.block_size), p.block_size);
          }
        }
        ++j;
        --left;
      };
      auto load = [&](Rows& r) {
        r.flags = at_flags;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          r.c[i][0] = r.c[i][1] = make_uint4(0, 0, 0, 0);
          r.par[i] = 0;
          if (at[i] >= 0) {
            const uint4* src = reinterpret_cast<const uint4*>(p.codes + at[i] * (kDim / 2));
            r.c[i][0] = __ldg(src);
            r.c[i][1] = __ldg(src + 1);
            r.par[i] = __ldg(reinterpret_cast<const uint32_t*>(p.params) + at[i]);
          }
        }
      };
      Rows cur, nxt;
      look();
      load(nxt);
      look();
      int vexp = 0;
      float vlim = 0.f, vscale = 1.f;
      for (int g = 0; (nxt.flags & 8) && !fail; ++g) {
        cur = nxt;
        load(nxt);
        look();
        const int st = g % kStages;
        if (g >= kStages && !warp_ok(mbar_wait(bar_free + st, (g / kStages - 1) & 1))) {
          fail = true;
          break;
        }
        Factors& f = fac[st];
        const uint32_t tile = ring + st * kKvTile;
        const float2 p0 = unpack2<T>(cur.par[0]), p1 = unpack2<T>(cur.par[1]);
        if (!is_v) {
          // 128 + c (bf16) or 1024 + c (f16), elements in order
          constexpr float kOff = Elem<T>::code == PSB_BF16 ? 135.5f : 1031.5f;
          constexpr uint32_t kHigh = Elem<T>::code == PSB_BF16 ? 0x43434343u : 0x64646464u;
          const float sc = p.scale_log2;
          f.ks[lane] = p0.x * sc;
          f.ks[lane + 32] = p1.x * sc;
          f.km[lane] = fmaf(p0.x, -kOff, p0.y) * sc;
          f.km[lane + 32] = fmaf(p1.x, -kOff, p1.y) * sc;
          const uint32_t bad0 = __ballot_sync(0xffffffffu, cur.flags & 1), bad1 = __ballot_sync(0xffffffffu, cur.flags & 2);
          if (lane == 0) {
            f.bad[0] = bad0;
            f.bad[1] = bad1;
            if (bad0 | bad1) flag_error(p.err, PSB_DEVERR_BLOCK_RANGE);
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int r = lane + 32 * i;
            const uint32_t* w = &cur.c[i][0].x;
#pragma unroll
            for (int c = 0; c < 8; ++c) {
              const uint32_t x = w[c], t = x & 0x0f0f0f0fu, u = (x >> 4) & 0x0f0f0f0fu;
              const uint32_t m0 = __byte_perm(t, u, 0x5140), m1 = __byte_perm(t, u, 0x7362);
              st_shared_v4(tile + r * 128 + ((c ^ (r & 7)) << 4), __byte_perm(m0, kHigh, 0x4140),
                           __byte_perm(m0, kHigh, 0x4342), __byte_perm(m1, kHigh, 0x4140),
                           __byte_perm(m1, kHigh, 0x4342));
            }
          }
        } else {
          if (cur.flags & 4) {  // a run's first step
            vlim = 0.f;
            vexp = 0;
            vscale = 1.f;
          }
          if (__any_sync(0xffffffffu, fmaxf(p0.x, p1.x) > vlim)) {
            float top = fmaxf(p0.x, p1.x);
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            vexp = max(-100, ilogb_f32(top)) + 1;  // top < 2^vexp
            vlim = exp2_int(min(vexp, 127));
            vscale = exp2_int(kPBits - vexp);
          }
          f.vs[lane] = p0.x * vscale;
          f.vs[lane + 32] = p1.x * vscale;
          f.vm[lane] = p0.y;
          f.vm[lane + 32] = p1.y;
          if (lane == 0) f.vexp = vexp;
          // (c - 7.5) 2^-9 in f16: the nibble pairs (i, i + 4) are the subnormals
          // c 2^-24 (even i) and c 2^-20 (odd i); element 8 w + i + 4 h of a row
          // sits at 8 w + 2 i + h
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int r = lane + 32 * i;
            const uint32_t* w = &cur.c[i][0].x;
#pragma unroll
            for (int c = 0; c < 8; ++c) {
              const uint32_t x = w[c], y = x >> 8;
              // 2^15, 2^11 and - 7.5 / 512 as f16 pairs
              st_shared_v4(tile + r * 128 + ((c ^ (r & 7)) << 4), hfma2(x & 0x000f000fu, 0x78007800u, 0xa380a380u),
                           hfma2(x & 0x00f000f0u, 0x68006800u, 0xa380a380u),
                           hfma2(y & 0x000f000fu, 0x78007800u, 0xa380a380u),
                           hfma2(y & 0x00f000f0u, 0x68006800u, 0xa380a380u));
            }
          }
        }
        fence_proxy_async_smem();  // visible to the tensor core
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_full + st);
      }
      if (fail && lane == 0) flag_error(p.err, PSB_DEVERR_TIMEOUT);
    }
  } else {
    reg_inc<168>();
    // ---- softmax warps ------------------------------------------------------
    const int row = warp * 32 + lane;
    const int rtok = row / group, rhead = row - rtok * group;
    const uint32_t t_lane = tmem + (static_cast<uint32_t>(warp * 32) << 16);
    const bool out16 = reinterpret_cast<uintptr_t>(p.out) % 16 == 0 && p.ost % 8 == 0 && p.osh % 8 == 0;
    // a run's output is written after the next run's first step (or at the
    // end): by then its last P V is normally done
    int pend_k = -1, pend_exp = 0;
    float pend_l = 0.f, pend_z = 0.f, pend_m = 0.f;
    Seg pend{};
    auto write_pending = [&](int pg) -> bool {
      if (!warp_ok(mbar_wait(bar_pv + (pg & 1), (pg >> 1) & 1))) return false;
      tc_fence_after();
      const uint32_t t_po = t_lane + kOCol + (pend_k & 1) * kDim;
      const bool whole = pend.j0 == 0 && pend.n == pend.n_kv;
      const int tok = pend.qt * TQ + rtok;
      const bool live = rtok < TQ && tok < plan.len[pend.seq];
      const float back = exp2_int(max(-126, min(127, pend_exp - kPBits))) * kVBack;  // of one unit of O
      const float inv = !whole ? 1.f : pend_l == 0.f ? 0.f : 1.f / pend_l;
      const float scale = back * inv, base = pend_z * inv;
      float* const dst = part + static_cast<int64_t>(2 * cta + (pend.j0 > 0 ? 0 : 1)) * kPartFloats;
      T* const out = reinterpret_cast<T*>(p.out) + static_cast<int64_t>(plan.q0[pend.seq] + tok) * p.ost +
                     static_cast<int64_t>(pend.kvh * group + rhead) * p.osh;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t ot[32];
        tmem_ld32(t_po + 32 * h, ot);
        tmem_wait_ld();
        float o[32];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {  // columns 2 i, 2 i + 1 of a word are its elements i, i + 4
            o[8 * w + i] = fmaf(__uint_as_float(ot[8 * w + 2 * i]), scale, base);
            o[8 * w + i + 4] = fmaf(__uint_as_float(ot[8 * w + 2 * i + 1]), scale, base);
          }
        }
        if (!whole) {
          if (live)
#pragma unroll
            for (int d = 0; d < 32; d += 4)
              *reinterpret_cast<float4*>(dst + row * kDim + 32 * h + d) = make_float4(o[d], o[d + 1], o[d + 2], o[d + 3]);
        } else if (live) {
          if (out16) {
#pragma unroll
            for (int d = 0; d < 32; d += 8)
              *reinterpret_cast<uint4*>(out + 32 * h + d) = make_uint4(pack2<T>(o[d], o[d + 1]), pack2<T>(o[d + 2], o[d + 3]),
                                                                       pack2<T>(o[d + 4], o[d + 5]), pack2<T>(o[d + 6], o[d + 7]));
          } else {
#pragma unroll
            for (int d = 0; d < 32; ++d) out[32 * h + d] = Elem<T>::from_float(o[d]);
          }
        }
      }
      if (!whole) *reinterpret_cast<float2*>(dst + kRows * kDim + 2 * row) = make_float2(pend_m, pend_l);
      tc_fence_before();
      pend_k = -1;
      return true;
    };
    Cursor cc(plan, my_a, my_e);
    int g = 0;
    for (int k = 0; cc.more() && !fail; ++k) {
      const Seg s = cc.take();
      const int ctx = plan.ctx[s.seq], start = ctx - plan.len[s.seq];
      const int tok = s.qt * TQ + rtok;
      // last key of this row; rows past the tile's tokens see none
      const int last = rtok < TQ && tok < plan.len[s.seq] ? start + tok : -1;
      const uint32_t t_o = t_lane + kOCol + (k & 1) * kDim;
      // sum of the row's q
      if (!warp_ok(mbar_wait(bar_q + (k & 1), (k >> 1) & 1))) {
        fail = true;
        break;
      }
      float qsum = 0.f;
      {
        const uint32_t qrow = s_base + (k & 1) * kQTile + row * 128;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const uint4 v = ld_shared_v4(qrow + (((c + lane) & 7) << 4));
          const float2 a = unpack2<T>(v.x), b = unpack2<T>(v.y), d = unpack2<T>(v.z), e = unpack2<T>(v.w);
          qsum += ((a.x + a.y) + (b.x + b.y)) + ((d.x + d.y) + (e.x + e.y));
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_qread + (k & 1));
      float ref = 0.f, l = 0.f, z = 0.f;  // the exponents' reference; sums of p and p mid
      bool fresh = true;
      int vexp = 0;
      auto step = [&](int i) -> bool {
        const int st = g % kStages;
        const uint32_t ph = (g / kStages) & 1;
        if (!warp_ok(mbar_wait(bar_s + (g & 1), (g >> 1) & 1) && mbar_wait(bar_k + st, ph) && mbar_wait(bar_v + st, ph)))
          return false;
        tc_fence_after();
        const Factors& f = fac[st];
        uint32_t sr[kBN];
        tmem_ld32(t_lane + kSCol + (g & 1) * kBN, sr);
        tmem_ld32(t_lane + kSCol + (g & 1) * kBN + 32, sr + 32);
        tmem_wait_ld();
        // scores minus reference
        const uint64_t qs2 = f2_pack(qsum, qsum), nref2 = f2_pack(-ref, -ref);
#pragma unroll
        for (int c = 0; c < kBN; c += 4) {
          const float4 ks = ld_shared_f4(f.ks + c), km = ld_shared_f4(f.km + c);
          const float2 a = f2_unpack(f2_fma(f2_pack(ks.x, ks.y), f2_pack(__uint_as_float(sr[c]), __uint_as_float(sr[c + 1])),
                                            f2_fma(f2_pack(km.x, km.y), qs2, nref2)));
          const float2 b = f2_unpack(f2_fma(f2_pack(ks.z, ks.w), f2_pack(__uint_as_float(sr[c + 2]), __uint_as_float(sr[c + 3])),
                                            f2_fma(f2_pack(km.z, km.w), qs2, nref2)));
          sr[c] = __float_as_uint(a.x);
          sr[c + 1] = __float_as_uint(a.y);
          sr[c + 2] = __float_as_uint(b.x);
          sr[c + 3] = __float_as_uint(b.y);
        }
        const int lim = last - (s.j0 + i) * kBN;  // last valid column
        if (lim < kBN - 1) {
#pragma unroll
          for (int c = 0; c < kBN; ++c)
            if (c > lim) sr[c] = __float_as_uint(-INFINITY);
        }
        const uint32_t bad0 = f.bad[0], bad1 = f.bad[1];
        if (bad0 | bad1) {
#pragma unroll
          for (int c = 0; c < kBN; ++c)
            if ((c < 32 ? bad0 : bad1) >> (c & 31) & 1) sr[c] = __float_as_uint(-INFINITY);
        }
        float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
        for (int c = 0; c < kBN; c += 4) {
          mx0 = fmax3(mx0, __uint_as_float(sr[c]), __uint_as_float(sr[c + 1]));
          mx1 = fmax3(mx1, __uint_as_float(sr[c + 2]), __uint_as_float(sr[c + 3]));
        }
        const float mx = fmaxf(mx0, mx1);
        // A row's reference moves when a score is above it by more than the
        // limit, or at its first score; O is rescaled then, or when the scale
        // of p step changed.  The warp's TMEM access is collective.
        const int ve = f.vexp;
        const bool grow = mx > (fresh ? -INFINITY : kGrowth);
        if (__any_sync(0xffffffffu, grow) || (i > 0 && ve != vexp)) {
          const float up = grow ? fminf(fmaxf(mx, -3e38f), 3e38f) : 0.f;
          const float al = grow ? (fresh ? 0.f : ex2_approx(-up)) : 1.f;
          if (i > 0) {  // O holds P V of the earlier steps once the last of them is done
            if (!warp_ok(mbar_wait(bar_pv + ((g - 1) & 1), ((g - 1) >> 1) & 1))) return false;
            tc_fence_after();
            const float ao = al * exp2_int(max(-126, vexp - ve));
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t ot[32];
              tmem_ld32(t_o + 32 * h, ot);
              tmem_wait_ld();
#pragma unroll
              for (int d = 0; d < 32; ++d) ot[d] = __float_as_uint(__uint_as_float(ot[d]) * ao);
              tmem_st32(t_o + 32 * h, ot);
            }
            tmem_wait_st();
          }
          l *= al;
          z *= al;
          ref += up;
          fresh = fresh && !grow;
#pragma unroll
          for (int c = 0; c < kBN; ++c) sr[c] = __float_as_uint(__uint_as_float(sr[c]) - up);
        }
        vexp = ve;
        uint32_t pk[kBN / 2];
        uint64_t l2 = f2_pack(0.f, 0.f), z2 = f2_pack(0.f, 0.f);
#pragma unroll
        for (int c = 0; c < kBN; c += 4) {
          const float4 vs = ld_shared_f4(f.vs + c), vm = ld_shared_f4(f.vm + c);
          const uint64_t a = f2_pack(ex2_approx(__uint_as_float(sr[c])), ex2_approx(__uint_as_float(sr[c + 1])));
          const uint64_t b = f2_pack(ex2_approx(__uint_as_float(sr[c + 2])), ex2_approx(__uint_as_float(sr[c + 3])));
          l2 = f2_add(l2, f2_add(a, b));
          z2 = f2_fma(a, f2_pack(vm.x, vm.y), z2);
          z2 = f2_fma(b, f2_pack(vm.z, vm.w), z2);
          const float2 pa = f2_unpack(f2_mul(a, f2_pack(vs.x, vs.y))), pb = f2_unpack(f2_mul(b, f2_pack(vs.z, vs.w)));
          pk[c / 2] = pack2<__half>(pa.x, pa.y);
          pk[c / 2 + 1] = pack2<__half>(pb.x, pb.y);
        }
        const float2 lf = f2_unpack(l2), zf = f2_unpack(z2);
        l += lf.x + lf.y;
        z += zf.x + zf.y;
        tmem_st32(t_lane + kSCol + (g & 1) * kBN, pk);
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(bar_p + (g & 1));
        __syncwarp();  // every lane has read the factors
        if (lane == 0) mbar_arrive(bar_kfree + st);
        return true;
      };
      if (!step(0) || (pend_k >= 0 && !write_pending(g - 1))) {
        fail = true;
        break;
      }
      ++g;
      for (int i = 1; i < s.n; ++i, ++g) {
        if (!step(i)) {
          fail = true;
          break;
        }
      }
      if (fail) break;
      pend_k = k;
      pend = s;
      pend_l = l;
      pend_z = z;
      pend_exp = vexp;
      pend_m = fresh ? -INFINITY : ref;
    }
    if (!fail && pend_k >= 0 && !write_pending(g - 1)) fail = true;
    if (fail && lane == 0) flag_error(p.err, PSB_DEVERR_TIMEOUT);
    if (warp == 0) {
      // the tile that begins here and runs past the CTA's end, if any
      Cut c{0, 0, 0, 0};
      const int64_t at = my_e - 1;
      const int kvh = static_cast<int>(at / n_steps);
      const int tile = last_le(s_sfirst, n_tiles, static_cast<int>(at - static_cast<int64_t>(kvh) * n_steps));
      const int64_t t_a = static_cast<int64_t>(kvh) * n_steps + s_sfirst[tile];
      const int64_t t_e = static_cast<int64_t>(kvh) * n_steps + s_sfirst[tile + 1];
      if (t_a >= my_a && t_e > my_e) {
        const int seq = last_le(s_tfirst, p.num_seqs, tile), first = (tile - s_tfirst[seq]) * TQ;
        c.kvh = kvh;
        c.row0 = s_q0[seq] + first;
        c.tokens = min(TQ, s_len[seq] - first);
        c.c1 = cta;
        for (int c0 = cta + 1; c0 < act; c0 += 32) {  // CTAs that start before its end
          const bool in = c0 + lane < act && cta_start(min(c0 + lane, act)) < t_e;
          const int n = __popc(__ballot_sync(0xffffffffu, in));
          c.c1 += n;
          if (n < 32) break;
        }
      }
      if (lane == 0) cuts[cta] = c;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// Joins the partials of the tile that CTA blockIdx.x left cut at its end: a
// quarter of the tile's rows per CTA, kWarpRows rows per warp, two elements a
// lane, kBatch partials in flight.
constexpr int kCombineRows = 32, kWarpRows = kCombineRows / (kThreads / 32), kBatch = 4;

template <typename T>
__global__ void __launch_bounds__(kThreads) int4_prefill_combine_kernel(const TcParams tp) {
  const Int4PrefillParams& p = tp.a;
  pdl_wait();
  pdl_launch_dependents();
  const int c0 = blockIdx.x, lane = threadIdx.x & 31;
  const int4 cut = __ldcg(reinterpret_cast<const int4*>(tp.part) + c0);
  const int row0 = blockIdx.y * kCombineRows + (threadIdx.x >> 5) * kWarpRows;
  if (cut.z <= c0 || row0 >= cut.w * tp.group) return;
  const float* const part = tp.part + kMaxCtas * (sizeof(Cut) / sizeof(float));
  auto piece_of = [&](int c) { return part + static_cast<int64_t>(2 * c + (c == c0 ? 1 : 0)) * kPartFloats; };
  float m[kWarpRows], l[kWarpRows];
  float2 o[kWarpRows];
#pragma unroll
  for (int r = 0; r < kWarpRows; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
    o[r] = make_float2(0.f, 0.f);
  }
  for (int c = c0; c <= cut.z; c += kBatch) {
    float2 ml[kBatch][kWarpRows], v[kBatch][kWarpRows];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
#pragma unroll
      for (int r = 0; r < kWarpRows; ++r) {
        ml[j][r] = make_float2(-INFINITY, 0.f);
        v[j][r] = make_float2(0.f, 0.f);
        if (c + j <= cut.z) {
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
    if (rtok >= cut.w) continue;
    const float inv = l[r] == 0.f ? 0.f : 1.f / l[r];
    T* out = reinterpret_cast<T*>(p.out) + static_cast<int64_t>(cut.y + rtok) * p.ost +
             static_cast<int64_t>(cut.x * tp.group + rhead) * p.osh + 2 * lane;
    out[0] = Elem<T>::from_float(o[r].x * inv);
    out[1] = Elem<T>::from_float(o[r].y * inv);
  }
}

size_t tc_smem(int num_seqs, int max_tiles) {
  return 1024 + kOffTab + sizeof(int32_t) * (4 * static_cast<size_t>(num_seqs) + 1 + max_tiles + 1);
}

int64_t tiles_bound(int total, int num_seqs, int tq) { return static_cast<int64_t>(total) / tq + num_seqs; }

}  // namespace

bool int4_prefill_tc_geometry(int dtype, int total, int num_seqs, int q_heads, int hkv, int head_dim, int block_size,
                              int max_context) {
  const int group = q_heads / hkv;
  if (!(dtype == PSB_BF16 || dtype == PSB_F16) || head_dim != kDim || group > kRows) return false;
  return num_seqs <= kMaxSeqs && tiles_bound(total, num_seqs, kRows / group) <= kMaxTiles &&
         static_cast<int64_t>(max_context + kBN) * block_size < (int64_t(1) << 32) &&
         tiles_bound(total, num_seqs, kRows / group) * (max_context / kBN + 1) < (int64_t(1) << 31);
}

size_t int4_prefill_tc_workspace() { return sizeof(Cut) * kMaxCtas + sizeof(float) * 2 * kMaxCtas * kPartFloats; }

int int4_prefill_tc_launch(const Int4PrefillParams& p, int dtype, float* workspace, cudaStream_t s) {
  TcParams tp;
  tp.a = p;
  tp.group = p.hq / p.hkv;
  tp.tq = kRows / tp.group;
  tp.max_tiles = static_cast<int32_t>(tiles_bound(p.total, p.num_seqs, tp.tq));
  tp.block_div = ((uint64_t(1) << 32) + p.block_size - 1) / p.block_size;
  tp.part = workspace;
  CUtensorMap tq;
  if (!encode_row_groups_map(&tq, p.q, p.total, p.hq, kDim, p.qst, p.qsh, tp.group, tp.tq,
                             dtype == PSB_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16))
    return PSB_ERR_CUDA;
  const int sms = device_sm_count();
  if (sms <= 0) return PSB_ERR_CUDA;
  const auto kern = dtype == PSB_BF16 ? int4_prefill_tc_kernel<__nv_bfloat16> : int4_prefill_tc_kernel<__half>;
  const auto comb = dtype == PSB_BF16 ? int4_prefill_combine_kernel<__nv_bfloat16> : int4_prefill_combine_kernel<__half>;
  const size_t smem = tc_smem(p.num_seqs, tp.max_tiles);
  // the register split draws on what the block was launched with
  static_assert(168 + 88 == 2 * 128, "two warpgroups' shares");
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
  // an upper bound of the steps
  const int64_t steps = static_cast<int64_t>(tp.max_tiles) * p.hkv * ((p.max_context + kBN - 1) / kBN);
  const int64_t grid = std::min<int64_t>(std::min<int64_t>(steps, kMaxCtas), static_cast<int64_t>(sms) * std::min(occ, 2));
  discard_stale_error();
  cudaError_t e = launch_pdl(kern, dim3(static_cast<unsigned>(grid)), dim3(kThreads), smem, s, tp, tq);
  if (e != cudaSuccess) return record_cuda_error(e);
  if (grid > 1) {
    e = launch_pdl(comb, dim3(static_cast<unsigned>(grid - 1), kRows / kCombineRows), dim3(kThreads), 0, s, tp);
    if (e != cudaSuccess) return record_cuda_error(e);
  }
  return check_launch();
}

}  // namespace psb
