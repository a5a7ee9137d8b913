// Decode attention for a batch whose sequences share long prefixes.
//
// Sequences cu[g] .. cu[g + 1] - 1 are group g and agree in their first
// prefix[g] tokens.  Softmax over a sequence's tokens splits into the part over
// the shared ones and the part over its own:
//   m = max(m1, m2),  l = l1 2^(m1 - m) + l2 2^(m2 - m),
//   o = (o1 2^(m1 - m) + o2 2^(m2 - m)) / l,
// so the shared part is computed for all of a group's query rows at once, where
// it is a matrix product (tcgen05), and each sequence's own part by itself, where
// it is a stream from HBM (mma.sync, as the plain decode).  Three launches:
//
//  shared_prefix_kernel  a tile is 128 rows: TQ = 128 / heads consecutive
//    sequences of a group times the q heads of one kv head (one TMA box of
//    [TQ, heads, 64]).  The steps (64 keys) of all tiles, in (kv head, group,
//    tile, step) order, are dealt evenly over a persistent grid; every run of
//    steps leaves an fp32 partial.
//  shared_own_kernel     the 16-token slices of what is each sequence's own, in
//    (kv heads, sequence, slice) order, dealt evenly over the warps of the grid;
//    every run of slices leaves an fp32 partial.
//  shared_join_kernel    joins the partials of each row.
//
// The first two do not depend on each other: the second starts while the first
// runs (it needs no tensor memory, and its registers and shared memory fit
// beside two CTAs of the first), so the stream from HBM goes on under the
// matrix products.
//
// Which of a group's tables the prefix is read through: that of the sequence
// with the most tokens (the first of those), and the prefix ends with it.  A
// sequence that is shorter than the prefix is read on its own (an idle row of a
// captured batch has no tokens at all): keys that it does not see, masked in the
// tile, would still meet its probabilities of 0, and 0 times infinity is no number.
#include <algorithm>
#include <climits>
#include <cmath>

#include "common.cuh"
#include "host_util.h"
#include "packed_f32.cuh"

namespace psb {
namespace {

constexpr int kMaxBatch = 2048;      // sequences (and groups) whose plan fits shared memory beside the rings
constexpr int kTcThreads = 192;      // warps 0-3: softmax; warp 4: products; warp 5: copies
constexpr int kRows = 128;           // rows of a tile
constexpr int kBN = 64;              // keys per step
constexpr int kHalf = 64;            // dims of one 128-byte line
constexpr uint32_t kQHalf = kRows * 128;   // bytes of 64 dims of a Q tile
constexpr uint32_t kKvHalf = kBN * 128;    // of a K or V tile
constexpr uint32_t kTmemCols = 256;
constexpr uint32_t kSCol = 0, kOCol = 128;
constexpr float kRescaleLog2 = 8.f;  // O is rescaled when a row's maximum grows by more than 2^8
constexpr int kMinSteps = 4;         // steps per CTA below which the grid shrinks
constexpr int kMaxTcCtas = 320;

constexpr int kOwnWarps = 4, kOwnThreads = kOwnWarps * 32;
constexpr int kOwnMinItems = 4;      // slices per warp below which fewer warps work
constexpr int kMaxOwnCtas = 320;

template <int D>
struct TcGeom {
  static constexpr int kH = D / kHalf;
  static constexpr int kStages = D == 64 ? 3 : 2;
  static constexpr uint32_t kOffK = kH * kQHalf;
  static constexpr uint32_t kOffV = kOffK + kStages * kH * kKvHalf;
  static constexpr uint32_t kOffBars = kOffV + kStages * kH * kKvHalf;
  static constexpr uint32_t kOffPlan = kOffBars + 256;
};

template <int D, int HP>
struct OwnGeom {
  static constexpr int kRing = 2;                 // slots per warp
  static constexpr int kTile = 16 * D * 2;        // 16 tokens of one kv head
  static constexpr int kKV = HP * kTile;
  static constexpr int kSlot = 2 * kKV;
  static constexpr int kBytes = kOwnWarps * kRing * kSlot;
};

struct SharedParams {
  const char* q;
  int64_t qsb, qsh;  // elements
  char* out;
  int64_t osb, osh;
  const char* k_cache;
  const char* v_cache;
  const int32_t* tables;
  int64_t table_stride;
  const int32_t* ctx;
  const int32_t* cu;
  const int32_t* prefix;
  int32_t batch, groups, hkv, group, layer, block_size, max_context;
  int32_t tq;          // sequences per tile
  int32_t max_tiles;   // tiles of one kv head there is room for
  int32_t max_warps;   // warps of the own kernel
  int64_t num_blocks;
  float scale_log2;    // scale log2(e), positive
  // workspace
  int2* tile_info;     // [hkv * max_tiles] a tile's first partial and how many
  int2* seq_info;      // [batch] a sequence's tile in each kv head (-1: none) and its place there
  int2* own_info;      // [hkv * batch] a (kv heads, sequence) pair's first partial and how many
  float* tile_part;    // partials of the tiles: [D / 4][128] x 4 sums, then [128] (maximum, sum)
  float* own_part;     // partials of the pairs: [16][D] sums, then [16] (maximum, sum)
  int32_t* err;
};

constexpr int tile_floats(int d) { return kRows * (d + 2); }
constexpr int own_floats(int d) { return 16 * (d + 2); }

__device__ __forceinline__ int last_le(const int32_t* v, int n, int x) {  // last i < n with v[i] <= x
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (v[mid] <= x) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// ---------------------------------------------------------------------------
// the plan: what both kernels know of the batch, built by every CTA
// ---------------------------------------------------------------------------
struct Plan {
  int32_t* ctx;     // [batch] tokens
  int32_t* cu;      // [groups + 1]
  int32_t* pre;     // [groups] shared tokens (0: the group's sequences are on their own)
  int32_t* lead;    // [groups] the sequence whose table holds them
  __host__ __device__ static size_t ints(int batch, int groups) {
    return static_cast<size_t>(batch) + 3 * static_cast<size_t>(groups) + 1;
  }
  __device__ Plan(int32_t* at, int batch, int groups) : ctx(at), cu(at + batch), pre(cu + groups + 1), lead(pre + groups) {}
};

template <int THREADS>
__device__ void build_plan(const SharedParams& p, const Plan& pl) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const bool report = blockIdx.x == 0;
  for (int b = tid; b < p.batch; b += THREADS) {
    int n = __ldcg(p.ctx + b);
    if (n < 0 || n > p.max_context) {
      if (report) flag_error(p.err, PSB_DEVERR_CONTEXT);
      n = n < 0 ? 0 : p.max_context;
    }
    pl.ctx[b] = n;
  }
  bool bad = false;
  for (int g = tid; g <= p.groups; g += THREADS) {
    const int a = __ldcg(p.cu + g), prev = g == 0 ? 0 : __ldcg(p.cu + g - 1);
    bad = bad || a < prev || prev < 0 || a > p.batch;
    pl.cu[g] = a;
  }
  bad = __syncthreads_or(bad) != 0;
  if (bad && report && tid == 0) flag_error(p.err, PSB_DEVERR_SEQLENS);
  for (int g = warp; g < p.groups; g += THREADS / 32) {
    // malformed groups: every sequence on its own
    const int b0 = bad ? 0 : pl.cu[g], b1 = bad ? 0 : pl.cu[g + 1];
    int best = -1, at = 0;
    for (int b = b0 + lane; b < b1; b += 32) {
      if (pl.ctx[b] > best) {
        best = pl.ctx[b];
        at = b;
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const int x = __shfl_xor_sync(0xffffffffu, best, o), y = __shfl_xor_sync(0xffffffffu, at, o);
      if (x > best || (x == best && y < at)) {
        best = x;
        at = y;
      }
    }
    if (lane == 0) {
      const int n = __ldcg(p.prefix + g);
      if (n < 0 && report) flag_error(p.err, PSB_DEVERR_CONTEXT);
      // one sequence shares with nobody: all of it is its own
      pl.pre[g] = b1 - b0 < 2 ? 0 : max(0, min(n, best));
      pl.lead[g] = at;
    }
  }
  __syncthreads();
}

// Exclusive scan of one value per thread over the CTA, and the total.
template <int THREADS>
__device__ __forceinline__ int scan_cta(int v, int& total) {
  __shared__ int32_t sums[THREADS / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += x;
  }
  __syncthreads();
  if (lane == 31) sums[warp] = incl;
  __syncthreads();
  int run = incl - v;
  total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) run += sums[w];
    total += sums[w];
  }
  return run;
}

// ---------------------------------------------------------------------------
// the shared part
// ---------------------------------------------------------------------------
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// The products and their commits, by the one lane for which ``on`` holds, in code
// that the whole warp runs through: operands then stay in uniform registers (issued
// from a branch of one lane, each product took 70 cycles for its operands' moves).
__device__ __forceinline__ void mma_ss(bool on, uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(static_cast<uint32_t>(accumulate)), "r"(static_cast<uint32_t>(on))
      : "memory");
}
__device__ __forceinline__ void mma_ts(bool on, uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(static_cast<uint32_t>(accumulate)), "r"(static_cast<uint32_t>(on))
      : "memory");
}
__device__ __forceinline__ void mma_commit(bool on, uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar), "r"(static_cast<uint32_t>(on))
      : "memory");
}
__device__ __forceinline__ bool elect_one() {
  uint32_t on;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(on));
  return on != 0;
}
// mbar_wait by a whole warp: its lanes give up together or not at all.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity)); }

// A run of steps of one tile.
struct Run {
  int kvh, tile, grp, b0, n_seq;  // tile of its kv head, group, first sequence and how many
  int j0, n;                      // its steps
};

// Walks a CTA's steps tile by tile.
struct Cursor {
  int kvh, tile, grp, in_grp, j0, left;
  __device__ Run take(const Plan& pl, const int32_t* tfirst, int tq, int groups, int n_tiles) {
    Run r;
    r.kvh = kvh;
    r.tile = tile;
    r.grp = grp;
    r.b0 = pl.cu[grp] + in_grp * tq;
    r.n_seq = min(tq, pl.cu[grp + 1] - r.b0);
    r.j0 = j0;
    r.n = min((pl.pre[grp] + kBN - 1) / kBN - j0, left);
    left -= r.n;
    j0 = 0;
    if (left > 0) {
      ++in_grp;
      if (++tile == n_tiles) {
        tile = 0;
        grp = 0;
        in_grp = 0;
        ++kvh;
      }
      while (tile >= tfirst[grp + 1]) {  // groups without tiles are passed over
        ++grp;
        in_grp = 0;
      }
    }
    return r;
  }
};

template <typename T, int D>
__global__ void __launch_bounds__(kTcThreads, 2)
    shared_prefix_kernel(const SharedParams p, const __grid_constant__ CUtensorMap tm_q,
                         const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v) {
  using Geo = TcGeom<D>;
  constexpr int kH = Geo::kH, kStages = Geo::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const smem = smem_raw + ((0u - smem_u32(smem_raw)) & 1023u);
  uint64_t* const bar_q = reinterpret_cast<uint64_t*>(smem + Geo::kOffBars);
  // of step x, its stage x % kStages (a barrier's next phase needs this one's products):
  uint64_t* const bar_k = bar_q + 1;               // [kStages] K landed
  uint64_t* const bar_s = bar_k + kStages;         // [kStages] Q K^T done: S written, the stage's K free
  uint64_t* const bar_v = bar_s + kStages;         // [kStages] V landed
  uint64_t* const bar_pv = bar_v + kStages;        // [kStages] P V done: the stage's V free
  uint64_t* const bar_p = bar_pv + kStages;        // [2] P written over S, in S buffer x & 1
  uint64_t* const bar_drain = bar_p + 2;           // after a failed wait: every product issued so far is done
  uint32_t* const s_tmem = reinterpret_cast<uint32_t*>(bar_drain + 1);
  static_assert((4 + 4 * kStages) * 8 + 4 <= 256, "barriers fit their area");
  const Plan plan(reinterpret_cast<int32_t*>(smem + Geo::kOffPlan), p.batch, p.groups);
  int32_t* const tfirst = plan.lead + p.groups;    // [groups + 1] tiles before a group, of one kv head
  int32_t* const sfirst = tfirst + p.groups + 1;   // [groups + 1] steps before a group, of one kv head
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int TQ = p.tq, group = p.group;
  if (tid == 0) {
    mbar_init(bar_q, 1);
    for (int i = 0; i < kStages; ++i) {
      mbar_init(bar_k + i, 1);
      mbar_init(bar_s + i, 1);
      mbar_init(bar_v + i, 1);
      mbar_init(bar_pv + i, 1);
    }
    for (int i = 0; i < 2; ++i) mbar_init(bar_p + i, kRows);
    mbar_init(bar_drain, 1);
    fence_barrier_init();
  }
  if (warp == 0) {
    tmem_alloc(s_tmem, kTmemCols);
    tmem_relinquish();
  }
  pdl_wait();  // lengths, groups, tables, q and the pools may come from the stream predecessor
  pdl_launch_dependents();  // (after the wait: the own kernel counts on it)

  build_plan<kTcThreads>(p, plan);
  int n_tiles, n_steps;
  {
    const int per = (p.groups + kTcThreads - 1) / kTcThreads;
    const int g0 = min(tid * per, p.groups), g1 = min(g0 + per, p.groups);
    auto tiles_of = [&](int g) { return plan.pre[g] > 0 ? (plan.cu[g + 1] - plan.cu[g] + TQ - 1) / TQ : 0; };
    auto steps_of = [&](int g) { return tiles_of(g) * ((plan.pre[g] + kBN - 1) / kBN); };
    int tiles = 0, steps = 0;
    for (int g = g0; g < g1; ++g) {
      tiles += tiles_of(g);
      steps += steps_of(g);
    }
    int t = scan_cta<kTcThreads>(tiles, n_tiles), s = scan_cta<kTcThreads>(steps, n_steps);
    for (int g = g0; g < g1; ++g) {
      tfirst[g] = t;
      sfirst[g] = s;
      t += tiles_of(g);
      s += steps_of(g);
    }
    if (tid == 0) {
      tfirst[p.groups] = n_tiles;
      sfirst[p.groups] = n_steps;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;
  const uint32_t total = static_cast<uint32_t>(n_steps) * p.hkv;  // below 2^31
  const uint32_t act = min(gridDim.x, (total + kMinSteps - 1) / kMinSteps), cta = blockIdx.x;
  if (cta >= act) {
    __syncthreads();  // every warp has read the address
    if (warp == 0) tmem_dealloc(tmem, kTmemCols);
    return;
  }
  const uint32_t share = total / act, extra = total - share * act;
  const uint32_t my_a = share * cta + min(cta, extra);
  const int n_mine = static_cast<int>(share + (cta < extra ? 1 : 0));
  auto cta_of = [&](uint32_t step) {  // the CTA a step was dealt to
    const uint32_t head = extra * (share + 1);
    return step < head ? step / (share + 1) : extra + (step - head) / share;
  };
  Cursor first;
  {
    first.kvh = static_cast<int>(my_a / n_steps);
    const int r = static_cast<int>(my_a - static_cast<uint32_t>(first.kvh) * n_steps);
    first.grp = last_le(sfirst, p.groups, r);  // (of groups without steps the last: it has some)
    const int n = (plan.pre[first.grp] + kBN - 1) / kBN;
    first.in_grp = (r - sfirst[first.grp]) / n;
    first.j0 = r - sfirst[first.grp] - first.in_grp * n;
    first.tile = tfirst[first.grp] + first.in_grp;
    first.left = n_mine;
  }
  bool fail = false;

  if (warp == 4) {
    // ---- products ----
    constexpr int kFmt = Elem<T>::code == PSB_BF16 ? 1 : 0;
    constexpr uint32_t idesc_s = umma_idesc_f16(kFmt, kRows, kBN, 0, 0), idesc_o = umma_idesc_f16(kFmt, kRows, D, 0, 1);
    const bool on = elect_one();
    const uint32_t s_base = smem_u32(smem);
    const uint64_t dq = umma_desc_sw128(s_base, 1024, 16);
    const uint64_t dk = umma_desc_sw128(s_base + Geo::kOffK, 1024, 16);
    const uint64_t dv = umma_desc_sw128(s_base + Geo::kOffV, 1024, kKvHalf);  // (of D 128 the second half's dims lie a half tile on)
    if (on) prefetch_tmap(&tm_q);
    const uint32_t box = static_cast<uint32_t>(TQ * group) * 128 * kH;
    Cursor sc = first, oc = first;
    int s_left = 0, o_left = 0, q_seen = 0;
    uint32_t k_st = 0, k_ph = 0, v_st = 0, v_ph = 0;
    bool begins = false, q_flight = false;
    // step i uses S buffer i & 1, for the (i >> 1)-th time; S runs two steps ahead of O
#pragma unroll 1
    for (int i = -2; i < n_mine; ++i) {
      if (i >= 0) {  // P V of step i
        if (o_left == 0) {
          o_left = oc.take(plan, tfirst, TQ, p.groups, n_tiles).n;
          begins = true;
        }
        if (!warp_wait(bar_v + v_st, v_ph) || !warp_wait(bar_p + (i & 1), (i >> 1) & 1)) {
          fail = true;
          break;
        }
        tc_fence_after();
        const uint32_t pcol = tmem + kSCol + (i & 1) * kBN;
        const uint64_t vd = dv + static_cast<uint64_t>(v_st * kH * (kKvHalf >> 4));
#pragma unroll
        for (int kk = 0; kk < kBN / 16; ++kk) mma_ts(on, tmem + kOCol, pcol + 8 * kk, vd + 128 * kk, idesc_o, !begins || kk > 0);
        mma_commit(on, smem_u32(bar_pv + v_st));
        --o_left;
        begins = false;
      }
      if (i + 2 < n_mine) {  // S of step i + 2, whose buffer held S and then P of step i
        if (i >= 0 && !warp_wait(bar_pv + v_st, v_ph)) {
          fail = true;
          break;
        }
        if (s_left == 0) {  // a run begins: its Q, once the last S of the run before (step i + 1) is done
          const uint32_t b_st = k_st == 0 ? kStages - 1 : k_st - 1, b_ph = k_st == 0 ? k_ph ^ 1 : k_ph;
          if (i > -2 && !warp_wait(bar_s + b_st, b_ph)) {
            fail = true;
            break;
          }
          const Run r = sc.take(plan, tfirst, TQ, p.groups, n_tiles);
          s_left = r.n;
          if (on) {
            mbar_arrive_expect_tx(bar_q, box);
#pragma unroll
            for (int h = 0; h < kH; ++h) tma_load_3d(smem + h * kQHalf, &tm_q, h * kHalf, r.kvh * group, r.b0, bar_q);
          }
          q_flight = true;
          if (!warp_wait(bar_q, q_seen & 1)) {
            fail = true;
            break;
          }
          ++q_seen;
          q_flight = false;
        }
        if (!warp_wait(bar_k + k_st, k_ph)) {
          fail = true;
          break;
        }
        tc_fence_after();
        const uint64_t kd = dk + static_cast<uint64_t>(k_st * kH * (kKvHalf >> 4));
#pragma unroll
        for (int h = 0; h < kH; ++h) {
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            mma_ss(on, tmem + kSCol + (i & 1) * kBN, dq + h * (kQHalf >> 4) + 2 * kk, kd + h * (kKvHalf >> 4) + 2 * kk, idesc_s, h > 0 || kk > 0);
        }
        mma_commit(on, smem_u32(bar_s + k_st));
        if (++k_st == kStages) {
          k_st = 0;
          k_ph ^= 1;
        }
        --s_left;
      }
      if (i >= 0 && ++v_st == kStages) {
        v_st = 0;
        v_ph ^= 1;
      }
    }
    if (fail) {
      if (on) flag_error(p.err, PSB_DEVERR_TIMEOUT);
      // let the copy and the products in flight land before shared memory and TMEM are released
      if (q_flight) (void)warp_wait(bar_q, q_seen & 1);
      mma_commit(on, smem_u32(bar_drain));
      (void)warp_wait(bar_drain, 0);
    }
  } else if (warp == 5) {
    // ---- copies: K of step x, then V of step x - 1 (the products need V later) ----
    if (lane == 0) {
      prefetch_tmap(&tm_k);
      prefetch_tmap(&tm_v);
    }
    const int bs = p.block_size, box_rows = min(bs, kBN), boxes = kBN / box_rows;
    const int64_t layer0 = static_cast<int64_t>(p.layer) * p.num_blocks;
    struct Walk {
      Cursor c;
      int left, j, kvh, n_blk, chunk;  // steps left of the run, its next step; entries of the prefix, chunk of 32 at hand
      const int32_t* row;
      int32_t id;                      // this lane's entry of the chunk
    };
    Walk wk{first, 0, 0, 0, 0, -1, nullptr, 0}, wv = wk;
    auto issue = [&](Walk& w, int x, const CUtensorMap* tm, uint64_t* bar, uint64_t* bar_free, uint32_t off) -> bool {
      if (w.left == 0) {
        const Run r = w.c.take(plan, tfirst, TQ, p.groups, n_tiles);
        w.left = r.n;
        w.j = r.j0;
        w.kvh = r.kvh;
        w.n_blk = (plan.pre[r.grp] + bs - 1) / bs;
        w.row = p.tables + static_cast<int64_t>(plan.lead[r.grp]) * p.table_stride;
        w.chunk = -1;
      }
      const int st = x % kStages;
      if (x >= kStages && !__all_sync(0xffffffffu, mbar_wait(bar_free + st, (x / kStages - 1) & 1))) return false;
      // the step's blocks, from block i0 on at row y (a block of more than a step's keys: a part of one)
      const int i0 = w.j * kBN / bs, y = bs > kBN ? w.j * kBN - i0 * bs : 0;
      const int n = min(boxes, w.n_blk - i0);  // blocks behind the prefix are not loaded: their keys are masked
      if (lane == 0) mbar_arrive_expect_tx(bar + st, static_cast<uint32_t>(n * box_rows) * 128 * kH);
      for (int b = 0; b < n; ++b) {
        const int i = i0 + b;
        if ((i >> 5) != w.chunk) {
          w.chunk = i >> 5;
          const int mine = w.chunk * 32 + lane;
          w.id = 0;
          if (mine < w.n_blk) {
            w.id = __ldcg(w.row + mine);
            if (w.id < 0 || w.id >= p.num_blocks) {  // flagged, and another block's keys read in its place
              flag_error(p.err, PSB_DEVERR_BLOCK_RANGE);
              w.id = 0;
            }
          }
        }
        const int32_t blk = __shfl_sync(0xffffffffu, w.id, i & 31);
        if (lane == 0) {
          const int32_t tile = static_cast<int32_t>((layer0 + blk) * p.hkv + w.kvh);
#pragma unroll
          for (int h = 0; h < kH; ++h)
            tma_load_3d(smem + off + (st * kH + h) * kKvHalf + b * box_rows * 128, tm, h * kHalf, y, tile, bar + st);
        }
      }
      ++w.j;
      --w.left;
      return true;
    };
    int x = 0;
    for (; x <= n_mine; ++x) {
      if (x < n_mine && !issue(wk, x, &tm_k, bar_k, bar_s, Geo::kOffK)) {
        fail = true;
        break;
      }
      if (x > 0 && !issue(wv, x - 1, &tm_v, bar_v, bar_pv, Geo::kOffV)) {
        fail = true;
        ++x;  // K of step x is on its way
        break;
      }
    }
    if (fail && lane == 0) {
      flag_error(p.err, PSB_DEVERR_TIMEOUT);
      // copies still in flight: the newest of each stage, K of the steps below x, V of those below x - 1
      for (int t = max(0, min(x, n_mine) - kStages); t < min(x, n_mine); ++t) (void)mbar_wait(bar_k + t % kStages, (t / kStages) & 1);
      for (int t = max(0, x - 1 - kStages); t < x - 1; ++t) (void)mbar_wait(bar_v + t % kStages, (t / kStages) & 1);
    }
  } else {
    // ---- softmax: thread r is row r of the tile and lane r of TMEM ----
    const int row = warp * 32 + lane;
    const int rseq = row / group;
    const uint32_t t_lane = tmem + (static_cast<uint32_t>(warp * 32) << 16);
    const float sc = p.scale_log2;
    Cursor cc = first;
    int g = 0;
    while (cc.left > 0 && !fail) {
      const Run r = cc.take(plan, tfirst, TQ, p.groups, n_tiles);
      const int pre = plan.pre[r.grp];
      const bool live = rseq < r.n_seq;
      int have = pre - r.j0 * kBN;  // keys there are, from the run's first on
      float ms = -INFINITY, l = 0.f;  // the exponents' reference (times sc), the sum
      for (int j = 0; j < r.n; ++j, ++g, have -= kBN) {
        const uint32_t st = g % kStages, ph = (g / kStages) & 1;
        if (!mbar_wait(bar_s + st, ph)) {
          fail = true;
          break;
        }
        tc_fence_after();
        const uint32_t t_s = t_lane + kSCol + (g & 1) * kBN;
        uint32_t sr[kBN];
        tmem_ld32(t_s, sr);
        tmem_ld32(t_s + 32, sr + 32);
        tmem_wait_ld();
        if (have < kBN) {
          // V rows behind the prefix (another token's, or never loaded) must
          // not reach P V, where 0 * NaN would be NaN: this thread's arrival
          // lets P V read the stage
          if (!mbar_wait(bar_v + st, ph)) {
            fail = true;
            break;
          }
          if (row < kBN && row >= have) {
#pragma unroll
            for (int h = 0; h < kH; ++h) {
              const uint32_t vrow = smem_u32(smem) + Geo::kOffV + (st * kH + h) * kKvHalf + row * 128;
#pragma unroll
              for (int c = 0; c < 128; c += 16) st_shared_zero16(vrow + c);
            }
            fence_proxy_async_smem();  // visible to the tensor core
          }
#pragma unroll
          for (int c = 0; c < kBN; ++c)
            if (c >= have) sr[c] = __float_as_uint(-INFINITY);
        }
        float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
        for (int c = 0; c < kBN; c += 4) {
          mx0 = max3(mx0, __uint_as_float(sr[c]), __uint_as_float(sr[c + 1]));
          mx1 = max3(mx1, __uint_as_float(sr[c + 2]), __uint_as_float(sr[c + 3]));
        }
        const float mxs = fmaxf(mx0, mx1) * sc;
        const bool grow = mxs > ms + kRescaleLog2;
        if (__any_sync(0xffffffffu, grow)) {  // (the warp's TMEM access is collective)
          const float ms_new = grow ? mxs : ms;
          const float alpha = ms == -INFINITY ? 0.f : ex2_approx(ms - ms_new);  // (a step has at least one key)
          if (j > 0) {  // O holds P V of the earlier steps once the last of them is done
            if (!mbar_wait(bar_pv + (g - 1) % kStages, ((g - 1) / kStages) & 1)) {
              fail = true;
              break;
            }
            tc_fence_after();
#pragma unroll 1
            for (int q = 0; q < D; q += 32) {
              uint32_t ot[32];
              tmem_ld32(t_lane + kOCol + q, ot);
              tmem_wait_ld();
#pragma unroll
              for (int d = 0; d < 32; ++d) ot[d] = __float_as_uint(__uint_as_float(ot[d]) * alpha);
              tmem_st32(t_lane + kOCol + q, ot);
            }
            tmem_wait_st();
          }
          l *= alpha;
          ms = ms_new;
        }
        const float mu = ms == -INFINITY ? 0.f : ms;
        uint32_t pk[kBN / 2];
        const uint64_t sc2 = pair2(sc, sc), nmu2 = pair2(-mu, -mu);
        uint64_t rs2 = pair2(0.f, 0.f);
#pragma unroll
        for (int c = 0; c < kBN; c += 2) {
          const float2 a = unpair2(fma2(pair2(__uint_as_float(sr[c]), __uint_as_float(sr[c + 1])), sc2, nmu2));
          const float x0 = ex2_approx(a.x), x1 = ex2_approx(a.y);
          rs2 = add2(rs2, pair2(x0, x1));
          pk[c / 2] = pack2<T>(x0, x1);
        }
        const float2 rs = unpair2(rs2);
        l += rs.x + rs.y;
        tmem_st32(t_s, pk);
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(bar_p + (g & 1));
      }
      if (fail) break;
      // the run's partial; the next run's first P V comes after its P
      if (!warp_wait(bar_pv + (g - 1) % kStages, ((g - 1) / kStages) & 1)) {
        fail = true;
        break;
      }
      tc_fence_after();
      const int ord = r.kvh * n_tiles + r.tile;
      float* const part = p.tile_part + static_cast<int64_t>(cta + ord) * tile_floats(D);
#pragma unroll 1
      for (int q = 0; q < D; q += 32) {
        uint32_t ot[32];
        tmem_ld32(t_lane + kOCol + q, ot);
        tmem_wait_ld();
        if (live) {
#pragma unroll
          for (int d = 0; d < 32; d += 4)
            reinterpret_cast<float4*>(part)[((q + d) >> 2) * kRows + row] =
                make_float4(__uint_as_float(ot[d]), __uint_as_float(ot[d + 1]), __uint_as_float(ot[d + 2]), __uint_as_float(ot[d + 3]));
        }
        __syncwarp();
      }
      if (live) reinterpret_cast<float2*>(part + kRows * D)[row] = make_float2(ms, l);
      if (r.j0 == 0 && tid == 0) {
        const uint32_t end = my_a + static_cast<uint32_t>(g) - r.n + (pre + kBN - 1) / kBN;  // the tile's last step + 1
        p.tile_info[r.kvh * p.max_tiles + r.tile] = make_int2(static_cast<int>(cta) + ord, static_cast<int>(cta_of(end - 1) - cta) + 1);
      }
      tc_fence_before();
    }
    if (fail && lane == 0) flag_error(p.err, PSB_DEVERR_TIMEOUT);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// ---------------------------------------------------------------------------
// each sequence's own part
// ---------------------------------------------------------------------------
// As the plain decode: a warp streams its slices (16 tokens of HP kv heads)
// through a ring of its own with 16-byte cp.async copies.  HP = 2 (up to 8 q
// heads per kv head): rows 0-7 of the m16n8k16 tile are one kv head's q heads,
// rows 8-15 the next one's.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, uint64_t policy) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "l"(policy) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// floor(n w / warps) and its reverse, for items dealt over warps
struct Deal {
  int64_t n;
  int warps;
  __device__ __forceinline__ int64_t start(int w) const { return n * w / warps; }
  __device__ __forceinline__ int warp_of(int64_t item) const { return static_cast<int>(((item + 1) * warps - 1) / n); }
};

template <typename T, int D, int HP>
__global__ void __launch_bounds__(kOwnThreads) shared_own_kernel(const SharedParams p) {
  using Geo = OwnGeom<D, HP>;
  constexpr int kRing = Geo::kRing, kSteps = D / 16, kCols = D / 8;  // k steps; 16-byte columns of a row
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const ring_all = smem_raw + ((0u - smem_u32(smem_raw)) & 1023u);
  const Plan plan(reinterpret_cast<int32_t*>(ring_all + Geo::kBytes), p.batch, p.groups);
  int32_t* const s_start = plan.lead + p.groups;  // [batch] first token of its own
  int32_t* const bpre = s_start + p.batch;        // [batch + 1] slices before a sequence
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int gq = lane >> 2, t = lane & 3;
  const int G = p.group, B = p.batch, hgs = p.hkv / HP;
  // No wait for the stream predecessor here: this launch begins once every CTA
  // of shared_prefix_kernel has begun, which each does behind a wait for what
  // came before (and everything is read through L2).  What it waits for, at its
  // end, is that kernel itself, so that its own end is the end of both.
  pdl_launch_dependents();
  build_plan<kOwnThreads>(p, plan);
  for (int b = tid; b < B; b += kOwnThreads) s_start[b] = 0;
  __syncthreads();
  for (int g = warp; g < p.groups; g += kOwnWarps)
    if (plan.pre[g] > 0)
      for (int b = plan.cu[g] + lane; b < plan.cu[g + 1]; b += 32)
        if (plan.ctx[b] >= plan.pre[g]) s_start[b] = plan.pre[g];
  __syncthreads();
  auto slices_of = [&](int b) { return max(0, (plan.ctx[b] + 15) / 16 - s_start[b] / 16) * (plan.ctx[b] > s_start[b] ? 1 : 0); };
  int n_slices;
  {
    const int per = (B + kOwnThreads - 1) / kOwnThreads;
    const int b0 = min(tid * per, B), b1 = min(b0 + per, B);
    int n = 0;
    for (int b = b0; b < b1; ++b) n += slices_of(b);
    int run = scan_cta<kOwnThreads>(n, n_slices);
    for (int b = b0; b < b1; ++b) {
      bpre[b] = run;
      run += slices_of(b);
    }
    if (tid == 0) bpre[B] = n_slices;
    __syncthreads();
  }
  const int64_t items = static_cast<int64_t>(n_slices) * hgs;
  const Deal deal{items, static_cast<int>(min(static_cast<int64_t>(gridDim.x * kOwnWarps), max(int64_t(1), items / kOwnMinItems)))};
  // warps in order of their place in a CTA: few warps are spread over the SMs
  const int gw = warp * gridDim.x + blockIdx.x;
  // what the join needs: tiles of the sequences, partials of the pairs
  const int gt = blockIdx.x * kOwnThreads + tid, gts = gridDim.x * kOwnThreads;
  if (gt < B) {
    for (int b = gt; b < B; b += gts) {
      int2 at = make_int2(-1, 0);
      if (s_start[b] > 0) {
        int g = last_le(plan.cu, p.groups, b), tiles = 0;  // (of empty groups the last: it holds b)
        for (int i = 0; i < g; ++i)
          if (plan.pre[i] > 0) tiles += (plan.cu[i + 1] - plan.cu[i] + p.tq - 1) / p.tq;
        const int m = b - plan.cu[g];
        at = make_int2(tiles + m / p.tq, m % p.tq);
      }
      p.seq_info[b] = at;
    }
  }
  for (int s = gt; s < B * hgs; s += gts) {
    const int hg = s / B, b = s - hg * B;
    int2 at = make_int2(0, 0);
    if (bpre[b + 1] > bpre[b]) {
      const int64_t a = static_cast<int64_t>(hg) * n_slices + bpre[b], e = static_cast<int64_t>(hg) * n_slices + bpre[b + 1];
      const int w0 = deal.warp_of(a), w1 = deal.warp_of(e - 1);
      at = make_int2(w0 + s, w1 - w0 + 1);
    }
    p.own_info[s] = at;
  }

  const bool works = gw < deal.warps && items > 0;
  const int64_t my_a = works ? deal.start(gw) : 0, my_e = works ? deal.start(gw + 1) : 0;
  uint8_t* const ring = ring_all + warp * kRing * Geo::kSlot;
  const uint32_t ring_u = smem_u32(ring);
  const uint64_t policy = l2_policy_evict_first();
  const int64_t layer0 = static_cast<int64_t>(p.layer) * p.num_blocks;
  const bool row_lo = gq < G, row_hi = HP == 2 ? gq < G : gq + 8 < G;

  // A chunk: up to 32 consecutive slices of the warp's range, one a lane: its
  // place in the pool (-1: its block is outside), the valid tokens [lo, hi), and
  // whether a pair or the range begins or ends with it.
  struct Chunk {
    int64_t beg;
    int n;
    int32_t blk, row, meta, pair;
  };
  auto build_chunk = [&](int64_t beg) -> Chunk {
    Chunk c;
    c.beg = beg;
    c.n = static_cast<int>(min(int64_t(32), my_e - beg));
    c.blk = -1;
    c.row = c.meta = c.pair = 0;
    if (lane < c.n) {
      const int64_t i = beg + lane;
      const int hg = static_cast<int>(i / n_slices), r = static_cast<int>(i - static_cast<int64_t>(hg) * n_slices);
      const int b = last_le(bpre, B, r);  // (of sequences without slices the last: it has some)
      const int j = r - bpre[b], pos = (s_start[b] / 16 + j) * 16;
      const int lo = max(0, s_start[b] - pos), hi = min(16, plan.ctx[b] - pos);
      const int bi = pos / p.block_size;
      c.row = pos - bi * p.block_size;
      c.blk = __ldcg(p.tables + static_cast<int64_t>(b) * p.table_stride + bi);
      if (c.blk < 0 || c.blk >= p.num_blocks) {
        flag_error(p.err, PSB_DEVERR_BLOCK_RANGE);
        c.blk = -1;
      }
      c.meta = lo | hi << 5 | (j == 0 || i == my_a ? 1 << 10 : 0) | (r + 1 == bpre[b + 1] || i == my_e - 1 ? 1 << 11 : 0);
      c.pair = hg * B + b;
    }
    return c;
  };
  Chunk cur{}, nxt{};
  bool c_ok = false, n_ok = false;
  if (my_e > my_a) {
    cur = build_chunk(my_a);
    c_ok = true;
    if (my_a + cur.n < my_e) {
      nxt = build_chunk(my_a + cur.n);
      n_ok = true;
    }
  }
  int ib = 0;
  uint32_t issued = 0, consumed = 0;
  int32_t meta = 0, meta_pair = 0;  // lane s: of ring slot s
  auto issue_one = [&]() {
    const uint32_t slot = issued % kRing;
    const uint32_t dst = ring_u + slot * Geo::kSlot;
    const int32_t blk = __shfl_sync(0xffffffffu, cur.blk, ib), r0 = __shfl_sync(0xffffffffu, cur.row, ib);
    const int32_t mt = __shfl_sync(0xffffffffu, cur.meta, ib), pair = __shfl_sync(0xffffffffu, cur.pair, ib);
    if (blk >= 0) {
      const int hg = pair / B;
#pragma unroll
      for (int hs = 0; hs < HP; ++hs) {
        const int64_t at = (((layer0 + blk) * p.hkv + hg * HP + hs) * p.block_size + r0) * (D * 2);
#pragma unroll
        for (int i = 0; i < 16 * kCols / 32; ++i) {
          const int c = lane + 32 * i, r = c / kCols, col = c % kCols;
          const uint32_t d = dst + hs * Geo::kTile + r * (D * 2) + ((col ^ (r & 7)) << 4);
          copy16(d, p.k_cache + at + c * 16, policy);
          copy16(d + Geo::kKV, p.v_cache + at + c * 16, policy);
        }
      }
    }
    copy_commit();
    if (lane == static_cast<int>(slot)) {
      meta = mt | (blk >= 0 ? 1 << 12 : 0);
      meta_pair = pair;
    }
    ++issued;
    if (++ib == cur.n) {
      c_ok = n_ok;
      cur = nxt;
      ib = 0;
      n_ok = false;
      if (c_ok && cur.beg + cur.n < my_e) {
        nxt = build_chunk(cur.beg + cur.n);
        n_ok = true;
      }
    }
  };
  while (c_ok && issued < static_cast<uint32_t>(kRing)) issue_one();

  uint32_t qa[kSteps][4];
  float o[kCols][4];
  float m_lo = -INFINITY, m_hi = -INFINITY, l_lo = 0.f, l_hi = 0.f;
  int32_t pair = 0;
  while (consumed != issued) {
    const uint32_t slot = consumed % kRing;
    const int32_t mt = __shfl_sync(0xffffffffu, meta, slot);
    const int lo = mt & 31, hi = (mt >> 5) & 31;
    const uint32_t base = ring_u + slot * Geo::kSlot;
    if ((mt >> 10) & 1) {  // a pair (or the range) begins: its q rows
      pair = __shfl_sync(0xffffffffu, meta_pair, slot);
      const int hg = pair / B, b = pair - hg * B;
      const T* qb = reinterpret_cast<const T*>(p.q) + b * p.qsb + 2 * t;
      const T* qlo = qb + static_cast<int64_t>(hg * HP * G + gq) * p.qsh;
      const T* qhi = qb + static_cast<int64_t>(HP == 2 ? (hg * 2 + 1) * G + gq : hg * G + gq + 8) * p.qsh;
#pragma unroll
      for (int ks = 0; ks < kSteps; ++ks) {
        qa[ks][0] = row_lo ? __ldcg(reinterpret_cast<const uint32_t*>(qlo + 16 * ks)) : 0u;
        qa[ks][1] = row_hi ? __ldcg(reinterpret_cast<const uint32_t*>(qhi + 16 * ks)) : 0u;
        qa[ks][2] = row_lo ? __ldcg(reinterpret_cast<const uint32_t*>(qlo + 16 * ks + 8)) : 0u;
        qa[ks][3] = row_hi ? __ldcg(reinterpret_cast<const uint32_t*>(qhi + 16 * ks + 8)) : 0u;
      }
      m_lo = m_hi = -INFINITY;
      l_lo = l_hi = 0.f;
#pragma unroll
      for (int n = 0; n < kCols; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
    }
    if (issued - consumed == static_cast<uint32_t>(kRing)) copy_wait<kRing - 1>(); else copy_wait<0>();
    __syncwarp();
    if ((mt >> 12) & 1) {
      float s[2][4];
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) {
        float acc[HP][4];
#pragma unroll
        for (int hs = 0; hs < HP; ++hs) {
          acc[hs][0] = acc[hs][1] = acc[hs][2] = acc[hs][3] = 0.f;  // (of its rows, half are the other head's: not used)
          const uint32_t krow = base + hs * Geo::kTile + (nt * 8 + (lane & 7)) * (D * 2);
#pragma unroll
          for (int kp = 0; kp < kSteps / 2; ++kp) {  // two k steps a load
            uint32_t b0, b1, b2, b3;
            ldsm_x4(krow + (((kp * 4 + (lane >> 3)) ^ (lane & 7)) << 4), b0, b1, b2, b3);
            mma_16816<T>(acc[hs], qa[2 * kp][0], qa[2 * kp][1], qa[2 * kp][2], qa[2 * kp][3], b0, b1);
            mma_16816<T>(acc[hs], qa[2 * kp + 1][0], qa[2 * kp + 1][1], qa[2 * kp + 1][2], qa[2 * kp + 1][3], b2, b3);
          }
        }
        s[nt][0] = acc[0][0];
        s[nt][1] = acc[0][1];
        s[nt][2] = acc[HP - 1][2];
        s[nt][3] = acc[HP - 1][3];
      }
      uint32_t keep[2] = {0xffffffffu, 0xffffffffu};  // of V's rows: what is masked may hold anything (even NaN)
      if (hi < 16 || lo > 0) {
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) {
          keep[nt] = 0;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int tok = nt * 8 + 2 * t + e;
            if (tok >= lo && tok < hi) {
              keep[nt] |= e == 0 ? 0x0000ffffu : 0xffff0000u;
            } else {
              s[nt][e] = -INFINITY;
              s[nt][2 + e] = -INFINITY;
            }
          }
        }
      }
      float mb_lo = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1]));
      float mb_hi = fmaxf(fmaxf(s[0][2], s[0][3]), fmaxf(s[1][2], s[1][3]));
      mb_lo = fmaxf(mb_lo, __shfl_xor_sync(0xffffffffu, mb_lo, 1));
      mb_hi = fmaxf(mb_hi, __shfl_xor_sync(0xffffffffu, mb_hi, 1));
      mb_lo = fmaxf(mb_lo, __shfl_xor_sync(0xffffffffu, mb_lo, 2));
      mb_hi = fmaxf(mb_hi, __shfl_xor_sync(0xffffffffu, mb_hi, 2));
      // every slice holds a valid token: the new maxima are finite (or the scores are not numbers)
      const float mn_lo = fmaxf(m_lo, mb_lo), mn_hi = fmaxf(m_hi, mb_hi);
      const float al_lo = ex2_approx((m_lo - mn_lo) * p.scale_log2), al_hi = ex2_approx((m_hi - mn_hi) * p.scale_log2);
      m_lo = mn_lo;
      m_hi = mn_hi;
      const float ms_lo = mn_lo * p.scale_log2, ms_hi = mn_hi * p.scale_log2;
      float pr[2][4];
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) {
        pr[nt][0] = ex2_approx(fmaf(s[nt][0], p.scale_log2, -ms_lo));
        pr[nt][1] = ex2_approx(fmaf(s[nt][1], p.scale_log2, -ms_lo));
        pr[nt][2] = ex2_approx(fmaf(s[nt][2], p.scale_log2, -ms_hi));
        pr[nt][3] = ex2_approx(fmaf(s[nt][3], p.scale_log2, -ms_hi));
      }
      l_lo = l_lo * al_lo + ((pr[0][0] + pr[0][1]) + (pr[1][0] + pr[1][1]));
      l_hi = l_hi * al_hi + ((pr[0][2] + pr[0][3]) + (pr[1][2] + pr[1][3]));
#pragma unroll
      for (int n = 0; n < kCols; ++n) {
        o[n][0] *= al_lo;
        o[n][1] *= al_lo;
        o[n][2] *= al_hi;
        o[n][3] *= al_hi;
      }
      const uint32_t pa0 = pack2<T>(pr[0][0], pr[0][1]), pa1 = pack2<T>(pr[0][2], pr[0][3]);
      const uint32_t pa2 = pack2<T>(pr[1][0], pr[1][1]), pa3 = pack2<T>(pr[1][2], pr[1][3]);
      const int vr = ((lane >> 3) & 1) * 8 + (lane & 7);
#pragma unroll
      for (int hs = 0; hs < HP; ++hs) {
        const uint32_t vrow = base + Geo::kKV + hs * Geo::kTile + vr * (D * 2);
#pragma unroll
        for (int dp = 0; dp < kCols / 2; ++dp) {
          uint32_t b0, b1, b2, b3;
          ldsm_x4_t(vrow + (((dp * 2 + (lane >> 4)) ^ (vr & 7)) << 4), b0, b1, b2, b3);
          b0 &= keep[0];
          b1 &= keep[1];
          b2 &= keep[0];
          b3 &= keep[1];
          if constexpr (HP == 1) {
            mma_16816<T>(o[2 * dp], pa0, pa1, pa2, pa3, b0, b1);
            mma_16816<T>(o[2 * dp + 1], pa0, pa1, pa2, pa3, b2, b3);
          } else {
            // the rows that are this head's, added in registers: zeros in the
            // other head's probabilities would still make NaN of an infinite value
            float x[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};
            mma_16816<T>(x, pa0, pa1, pa2, pa3, b0, b1);
            mma_16816<T>(y, pa0, pa1, pa2, pa3, b2, b3);
            o[2 * dp][2 * hs] += x[2 * hs];
            o[2 * dp][2 * hs + 1] += x[2 * hs + 1];
            o[2 * dp + 1][2 * hs] += y[2 * hs];
            o[2 * dp + 1][2 * hs + 1] += y[2 * hs + 1];
          }
        }
      }
    }
    __syncwarp();
    ++consumed;
    if (c_ok) issue_one();  // refill the slot just read
    if ((mt >> 11) & 1) {   // the pair's or the range's end: its partial
      float ll = l_lo, lh = l_hi;
      ll += __shfl_xor_sync(0xffffffffu, ll, 1);
      lh += __shfl_xor_sync(0xffffffffu, lh, 1);
      ll += __shfl_xor_sync(0xffffffffu, ll, 2);
      lh += __shfl_xor_sync(0xffffffffu, lh, 2);
      float* const part = p.own_part + static_cast<int64_t>(gw + pair) * own_floats(D);
      float2* const ml = reinterpret_cast<float2*>(part + 16 * D);
#pragma unroll
      for (int n = 0; n < kCols; ++n) {
        if (row_lo) *reinterpret_cast<float2*>(part + gq * D + 8 * n + 2 * t) = make_float2(o[n][0], o[n][1]);
        if (row_hi) *reinterpret_cast<float2*>(part + (gq + 8) * D + 8 * n + 2 * t) = make_float2(o[n][2], o[n][3]);
      }
      if (t == 0 && row_lo) ml[gq] = make_float2(m_lo * p.scale_log2, ll);
      if (t == 0 && row_hi) ml[gq + 8] = make_float2(m_hi * p.scale_log2, lh);
    }
  }
  pdl_wait();  // shared_prefix_kernel's end (see above)
}

// ---------------------------------------------------------------------------
// the join
// ---------------------------------------------------------------------------
// One row (a sequence's q head) per D / 4 lanes, four partials in flight (they
// come from L2: a round of loads costs more than their bytes).
constexpr int kJoinThreads = 128, kBatch = 4;

template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads) shared_join_kernel(const SharedParams p, int hp) {
  constexpr int kLanes = D / 4, kRowsWarp = 32 / kLanes;
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int64_t u = (static_cast<int64_t>(blockIdx.x) * (kJoinThreads / 32) + (threadIdx.x >> 5)) * kRowsWarp + lane / kLanes;
  const int hq = p.hkv * p.group;
  if (u >= static_cast<int64_t>(p.batch) * hq) return;
  const int c4 = lane % kLanes, b = static_cast<int>(u / hq), head = static_cast<int>(u - static_cast<int64_t>(b) * hq);
  const int kvh = head / p.group, gh = head - kvh * p.group;
  const int s = (kvh / hp) * p.batch + b;
  const int2 seq = __ldcg(p.seq_info + b), own = __ldcg(p.own_info + s);
  int2 tile = make_int2(0, 0);
  if (seq.x >= 0) tile = __ldcg(p.tile_info + kvh * p.max_tiles + seq.x);
  const int trow = seq.y * p.group + gh, orow = (hp == 2 ? (kvh & 1) * 8 : 0) + gh;
  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  const int n = tile.y + own.y;
  for (int i0 = 0; i0 < n; i0 += kBatch) {
    float2 ml[kBatch];
    float4 v[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int i = i0 + j;
      ml[j] = make_float2(-INFINITY, 0.f);
      v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (i < tile.y) {
        const float* part = p.tile_part + static_cast<int64_t>(tile.x + i) * tile_floats(D);
        ml[j] = __ldcg(reinterpret_cast<const float2*>(part + kRows * D) + trow);
        v[j] = __ldcg(reinterpret_cast<const float4*>(part) + c4 * kRows + trow);
      } else if (i < n) {
        const float* part = p.own_part + static_cast<int64_t>(own.x + i - tile.y) * own_floats(D);
        ml[j] = __ldcg(reinterpret_cast<const float2*>(part + 16 * D) + orow);
        v[j] = __ldcg(reinterpret_cast<const float4*>(part + orow * D) + c4);
      }
    }
    float mn = m;
#pragma unroll
    for (int j = 0; j < kBatch; ++j) mn = fmaxf(mn, ml[j].x);
    const float mu = mn == -INFINITY ? 0.f : mn, a = ex2_approx(m - mu);
    m = mn;
    l *= a;
    o.x *= a;
    o.y *= a;
    o.z *= a;
    o.w *= a;
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const float w = ex2_approx(ml[j].x - mu);
      l = fmaf(ml[j].y, w, l);
      o.x = fmaf(v[j].x, w, o.x);
      o.y = fmaf(v[j].y, w, o.y);
      o.z = fmaf(v[j].z, w, o.z);
      o.w = fmaf(v[j].w, w, o.w);
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  T* const out = reinterpret_cast<T*>(p.out) + b * p.osb + head * p.osh + 4 * c4;
  out[0] = Elem<T>::from_float(o.x * inv);
  out[1] = Elem<T>::from_float(o.y * inv);
  out[2] = Elem<T>::from_float(o.z * inv);
  out[3] = Elem<T>::from_float(o.w * inv);
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
bool takes(int batch, int groups, int q_heads, int hkv, int head_dim, int block_size, int dtype, int max_context) {
  if (!(dtype == PSB_BF16 || dtype == PSB_F16) || !(head_dim == 64 || head_dim == 128)) return false;
  if (batch <= 0 || batch > kMaxBatch || groups < 0 || groups > kMaxBatch || hkv <= 0 || q_heads <= 0 || q_heads % hkv) return false;
  const int group = q_heads / hkv;
  if (group > 16 || block_size < 16 || block_size % 16 || !(64 % block_size == 0 || block_size % 64 == 0)) return false;
  const int64_t steps = (static_cast<int64_t>(max_context) + kBN) / kBN, tiles = batch / (kRows / group) + std::min(groups, batch / 2) + 1;
  return static_cast<int64_t>(batch) * hkv < (1 << 24) && steps * tiles < (int64_t(1) << 31) / hkv &&
         static_cast<int64_t>(max_context) * batch / 16 < (int64_t(1) << 31) / 2;
}

struct Layout {
  int max_tiles;
  size_t tile_info, seq_info, own_info, tile_part, own_part, bytes;
  Layout(int batch, int groups, int group, int hkv, int d) {
    max_tiles = batch / (kRows / group) + std::min(groups, batch / 2) + 1;
    size_t at = 0;
    auto take = [&](size_t n) {
      const size_t r = at;
      at = align_up(at + n, 256);
      return r;
    };
    tile_info = take(sizeof(int2) * static_cast<size_t>(hkv) * max_tiles);
    seq_info = take(sizeof(int2) * static_cast<size_t>(batch));
    own_info = take(sizeof(int2) * static_cast<size_t>(hkv) * batch);
    tile_part = take(sizeof(float) * tile_floats(d) * (static_cast<size_t>(hkv) * max_tiles + kMaxTcCtas));
    own_part = take(sizeof(float) * own_floats(d) * (static_cast<size_t>(hkv) * batch + static_cast<size_t>(kMaxOwnCtas) * kOwnWarps));
    bytes = at;
  }
};

template <typename T, int D>
int launch(SharedParams p, int num_layers, cudaStream_t s) {
  const CUtensorMapDataType dt = Elem<T>::code == PSB_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const int sms = device_sm_count();
  if (sms <= 0) return PSB_ERR_CUDA;
  const bool two = D == 64 && p.group <= 8 && p.hkv % 2 == 0;  // (a tile of two heads of D 128 takes too many registers)
  CUtensorMap tq, tk, tv;
  const int64_t tiles = static_cast<int64_t>(num_layers) * p.num_blocks * p.hkv, hq = static_cast<int64_t>(p.hkv) * p.group;
  const int64_t qdims[3] = {D, hq, p.batch}, qstr[2] = {p.qsh * 2, p.qsb * 2}, kdims[3] = {D, p.block_size, tiles},
                kstr[2] = {D * 2, static_cast<int64_t>(p.block_size) * D * 2};
  const int qbox[3] = {kHalf, p.group, p.tq}, kbox[3] = {kHalf, std::min(p.block_size, kBN), 1};
  if (!encode_box_map(&tq, p.q, qdims, qstr, qbox, dt) || !encode_box_map(&tk, p.k_cache, kdims, kstr, kbox, dt) ||
      !encode_box_map(&tv, p.v_cache, kdims, kstr, kbox, dt))
    return PSB_ERR_CUDA;
  const auto pre = shared_prefix_kernel<T, D>;
  const auto own = two ? shared_own_kernel<T, D, D == 64 ? 2 : 1> : shared_own_kernel<T, D, 1>;
  const auto join = shared_join_kernel<T, D>;
  const size_t pre_smem = 1024 + TcGeom<D>::kOffPlan + sizeof(int32_t) * (Plan::ints(p.batch, p.groups) + 2 * (static_cast<size_t>(p.groups) + 1));
  const size_t own_smem = 1024 + (two ? OwnGeom<D, D == 64 ? 2 : 1>::kBytes : OwnGeom<D, 1>::kBytes) +
                          sizeof(int32_t) * (Plan::ints(p.batch, p.groups) + 2 * static_cast<size_t>(p.batch) + 1);
  int occ = 0, own_occ = 0;
  if (!kernel_occupancy(reinterpret_cast<const void*>(pre), kTcThreads, pre_smem, &occ) || occ < 1 ||
      !kernel_occupancy(reinterpret_cast<const void*>(own), kOwnThreads, own_smem, &own_occ) || own_occ < 1)
    return PSB_ERR_CUDA;
  discard_stale_error();
  const int pre_grid = std::min(kMaxTcCtas, sms * std::min(occ, 2));
  cudaError_t e = launch_pdl(pre, dim3(pre_grid), dim3(kTcThreads), pre_smem, s, p, tq, tk, tv);
  if (e != cudaSuccess) return record_cuda_error(e);
  const int own_grid = std::min(kMaxOwnCtas, sms * std::min(own_occ, 2));
  e = launch_pdl(own, dim3(own_grid), dim3(kOwnThreads), own_smem, s, p);
  if (e != cudaSuccess) return record_cuda_error(e);
  const int64_t rows = static_cast<int64_t>(p.batch) * hq, per = kJoinThreads / (D / 4);
  e = launch_pdl(join, dim3(static_cast<unsigned>((rows + per - 1) / per)), dim3(kJoinThreads), 0, s, p, two ? 2 : 1);
  if (e != cudaSuccess) return record_cuda_error(e);
  return check_launch();
}

}  // namespace
}  // namespace psb

using namespace psb;

extern "C" size_t psb_paged_decode_shared_workspace_size(int32_t batch, int32_t num_groups, int32_t q_heads, int32_t num_kv_heads,
                                                         int32_t head_dim, int32_t block_size, int32_t max_context, int32_t dtype) {
  if (max_context < 0 || !takes(batch, num_groups, q_heads, num_kv_heads, head_dim, block_size, dtype, max_context)) return 0;
  return Layout(batch, num_groups, q_heads / num_kv_heads, num_kv_heads, head_dim).bytes;
}

extern "C" int psb_paged_decode_shared(const void* query, int64_t q_stride_b, int64_t q_stride_h, void* out, int64_t o_stride_b,
                                       int64_t o_stride_h, const void* k_cache, const void* v_cache, const int32_t* block_tables,
                                       int64_t table_stride, const int32_t* context_lens, const int32_t* cu_groups,
                                       const int32_t* prefix_lens, int32_t batch, int32_t num_groups, int32_t q_heads,
                                       int32_t layer, int32_t num_layers, int64_t num_blocks, int32_t num_kv_heads,
                                       int32_t block_size, int32_t head_dim, int32_t dtype, int32_t max_context, float scale,
                                       void* workspace, size_t workspace_bytes, int32_t* error_flag, psb_stream_t stream) {
  if (batch < 0 || num_groups < 0 || q_heads <= 0 || num_kv_heads <= 0 || q_heads % num_kv_heads || block_size <= 0 ||
      head_dim <= 0 || layer < 0 || layer >= num_layers || num_blocks <= 0 || max_context < 0 || table_stride < 0 ||
      !(dtype == PSB_F32 || dtype == PSB_F16 || dtype == PSB_BF16) || !(scale > 0.f) || !(scale < INFINITY))
    return PSB_ERR_INVALID;
  if (batch == 0) return PSB_OK;
  if (!query || !out || !k_cache || !v_cache || !block_tables || !context_lens || (num_groups > 0 && (!cu_groups || !prefix_lens)))
    return PSB_ERR_INVALID;
  auto al16 = [](const void* x) { return reinterpret_cast<uintptr_t>(x) % 16 == 0; };
  if (!takes(batch, num_groups, q_heads, num_kv_heads, head_dim, block_size, dtype, max_context) || !al16(query) || !al16(k_cache) ||
      !al16(v_cache) || q_stride_b % 8 || q_stride_h % 8 || q_stride_b <= 0 || q_stride_h <= 0 ||
      static_cast<int64_t>(num_layers) * num_blocks * num_kv_heads > INT32_MAX)
    return PSB_ERR_UNSUPPORTED;
  const int group = q_heads / num_kv_heads;
  const Layout lay(batch, num_groups, group, num_kv_heads, head_dim);
  if (!workspace || !al16(workspace) || workspace_bytes < lay.bytes) return PSB_ERR_WORKSPACE;
  SharedParams p{};
  p.q = static_cast<const char*>(query);
  p.qsb = q_stride_b;
  p.qsh = q_stride_h;
  p.out = static_cast<char*>(out);
  p.osb = o_stride_b;
  p.osh = o_stride_h;
  p.k_cache = static_cast<const char*>(k_cache);
  p.v_cache = static_cast<const char*>(v_cache);
  p.tables = block_tables;
  p.table_stride = table_stride;
  p.ctx = context_lens;
  p.cu = cu_groups;
  p.prefix = prefix_lens;
  p.batch = batch;
  p.groups = num_groups;
  p.hkv = num_kv_heads;
  p.group = group;
  p.layer = layer;
  p.block_size = block_size;
  p.max_context = max_context;
  p.tq = kRows / group;
  p.max_tiles = lay.max_tiles;
  p.num_blocks = num_blocks;
  p.scale_log2 = scale * 1.4426950408889634f;
  char* const ws = static_cast<char*>(workspace);
  p.tile_info = reinterpret_cast<int2*>(ws + lay.tile_info);
  p.seq_info = reinterpret_cast<int2*>(ws + lay.seq_info);
  p.own_info = reinterpret_cast<int2*>(ws + lay.own_info);
  p.tile_part = reinterpret_cast<float*>(ws + lay.tile_part);
  p.own_part = reinterpret_cast<float*>(ws + lay.own_part);
  p.err = error_flag;
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (head_dim == 64) return dtype == PSB_BF16 ? launch<__nv_bfloat16, 64>(p, num_layers, s) : launch<__half, 64>(p, num_layers, s);
  return dtype == PSB_BF16 ? launch<__nv_bfloat16, 128>(p, num_layers, s) : launch<__half, 128>(p, num_layers, s);
}
