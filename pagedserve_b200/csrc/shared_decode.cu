// Decode attention for a batch whose sequences share long prefixes.
//
// Sequences cu[g] .. cu[g + 1] - 1 are group g and agree in their first
// prefix[g] tokens.  Softmax over a sequence's tokens splits into the part over
// the shared ones and the part over its own:
//   m = max(m1, m2),  l = l1 2^(m1 - m) + l2 2^(m2 - m),
//   o = (o1 2^(m1 - m) + o2 2^(m2 - m)) / l,
// so the shared part is computed for all of a group's query rows at once, where
// it is a matrix product (tcgen05), and each sequence's own part by itself, where
// it is a stream from HBM (mma.sync, as the plain decode).  shared_main_kernel does both
// in one grid of one CTA per SM, so that the stream goes on under the products (and a
// short call pays one launch and one plan for both); each leaves fp32 partials, which
// shared_join_kernel joins.
//
//  Prefixes: a tile is 128 rows: TQ = 128 / heads consecutive sequences of a group
//    times the q heads of one kv head (one TMA box of [TQ, heads, 64]).  Two
//    consecutive tiles make a pair and share each step's 64 keys (a tile by itself reads
//    a step's K and V, 32 KB for D 128, in the time of its products: beyond what L2
//    gives all SMs); of a pair with one tile, the two streams below take the steps in
//    turn.  The steps of all pairs, in (kv head, group, pair, step) order, are dealt
//    evenly, by what they cost, over the CTAs; every run of steps leaves partials.
//  Own parts: the 16-token slices of what is each sequence's own, in (kv heads,
//    sequence, slice) order, are dealt evenly over four warps of every CTA; every run
//    of slices leaves a partial.
//
// A CTA's 16 warps: two streams of four are the softmax (thread r is row r of a tile and
// lane r of TMEM); two issue the products of a stream each (one warp for both spent 1400
// cycles a stream and step on waits and operands, the softmax takes 1050), one the
// copies of K, one those of V; four have the own parts.  A stream has two S buffers in
// TMEM: S = Q K^T of its next step but one is issued behind O += P V of this one, whose
// P, two keys a column, was written over S.
//
// Measured (a call among others, of which 5 us are the two launches and 3 to 4 the plan): 8
// sequences on 1 K shared tokens 12 us, 64 on 4 K 20, 32 groups of 8 on 1.5 K 27; 256 on 2 K
// with 1 K each of their own 40, its 130 MB in 30 at 4.3 TB/s (the plain decode of the
// same contexts: 720 MB); 96 on 30 K, D 128, 86, its 47 GFLOP in 66: a pair's step takes 2050
// cycles where its exponentials are 1024 and its products 1300 (64 keys a step: Q is
// read from shared memory again for each; two S of 128 keys and two O of 128 dims fill TMEM,
// so 128 keys a step would leave each stream one S to write and read in turn).  Tried
// and not faster: a third stage of V, boxes asked into L2 ahead, the products' bookkeeping
// moved behind P V's issue, own slices of 32 tokens.
//
// Which of a group's tables the prefix is read through: that of the sequence
// with the most tokens (the first of those), and the prefix ends with it.  A
// sequence that is shorter than the prefix is read on its own (an idle row of a
// captured batch has no tokens at all): keys that it does not see, masked in the
// tile, would still meet its probabilities of 0, and 0 times infinity is no number.
#include <algorithm>
#include <atomic>
#include <cfloat>
#include <climits>
#include <cmath>

#include "common.cuh"
#include "host_util.h"
#include "packed_f32.cuh"

namespace psb {
namespace {

constexpr int kMaxBatch = 2048;      // sequences, and groups (fewer where their plan does not fit shared memory beside the rings)
constexpr size_t kMaxSmem = 227 * 1024;
constexpr int kOwnWarps = 4, kFirstOwn = 12;  // warps 0-7: softmax, two streams; 8, 9: their products; 10, 11: copies of K, of V; 12-15: own parts
constexpr int kThreads = 512;
// Registers: 128 a thread at launch, and the shares they are dealt anew in.
constexpr int kSoftmaxRegs = 136, kOtherRegs = 112, kOwnRegs = 128;
static_assert(256 * kSoftmaxRegs + 128 * kOtherRegs + 128 * kOwnRegs <= kThreads * 128, "the shares fit the launch");
constexpr int kRows = 128;           // rows of a tile
constexpr int kBN = 64;              // keys per step
constexpr int kHalf = 64;            // dims of one 128-byte line
constexpr uint32_t kQHalf = kRows * 128;   // bytes of 64 dims of a Q tile
constexpr uint32_t kKvHalf = kBN * 128;    // of a K or V tile
// TMEM: of each stream two S buffers, then each stream's O
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kSCol = 0, kOCol = 4 * kBN;
constexpr float kRescaleLog2 = 8.f;  // O is rescaled when a row's maximum grows by more than 2^8
// What a step costs, of a pair of tiles and of a single one: D 128 1.40 and 0.97 us over 30 K
// keys (by tiles, CTAs of singles alone end 10 us after those of pairs; all of it 88.5 us, so
// 84.5); D 64 by tiles (256 on 2 K 46.0 us, as D 128 46.7).
// kMin: cost per CTA below which the grid shrinks, beyond a quarter of the SMs and below
// (kMinFew; at least two pairs' steps less one: see Cursor).  Fewer steps are more partials:
// 256 sequences on 2 K take 2 us more with the lower one everywhere, 8 on 1 K 2 us more
// with the higher one.
template <int D>
struct Cost {
  static constexpr int kPair = D == 64 ? 2 : 3, kTile = D == 64 ? 1 : 2;
  static constexpr int kMin = 4 * kPair, kMinFew = 4 * kTile;
  static_assert(kMinFew >= 2 * kPair - 1 && kMin >= kMinFew, "every CTA has a step");
};
constexpr int kOwnMinItems = 2;      // slices per warp below which fewer warps work
constexpr int kMaxCtas = 160;        // (B200 has 148 SMs)

template <int D>
struct TcGeom {
  static constexpr int kH = D / kHalf;
  static constexpr int kStages = D == 64 ? 4 : 2;
  static constexpr uint32_t kOffK = 2 * kH * kQHalf;  // behind a Q tile for each stream
  static constexpr uint32_t kOffV = kOffK + kStages * kH * kKvHalf;
  static constexpr uint32_t kBarBytes = 384;
  static constexpr uint32_t kOffBars = kOffV + kStages * kH * kKvHalf;
  static constexpr uint32_t kOffRing = (kOffBars + kBarBytes + 1023) / 1024 * 1024;
};

template <int D, int HP>
struct OwnGeom {
  static constexpr int kRing = D == 64 ? 3 : 2;  // slots per warp
  static constexpr int kBox = 16 * 128;          // 16 tokens of one kv head, 64 dims
  static constexpr int kTile = D / kHalf * kBox;
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
  int32_t max_tiles;   // of one kv head there is room for
  int64_t num_blocks;
  float scale_log2;    // scale log2(e), positive
  // workspace
  int2* tile_info;     // [hkv * max_tiles] a tile's first partial, how many, how far apart (<< 16)
  int2* seq_info;      // [batch] a sequence's tile in each kv head (-1: none) and its place there
  int2* own_info;      // [hkv * batch] a (kv heads, sequence) pair's first partial and how many
  float* tile_part;    // partials of the tiles: [D / 4][128] x 4 sums, then [128] (maximum, sum)
  float* own_part;     // partials of the (kv heads, sequence) pairs: [D / 4][16] x 4 sums, then [16] (maximum, sum)
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
// the plan: what every CTA knows of the batch
// ---------------------------------------------------------------------------
struct Plan {
  int32_t* ctx;     // [batch] tokens
  int32_t* start;   // [batch] first token of a sequence's own part
  int32_t* slices;  // [batch + 1] slices before a sequence, of one (kv heads)
  int32_t* cu;      // [groups + 1]
  int32_t* pre;     // [groups] shared tokens (0: the group's sequences are on their own)
  int32_t* lead;    // [groups] the sequence whose table holds them
  // before a group, of one kv head:
  int32_t* tiles;   // [groups + 1]
  int32_t* pairs;   // [groups + 1]
  int32_t* cost;    // [groups + 1]
  int groups, tq, n_pairs, n_cost, n_slices;
  __host__ __device__ static size_t ints(int batch, int groups) { return 3 * static_cast<size_t>(batch) + 1 + 6 * static_cast<size_t>(groups) + 4; }
  __device__ Plan(int32_t* at, int batch, int n, int q) : groups(n), tq(q) {
    ctx = at;
    start = ctx + batch;
    slices = start + batch;
    cu = slices + batch + 1;
    pre = cu + n + 1;
    lead = pre + n;
    tiles = lead + n;
    pairs = tiles + n + 1;
    cost = pairs + n + 1;
  }
  __device__ __forceinline__ int steps_of(int g) const { return (pre[g] + kBN - 1) / kBN; }
};

// A warp's exclusive scans of N values a lane, and the totals.
template <int N>
__device__ __forceinline__ void scan_warp(int (&v)[N], int (&total)[N]) {
  int incl[N];
#pragma unroll
  for (int i = 0; i < N; ++i) incl[i] = v[i];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    int x[N];
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = __shfl_up_sync(0xffffffffu, incl[i], o);
    if ((threadIdx.x & 31) >= o) {
#pragma unroll
      for (int i = 0; i < N; ++i) incl[i] += x[i];
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    total[i] = __shfl_sync(0xffffffffu, incl[i], 31);
    v[i] = incl[i] - v[i];
  }
}

template <int D>
__device__ void build_plan(const SharedParams& p, Plan& pl) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const bool report = blockIdx.x == 0;
  bool bad = false;
  for (int b = tid; b < p.batch; b += kThreads) {
    int n = __ldcg(p.ctx + b);
    if (n < 0 || n > p.max_context) {
      if (report) flag_error(p.err, PSB_DEVERR_CONTEXT);
      n = n < 0 ? 0 : p.max_context;
    }
    pl.ctx[b] = n;
    pl.start[b] = 0;
  }
  for (int g = kThreads - 1 - tid; g <= p.groups; g += kThreads) {  // (from the other end: in the same round of loads)
    const int a = __ldcg(p.cu + g), prev = g == 0 ? 0 : __ldcg(p.cu + g - 1);
    bad = bad || a < prev || prev < 0 || a > p.batch;
    pl.cu[g] = a;
    if (g < p.groups) pl.pre[g] = __ldcg(p.prefix + g);
  }
  bad = __syncthreads_or(bad) != 0;
  if (bad && report && tid == 0) flag_error(p.err, PSB_DEVERR_SEQLENS);
  for (int g = warp; g < p.groups; g += kThreads / 32) {
    // malformed groups: every sequence on its own
    const int b0 = bad ? 0 : pl.cu[g], b1 = bad ? 0 : pl.cu[g + 1], n = pl.pre[g];
    int best = -1, at = 0;
    for (int b = b0 + lane; b < b1; b += 32) {
      if (pl.ctx[b] > best) {
        best = pl.ctx[b];
        at = b;
      }
    }
    const int most = __reduce_max_sync(0xffffffffu, best);
    at = __reduce_min_sync(0xffffffffu, best == most ? at : INT_MAX);
    // one sequence shares with nobody: all of it is its own
    const int pre = b1 - b0 < 2 ? 0 : max(0, min(n, most));
    if (pre > 0)
      for (int b = b0 + lane; b < b1; b += 32)
        if (pl.ctx[b] >= pre) pl.start[b] = pre;
    __syncwarp();
    if (lane == 0) {
      if (n < 0 && report) flag_error(p.err, PSB_DEVERR_CONTEXT);
      pl.pre[g] = pre;
      pl.lead[g] = at;
    }
  }
  __syncthreads();
  if (warp == 0) {  // the groups' tiles
    const int per = (p.groups + 31) / 32, g0 = min(lane * per, p.groups), g1 = min(g0 + per, p.groups);
    auto tiles_of = [&](int g) { return pl.pre[g] > 0 ? (pl.cu[g + 1] - pl.cu[g] + p.tq - 1) / p.tq : 0; };
    auto cost_of = [](int n) { return (n >> 1) * Cost<D>::kPair + (n & 1) * Cost<D>::kTile; };  // a step of n tiles
    int v[3] = {0, 0, 0}, all[3];  // tiles, pairs, cost
    for (int g = g0; g < g1; ++g) {
      const int n = tiles_of(g);
      v[0] += n;
      v[1] += (n + 1) >> 1;
      v[2] += cost_of(n) * pl.steps_of(g);
    }
    scan_warp(v, all);
    for (int g = g0; g < g1; ++g) {
      pl.tiles[g] = v[0];
      pl.pairs[g] = v[1];
      pl.cost[g] = v[2];
      const int n = tiles_of(g);
      v[0] += n;
      v[1] += (n + 1) >> 1;
      v[2] += cost_of(n) * pl.steps_of(g);
    }
    if (lane == 0) {
      pl.tiles[p.groups] = all[0];
      pl.pairs[p.groups] = all[1];
      pl.cost[p.groups] = all[2];
    }
  } else if (warp == 1) {  // the sequences' slices
    const int per = (p.batch + 31) / 32, b0 = min(lane * per, p.batch), b1 = min(b0 + per, p.batch);
    auto slices_of = [&](int b) { return pl.ctx[b] > pl.start[b] ? (pl.ctx[b] + 15) / 16 - pl.start[b] / 16 : 0; };
    int n[1] = {0}, all[1];
    for (int b = b0; b < b1; ++b) n[0] += slices_of(b);
    scan_warp(n, all);
    for (int b = b0; b < b1; ++b) {
      pl.slices[b] = n[0];
      n[0] += slices_of(b);
    }
    if (lane == 0) pl.slices[p.batch] = all[0];
  }
  __syncthreads();
  pl.n_pairs = pl.pairs[p.groups];
  pl.n_cost = pl.cost[p.groups];
  pl.n_slices = pl.slices[p.batch];
}

// ``n`` units dealt evenly over ``parts``: part i has [start(i), start(i + 1)).
struct Deal {
  uint32_t n, parts, share, extra;
  __device__ Deal(uint32_t units, uint32_t over) : n(units), parts(over), share(over ? units / over : 0), extra(over ? units - share * over : 0) {}
  __device__ __forceinline__ uint32_t start(uint32_t i) const { return share * i + min(i, extra); }
  __device__ __forceinline__ uint32_t part_of(uint32_t unit) const {
    const uint32_t head = extra * (share + 1);
    return unit < head ? unit / (share + 1) : extra + (unit - head) / share;
  }
};

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
__device__ __forceinline__ void box_load(bool on, uint32_t dst, const CUtensorMap* map, int32_t x, int32_t y, int32_t z, uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %6, 0;\n\t"
      "@q cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n\t}" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar), "r"(static_cast<uint32_t>(on))
      : "memory");
}
// the same, of what is read once
__device__ __forceinline__ void box_load_once(bool on, uint32_t dst, const CUtensorMap* map, int32_t x, int32_t y, int32_t z, uint32_t bar, uint64_t policy) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %6, 0;\n\t"
      "@q cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%2, %3, %4}], [%5], %7;\n\t}" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar), "r"(static_cast<uint32_t>(on)), "l"(policy)
      : "memory");
}
__device__ __forceinline__ void expect_bytes(bool on, uint32_t bar, uint32_t bytes) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %2, 0;\n\t"
      "@q mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n\t}" ::"r"(bar), "r"(bytes), "r"(static_cast<uint32_t>(on))
      : "memory");
}
__device__ __forceinline__ uint64_t desc_of(uint32_t lo, uint32_t hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "r"(hi));
  return d;
}
// A value that every lane has alike, where the compiler cannot tell.
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __reduce_or_sync(0xffffffffu, x); }
__device__ __forceinline__ bool elect_one() {
  uint32_t on;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(on));
  return on != 0;
}
// mbar_wait by a whole warp: its lanes give up together or not at all.
__device__ __forceinline__ bool warp_wait_at(uint32_t bar, uint32_t parity) {
  uint64_t t0 = 0;
#pragma unroll 1
  while (!__all_sync(0xffffffffu, mbar_try_wait_sleep(bar, parity, 100000u))) {
    const uint64_t t = globaltimer_ns();
    if (t0 == 0) t0 = t;
    if (__all_sync(0xffffffffu, t - t0 > kWaitLimitNs)) return false;
  }
  return true;
}
template <int S>
struct Int {
  static constexpr int value = S;
};
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity)); }

// A run of steps of one pair of tiles.
struct Run {
  int kvh, pair, tile, grp;  // pair of its kv head and its first tile, group
  int b0, n_seq;             // first sequence, sequences from it to the group's end
  int j0, n;                 // its steps
  int in_grp;                // pair of its group
  bool two;                  // there is a second tile
};

// Walks a CTA's steps pair by pair.  A step belongs to the CTA that its last unit of cost
// was dealt to: a CTA that was dealt a step's cost or more in a pair has steps there.
template <int D>
struct Cursor {
  static constexpr int kPairCost = Cost<D>::kPair, kTileCost = Cost<D>::kTile;
  int kvh, grp, in_grp, j0, left;  // left: cost
  // To the step that the unit at ``pos`` of the whole list is in, or begins; returns its first unit.
  __device__ uint32_t seek(const Plan& pl, uint32_t pos) {
    kvh = static_cast<int>(pos / pl.n_cost);
    const int r = static_cast<int>(pos - static_cast<uint32_t>(kvh) * pl.n_cost);
    grp = last_le(pl.cost, pl.groups, r);  // (of groups without steps the last: it has some)
    const int steps = pl.steps_of(grp), off = r - pl.cost[grp];
    in_grp = off / (kPairCost * steps);
    const int in_pair = off - in_grp * kPairCost * steps, of_step = two(pl) ? kPairCost : kTileCost;
    j0 = in_pair / of_step;
    return pos - (in_pair - j0 * of_step);
  }
  __device__ bool two(const Plan& pl) const { return 2 * in_grp + 1 < pl.tiles[grp + 1] - pl.tiles[grp]; }
  __device__ Run take(const Plan& pl) {  // the next run (left > 0)
    Run r;
    r.kvh = kvh;
    r.pair = pl.pairs[grp] + in_grp;
    r.tile = pl.tiles[grp] + 2 * in_grp;
    r.grp = grp;
    r.in_grp = in_grp;
    r.b0 = pl.cu[grp] + in_grp * 2 * pl.tq;
    r.n_seq = pl.cu[grp + 1] - r.b0;
    r.two = two(pl);
    r.j0 = j0;
    r.n = min(pl.steps_of(grp) - j0, r.two ? left / kPairCost : left / kTileCost);
    left -= r.n * (r.two ? kPairCost : kTileCost);
    j0 = 0;
    if (left > 0) {
      ++in_grp;
      if (pl.pairs[grp] + in_grp == pl.n_pairs) {
        grp = 0;
        in_grp = 0;
        ++kvh;
      }
      while (pl.pairs[grp] + in_grp >= pl.pairs[grp + 1]) {  // groups without pairs are passed over
        ++grp;
        in_grp = 0;
      }
    }
    return r;
  }
};

// One stream's steps of a CTA, in order: of pairs of tiles every step, of single tiles
// those whose number, counted in half-steps (a step of one stream) of the CTA, is its own.
template <int D>
struct Steps {
  Cursor<D> c;
  Run r;
  int x, half, g0;  // step of the run; half-steps and steps of the CTA before the run
  bool begins;      // the first of the run
  __device__ explicit Steps(const Cursor<D>& first) : c(first), x(0), half(0), g0(0), begins(true) {
    r.n = 0;
    r.two = false;
  }
  // Takes the next run up when this one's steps are through; false: there is none.
  __device__ __forceinline__ bool more(const Plan& pl, int s) {
    while (x >= r.n) {
      if (c.left == 0) return false;
      half += r.two ? 2 * r.n : r.n;
      g0 += r.n;
      r = c.take(pl);
      x = r.two ? 0 : (half + s) & 1;
      begins = true;
    }
    return true;
  }
  __device__ __forceinline__ void next() {
    x += r.two ? 1 : 2;
    begins = false;
  }
};

// An 8 by 8 tile of 16-bit values, row i / 4 and columns 2 (i % 4), + 1 in lane i, transposed.
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
template <int N>
__device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// ---------------------------------------------------------------------------
// each sequence's own part
// ---------------------------------------------------------------------------
// A warp streams its slices (16 tokens of HP kv heads) through a ring of its own, by
// boxes of 16 tokens, 64 dims and the HP heads (with 16 bytes a lane and instruction,
// half of a warp's time and more went into issuing the copies).  Its products are
//   S^T = K Q^T   of 16 tokens by 8 q heads,   O^T += V^T P^T   of 16 dims by 8 q heads,
// (m16n8k16; P^T by an 8 by 8 transposition in registers): q heads as columns, because
// their tile is the narrower side, and a kv head has as few as 4 of them.  NT: such
// tiles of a kv head (1 or 2).
template <typename T, int D, int HP, int NT>
__device__ __forceinline__ void own_parts(const SharedParams& p, const Plan& plan, const CUtensorMap* tm_k, const CUtensorMap* tm_v, uint8_t* ring_all, uint64_t* bars_all) {
  using Geo = OwnGeom<D, HP>;
  constexpr int kRing = Geo::kRing, kH = D / kHalf, kSteps = D / 16;  // steps of 16 dims
  const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) - kFirstOwn;
  const int gq = lane >> 2, t = lane & 3;
  const int G = p.group, B = p.batch, hgs = p.hkv / HP;
  const uint32_t items = static_cast<uint32_t>(plan.n_slices) * hgs;  // below 2^31
  const Deal deal(items, min(gridDim.x * kOwnWarps, (items + kOwnMinItems - 1) / kOwnMinItems));
  // warps in order of their place in a CTA: few are spread over the SMs
  const uint32_t gw = warp * gridDim.x + blockIdx.x;
  const uint32_t my_a = gw < deal.parts ? deal.start(gw) : 0, my_e = gw < deal.parts ? deal.start(gw + 1) : 0;
  const uint32_t ring_u = smem_u32(ring_all) + warp * kRing * Geo::kSlot;
  const uint32_t bars = smem_u32(bars_all) + warp * kRing * 8;  // a slot's copies landed
  const bool on = elect_one();
  if (on) {
    prefetch_tmap(tm_k);
    prefetch_tmap(tm_v);
  }
  const uint64_t policy = l2_policy_evict_first();
  const int64_t layer0 = static_cast<int64_t>(p.layer) * p.num_blocks;

  // A chunk: up to 32 consecutive slices of the warp's range, one a lane: its
  // place in the pool (-1: its block is outside), the valid tokens [lo, hi), and
  // whether a pair or the range begins or ends with it.
  struct Chunk {
    uint32_t beg;
    int n;
    int32_t blk, row, meta, pair;
  };
  auto build_chunk = [&](uint32_t beg) -> Chunk {
    Chunk c;
    c.beg = beg;
    c.n = static_cast<int>(min(32u, my_e - beg));
    c.blk = -1;
    c.row = c.meta = c.pair = 0;
    if (lane < c.n) {
      const uint32_t i = beg + lane, hg = i / plan.n_slices;
      const int r = static_cast<int>(i - hg * plan.n_slices);
      const int b = last_le(plan.slices, B, r);  // (of sequences without slices the last: it has some)
      const int j = r - plan.slices[b], pos = (plan.start[b] / 16 + j) * 16;
      const int lo = max(0, plan.start[b] - pos), hi = min(16, plan.ctx[b] - pos);
      const int bi = pos / p.block_size;
      c.row = pos - bi * p.block_size;
      c.blk = __ldcg(p.tables + static_cast<int64_t>(b) * p.table_stride + bi);
      if (c.blk < 0 || c.blk >= p.num_blocks) {
        flag_error(p.err, PSB_DEVERR_BLOCK_RANGE);
        c.blk = -1;
      }
      c.meta = lo | hi << 5 | (j == 0 || i == my_a ? 1 << 10 : 0) | (r + 1 == plan.slices[b + 1] || i == my_e - 1 ? 1 << 11 : 0);
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
    const uint32_t bar = bars + slot * 8;
    expect_bytes(on, bar, blk >= 0 ? Geo::kSlot : 0);
    if (blk >= 0) {
      const int32_t tile = static_cast<int32_t>((layer0 + blk) * p.hkv + pair / B * HP);
#pragma unroll
      for (int h = 0; h < kH; ++h) {
        box_load_once(on, dst + h * Geo::kBox, tm_k, h * kHalf, r0, tile, bar, policy);
        box_load_once(on, dst + Geo::kKV + h * Geo::kBox, tm_v, h * kHalf, r0, tile, bar, policy);
      }
    }
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
  // (while the first copies are on their way) what the join needs: the partials of
  // the pairs, the tiles of the sequences
  const int gt = blockIdx.x * (kOwnWarps * 32) + warp * 32 + lane, gts = gridDim.x * (kOwnWarps * 32);
  for (int s = gt; s < B * hgs; s += gts) {
    const int hg = s / B, b = s - hg * B;
    int2 at = make_int2(0, 0);
    if (plan.slices[b + 1] > plan.slices[b]) {
      const uint32_t before = static_cast<uint32_t>(hg) * plan.n_slices;
      const uint32_t w0 = deal.part_of(before + plan.slices[b]), w1 = deal.part_of(before + plan.slices[b + 1] - 1);
      at = make_int2(static_cast<int>(w0) + s, static_cast<int>(w1 - w0) + 1);
    }
    p.own_info[s] = at;
  }
  for (int b = gt; b < B; b += gts) {
    int2 at = make_int2(-1, 0);
    if (plan.start[b] > 0) {
      const int g = last_le(plan.cu, p.groups, b);  // (of empty groups the last: it holds b)
      const int m = b - plan.cu[g];
      at = make_int2(plan.tiles[g] + m / p.tq, m % p.tq);
    }
    p.seq_info[b] = at;
  }

  uint32_t q[HP][NT][kSteps][2];  // columns: q heads gq (+ 8)
  float o[HP][NT][kSteps][4];     // dims gq, gq + 8 of 16, of q heads 2 t, 2 t + 1 (+ 8)
  float m[HP][NT][2], l[HP][NT][2];  // of these heads: the exponents' reference (a maximum, scaled), this lane's share of the sum
  int32_t pair = 0;
  while (consumed != issued) {
    const uint32_t slot = consumed % kRing;
    const int32_t mt = __shfl_sync(0xffffffffu, meta, slot);
    const int lo = mt & 31, hi = (mt >> 5) & 31;
    const uint32_t base = ring_u + slot * Geo::kSlot;
    if ((mt >> 10) & 1) {  // a pair (or the range) begins: its q rows
      pair = __shfl_sync(0xffffffffu, meta_pair, slot);
      const int hg = pair / B, b = pair - hg * B;
      const T* const qb = reinterpret_cast<const T*>(p.q) + b * p.qsb + 2 * t;
#pragma unroll
      for (int hs = 0; hs < HP; ++hs) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const int h = nt * 8 + gq;
          const T* const row = qb + static_cast<int64_t>((hg * HP + hs) * G + h) * p.qsh;
#pragma unroll
          for (int ks = 0; ks < kSteps; ++ks) {
            q[hs][nt][ks][0] = h < G ? __ldcg(reinterpret_cast<const uint32_t*>(row + 16 * ks)) : 0u;
            q[hs][nt][ks][1] = h < G ? __ldcg(reinterpret_cast<const uint32_t*>(row + 16 * ks + 8)) : 0u;
            o[hs][nt][ks][0] = o[hs][nt][ks][1] = o[hs][nt][ks][2] = o[hs][nt][ks][3] = 0.f;
          }
          m[hs][nt][0] = m[hs][nt][1] = -FLT_MAX;  // (not -infinity: beside it a score of -infinity would be no number)
          l[hs][nt][0] = l[hs][nt][1] = 0.f;
        }
      }
    }
    if (!warp_wait_at(bars + slot * 8, (consumed / kRing) & 1)) {
      if (on) flag_error(p.err, PSB_DEVERR_TIMEOUT);
      for (uint32_t i = consumed + 1; i != issued; ++i) (void)warp_wait_at(bars + i % kRing * 8, (i / kRing) & 1);  // the other copies in flight
      return;
    }
    if ((mt >> 12) & 1) {
      float s[HP][NT][4];  // tokens gq, gq + 8 of q heads 2 t, 2 t + 1 (+ 8)
#pragma unroll
      for (int hs = 0; hs < HP; ++hs) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) s[hs][nt][0] = s[hs][nt][1] = s[hs][nt][2] = s[hs][nt][3] = 0.f;
      }
#pragma unroll
      for (int ks = 0; ks < kSteps; ++ks) {
#pragma unroll
        for (int hs = 0; hs < HP; ++hs) {
          uint32_t a0, a1, a2, a3;
          ldsm_x4(base + ((ks >> 2) * HP + hs) * Geo::kBox + (((lane >> 3) & 1) * 8 + (lane & 7)) * 128 +
                      ((((ks & 3) * 2 + (lane >> 4)) ^ (lane & 7)) << 4), a0, a1, a2, a3);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_16816<T>(s[hs][nt], a0, a1, a2, a3, q[hs][nt][ks][0], q[hs][nt][ks][1]);
        }
      }
      uint32_t keep[2] = {0xffffffffu, 0xffffffffu};  // of V's rows 2 t, + 1 and 8 + 2 t, + 1: what is masked may hold anything (even NaN)
      if (hi < 16 || lo > 0) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int k = 8 * e + 2 * t;
          keep[e] = (k >= lo && k < hi ? 0x0000ffffu : 0u) | (k + 1 >= lo && k + 1 < hi ? 0xffff0000u : 0u);
          const int row = 8 * e + gq;
          if (row < lo || row >= hi) {
#pragma unroll
            for (int hs = 0; hs < HP; ++hs) {
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) s[hs][nt][2 * e] = s[hs][nt][2 * e + 1] = -INFINITY;
            }
          }
        }
      }
      // A new reference, and O and the sums brought to it, where a score is above the old
      // one by more than 2^8 (nearly always the first slices alone)
      bool grow = false;
#pragma unroll
      for (int hs = 0; hs < HP; ++hs) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int e = 0; e < 2; ++e) grow = grow || fmaxf(s[hs][nt][e], s[hs][nt][2 + e]) * p.scale_log2 > m[hs][nt][e] + kRescaleLog2;
        }
      }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int hs = 0; hs < HP; ++hs) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float mx = fmaxf(s[hs][nt][e], s[hs][nt][2 + e]);
#pragma unroll
              for (int x = 4; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
              const float mn = fmaxf(m[hs][nt][e], mx * p.scale_log2), alpha = ex2_approx(m[hs][nt][e] - mn);
              m[hs][nt][e] = mn;
              l[hs][nt][e] *= alpha;
#pragma unroll
              for (int ks = 0; ks < kSteps; ++ks) {
                o[hs][nt][ks][e] *= alpha;
                o[hs][nt][ks][2 + e] *= alpha;
              }
            }
          }
        }
      }
      uint32_t pr[HP][NT][2];  // P^T: tokens 2 t, + 1 (+ 8) of q head gq
#pragma unroll
      for (int hs = 0; hs < HP; ++hs) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float ex[4];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            ex[e] = ex2_approx(fmaf(s[hs][nt][e], p.scale_log2, -m[hs][nt][e]));
            ex[2 + e] = ex2_approx(fmaf(s[hs][nt][2 + e], p.scale_log2, -m[hs][nt][e]));
            l[hs][nt][e] += ex[e] + ex[2 + e];
          }
          pr[hs][nt][0] = transposed(pack2<T>(ex[0], ex[1]));
          pr[hs][nt][1] = transposed(pack2<T>(ex[2], ex[3]));
        }
      }
#pragma unroll
      for (int ks = 0; ks < kSteps; ++ks) {
#pragma unroll
        for (int hs = 0; hs < HP; ++hs) {
          uint32_t a0, a1, a2, a3;
          ldsm_x4_t(base + Geo::kKV + ((ks >> 2) * HP + hs) * Geo::kBox + ((lane >> 4) * 8 + (lane & 7)) * 128 +
                        ((((ks & 3) * 2 + ((lane >> 3) & 1)) ^ (lane & 7)) << 4), a0, a1, a2, a3);
          a0 &= keep[0];
          a1 &= keep[0];
          a2 &= keep[1];
          a3 &= keep[1];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_16816<T>(o[hs][nt][ks], a0, a1, a2, a3, pr[hs][nt][0], pr[hs][nt][1]);
        }
      }
    }
    __syncwarp();
    ++consumed;
    if (c_ok) issue_one();  // refill the slot just read
    if ((mt >> 11) & 1) {   // the pair's or the range's end: its partial
      float* const part = p.own_part + static_cast<int64_t>(gw + pair) * own_floats(D);
      float2* const ml = reinterpret_cast<float2*>(part + 16 * D);
#pragma unroll
      for (int hs = 0; hs < HP; ++hs) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float sum = l[hs][nt][e];
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
            const int h = nt * 8 + 2 * t + e, row = hs * 8 + h;
            if (h >= G) continue;
#pragma unroll
            for (int ks = 0; ks < kSteps; ++ks) {
#pragma unroll
              for (int u = 0; u < 2; ++u) part[(4 * ks + 2 * u + (gq >> 2)) * 64 + 4 * row + (gq & 3)] = o[hs][nt][ks][2 * u + e];
            }
            if (gq == 0) ml[row] = make_float2(m[hs][nt][e], sum);
          }
        }
      }
    }
  }
}

template <typename T, int D, int HP, int NT>
__global__ void __launch_bounds__(kThreads, 1)
    shared_main_kernel(const SharedParams p, const __grid_constant__ CUtensorMap tm_q,
                       const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                       const __grid_constant__ CUtensorMap tm_ko, const __grid_constant__ CUtensorMap tm_vo) {
  using Geo = TcGeom<D>;
  constexpr int kH = Geo::kH, kStages = Geo::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const smem = smem_raw + ((0u - smem_u32(smem_raw)) & 1023u);
  uint64_t* const bar_q = reinterpret_cast<uint64_t*>(smem + Geo::kOffBars);  // [2] a stream's Q landed
  uint64_t* const bar_k = bar_q + 2;               // [kStages] K landed
  uint64_t* const bar_kfree = bar_k + kStages;     // [kStages] Q K^T of the step done (two arrivals: both streams', or its one's twice)
  uint64_t* const bar_v = bar_kfree + kStages;     // [kStages] V landed
  uint64_t* const bar_vfree = bar_v + kStages;     // [kStages] P V of the step done (the same)
  // of each stream, two in turn (a barrier's next phase needs this one's products):
  uint64_t* const bar_s = bar_vfree + kStages;     // [2][2] S written
  uint64_t* const bar_p = bar_s + 4;               // [2][2] P written over it
  uint64_t* const bar_pv = bar_p + 4;              // [2][2] P V done
  uint64_t* const bar_drain = bar_pv + 4;          // [2] every product of the stream is done
  uint64_t* const bar_own = bar_drain + 2;         // [4][ring] of the own parts' warps: a slot's copies landed
  constexpr int kOwnBars = kOwnWarps * OwnGeom<D, HP>::kRing;
  uint32_t* const s_tmem = reinterpret_cast<uint32_t*>(bar_own + kOwnBars);
  static_assert((16 + 4 * kStages + kOwnBars) * 8 + 4 <= Geo::kBarBytes, "barriers fit their area");
  Plan plan(reinterpret_cast<int32_t*>(smem + Geo::kOffRing + OwnGeom<D, HP>::kBytes), p.batch, p.groups, p.tq);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int TQ = p.tq, group = p.group;
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(bar_k + i, 1);
      mbar_init(bar_kfree + i, 2);
      mbar_init(bar_v + i, 1);
      mbar_init(bar_vfree + i, 2);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar_q + i, 1);
      mbar_init(bar_drain + i, 1);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(bar_s + i, 1);
      mbar_init(bar_p + i, kRows);
      mbar_init(bar_pv + i, 1);
    }
    for (int i = 0; i < kOwnBars; ++i) mbar_init(bar_own + i, 1);
    fence_barrier_init();
  }
  if (warp == 0) {
    tmem_alloc(s_tmem, kTmemCols);
    tmem_relinquish();
  }
  pdl_wait();  // lengths, groups, tables, q and the pools may come from the stream predecessor
  pdl_launch_dependents();
  tc_fence_before();
  build_plan<D>(p, plan);  // (its barriers are also those behind the set-up above)
  tc_fence_after();
  const uint32_t tmem = *s_tmem;
  using C = Cost<D>;
  const uint32_t total = static_cast<uint32_t>(plan.n_cost) * p.hkv;  // below 2^31
  const Deal deal(total, min(gridDim.x, max((total + C::kMin - 1) / C::kMin, min((total + C::kMinFew - 1) / C::kMinFew, gridDim.x / 4))));
  const uint32_t cta = blockIdx.x;
  Cursor<D> first;
  first.left = 0;
  if (cta < deal.parts) {  // odd lanes look where the CTA's steps end, even ones where they begin
    const uint32_t at = deal.start(cta + (lane & 1));
    Cursor<D> c;
    const uint32_t unit = at == total ? total : c.seek(plan, at);
    first.kvh = __shfl_sync(0xffffffffu, c.kvh, 0);
    first.grp = __shfl_sync(0xffffffffu, c.grp, 0);
    first.in_grp = __shfl_sync(0xffffffffu, c.in_grp, 0);
    first.j0 = __shfl_sync(0xffffffffu, c.j0, 0);
    first.left = static_cast<int>(__shfl_sync(0xffffffffu, unit, 1) - __shfl_sync(0xffffffffu, unit, 0));
  }
  bool fail = false;

  // ---- products of stream s ----
  auto products = [&](auto stream) {
    constexpr int s = decltype(stream)::value;
    constexpr int kFmt = Elem<T>::code == PSB_BF16 ? 1 : 0;
    constexpr uint32_t idesc_s = umma_idesc_f16(kFmt, kRows, kBN, 0, 0), idesc_o = umma_idesc_f16(kFmt, kRows, D, 0, 1);
    const bool on = elect_one();
    const uint32_t s_base = smem_u32(smem);
    // descriptors: their low words (addresses) move, their high ones do not
    const uint64_t dq = umma_desc_sw128(s_base + s * kH * kQHalf, 1024, 16);
    const uint64_t dk = umma_desc_sw128(s_base + Geo::kOffK, 1024, 16);
    const uint64_t dv = umma_desc_sw128(s_base + Geo::kOffV, 1024, kKvHalf);  // (of D 128 the second half's dims lie a half tile on)
    const uint32_t qlo = static_cast<uint32_t>(dq), klo = static_cast<uint32_t>(dk), vlo = static_cast<uint32_t>(dv);
    const uint32_t khi = static_cast<uint32_t>(dk >> 32), vhi = static_cast<uint32_t>(dv >> 32);  // (Q's is K's)
    const uint32_t a_q = smem_u32(bar_q + s), a_k = smem_u32(bar_k), a_kfree = smem_u32(bar_kfree), a_v = smem_u32(bar_v),
                   a_vfree = smem_u32(bar_vfree), a_s = smem_u32(bar_s + 2 * s), a_p = smem_u32(bar_p + 2 * s), a_pv = smem_u32(bar_pv + 2 * s);
    if (on) prefetch_tmap(&tm_q);
    const uint32_t box = static_cast<uint32_t>(TQ * group) * 128 * kH;
    const uint32_t ocol = tmem + kOCol + s * D, scol = tmem + kSCol + 2 * s * kBN;
    // Until a stage's copies of ``round`` have landed.  Its use before may have been
    // the other stream's, and a wait for a barrier's phase passes while the phase before
    // is still open; so first until that use is over.  (That wait is of one phase at a
    // time: this stream's step before, two back at most, had landed, and was asked for
    // when the use before the last was over.  The next phase needs this step.)
    auto landed = [&](uint32_t full, uint32_t free, uint32_t st, uint32_t round) {
      return (round == 0 || warp_wait_at(free + 8 * st, (round - 1) & 1)) && warp_wait_at(full + 8 * st, round & 1);
    };
    Steps<D> hs(first);
    // What P V has to know of a step, from its S two steps before: its number in the
    // CTA's list, how many of its keys there are (bits 24 to 29; 0: all), whether the run
    // begins (bit 30) and is a pair's (bit 31); of none: kNone.
    constexpr uint32_t kNone = 0xffffffffu, kStep = (1u << 24) - 1, kBegins = 1u << 30, kTwo = 1u << 31;
    uint32_t now = kNone, then = kNone, q_ph = 0;
    bool q_flight = false;
#pragma unroll 1
    for (int k = -2;; ++k) {
      const uint32_t b = k & 1, ph = (k >> 1) & 1;
      if (k >= 0) {  // P V of step k
        if (now == kNone) break;
        const uint32_t g = now & kStep, st = g % kStages, round = g / kStages;
        if (!landed(a_v, a_vfree, st, round) || !warp_wait_at(a_p + 8 * b, ph)) {
          fail = true;
          break;
        }
        const uint32_t have = (now >> 24) & 63;
        if (have != 0) {
          // V rows behind the prefix (another token's, or never loaded) must not reach
          // P V, where 0 * NaN would be NaN
          const uint32_t v0 = s_base + Geo::kOffV + st * (kH * kKvHalf);
          for (uint32_t c = have * 8 + lane; c < kBN * 8; c += 32) {
#pragma unroll
            for (int h = 0; h < kH; ++h) st_shared_zero16(v0 + h * kKvHalf + c * 16);
          }
          fence_proxy_async_smem();  // visible to the tensor core
          __syncwarp();
        }
        tc_fence_after();
        const uint32_t pcol = scol + b * kBN, vd = vlo + st * (kH * kKvHalf >> 4);
#pragma unroll
        for (int kk = 0; kk < kBN / 16; ++kk) mma_ts(on, ocol, pcol + 8 * kk, desc_of(vd + 128 * kk, vhi), idesc_o, (now & kBegins) == 0 || kk > 0);
        mma_commit(on, a_pv + 8 * b);
        mma_commit(on, a_vfree + 8 * st);
        if ((now & kTwo) == 0) mma_commit(on, a_vfree + 8 * st);
      }
      now = then;
      then = kNone;
      if (hs.more(plan, s)) {  // S of step k + 2, whose buffer held P of step k
        if (hs.begins) {  // the run's Q, once the last S of the run before (step k + 1) is done
          if (k >= -1 && !warp_wait_at(a_s + 8 * (b ^ 1), ((k + 1) >> 1) & 1)) {
            fail = true;
            break;
          }
          expect_bytes(on, a_q, box);
#pragma unroll
          for (int h = 0; h < kH; ++h)
            box_load(on, s_base + (s * kH + h) * kQHalf, &tm_q, h * kHalf, hs.r.kvh * group, hs.r.b0 + (hs.r.two ? s * TQ : 0), a_q);
          q_flight = true;
          if (!warp_wait_at(a_q, q_ph)) {
            fail = true;
            break;
          }
          q_ph ^= 1;
          q_flight = false;
        }
        const uint32_t g = uniform(hs.g0 + hs.x), st = g % kStages, round = g / kStages;
        const int have = plan.pre[hs.r.grp] - (hs.r.j0 + hs.x) * kBN;
        then = uniform(g | (have < kBN ? have << 24 : 0) | (hs.begins ? kBegins : 0) | (hs.r.two ? kTwo : 0));
        if (!landed(a_k, a_kfree, st, round) || (k >= 0 && !warp_wait_at(a_pv + 8 * b, ph))) {
          fail = true;
          break;
        }
        tc_fence_after();
        const uint32_t kd = klo + st * (kH * kKvHalf >> 4);
#pragma unroll
        for (int h = 0; h < kH; ++h) {
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            mma_ss(on, scol + b * kBN, desc_of(qlo + h * (kQHalf >> 4) + 2 * kk, khi), desc_of(kd + h * (kKvHalf >> 4) + 2 * kk, khi), idesc_s, h > 0 || kk > 0);
        }
        mma_commit(on, a_s + 8 * b);
        mma_commit(on, a_kfree + 8 * st);
        if ((then & kTwo) == 0) mma_commit(on, a_kfree + 8 * st);
        hs.next();
      }
    }
    if (fail) {
      if (on) flag_error(p.err, PSB_DEVERR_TIMEOUT);
      if (q_flight) (void)warp_wait_at(a_q, q_ph);
    }
    // the copy, the products and their commits in flight land before shared memory and TMEM are released
    mma_commit(on, smem_u32(bar_drain + s));
    (void)warp_wait_at(smem_u32(bar_drain + s), 0);
  };
  auto copies = [&]() {
    // ---- copies: of K, or of V ----
    const CUtensorMap* const tm = warp == 10 ? &tm_k : &tm_v;
    const uint32_t a_full = smem_u32(warp == 10 ? bar_k : bar_v), a_free = smem_u32(warp == 10 ? bar_kfree : bar_vfree);
    const uint32_t ring = smem_u32(smem) + (warp == 10 ? Geo::kOffK : Geo::kOffV);
    const bool on = elect_one();
    if (on) prefetch_tmap(tm);
    const int bs = p.block_size, box_rows = min(bs, kBN), boxes = kBN / box_rows;
    const int64_t layer0 = static_cast<int64_t>(p.layer) * p.num_blocks;
    const uint32_t box_bytes = static_cast<uint32_t>(box_rows) * 128;
    Cursor<D> cc = first;
    uint32_t g = 0;  // steps so far
#pragma unroll 1
    while (cc.left > 0 && !fail) {
      const Run r = cc.take(plan);
      int i0 = r.j0 * kBN / bs, y = r.j0 * kBN - i0 * bs;  // the next step's first block, and its row there (a block of more than a step's keys)
      const int n_blk = (plan.pre[r.grp] + bs - 1) / bs;
      const int32_t* const row = p.tables + static_cast<int64_t>(plan.lead[r.grp]) * p.table_stride;
      int chunk = -1;   // 32 entries of the table at hand, one a lane
      int32_t id = 0;
#pragma unroll 1
      for (int x = 0; x < r.n; ++x, ++g) {
        const uint32_t st = uniform(g) % kStages;
        if (g >= kStages && !warp_wait_at(a_free + 8 * st, (g / kStages - 1) & 1)) {
          fail = true;
          break;
        }
        const int n = min(boxes, n_blk - i0);  // blocks behind the prefix are not loaded: their keys are masked
        expect_bytes(on, a_full + 8 * st, static_cast<uint32_t>(n) * box_bytes * kH);
        uint32_t dst = ring + st * (kH * kKvHalf);
#pragma unroll 1
        for (int b = 0; b < n; ++b, dst += box_bytes) {
          const int i = i0 + b;
          if ((i >> 5) != chunk) {
            chunk = i >> 5;
            const int mine = chunk * 32 + lane;
            id = 0;
            if (mine < n_blk) {
              id = __ldcg(row + mine);
              if (id < 0 || id >= p.num_blocks) {  // flagged, and another block's keys read in its place
                flag_error(p.err, PSB_DEVERR_BLOCK_RANGE);
                id = 0;
              }
            }
            __syncwarp();
          }
          const int32_t tile = static_cast<int32_t>((layer0 + __shfl_sync(0xffffffffu, id, i & 31)) * p.hkv + r.kvh);
#pragma unroll
          for (int h = 0; h < kH; ++h) box_load(on, dst + h * kKvHalf, tm, h * kHalf, y, tile, a_full + 8 * st);
        }
        if (bs > kBN) {
          y += kBN;
          if (y == bs) {
            y = 0;
            ++i0;
          }
        } else {
          i0 += boxes;
        }
      }
    }
    if (fail && on) flag_error(p.err, PSB_DEVERR_TIMEOUT);
    // the newest copies of each stage land before the CTA ends, also where the products gave up waiting for others
    for (uint32_t t = g > kStages ? g - kStages : 0; t < g; ++t) (void)warp_wait_at(a_full + 8 * (t % kStages), (t / kStages) & 1);
  };
  if (warp >= kFirstOwn) {
    own_parts<T, D, HP, NT>(p, plan, &tm_ko, &tm_vo, smem + Geo::kOffRing, bar_own);
  } else if (warp >= 8) {
    fewer_registers<kOtherRegs>();
    if (warp == 8) products(Int<0>());
    else if (warp == 9) products(Int<1>());
    else copies();
  } else {
    more_registers<kSoftmaxRegs>();
    // ---- softmax: thread r of a stream is row r of the tile and lane r of TMEM ----
    const int s = warp >> 2, row = tid - 128 * s;
    const int rseq = row / group;
    const uint32_t t_lane = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const float sc = p.scale_log2;
    Cursor<D> cc = first;
    int half = 0, k = 0;  // half-steps before the run, this stream's steps so far
    while (cc.left > 0 && !fail) {
      const Run r = cc.take(plan);
      const int pre = plan.pre[r.grp];
      const int mine = (half + s) & 1;  // which of each two half-steps is this stream's
      const bool live = rseq < TQ && rseq + (r.two ? s * TQ : 0) < r.n_seq;
      float ms = -INFINITY, l = 0.f;    // the exponents' reference (times sc), the sum
      bool begun = false;
      for (int x = r.two ? 0 : mine; x < r.n; x += r.two ? 1 : 2, ++k) {
        const int b = k & 1;
        const uint32_t ph = (k >> 1) & 1;
        // (by whole warps, here and below: lanes that gave up by themselves would leave the others' TMEM access short of them)
        if (!warp_wait(bar_s + 2 * s + b, ph)) {
          fail = true;
          break;
        }
        tc_fence_after();
        const uint32_t t_s = t_lane + kSCol + (2 * s + b) * kBN, t_o = t_lane + kOCol + s * D;
        const int have = pre - (r.j0 + x) * kBN;  // keys there are, from the step's first on
        uint32_t sr[kBN];
        tmem_ld32(t_s, sr);
        tmem_ld32(t_s + 32, sr + 32);
        tmem_wait_ld();
        if (have < kBN) {
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
          if (begun) {  // O holds P V of the earlier half-steps once the last of them is done
            if (!warp_wait(bar_pv + 2 * s + (b ^ 1), ((k - 1) >> 1) & 1)) {
              fail = true;
              break;
            }
            tc_fence_after();
#pragma unroll 1
            for (int q = 0; q < D; q += 32) {
              uint32_t ot[32];
              tmem_ld32(t_o + q, ot);
              tmem_wait_ld();
#pragma unroll
              for (int d = 0; d < 32; ++d) ot[d] = __float_as_uint(__uint_as_float(ot[d]) * alpha);
              tmem_st32(t_o + q, ot);
            }
            tmem_wait_st();
          }
          l *= alpha;
          ms = ms_new;
        }
        begun = true;
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
        mbar_arrive(bar_p + 2 * s + b);
      }
      if (fail) break;
      // the run's partial; the next run's first P V comes after its P
      const int ord = r.kvh * plan.n_pairs + r.pair;
      float* const part = p.tile_part + static_cast<int64_t>(2 * (cta + ord) + s) * tile_floats(D);
      if (begun) {
        if (!warp_wait(bar_pv + 2 * s + ((k - 1) & 1), ((k - 1) >> 1) & 1)) {
          fail = true;
          break;
        }
        tc_fence_after();
#pragma unroll 1
        for (int q = 0; q < D; q += 32) {
          uint32_t ot[32];
          tmem_ld32(t_lane + kOCol + s * D + q, ot);
          tmem_wait_ld();
          if (live) {
#pragma unroll
            for (int d = 0; d < 32; d += 4)
              reinterpret_cast<float4*>(part)[((q + d) >> 2) * kRows + row] =
                  make_float4(__uint_as_float(ot[d]), __uint_as_float(ot[d + 1]), __uint_as_float(ot[d + 2]), __uint_as_float(ot[d + 3]));
          }
          __syncwarp();
        }
        tc_fence_before();
      }
      if (live) reinterpret_cast<float2*>(part + kRows * D)[row] = make_float2(ms, l);  // (of a stream without steps: none)
      if (r.j0 == 0 && tid == 0) {
        const int steps = plan.steps_of(r.grp);
        const uint32_t begin = static_cast<uint32_t>(r.kvh) * plan.n_cost + plan.cost[r.grp] + C::kPair * r.in_grp * steps;
        const int ctas = static_cast<int>(deal.part_of(begin + (r.two ? C::kPair : C::kTile) * steps - 1) - cta) + 1;
        int2* const info = p.tile_info + r.kvh * p.max_tiles + r.tile;
        const int slot = 2 * static_cast<int>(cta + ord);
        info[0] = r.two ? make_int2(slot, ctas | 2 << 16) : make_int2(slot, 2 * ctas | 1 << 16);
        if (r.two) info[1] = make_int2(slot + 1, ctas | 2 << 16);
      }
      half += r.two ? 2 * r.n : r.n;
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
// the join
// ---------------------------------------------------------------------------
// A lane has a row (a sequence's q head of one kv head) and four of its dims, a warp 32
// consecutive rows, whose partials lie side by side; a CTA's four warps take a quarter
// of the partials each (they come from L2: rounds of loads, not bytes, are what it
// costs; one warp for all of 33 partials took 10 us).  BATCH: a warp's partials in flight,
// eight of a few CTAs (those 33: 2 us less than with four), four of many (3000 CTAs: the
// registers of eight would cost 3 us).
constexpr int kJoinThreads = 128, kJoinWarps = kJoinThreads / 32;

template <typename T, int D, int BATCH>
__global__ void __launch_bounds__(kJoinThreads) shared_join_kernel(const SharedParams p, int hp) {
  __shared__ float2 s_ml[kJoinWarps][32];
  __shared__ float4 s_o[kJoinWarps][32];
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c4 = blockIdx.y, kvh = blockIdx.z;
  const int u = min(static_cast<int>(blockIdx.x) * 32 + lane, p.batch * p.group - 1);  // (the last row again behind the last)
  const int b = u / p.group, gh = u - b * p.group;
  const int s = (kvh / hp) * p.batch + b;
  const int2 seq = __ldcg(p.seq_info + b), own = __ldcg(p.own_info + s);
  int2 tile = make_int2(0, 0);
  if (seq.x >= 0) tile = __ldcg(p.tile_info + kvh * p.max_tiles + seq.x);
  const int trow = seq.y * p.group + gh, orow = (hp == 2 ? (kvh & 1) * 8 : 0) + gh;
  const int tiles = tile.y & 0xffff, apart = tile.y >> 16, n = tiles + own.y;
  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](auto batch, const float2* ml, const float4* v) {
    constexpr int kBatch = decltype(batch)::value;
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
      // nothing was summed (nor written); a sum that is no number, of scores that are none, is not nothing
      if (ml[j].x == -INFINITY && ml[j].y == 0.f) continue;
      const float w = ex2_approx(ml[j].x - mu);
      l = fmaf(ml[j].y, w, l);
      o.x = fmaf(v[j].x, w, o.x);
      o.y = fmaf(v[j].y, w, o.y);
      o.z = fmaf(v[j].z, w, o.z);
      o.w = fmaf(v[j].w, w, o.w);
    }
  };
  // partials i0, i0 + 4, .. of the row, ``batch`` in flight
  auto round = [&](auto batch, int i0) {
    constexpr int kBatch = decltype(batch)::value;
    float2 ml[kBatch];
    float4 v[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int i = i0 + j * kJoinWarps;
      ml[j] = make_float2(-INFINITY, 0.f);
      v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (i < n) {
        const bool of_tile = i < tiles;
        const float* const part = of_tile ? p.tile_part + static_cast<int64_t>(tile.x + i * apart) * tile_floats(D)
                                          : p.own_part + static_cast<int64_t>(own.x + i - tiles) * own_floats(D);
        const int rows = of_tile ? kRows : 16, row = of_tile ? trow : orow;
        ml[j] = __ldcg(reinterpret_cast<const float2*>(part + rows * D) + row);
        v[j] = __ldcg(reinterpret_cast<const float4*>(part) + c4 * rows + row);
      }
    }
    add(batch, ml, v);
  };
#pragma unroll 1
  for (int i0 = warp; i0 < n; i0 += BATCH * kJoinWarps) round(Int<BATCH>(), i0);
  s_ml[warp][lane] = make_float2(m, l);
  s_o[warp][lane] = o;
  __syncthreads();
  if (warp != 0 || static_cast<int>(blockIdx.x) * 32 + lane >= p.batch * p.group) return;
  {
    float2 ml[kJoinWarps - 1];
    float4 v[kJoinWarps - 1];
#pragma unroll
    for (int j = 0; j < kJoinWarps - 1; ++j) {
      ml[j] = s_ml[j + 1][lane];
      v[j] = s_o[j + 1][lane];
    }
    add(Int<kJoinWarps - 1>(), ml, v);
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  T* const out = reinterpret_cast<T*>(p.out) + b * p.osb + (kvh * p.group + gh) * p.osh + 4 * c4;
  const uint32_t lo = pack2<T>(o.x * inv, o.y * inv), hi = pack2<T>(o.z * inv, o.w * inv);
  if (reinterpret_cast<uintptr_t>(out) % 8 == 0) {
    *reinterpret_cast<uint2*>(out) = make_uint2(lo, hi);
  } else {
    uint16_t* const o16 = reinterpret_cast<uint16_t*>(out);
    o16[0] = static_cast<uint16_t>(lo);
    o16[1] = static_cast<uint16_t>(lo >> 16);
    o16[2] = static_cast<uint16_t>(hi);
    o16[3] = static_cast<uint16_t>(hi >> 16);
  }
}

// The groups' checks by themselves, as build_plan makes them.
__global__ void check_groups_kernel(const int32_t* cu, const int32_t* prefix, int32_t batch, int32_t groups, int32_t* err) {
  int32_t bits = 0;
  for (int g = threadIdx.x; g <= groups; g += blockDim.x) {
    const int a = cu[g], prev = g == 0 ? 0 : cu[g - 1];
    if (a < prev || prev < 0 || a > batch) bits |= PSB_DEVERR_SEQLENS;
    if (g < groups && prefix[g] < 0) bits |= PSB_DEVERR_CONTEXT;
  }
  if (bits != 0) flag_error(err, bits);
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
bool two_heads(int group, int hkv, int d) { return d == 64 && group <= 8 && hkv % 2 == 0; }  // (D 128: too many registers)

size_t main_smem(int batch, int groups, int group, int hkv, int d) {
  const size_t fixed = d == 128 ? TcGeom<128>::kOffRing + OwnGeom<128, 1>::kBytes
                                : TcGeom<64>::kOffRing + (two_heads(group, hkv, d) ? OwnGeom<64, 2>::kBytes : OwnGeom<64, 1>::kBytes);
  return 1024 + fixed + sizeof(int32_t) * Plan::ints(batch, groups);
}

bool takes(int batch, int groups, int q_heads, int hkv, int head_dim, int block_size, int dtype, int max_context) {
  if (!(dtype == PSB_BF16 || dtype == PSB_F16) || !(head_dim == 64 || head_dim == 128)) return false;
  if (batch <= 0 || batch > kMaxBatch || groups < 0 || groups > kMaxBatch || hkv <= 0 || q_heads <= 0 || q_heads % hkv) return false;
  const int group = q_heads / hkv;
  if (group > 16 || block_size < 16 || block_size % 16 || !(64 % block_size == 0 || block_size % 64 == 0)) return false;
  if (main_smem(batch, groups, group, hkv, head_dim) > kMaxSmem || hkv > 65535) return false;
  const int64_t steps = (static_cast<int64_t>(max_context) + kBN) / kBN, tiles = batch / (kRows / group) + std::min(groups, batch / 2) + 1;
  return static_cast<int64_t>(batch) * hkv < (1 << 24) && steps * tiles < (int64_t(1) << 30) / hkv &&
         (static_cast<int64_t>(max_context) / 16 + 2) * batch < (int64_t(1) << 31) / hkv;
}

struct Layout {
  int max_tiles, max_pairs;
  size_t tile_info, seq_info, own_info, tile_part, own_part, bytes;
  Layout(int batch, int groups, int group, int hkv, int d) {
    max_tiles = batch / (kRows / group) + std::min(groups, batch / 2) + 1;
    max_pairs = batch / (2 * (kRows / group)) + std::min(groups, batch / 2) + 1;
    size_t at = 0;
    auto take = [&](size_t n) {
      const size_t r = at;
      at = align_up(at + n, 256);
      return r;
    };
    tile_info = take(sizeof(int2) * static_cast<size_t>(hkv) * max_tiles);
    seq_info = take(sizeof(int2) * static_cast<size_t>(batch));
    own_info = take(sizeof(int2) * static_cast<size_t>(hkv) * batch);
    tile_part = take(sizeof(float) * tile_floats(d) * 2 * (static_cast<size_t>(hkv) * max_pairs + kMaxCtas));
    own_part = take(sizeof(float) * own_floats(d) * (static_cast<size_t>(hkv) * batch + static_cast<size_t>(kMaxCtas) * kOwnWarps));
    bytes = at;
  }
};

template <typename T, int D>
int launch(SharedParams p, int num_layers, cudaStream_t s) {
  const CUtensorMapDataType dt = Elem<T>::code == PSB_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const int sms = device_sm_count();
  if (sms <= 0) return PSB_ERR_CUDA;
  const bool two = two_heads(p.group, p.hkv, D);
  CUtensorMap tq, tk, tv, tko, tvo;
  const int64_t tiles = static_cast<int64_t>(num_layers) * p.num_blocks * p.hkv, hq = static_cast<int64_t>(p.hkv) * p.group;
  const int64_t qdims[3] = {D, hq, p.batch}, qstr[2] = {p.qsh * 2, p.qsb * 2}, kdims[3] = {D, p.block_size, tiles},
                kstr[2] = {D * 2, static_cast<int64_t>(p.block_size) * D * 2};
  const int qbox[3] = {kHalf, p.group, p.tq}, kbox[3] = {kHalf, std::min(p.block_size, kBN), 1}, obox[3] = {kHalf, 16, two ? 2 : 1};
  if (!encode_box_map(&tq, p.q, qdims, qstr, qbox, dt) || !encode_box_map(&tk, p.k_cache, kdims, kstr, kbox, dt) ||
      !encode_box_map(&tv, p.v_cache, kdims, kstr, kbox, dt) || !encode_box_map(&tko, p.k_cache, kdims, kstr, obox, dt) ||
      !encode_box_map(&tvo, p.v_cache, kdims, kstr, obox, dt))
    return PSB_ERR_CUDA;
  // (a tile of two heads of D 128 takes too many registers; that of 9 to 16 q heads spills 240 bytes a
  // thread there, 32 sequences of 32 / 2 heads on 4 K with 256 each of their own in 25 us: paged_decode 1660)
  const bool hi = !two && p.group > 8;
  const auto kern = two ? shared_main_kernel<T, D, D == 64 ? 2 : 1, 1> : hi ? shared_main_kernel<T, D, 1, 2> : shared_main_kernel<T, D, 1, 1>;
  const void* const f = reinterpret_cast<const void*>(kern);
  static std::atomic<bool> checked[3];  // (of each instantiation) the shares draw on the launch's registers
  if (!checked[two ? 2 : hi].load(std::memory_order_relaxed)) {
    cudaFuncAttributes fa;
    const cudaError_t fe = cudaFuncGetAttributes(&fa, f);
    if (fe != cudaSuccess) return record_cuda_error(fe);
    if (fa.numRegs != 128) return PSB_ERR_UNSUPPORTED;
    checked[two ? 2 : hi].store(true, std::memory_order_relaxed);
  }
  const size_t smem = main_smem(p.batch, p.groups, p.group, p.hkv, D);
  int occ = 0;
  if (!kernel_occupancy(f, kThreads, smem, &occ)) return PSB_ERR_CUDA;
  if (occ < 1) return PSB_ERR_UNSUPPORTED;
  discard_stale_error();
  cudaError_t e = launch_pdl(kern, dim3(std::min(kMaxCtas, sms)), dim3(kThreads), smem, s, p, tq, tk, tv, tko, tvo);
  if (e != cudaSuccess) return record_cuda_error(e);
  const dim3 join((p.batch * p.group + 31) / 32, D / 4, p.hkv);
  const bool few = static_cast<int64_t>(join.x) * join.y * join.z <= 4 * sms;
  e = launch_pdl(few ? shared_join_kernel<T, D, 8> : shared_join_kernel<T, D, 4>, join, dim3(kJoinThreads), 0, s, p, two ? 2 : 1);
  if (e != cudaSuccess) return record_cuda_error(e);
  return check_launch();
}

}  // namespace
}  // namespace psb

using namespace psb;

extern "C" int psb_check_groups(const int32_t* cu_groups, const int32_t* prefix_lens, int32_t batch, int32_t num_groups, int32_t* error_flag,
                                psb_stream_t stream) {
  if (batch < 0 || num_groups < 0 || !cu_groups || (num_groups > 0 && !prefix_lens)) return PSB_ERR_INVALID;
  if (!error_flag) return PSB_OK;
  discard_stale_error();
  check_groups_kernel<<<1, 256, 0, reinterpret_cast<cudaStream_t>(stream)>>>(cu_groups, prefix_lens, batch, num_groups, error_flag);
  return check_launch();
}

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
  if (!query || !out || !k_cache || !v_cache || !block_tables || !context_lens || !cu_groups || (num_groups > 0 && !prefix_lens))
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
