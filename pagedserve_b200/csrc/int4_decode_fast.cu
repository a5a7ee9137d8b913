// Paged GQA decode attention over the 4-bit KV pool: the tensor-core path
// (bf16/f16, head_dim 64 or 128, block_size a multiple of 16).
//
// Mathematics.  Token t's key is mid_t + step_t (c_t - 7.5) with 4-bit codes
// c_t, so its score is  step_t (q . (c_t - 7.5)) + mid_t sum(q): the codes
// enter the matrix product as small exact integers and step, mid act on the
// fp32 result.  Likewise sum_t p_t v_t = sum_t (p_t step_t)(c_t - 7.5) +
// sum_t p_t mid_t: p_t step_t is rounded to the 16-bit type (the one rounding
// below fp32; probabilities are rounded there by every 16-bit attention of
// this library), the second sum is a scalar per head in fp32.
//
// Products.  mma.sync m16n8k16 in f16 with the tokens of a 16-token tile as
// rows of S^T = K Q^T (8 q heads are the 8 columns) and head_dim as rows of
// O^T = V^T P^T.  The codes are the A operand in both, so a lane needs no more
// than its own words of a code row: which element of head_dim an index k or a
// row stands for is free as long as q (loaded once) and the output agree.  A
// code becomes an operand by one AND: (w >> 8 i) & 0x000f000f is the pair of
// f16 subnormals c 2^-24, & 0x00f000f0 the pair c 2^-20, both exact.  The
// other operand is brought to f16 whatever T is, without losing anything T
// keeps: q times the power of two that takes the head tile's largest |q| to
// 2^14 (what falls below f16's range then is under 2^-38 of that largest);
// p step times a power of two that keeps it below 2^15, so it has f16's 11
// bits down to 2^-29 of the largest so far.  That one rounding is the only one
// below fp32.  A product with ones sums the rounded p step for the -7.5.
// P^T is S^T's accumulator layout transposed: two movmatrix per tile.
//
// What bounds it.  A 16-token tile of head_dim 64 is 1152 bytes against 4096
// in bf16, so the same bytes per second need 3.6 times the instructions of
// paged_decode (about 150 a tile): hence codes by AND, two tiles at a time
// (independent work, one vote and one set of loop instructions for both), each
// token's four factors worked out by one lane and handed round through shared
// memory, the exponents' reference folded into the score's multiply-add, and
// addresses and validity worked out for 32 items at once, one per lane.  They
// take 43% of the issue slots now (37% at head_dim 128, ALU 40%): what is left is
// latency.  A scheduler has three warps (two at head_dim 128) to cover it, each
// with one item's codes on their way; the stalls per issue are loads 1.8 (long
// scoreboard), fixed-latency results 1.3, shared memory 0.6.  Measured: 256
// sequences of 62 MB of cache 26.2 us (2.4 TB/s; the 16-bit pool's paged_decode
// 39 us), of which some 7 us do not depend on the length; 3 sequences of 32 K
// tokens 13.4 us, of 128 K 10 us more (4 TB/s); 64 sequences of 4 K at head_dim
// 128 43.7 us (3.5 TB/s).  Reading lengths and
// tables before the wait for the stream predecessor saved 0.6 to 1.5 us a call,
// but a predecessor that starts its dependents early (or has just left the GPU)
// may not have written them yet.
//
// Split.  The items (32 tokens) of all sequences, in (kv head, sequence,
// position) order, are dealt evenly over the warps of the grid (one CTA per
// SM).  A warp loads its codes straight into registers, each part of the next
// item as soon as this item's part has been used: bulk copies by a warp of
// their own through shared memory took 2.5 times as long, a ring filled by
// cp.async 187 instructions a tile, prefetches to L2 gained nothing.  12 warps
// of 164 registers beat 8 of 244 where the tile fits (26.0 against 28.1 us).  A
// sequence inside one warp's run is written at once; pieces of one sequence
// within a CTA are joined in shared memory, and only a sequence cut by a CTA
// boundary (at most one per CTA) leaves partials, for int4_combine_kernel.
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "host_util.h"
#include "int4_attention.h"
#include "int4_cache.cuh"

namespace psb {
namespace {

constexpr int kMaxCtas = 160;       // grid limit (one CTA per SM; B200 has 148)
constexpr int kMaxBatch = 2560;     // sequences whose lengths fit in shared memory

template <int D, int HT>
struct Geo {
  static constexpr int kWarps = D * HT == 64 ? 12 : 8;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kRows = 8 * HT;                  // q heads of a tile
  static constexpr int kCodeBytes = 16 * D / 2;         // K (or V) codes of 16 tokens
  static constexpr int kPartFloats = kRows * (D + 2);   // one piece: [rows][D] output, [rows][2] max, sum
  static constexpr int kFactors = 32 * 16;              // (K step, K mid, V step, V mid) of an item's tokens
  // per warp: first piece | last piece | factors; then the join's weights [rows][2 warps] and (max, sum)
  static constexpr size_t per_warp() { return 2 * kPartFloats * 4 + kFactors; }
  static constexpr size_t fixed_smem() { return kWarps * per_warp() + sizeof(float) * kRows * 2 * kWarps * 3; }
  static size_t smem(int batch) { return fixed_smem() + sizeof(int32_t) * (2 * static_cast<size_t>(batch) + 1); }
};

// What a CTA leaves for int4_combine_kernel: the sequence cut at its end that
// began in it (c1: the last CTA with a piece; 0: none).
struct Cut {
  int32_t grp, b, c1, pad;
};

__device__ __forceinline__ uint32_t movmatrix_t(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
// max(a, |x|) of packed pairs, a NaN in x passed over
template <typename T>
__device__ __forceinline__ uint32_t abs_max2(uint32_t a, uint32_t x);
template <>
__device__ __forceinline__ uint32_t abs_max2<__nv_bfloat16>(uint32_t a, uint32_t x) {
  uint32_t d;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(x & 0x7fff7fffu));
  return d;
}
template <>
__device__ __forceinline__ uint32_t abs_max2<__half>(uint32_t a, uint32_t x) {
  uint32_t d;
  asm("max.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(x & 0x7fff7fffu));
  return d;
}

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) { return __byte_perm(a, b, sel); }

// Pair i (0 .. 3) of a code word, its nibbles i and i + 4, as two f16: c 2^-24
// for even i, c 2^-20 for odd i.
__device__ __forceinline__ uint32_t code_pair(uint32_t w, uint32_t w8, int i) {
  return (i < 2 ? w : w8) & (i & 1 ? 0x00f000f0u : 0x000f000fu);
}

// d = a b (the accumulator starts at zero)
__device__ __forceinline__ void mma_f16_first(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

constexpr float kGrowth = 4.f;     // a score may exceed the exponents' reference by this (log2) before it is moved
constexpr int kPBits = 11;         // p step is scaled to at most 2^kGrowth 2^kPBits = 2^15
constexpr float kTwo24 = 16777216.f;
constexpr float kUnit = 1024.f;    // 2^24 (codes) over 2^14 (the largest |q|): of a unit of the scores' accumulator

__device__ __forceinline__ int items_of(int ctx) { return ctx <= 0 ? 1 : (ctx + 31) >> 5; }

// s_ctx[b] = clamped context, pre[b] = items before sequence b, pre[B] = all.
// Called by every thread of a CTA.
__device__ int build_prefix(const Int4DecodeParams& p, int32_t* pre, int32_t* s_ctx, bool flag) {
  __shared__ int32_t warp_sums[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nthr = blockDim.x;
  const int per = (p.batch + nthr - 1) / nthr;
  const int begin = min(tid * per, p.batch), end = min(begin + per, p.batch);
  int local = 0;
  for (int b = begin; b < end; ++b) {
    int n = p.ctx[b];
    if (n < 0 || n > p.max_context) {
      if (flag) flag_error(p.err, PSB_DEVERR_CONTEXT);
      n = n < 0 ? 0 : p.max_context;
    }
    s_ctx[b] = n;
    local += items_of(n);
  }
  int incl = local;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) warp_sums[warp] = incl;
  __syncthreads();
  int sums = lane < nthr / 32 ? warp_sums[lane] : 0;  // every warp scans the warps' sums
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, sums, o);
    if (lane >= o) sums += v;
  }
  const int total = __shfl_sync(0xffffffffu, sums, 31);
  int run = incl - local + (warp ? __shfl_sync(0xffffffffu, sums, warp - 1) : 0);
  for (int b = begin; b < end; ++b) {
    pre[b] = run;
    run += items_of(s_ctx[b]);
  }
  if (tid == 0) pre[p.batch] = total;
  __syncthreads();
  return total;
}

// Last b with pre[b] <= i.
__device__ __forceinline__ int find_seq(const int32_t* pre, int batch, int i) {
  int lo = 0, hi = batch - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (pre[mid] <= i) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// The item list dealt over ``parts``: part w starts at floor(n w / parts).
struct Deal {
  uint32_t q, r, parts;
  __device__ Deal(int n, int parts_) : q(static_cast<uint32_t>(n) / parts_), r(n - q * parts_), parts(parts_) {}
  __device__ int start(uint32_t w) const { return w * q + (r * w) / parts; }  // r, w <= 2560: no overflow
};

template <typename T, int D, int HT>
__global__ void __launch_bounds__(Geo<D, HT>::kThreads, 1) int4_decode_kernel(const Int4DecodeParams p) {
  using G = Geo<D, HT>;
  constexpr int kW = G::kWarps, kRows = G::kRows;
  constexpr int kM = D / 16;      // products per 16 tokens, K and V alike
  constexpr int kWords = D / 32;  // code words per lane: K per row, V per token / 2
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int32_t s_grp[2 * kW], s_seq[2 * kW];  // (head tile, sequence) of each warp's first and last piece, -1: none
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  float* const pieces = reinterpret_cast<float*>(smem);  // [warps][first, last]
  float4* const factors = reinterpret_cast<float4*>(smem + kW * 2 * G::kPartFloats * 4) + warp * 32;
  float* const s_w = reinterpret_cast<float*>(smem + kW * G::per_warp());  // [rows][2 kW] weights of the pieces
  float2* const s_ml = reinterpret_cast<float2*>(s_w + kRows * 2 * kW);    // [rows][2 kW] (max, sum) at a run's first piece
  int32_t* const pre = reinterpret_cast<int32_t*>(smem + G::fixed_smem());
  int32_t* const s_ctx = pre + p.batch + 1;

  const int B = p.batch, BS = p.block_size;
  const int hgroups = (p.group + kRows - 1) / kRows;  // head tiles per kv head
  if (tid < 2 * kW) s_grp[tid] = -1;
  pdl_wait();
  pdl_launch_dependents();
  const int n_seq = build_prefix(p, pre, s_ctx, blockIdx.x == 0);
  const int n_items = n_seq * (p.hkv * hgroups);
  const int act = min(static_cast<int>(gridDim.x), (n_items + kW - 1) / kW);
  Cut* const cuts = reinterpret_cast<Cut*>(p.part);
  float* const part = p.part + kMaxCtas * (sizeof(Cut) / sizeof(float));
  if (static_cast<int>(blockIdx.x) >= act) {
    if (tid == 0) cuts[blockIdx.x] = Cut{0, 0, 0, 0};
    return;
  }
  const Deal deal(n_items, act * kW);
  const int starts = deal.start(blockIdx.x * kW + min(lane, kW));  // lane w: of the CTA's warp w
  const int cta_a = __shfl_sync(0xffffffffu, starts, 0), cta_e = __shfl_sync(0xffffffffu, starts, kW);

  const int my_a = __shfl_sync(0xffffffffu, starts, warp), my_e = __shfl_sync(0xffffffffu, starts, warp + 1);

  // ---- 32 items at a time, one per lane: where their tiles are ---------------
  // row16: pool rows / 16 of the two K tiles (below 2^31; 0 where there is
  // none: it is read all the same and masked), the top bit set where the
  // tile's block is outside the pool; any_bad: some tile of the run is
  struct Chunk {
    uint32_t row16[2];
  };
  constexpr uint32_t kBad = 1u << 31;
  bool any_bad = false;
  int seg_grp = 0, seg_b = 0, seg_j = 0;  // head tile, sequence and item in it of the warp's next share
  auto build_chunk = [&](int beg) -> Chunk {
    Chunk c{{0u, 0u}};
    const int i = beg + lane;
    if (i < my_e) {
      const int grp = static_cast<uint32_t>(i) / static_cast<uint32_t>(n_seq);
      const int r = i - grp * n_seq;
      const int b = find_seq(pre, B, r), j = r - pre[b], ctx = s_ctx[b];
      const int kvh = hgroups == 1 ? grp : grp / hgroups;
      const int32_t* row = p.tables + static_cast<int64_t>(b) * p.table_stride;
      int blk[2];
      uint32_t sub[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint32_t tile = 2 * j + k;  // tile of the sequence; BS / 16 tiles a block
        const uint32_t bi = static_cast<uint32_t>((static_cast<uint64_t>(tile) * p.tile_div) >> 32);
        blk[k] = 16 * static_cast<int>(tile) < ctx ? __ldg(row + bi) : -1;
        sub[k] = tile - bi * (BS >> 4);
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        if (blk[k] >= 0 && blk[k] < p.num_blocks) {
          // rows of (layer, block, kv head) in the pool: 2 BS of K and V
          c.row16[k] = static_cast<uint32_t>((p.layer_tiles + static_cast<int64_t>(blk[k]) * p.hkv + kvh) * (BS >> 3)) + sub[k];
        } else if (16 * (2 * j + k) < ctx) {
          flag_error(p.err, PSB_DEVERR_BLOCK_RANGE);
          c.row16[k] = kBad;
        } else if (k == 1) {
          c.row16[1] = c.row16[0] & ~kBad;  // no second tile: the first one again
        }
      }
      if (i == my_a) {
        seg_grp = grp;
        seg_b = b;
        seg_j = j;
      }
    }
    any_bad = any_bad || __any_sync(0xffffffffu, (c.row16[0] | c.row16[1]) & kBad);
    return c;
  };
  Chunk cur{}, nxt{};
  if (my_a < my_e) {
    cur = build_chunk(my_a);
    seg_grp = __shfl_sync(0xffffffffu, seg_grp, 0);
    seg_b = __shfl_sync(0xffffffffu, seg_b, 0);
    seg_j = __shfl_sync(0xffffffffu, seg_j, 0);
    if (my_e - my_a > 32) nxt = build_chunk(my_a + 32);
  }

  // Row pi(r) of a tile is the token at index r (0 .. 7; those of 8 .. 15 are 8
  // rows on) of the products: the four tokens of a lane group's V load are
  // adjacent rows, one run of memory.
  auto pi = [](int r) { return (r >> 1) + 4 * (r & 1); };
  uint32_t qb[HT][kM][2];         // B fragments of q
  float qs[HT][2];                // sum(q) 2^(14 - qe) of heads 2 t, 2 t + 1
  float o[HT][kM][4];             // (element of row g | g + 8) x (head 2 t | 2 t + 1)
  float sp[HT][4];                // sums of the rounded, scaled p step
  float nref[HT][2];              // minus the exponents' reference
  float l[HT][2], z[HT][2];       // sum p, sum p mid
  // A unit of the accumulator is a score of 2^24 2^-14 2^qe sc per step, a unit of
  // sum(q) 2^-14 2^qe sc per unit of the value: 2^qe (the head tile's largest |q|)
  // last, as it may be anything bf16 holds.  (The former is up to 2^10 times the
  // scores it makes up: those end at 2^117.)
  float kexp = 1.f;               // 2^qe
  float vscale = 1.f, vlim = 0.f; // scale of p step; the largest step it allows
  int n_pieces = 0;
  const float sc = p.scale_log2;
  const int row0 = pi(g);         // tokens of rows g and g + 8: row0, 8 + row0

  // An item's codes and parameters live in registers; each part of the next
  // item is loaded as soon as this item's part has been used, so about one
  // item per warp (2.3 KB at D 64, 37 KB an SM) is always on its way.
  using KVec = typename std::conditional<D == 64, uint2, uint4>::type;
  using VVec = typename std::conditional<D == 64, uint32_t, uint2>::type;
  KVec kx[2][2];
  VVec vx[2][4];
  uint32_t kpar = 0, vpar = 0;    // parameters of token ``lane`` of the item
  uint32_t bad = 0, bad_next = 0; // bit k: tile k's block is outside the pool
  const uint8_t* const src_k = p.codes + row0 * (D / 2) + t * (D / 8);
  const uint8_t* const src_v = p.codes + static_cast<int64_t>(BS) * (D / 2) + pi(2 * t) * (D / 2) + g * (D / 16);
  const char* const src_par = reinterpret_cast<const char*>(p.params) + (lane & 15) * 4;
  const int64_t par_v = static_cast<int64_t>(BS) * 4;
  int next = my_a;                // next item to load
  uint32_t r0 = 0, r1 = 0;        // its tiles
  auto advance = [&]() {  // past the run's end: item 0 of the pool, read and not used
    if (next < my_e) {
      const int ib = (next - my_a) & 31;
      r0 = __shfl_sync(0xffffffffu, cur.row16[0], ib);
      r1 = __shfl_sync(0xffffffffu, cur.row16[1], ib);
      if (any_bad) {
        bad_next = (r0 >> 31) | (r1 >> 31) << 1;
        r0 &= ~kBad;
        r1 &= ~kBad;
      }
      ++next;
      if (ib == 31) {
        cur = nxt;
        if (my_e - next > 32) nxt = build_chunk(next + 32);
      }
    }
  };
  auto load_k = [&]() {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const uint8_t* src = src_k + static_cast<uint64_t>(k ? r1 : r0) * G::kCodeBytes;
      kx[k][0] = __ldcs(reinterpret_cast<const KVec*>(src));
      kx[k][1] = __ldcs(reinterpret_cast<const KVec*>(src + 8 * (D / 2)));
    }
  };
  auto load_v = [&]() {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const uint8_t* src = src_v + static_cast<uint64_t>(k ? r1 : r0) * G::kCodeBytes;
#pragma unroll
      for (int r = 0; r < 4; ++r)  // tokens of products 2 t, 2 t + 1, 2 t + 8, 2 t + 9
        vx[k][r] = __ldcs(reinterpret_cast<const VVec*>(src + ((r & 1) * 4 + (r >> 1) * 8) * (D / 2)));
    }
  };
  auto load_par = [&]() {
    const char* src = src_par + static_cast<uint64_t>(lane < 16 ? r0 : r1) * 64;
    kpar = __ldcs(reinterpret_cast<const uint32_t*>(src));
    vpar = __ldcs(reinterpret_cast<const uint32_t*>(src + par_v));
  };
  uint4 x[HT][kWords];  // q rows of a share: 8 elements a code word
  auto load_q = [&](int grp, int b) {
    const int kvh = hgroups == 1 ? grp : grp / hgroups, h0 = (grp - kvh * hgroups) * kRows;
#pragma unroll
    for (int ht = 0; ht < HT; ++ht) {
      const int hh = h0 + ht * 8 + g;
      const bool live = hh < p.group;
      const T* src = reinterpret_cast<const T*>(p.q) + b * p.qsb + (kvh * p.group + (live ? hh : 0)) * p.qsh + t * (D / 4);
#pragma unroll
      for (int w = 0; w < kWords; ++w) {
        x[ht][w] = make_uint4(0, 0, 0, 0);
        if (live) x[ht][w] = *reinterpret_cast<const uint4*>(src + 8 * w);
      }
    }
  };
  if (my_a < my_e) {
    load_q(seg_grp, seg_b);
    advance();
    bad = bad_next;
    load_par();
    load_k();
    load_v();
  }

  for (int at = my_a; at < my_e;) {
    // ---- the warp's share of one sequence: items seg_j .. of (seg_grp, seg_b) ----
    const int grp = seg_grp, b = seg_b, ctx = s_ctx[b], ni = items_of(ctx);
    if (at != my_a) load_q(grp, b);  // the first share's were loaded before its codes
    int todo = min(ni - seg_j, my_e - at);
    const bool whole = todo == ni;
    int tokens = ctx - 32 * seg_j;  // from this item on
    at += todo;
    seg_j = 0;
    if (++seg_b == B) {
      seg_b = 0;
      ++seg_grp;
    }
    bool fresh = true;  // no score seen yet
    const int kvh = hgroups == 1 ? grp : grp / hgroups, h0 = (grp - kvh * hgroups) * kRows;
    {
      uint32_t top2 = 0;
#pragma unroll
      for (int ht = 0; ht < HT; ++ht) {
#pragma unroll
        for (int w = 0; w < kWords; ++w) {
          const uint32_t* e = &x[ht][w].x;
#pragma unroll
          for (int i = 0; i < 4; ++i) top2 = abs_max2<T>(top2, e[i]);
        }
      }
      const float2 top_f = unpack2<T>(top2);
      float top = fmaxf(top_f.x, top_f.y);
      if (!finite_f32(top)) {  // an infinity: its own head's affair, the others keep their scale
        top = 0.f;
#pragma unroll
        for (int ht = 0; ht < HT; ++ht) {
#pragma unroll
          for (int w = 0; w < kWords; ++w) {
            const uint32_t* e = &x[ht][w].x;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float2 f = unpack2<T>(e[i]);
              if (finite_f32(f.x)) top = fmaxf(top, fabsf(f.x));
              if (finite_f32(f.y)) top = fmaxf(top, fabsf(f.y));
            }
          }
        }
      }
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
      const int qe = top > 0.f ? max(-113, ilogb_f32(top)) : 0;
      const float qsc = exp2_int(14 - qe);
      kexp = exp2_int(qe);
#pragma unroll
      for (int ht = 0; ht < HT; ++ht) {
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < kWords; ++w) {
          const float2 a0 = unpack2<T>(x[ht][w].x), a1 = unpack2<T>(x[ht][w].y), a2 = unpack2<T>(x[ht][w].z),
                       a3 = unpack2<T>(x[ht][w].w);
          // elements (i, i + 4) of the word, for products 4 (w / 2) + i; odd
          // products' codes are 16 times as large
          const float q16 = qsc * 0.0625f;
          const float2 b0 = make_float2(a0.x * qsc, a0.y * q16), b1 = make_float2(a1.x * qsc, a1.y * q16),
                       b2 = make_float2(a2.x * qsc, a2.y * q16), b3 = make_float2(a3.x * qsc, a3.y * q16);
          sum += (fmaf(16.f, b0.y, b0.x) + fmaf(16.f, b1.y, b1.x)) + (fmaf(16.f, b2.y, b2.x) + fmaf(16.f, b3.y, b3.x));
          qb[ht][4 * (w >> 1) + 0][w & 1] = pack2<__half>(b0.x, b2.x);
          qb[ht][4 * (w >> 1) + 1][w & 1] = pack2<__half>(b0.y, b2.y);
          qb[ht][4 * (w >> 1) + 2][w & 1] = pack2<__half>(b1.x, b3.x);
          qb[ht][4 * (w >> 1) + 3][w & 1] = pack2<__half>(b1.y, b3.y);
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        qs[ht][0] = __shfl_sync(0xffffffffu, sum, 8 * t);  // head 2 t is lanes 8 t .. 8 t + 3
        qs[ht][1] = __shfl_sync(0xffffffffu, sum, 8 * t + 4);
#pragma unroll
        for (int e = 0; e < 2; ++e) nref[ht][e] = l[ht][e] = z[ht][e] = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) sp[ht][e] = 0.f;
#pragma unroll
        for (int i = 0; i < kM; ++i) o[ht][i][0] = o[ht][i][1] = o[ht][i][2] = o[ht][i][3] = 0.f;
      }
      vscale = 1.f;
      vlim = 0.f;
    }
    for (; todo > 0; --todo, tokens -= 32) {
      const bool all = tokens >= 32 && bad == 0;
      int valid0 = 16, valid1 = 16;
      if (!all) {
        valid0 = bad & 1 ? 0 : max(0, min(16, tokens));
        valid1 = bad & 2 ? 0 : max(0, min(16, tokens - 16));
      }
      const bool some = valid0 + valid1 > 0;
      advance();
      bad = bad_next;
      // ---- the tokens' factors, one token a lane ---------------------------------
      {
        if (!all && (lane & 15) >= (lane < 16 ? valid0 : valid1)) kpar = vpar = 0;  // rows past the context may hold anything
        const float2 kp = unpack2<T>(kpar), vp = unpack2<T>(vpar);
        if (__any_sync(0xffffffffu, vp.x > vlim)) {  // a larger step than the scale of p step allows
          float top = vp.x;
#pragma unroll
          for (int d = 1; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
          const int e = max(-100, ilogb_f32(top)) + 1;  // top < 2^e
          const float nv = exp2_int(kPBits - e);
          if (!fresh) {
            const float ratio = nv / vscale;
#pragma unroll
            for (int ht = 0; ht < HT; ++ht) {
#pragma unroll
              for (int i = 0; i < kM; ++i) {
#pragma unroll
                for (int k = 0; k < 4; ++k) o[ht][i][k] *= ratio;
              }
              sp[ht][0] *= ratio;
              sp[ht][1] *= ratio;
            }
          }
          vlim = exp2_int(min(e, 127));
          vscale = nv;
        }
        // the code's -7.5 goes with mid
        factors[lane] = make_float4(kp.x * (sc * kUnit) * kexp, fmaf(kp.x, -7.5f, kp.y) * (sc * 0x1p-14f) * kexp,
                                    vp.x * vscale, vp.y);
        load_par();
      }
      // ---- S^T = K Q^T ---------------------------------------------------------
      float s[2][HT][4];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        uint32_t kw[2][kWords], kw8[2][kWords];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const uint32_t* x = reinterpret_cast<const uint32_t*>(&kx[k][r]);
#pragma unroll
          for (int w = 0; w < kWords; ++w) {
            kw[r][w] = x[w];
            kw8[r][w] = x[w] >> 8;
          }
        }
#pragma unroll
        for (int i = 0; i < kM; ++i) {
          const int w = 2 * (i >> 2), nb = i & 3;
          const uint32_t a0 = code_pair(kw[0][w], kw8[0][w], nb), a1 = code_pair(kw[1][w], kw8[1][w], nb);
          const uint32_t a2 = code_pair(kw[0][w + 1], kw8[0][w + 1], nb), a3 = code_pair(kw[1][w + 1], kw8[1][w + 1], nb);
#pragma unroll
          for (int ht = 0; ht < HT; ++ht) {
            if (i == 0) mma_f16_first(s[k][ht], a0, a1, a2, a3, qb[ht][i][0], qb[ht][i][1]);
            else mma_16816<__half>(s[k][ht], a0, a1, a2, a3, qb[ht][i][0], qb[ht][i][1]);
          }
        }
      }
      load_k();
      __syncwarp();  // factors written
      // ---- scores minus reference (log2 scale) -----------------------------------
      float vs[2][2], vm[2][2];
      float top[HT][2];
#pragma unroll
      for (int ht = 0; ht < HT; ++ht) top[ht][0] = top[ht][1] = -INFINITY;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float4 f = factors[16 * k + 8 * r + row0];
          vs[k][r] = f.z;
          vm[k][r] = f.w;
#pragma unroll
          for (int ht = 0; ht < HT; ++ht) {
#pragma unroll
            for (int e = 0; e < 2; ++e)
              s[k][ht][2 * r + e] = fmaf(f.x, s[k][ht][2 * r + e], fmaf(f.y, qs[ht][e], nref[ht][e]));
          }
        }
      }
      if (!all) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            if (row0 + 8 * r >= (k ? valid1 : valid0)) {
#pragma unroll
              for (int ht = 0; ht < HT; ++ht) s[k][ht][2 * r] = s[k][ht][2 * r + 1] = -INFINITY;
            }
          }
        }
      }
      // The reference moves only when some score is above it by more than the
      // limit: most items touch no accumulator.
      bool grow = fresh && some;
#pragma unroll
      for (int ht = 0; ht < HT; ++ht) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          top[ht][e] = fmaxf(fmaxf(s[0][ht][e], s[0][ht][2 + e]), fmaxf(s[1][ht][e], s[1][ht][2 + e]));
          grow = grow || top[ht][e] > kGrowth;
        }
      }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int ht = 0; ht < HT; ++ht) {
          float al[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float mx = top[ht][e];
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            // the first reference is the first maximum (finite whatever the scores are)
            mx = fresh ? fminf(fmaxf(mx, -3e38f), 3e38f) : fmaxf(mx, 0.f);
            al[e] = ex2_approx(-mx);
            nref[ht][e] -= mx;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              s[k][ht][e] -= mx;
              s[k][ht][2 + e] -= mx;
            }
          }
          if (!fresh) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              l[ht][e] *= al[e];
              z[ht][e] *= al[e];
            }
#pragma unroll
            for (int i = 0; i < kM; ++i) {
              o[ht][i][0] *= al[0];
              o[ht][i][1] *= al[1];
              o[ht][i][2] *= al[0];
              o[ht][i][3] *= al[1];
            }
            sp[ht][0] *= al[0];
            sp[ht][1] *= al[1];
          }
        }
        fresh = false;
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        // ---- probabilities, P^T ----------------------------------------------------
        uint32_t pb[HT][2];  // B fragments
#pragma unroll
        for (int r = 0; r < 2; ++r) {
#pragma unroll
          for (int ht = 0; ht < HT; ++ht) {
            float pr[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              pr[e] = ex2_approx(s[k][ht][2 * r + e]);
              l[ht][e] += pr[e];
              z[ht][e] = fmaf(pr[e], vm[k][r], z[ht][e]);
            }
            pb[ht][r] = movmatrix_t(pack2<__half>(pr[0] * vs[k][r], pr[1] * vs[k][r]));
          }
        }
        // ---- O^T += V^T P^T ----------------------------------------------------------
        uint32_t vw[4][D / 64];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const uint32_t* x = reinterpret_cast<const uint32_t*>(&vx[k][r]);
#pragma unroll
          for (int w = 0; w < D / 64; ++w) vw[r][w] = x[w];
        }
#pragma unroll
        for (int q = 0; q < D / 64; ++q) {
          const uint32_t x01 = prmt(vw[0][q], vw[1][q], 0x5410), y01 = prmt(vw[0][q], vw[1][q], 0x7632);
          const uint32_t x23 = prmt(vw[2][q], vw[3][q], 0x5410), y23 = prmt(vw[2][q], vw[3][q], 0x7632);
          const uint32_t x01h = x01 >> 8, y01h = y01 >> 8, x23h = x23 >> 8, y23h = y23 >> 8;
#pragma unroll
          for (int nb = 0; nb < 4; ++nb) {
            const uint32_t a0 = code_pair(x01, x01h, nb), a1 = code_pair(y01, y01h, nb), a2 = code_pair(x23, x23h, nb),
                           a3 = code_pair(y23, y23h, nb);
#pragma unroll
            for (int ht = 0; ht < HT; ++ht) mma_16816<__half>(o[ht][4 * q + nb], a0, a1, a2, a3, pb[ht][0], pb[ht][1]);
          }
        }
#pragma unroll
        for (int ht = 0; ht < HT; ++ht)
          mma_16816<__half>(sp[ht], 0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u, pb[ht][0], pb[ht][1]);
      }
      load_v();
      __syncwarp();  // factors read
    }
    {
      // ---- the warp's share of the sequence is done ----------------------------
      float* piece = nullptr;
      if (!whole) {
        const int k = n_pieces++;  // a run's first share and its last
        piece = pieces + (2 * warp + k) * G::kPartFloats;
        if (lane == 0) {
          s_grp[2 * warp + k] = grp;
          s_seq[2 * warp + k] = b;
        }
      }
      const float vinv = 1.f / vscale;  // a power of two: exact
#pragma unroll
      for (int ht = 0; ht < HT; ++ht) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            l[ht][e] += __shfl_xor_sync(0xffffffffu, l[ht][e], d);
            z[ht][e] += __shfl_xor_sync(0xffffffffu, z[ht][e], d);
          }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float base = -7.5f * sp[ht][e];
          // elements (D / 8) g + 8 q + {0 .. 7}: nibbles 0-3 are row g, 4-7 row g + 8
          float r[D / 8];
#pragma unroll
          for (int q = 0; q < D / 64; ++q) {
#pragma unroll
            for (int nb = 0; nb < 4; ++nb) {
              const float w = nb & 1 ? kTwo24 / 16.f : kTwo24;
              r[8 * q + nb] = fmaf(fmaf(o[ht][4 * q + nb][e], w, base), vinv, z[ht][e]);
              r[8 * q + 4 + nb] = fmaf(fmaf(o[ht][4 * q + nb][2 + e], w, base), vinv, z[ht][e]);
            }
          }
          const int hr = ht * 8 + 2 * t + e, hh = h0 + hr;
          if (!whole) {
            float4* dst = reinterpret_cast<float4*>(piece + hr * D + g * (D / 8));
#pragma unroll
            for (int q = 0; q < D / 32; ++q) dst[q] = make_float4(r[4 * q], r[4 * q + 1], r[4 * q + 2], r[4 * q + 3]);
            if (g == 0) {
              piece[kRows * D + 2 * hr] = fresh ? -INFINITY : -nref[ht][e];
              piece[kRows * D + 2 * hr + 1] = l[ht][e];
            }
          } else if (hh < p.group) {
            const float inv = l[ht][e] == 0.f ? 0.f : 1.f / l[ht][e];
            T* dst = reinterpret_cast<T*>(p.out) + b * p.osb + (kvh * p.group + hh) * p.osh + g * (D / 8);
#pragma unroll
            for (int q = 0; q < D / 64; ++q) {
              uint4 v;
              v.x = pack2<T>(r[8 * q] * inv, r[8 * q + 1] * inv);
              v.y = pack2<T>(r[8 * q + 2] * inv, r[8 * q + 3] * inv);
              v.z = pack2<T>(r[8 * q + 4] * inv, r[8 * q + 5] * inv);
              v.w = pack2<T>(r[8 * q + 6] * inv, r[8 * q + 7] * inv);
              reinterpret_cast<uint4*>(dst)[q] = v;
            }
          }
        }
      }
    }
  }


  // ---- join the pieces of this CTA ----------------------------------------------
  // Piece slot s = 2 warp + (0 | 1); slots are in item order, so the pieces of
  // one sequence are consecutive (with empty slots between).  First the
  // weights, a lane per slot and a warp per q head, then the outputs, a group
  // of threads per sequence.
  __syncthreads();
  const int my_grp = lane < 2 * kW ? s_grp[lane] : -1;
  const int my_b = my_grp >= 0 ? s_seq[lane] : 0;
  const uint32_t used = __ballot_sync(0xffffffffu, my_grp >= 0);
  const uint32_t below = used & ((1u << lane) - 1u);
  const int prev = below ? 31 - __clz(below) : lane;
  const int prev_grp = __shfl_sync(0xffffffffu, my_grp, prev), prev_b = __shfl_sync(0xffffffffu, my_b, prev);
  const bool same = below != 0 && prev_grp == my_grp && prev_b == my_b;
  const uint32_t leaders = __ballot_sync(0xffffffffu, my_grp >= 0 && !same);
  const uint32_t upto = leaders & ((2u << lane) - 1u);
  const int lead = upto ? 31 - __clz(upto) : 0;                // first slot of the lane's run
  const uint32_t after = leaders & ~((2u << lane) - 1u);
  const int last = after ? __ffs(after) - 2 : 31;              // its last slot (maybe an empty one)
  for (int hr = warp; hr < kRows; hr += kW) {
    float2 ml = make_float2(-INFINITY, 0.f);
    if (my_grp >= 0) ml = *reinterpret_cast<const float2*>(pieces + lane * G::kPartFloats + kRows * D + 2 * hr);
    float mx = ml.x;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const float v = __shfl_up_sync(0xffffffffu, mx, d);
      if (lane - d >= lead) mx = fmaxf(mx, v);
    }
    mx = __shfl_sync(0xffffffffu, mx, last);
    const float w = my_grp >= 0 ? ex2_approx(ml.x - (mx == -INFINITY ? 0.f : mx)) : 0.f;
    float sum = ml.y * w;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const float v = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane - d >= lead) sum += v;
    }
    sum = __shfl_sync(0xffffffffu, sum, last);
    if (lane < 2 * kW) {
      s_w[hr * 2 * kW + lane] = w;
      s_ml[hr * 2 * kW + lane] = make_float2(mx, sum);
    }
  }
  // extent of the lane's sequence in items; what it is cut by
  const int u_a = my_grp >= 0 ? my_grp * n_seq + pre[my_b] : 0;
  const int u_e = my_grp >= 0 ? my_grp * n_seq + pre[my_b + 1] : 0;
  const bool cut_a = u_a < cta_a, cut_e = u_e > cta_e;
  if (warp == kW - 1) {
    // the sequence that begins here and runs past the end of the CTA, if any
    const uint32_t tail = __ballot_sync(0xffffffffu, my_grp >= 0 && cut_e && !cut_a);
    Cut c{0, 0, 0, 0};
    if (tail) {
      const int src = __ffs(tail) - 1;
      const int end = __shfl_sync(0xffffffffu, u_e, src);
      c.grp = __shfl_sync(0xffffffffu, my_grp, src);
      c.b = __shfl_sync(0xffffffffu, my_b, src);
      c.c1 = blockIdx.x;
      for (int c0 = blockIdx.x + 1; c0 < act; c0 += 32) {  // CTAs that start before its end
        const bool in = c0 + lane < act && deal.start((c0 + lane) * kW) < end;
        const int n = __popc(__ballot_sync(0xffffffffu, in));
        c.c1 += n;
        if (n < 32) break;
      }
    }
    if (lane == 0) cuts[blockIdx.x] = c;
  }
  __syncthreads();
  // a group of kRows D / 4 threads per run, four elements a thread
  constexpr int kGroup = kRows * D / 4, kGroups = G::kThreads >= kGroup ? G::kThreads / kGroup : 1;
  const int my_group = kGroups == 1 ? 0 : tid / kGroup;
  uint32_t runs = leaders;
  for (int k = 0; runs; runs &= runs - 1, ++k) {
    const int r0s = __ffs(runs) - 1;
    const uint32_t later = runs & (runs - 1);
    const uint32_t run = used & (later ? (1u << (__ffs(later) - 1)) - 1u : ~0u) & ~((1u << r0s) - 1u);
    const int rg = __shfl_sync(0xffffffffu, my_grp, r0s), rb = __shfl_sync(0xffffffffu, my_b, r0s);
    const bool ca = __shfl_sync(0xffffffffu, cut_a, r0s), ce = __shfl_sync(0xffffffffu, cut_e, r0s);
    if (my_group >= kGroups || k % kGroups != my_group) continue;  // warp-uniform: a group is whole warps
    const int kvh = hgroups == 1 ? rg : rg / hgroups, h0 = (rg - kvh * hgroups) * kRows;
    for (int e = kGroups == 1 ? tid : tid - my_group * kGroup; e < kGroup; e += kGroups == 1 ? G::kThreads : kGroup) {
      const int hr = e / (D / 4), d = 4 * (e - hr * (D / 4));
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      for (uint32_t r = run; r; r &= r - 1) {
        const int sl = __ffs(r) - 1;
        const float w = s_w[hr * 2 * kW + sl];
        const float4 v = *reinterpret_cast<const float4*>(pieces + sl * G::kPartFloats + 4 * e);
        acc.x = fmaf(v.x, w, acc.x);
        acc.y = fmaf(v.y, w, acc.y);
        acc.z = fmaf(v.z, w, acc.z);
        acc.w = fmaf(v.w, w, acc.w);
      }
      const float2 ml = s_ml[hr * 2 * kW + r0s];
      if (!ca && !ce) {
        if (h0 + hr < p.group) {
          const float inv = ml.y == 0.f ? 0.f : 1.f / ml.y;
          uint2 v;
          v.x = pack2<T>(acc.x * inv, acc.y * inv);
          v.y = pack2<T>(acc.z * inv, acc.w * inv);
          *reinterpret_cast<uint2*>(reinterpret_cast<T*>(p.out) + rb * p.osb + (kvh * p.group + h0 + hr) * p.osh + d) = v;
        }
      } else {
        // cut at the CTA's start (slot 0) or only at its end (slot 1)
        float* dst = part + static_cast<int64_t>(2 * blockIdx.x + (ca ? 0 : 1)) * G::kPartFloats;
        *reinterpret_cast<float4*>(dst + 4 * e) = acc;
        if (d == 0) *reinterpret_cast<float2*>(dst + kRows * D + 2 * hr) = ml;
      }
    }
  }
}

// Joins the partials of the sequence that CTA blockIdx.x of the decode left
// cut at its end: kRows x kSplit warps, warp (row, k) takes every kSplit-th
// partial of q head ``row``, and the kSplit sums meet in shared memory.
constexpr int kCombineWarps = 32;

template <typename T, int D, int HT>
__global__ void __launch_bounds__(kCombineWarps * 32) int4_combine_kernel(const Int4DecodeParams p) {
  using G = Geo<D, HT>;
  constexpr int kRows = G::kRows, kSplit = kCombineWarps / kRows;
  __shared__ float s_acc[kCombineWarps][D];
  __shared__ float2 s_ml[kCombineWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, hr = warp % kRows, k = warp / kRows;
  const int hgroups = (p.group + kRows - 1) / kRows;
  const int c0 = blockIdx.x;
  pdl_wait();
  pdl_launch_dependents();
  const int4 cut = __ldcg(reinterpret_cast<const int4*>(p.part) + c0);
  const int grp = cut.x, b = cut.y, np = cut.z - c0 + 1;  // c0's own and those of the CTAs after it
  if (cut.z <= c0) return;
  const float* part = p.part + kMaxCtas * (sizeof(Cut) / sizeof(float));
  auto piece_of = [&](int i) { return part + static_cast<int64_t>(2 * (c0 + i) + (i == 0 ? 1 : 0)) * G::kPartFloats; };
  float mx = -INFINITY, ll = 0.f, acc[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i) acc[i] = 0.f;
  constexpr int kBatch = 8;
  for (int i0 = k; i0 < np; i0 += kSplit * kBatch) {
    float2 ml[kBatch];
    float v[kBatch][D / 32];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int i = i0 + j * kSplit;
      ml[j] = make_float2(-INFINITY, 0.f);
      if (i < np) {
        const float* pc = piece_of(i);
        ml[j] = __ldcg(reinterpret_cast<const float2*>(pc + kRows * D + 2 * hr));
#pragma unroll
        for (int q = 0; q < D / 32; ++q) v[j][q] = __ldcg(pc + hr * D + lane + 32 * q);
      } else {
#pragma unroll
        for (int q = 0; q < D / 32; ++q) v[j][q] = 0.f;
      }
    }
    float mn = mx;
#pragma unroll
    for (int j = 0; j < kBatch; ++j) mn = fmaxf(mn, ml[j].x);
    const float mu = mn == -INFINITY ? 0.f : mn;
    const float al = ex2_approx(mx - mu);  // 0 at first
    mx = mn;
    ll *= al;
#pragma unroll
    for (int q = 0; q < D / 32; ++q) acc[q] *= al;
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const float w = ex2_approx(ml[j].x - mu);
      ll = fmaf(ml[j].y, w, ll);
#pragma unroll
      for (int q = 0; q < D / 32; ++q) acc[q] = fmaf(v[j][q], w, acc[q]);
    }
  }
#pragma unroll
  for (int q = 0; q < D / 32; ++q) s_acc[warp][lane + 32 * q] = acc[q];
  if (lane == 0) s_ml[warp] = make_float2(mx, ll);
  __syncthreads();
  const int kvh = hgroups == 1 ? grp : grp / hgroups, hh = (grp - kvh * hgroups) * kRows + hr;
  if (k > 0 || hh >= p.group) return;
  float top = -INFINITY;
#pragma unroll
  for (int j = 0; j < kSplit; ++j) top = fmaxf(top, s_ml[j * kRows + hr].x);
  const float mu = top == -INFINITY ? 0.f : top;
  ll = 0.f;
#pragma unroll
  for (int q = 0; q < D / 32; ++q) acc[q] = 0.f;
#pragma unroll
  for (int j = 0; j < kSplit; ++j) {
    const float2 ml = s_ml[j * kRows + hr];
    const float w = ex2_approx(ml.x - mu);
    ll = fmaf(ml.y, w, ll);
#pragma unroll
    for (int q = 0; q < D / 32; ++q) acc[q] = fmaf(s_acc[j * kRows + hr][lane + 32 * q], w, acc[q]);
  }
  T* dst = reinterpret_cast<T*>(p.out) + b * p.osb + (kvh * p.group + hh) * p.osh;
#pragma unroll
  for (int q = 0; q < D / 32; ++q) dst[lane + 32 * q] = Elem<T>::from_float(ll == 0.f ? 0.f : acc[q] / ll);
}

// Upper bound of the items from the host-known longest context.
int64_t max_items(int batch, int hkv, int group, int rows, int max_context) {
  return static_cast<int64_t>(batch) * hkv * ((group + rows - 1) / rows) *
         std::max<int64_t>(1, (static_cast<int64_t>(max_context) + 31) / 32);
}

template <typename T, int D, int HT>
int launch_fast(const Int4DecodeParams& p, cudaStream_t stream, int sms) {
  using G = Geo<D, HT>;
  const size_t smem = G::smem(p.batch);
  const auto kern = int4_decode_kernel<T, D, HT>;
  const auto comb = int4_combine_kernel<T, D, HT>;
  int occ = 0;
  if (!kernel_occupancy(reinterpret_cast<const void*>(kern), G::kThreads, smem, &occ) || occ < 1) return PSB_ERR_CUDA;
  const int64_t items = max_items(p.batch, p.hkv, p.group, G::kRows, p.max_context);
  const int64_t want = (items + G::kWarps - 1) / G::kWarps;
  const int grid = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(want, std::min(sms, kMaxCtas))));
  discard_stale_error();
  cudaError_t e = launch_pdl(kern, dim3(static_cast<unsigned>(grid)), dim3(G::kThreads), smem, stream, p);
  if (e != cudaSuccess) return record_cuda_error(e);
  if (grid > 1) {
    if (!prefer_max_shared(reinterpret_cast<const void*>(comb))) return PSB_ERR_CUDA;
    e = launch_pdl(comb, dim3(static_cast<unsigned>(grid - 1)), dim3(kCombineWarps * 32), 0, stream, p);
    if (e != cudaSuccess) return record_cuda_error(e);
  }
  return check_launch();
}

int head_tiles(int group) { return group <= 8 ? 1 : 2; }

}  // namespace

bool int4_decode_fast_geometry(int dtype, int batch, int hkv, int group, int head_dim, int block_size,
                               int max_context, int num_layers, int64_t num_blocks) {
  const int rows = 8 * head_tiles(group);
  return (dtype == PSB_BF16 || dtype == PSB_F16) && (head_dim == 64 || head_dim == 128) && block_size % 16 == 0 &&
         batch <= kMaxBatch && max_items(batch, hkv, group, rows, max_context) < (int64_t(1) << 31) - 64 &&
         static_cast<int64_t>(num_layers) * num_blocks * hkv * 2 * (block_size / 16) < (int64_t(1) << 31) &&
         static_cast<int64_t>(max_context / 16 + 2) * (block_size / 16) < (int64_t(1) << 32);
}

size_t int4_decode_fast_workspace(int group, int head_dim) {
  return sizeof(Cut) * kMaxCtas + sizeof(float) * 2 * kMaxCtas * static_cast<size_t>(8 * head_tiles(group)) * (head_dim + 2);
}

int int4_decode_fast_launch(const Int4DecodeParams& p_in, int dtype, cudaStream_t s) {
  const int sms = device_sm_count();
  if (sms <= 0) return PSB_ERR_CUDA;
  Int4DecodeParams p = p_in;
  // floor(t / n) of a tile number t < 2^27 by n = block_size / 16 tiles a
  // block, as t ceil(2^32 / n) / 2^32: exact while t (n - 1) < 2^32
  const uint32_t n = static_cast<uint32_t>(p.block_size) / 16;
  p.tile_div = ((uint64_t(1) << 32) + n - 1) / n;
  const bool bf = dtype == PSB_BF16;
  if (head_tiles(p.group) == 1) {
    if (p.head_dim == 64)
      return bf ? launch_fast<__nv_bfloat16, 64, 1>(p, s, sms) : launch_fast<__half, 64, 1>(p, s, sms);
    return bf ? launch_fast<__nv_bfloat16, 128, 1>(p, s, sms) : launch_fast<__half, 128, 1>(p, s, sms);
  }
  if (p.head_dim == 64)
    return bf ? launch_fast<__nv_bfloat16, 64, 2>(p, s, sms) : launch_fast<__half, 64, 2>(p, s, sms);
  return bf ? launch_fast<__nv_bfloat16, 128, 2>(p, s, sms) : launch_fast<__half, 128, 2>(p, s, sms);
}

}  // namespace psb
