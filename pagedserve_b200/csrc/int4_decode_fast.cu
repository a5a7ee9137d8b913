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
// Products.  mma.sync m16n8k16 with the tokens of a 16-token tile as rows of
// S^T = K Q^T (8 q heads are the 8 columns) and head_dim as rows of
// O^T = V^T P^T.  The codes are the A operand in both, so a lane needs no more
// than its own words of a code row: which element of head_dim an index k or a
// row stands for is free as long as q (loaded once) and the output agree.  A
// code becomes a 16-bit operand without conversion instructions:
//   bf16: (w >> 4 i) & 0x000f000f | 0x4300 is 128 + c; for K the 128 is taken
//         out by starting the accumulator at -135.5 sum(q) (4 or 8 products
//         deep, so nothing builds up); for V, whose accumulator runs over the
//         whole context, one paired add makes it c - 8 exactly.
//   f16:  (w >> 8 i) & 0x000f000f is the subnormal c 2^-24 and & 0x00f000f0 is
//         c 2^-20, exactly; products of the two kinds go to accumulators of
//         their own (K) or rows of their own (V), and a product with ones sums
//         the rounded p_t step_t for the -7.5.
// P^T is S^T's accumulator layout transposed: two movmatrix per tile.
//
// What bounds it.  A tile of head_dim 64 is 1152 bytes against 4096 in bf16,
// so the same bytes per second need 3.6 times the instructions of
// paged_decode; at about 150 warp instructions a tile the four schedulers of
// an SM could issue some 30 bytes per clock, close to the SM's share of HBM.
//
// Split.  The tiles of all sequences, in (kv head, sequence, tile) order, are
// dealt evenly over the warps of the grid (one CTA of 16 warps per SM; 8 where
// two head tiles of 128 need the registers).  A warp streams its run through a
// private shared-memory ring (16-byte cp.async, one group per tile).  A
// sequence inside one warp's run is written at once; pieces of one sequence
// within a CTA are joined in shared memory, and only those cut by a CTA
// boundary (at most one per CTA) leave a partial for int4_combine_kernel.
#include <algorithm>

#include "common.cuh"
#include "host_util.h"
#include "int4_attention.h"
#include "int4_cache.cuh"

namespace psb {
namespace {

constexpr int kMaxCtas = 160;       // grid limit (one CTA per SM; B200 has 148)
constexpr int kMaxBatch = 4096;     // sequences whose lengths fit in shared memory
constexpr int kMinTiles = 2;        // tiles per warp below which fewer CTAs take part

template <int D, int HT>
struct Geo {
  static constexpr int kWarps = D * HT > 128 ? 8 : 16;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kStages = D == 64 ? 6 : (HT == 1 ? 3 : 4);
  static constexpr int kRows = 8 * HT;                  // q heads of a tile
  static constexpr int kCodeBytes = 16 * D / 2;         // K (or V) codes of 16 tokens
  static constexpr int kStage = 2 * kCodeBytes + 128;   // K codes, V codes, K params, V params
  static constexpr int kRing = kStages * kStage;
  static constexpr int kPartFloats = kRows * (D + 2);   // one piece: [rows][D] output, [rows][2] max, sum
  static_assert(kRing >= kPartFloats * 4, "a warp's last piece fits its ring");
  static constexpr size_t fixed_smem() { return static_cast<size_t>(kWarps) * (kRing + kPartFloats * 4); }
  static size_t smem(int batch) { return fixed_smem() + sizeof(int32_t) * (2 * static_cast<size_t>(batch) + 1); }
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async16_hint(uint32_t dst, const void* src, uint64_t pol) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "l"(pol)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ uint32_t movmatrix_t(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) { return __byte_perm(a, b, sel); }

// 4-bit codes as 16-bit operands; pair i (0 .. 3) of a word is its nibbles i
// and i + 4.
template <typename T> struct Nib;
template <> struct Nib<__nv_bfloat16> {
  static constexpr bool kSums = false;             // no product with ones
  static constexpr float kKStart = -(128.f + 7.5f);  // per unit of sum(q), in K's accumulator
  static constexpr float kVMid = 0.5f;             // V's codes enter as c - 8
  __device__ static uint32_t k(uint32_t w, int i) { return ((w >> (4 * i)) & 0x000f000fu) | 0x43004300u; }
  __device__ static uint32_t v(uint32_t w, int i) {
    uint32_t d;
    asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(k(w, i)), "r"(0xc308c308u));  // - 136
    return d;
  }
};
template <> struct Nib<__half> {
  static constexpr bool kSums = true;
  static constexpr float kKStart = 0.f;
  static constexpr float kVMid = 0.f;
  __device__ static uint32_t k(uint32_t w, int i) { return (w >> (8 * (i >> 1))) & (i & 1 ? 0x00f000f0u : 0x000f000fu); }
  __device__ static uint32_t v(uint32_t w, int i) { return k(w, i); }
};

template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<__half2*>(&w));
}

template <typename T>
__device__ __forceinline__ float growth_limit();  // log2 of how far a row's max may grow before it is moved
// p stays below 2^8 (bf16) or 2^2 (f16, where p step <= 4 * 8736 must stay finite)
template <> __device__ __forceinline__ float growth_limit<__nv_bfloat16>() { return 8.f; }
template <> __device__ __forceinline__ float growth_limit<__half>() { return 2.f; }

__device__ __forceinline__ int tiles_of(int ctx) { return ctx <= 0 ? 1 : (ctx + 15) >> 4; }

// s_ctx[b] = clamped context, pre[b] = tiles before sequence b, pre[B] = all.
// Called by every thread of a CTA of at most 32 warps.
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
    local += tiles_of(n);
  }
  int incl = local;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) warp_sums[warp] = incl;
  __syncthreads();
  int run = incl - local, total = 0;
  for (int w = 0; w < nthr / 32; ++w) {
    if (w < warp) run += warp_sums[w];
    total += warp_sums[w];
  }
  for (int b = begin; b < end; ++b) {
    pre[b] = run;
    run += tiles_of(s_ctx[b]);
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
  int q, r, parts;
  __device__ Deal(int n, int parts_) : q(n / parts_), r(n % parts_), parts(parts_) {}
  __device__ int start(int w) const { return w * q + (r * w) / parts; }  // r, w < 2560: no overflow
};

// CTAs that take part for n items.
__device__ __forceinline__ int active_ctas(int n, int warps, int grid) {
  return min(grid, max(1, (n + warps * kMinTiles - 1) / (warps * kMinTiles)));
}

template <typename T, int D, int HT>
__global__ void __launch_bounds__(Geo<D, HT>::kThreads, 1) int4_decode_kernel(const Int4DecodeParams p) {
  using G = Geo<D, HT>;
  constexpr int kW = G::kWarps, kS = G::kStages, kRows = G::kRows;
  constexpr int kM = D / 16;   // products per 16 tokens, K and V alike
  constexpr int kWords = D / 32;  // code words per lane: K per row, V per token / 2
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int32_t s_unit[2 * kW];  // the unit of each warp's first and last piece, -1: none
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  uint8_t* ring = smem + warp * G::kRing;
  float* first_piece = reinterpret_cast<float*>(smem + kW * G::kRing) + warp * G::kPartFloats;
  int32_t* pre = reinterpret_cast<int32_t*>(smem + G::fixed_smem());
  int32_t* s_ctx = pre + p.batch + 1;

  const int B = p.batch, BS = p.block_size;
  const int hgroups = (p.group + kRows - 1) / kRows;  // head tiles per kv head
  if (tid < 2 * kW) s_unit[tid] = -1;
  const int n_seq = build_prefix(p, pre, s_ctx, blockIdx.x == 0);
  const int n_items = n_seq * (p.hkv * hgroups);
  const int act = active_ctas(n_items, kW, gridDim.x);
  if (static_cast<int>(blockIdx.x) >= act) return;
  const Deal deal(n_items, act * kW);
  const int gw = blockIdx.x * kW + warp;
  const int my_a = deal.start(gw), my_e = deal.start(gw + 1);

  // ---- 32 items at a time, one per lane ------------------------------------
  // meta: bits 0-4 valid tokens, 5 first item of the warp's share of its unit,
  // 6 last of it, 7 first of the unit, 8 last of the unit
  struct Chunk {
    int beg, n, blk, meta, unit, sub;
  };
  auto build_chunk = [&](int beg) -> Chunk {
    Chunk c{beg, min(32, my_e - beg), -1, 0, 0, 0};
    if (lane < c.n) {
      const int i = beg + lane, grp = i / n_seq, r = i - grp * n_seq;
      const int b = find_seq(pre, B, r), j = r - pre[b];
      const int ctx = s_ctx[b], nt = tiles_of(ctx);
      const int valid = max(0, min(16, ctx - 16 * j));
      c.meta = valid | (j == 0 || i == my_a ? 32 : 0) | (j == nt - 1 || i == my_e - 1 ? 64 : 0) | (j == 0 ? 128 : 0) |
               (j == nt - 1 ? 256 : 0);
      c.unit = grp * B + b;
      const int pos = 16 * j;
      c.sub = pos % BS;
      if (valid > 0) c.blk = __ldg(p.tables + static_cast<int64_t>(b) * p.table_stride + pos / BS);
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
  int slot_meta = 0, slot_unit = 0;  // lane s: of ring stage s (bit 9 of the meta: data was copied)
  const uint32_t ring_u = smem_u32(ring);
  const uint64_t pol = l2_policy_evict_first();
  // Row pi(r) of a tile is the token at index r of the products: chosen so
  // that the lanes of one shared-memory phase read distinct banks - D 64: four
  // K rows of 32 bytes are 0, 1, 2, 3 modulo 4; D 128: two K rows differ in
  // parity; both: a V load's four tokens differ modulo 4.
  auto pi = [](int r) { return (r & 1) ? 4 + (((r >> 1) + (D == 64 ? 2 : 1)) & 3) : r >> 1; };
  // D 128: 16-byte column c of row r is kept at c ^ 2 ((r >> 1) & 1), so that
  // V's 8-byte reads of four tokens spread over all banks
  auto swz = [](int row) { return D == 128 ? ((row >> 1) & 1) << 1 : 0; };
  auto issue_one = [&]() {
    const uint32_t st = issued % kS;
    int blk = __shfl_sync(0xffffffffu, cur.blk, ib);
    int mt = __shfl_sync(0xffffffffu, cur.meta, ib);
    const int unit = __shfl_sync(0xffffffffu, cur.unit, ib);
    const int sub = __shfl_sync(0xffffffffu, cur.sub, ib);
    bool ok = (mt & 31) > 0;
    if (ok && (blk < 0 || blk >= p.num_blocks)) {
      if (lane == 0) flag_error(p.err, PSB_DEVERR_BLOCK_RANGE);
      ok = false;
    }
    if (ok) {
      const int kvh = (unit / B) / hgroups;
      const int64_t krow = int4_row(p.layer_tiles + static_cast<int64_t>(blk) * p.hkv + kvh, 0, sub, BS);
      const uint32_t dst = ring_u + st * G::kStage;
      const uint8_t* ks = p.codes + krow * (D / 2);
      const uint8_t* vs = ks + static_cast<int64_t>(BS) * (D / 2);
#pragma unroll
      for (int i = 0; i < D / 64; ++i) {
        const int ch = lane + 32 * i;  // 16-byte piece of the tile
        uint32_t o = ch * 16;
        if (D == 128) o = (ch >> 2) * 64 + (((ch & 3) ^ swz(ch >> 2)) << 4);
        cp_async16_hint(dst + o, ks + ch * 16, pol);
        cp_async16_hint(dst + G::kCodeBytes + o, vs + ch * 16, pol);
      }
      if (lane < 8) {
        const char* ps = reinterpret_cast<const char*>(p.params) + krow * 4 + (lane >> 2) * (static_cast<int64_t>(BS) * 4);
        cp_async16(dst + 2 * G::kCodeBytes + lane * 16, ps + (lane & 3) * 16);
      }
      mt |= 512;
    }
    cp_async_commit();
    if (lane == static_cast<int>(st)) {
      slot_meta = mt;
      slot_unit = unit;
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

  // Only lengths and tables have been read so far; the pool and q may still be
  // being written by the stream predecessor.
  pdl_wait();
  pdl_launch_dependents();
  while (c_ok && issued < kS) issue_one();

  uint32_t qb[HT][kM][2];         // B fragments of q
  float qs[HT][2];                // sum(q) of heads 2 t, 2 t + 1
  float o[HT][kM][4];             // (element of row g | g + 8) x (head 2 t | 2 t + 1)
  float sp[HT][4];                // sums of the rounded p step (f16)
  float m[HT][2], l[HT][2], z[HT][2];
  int unit = 0;
  bool whole = false;
  int pieces = 0;
  const float sc = p.scale_log2;
  constexpr float kTwo24 = 16777216.f;
  const int row0 = pi(g);         // tokens of rows g and g + 8: row0, 8 + row0

  while (consumed != issued) {
    const uint32_t st = consumed % kS;
    const int mt = __shfl_sync(0xffffffffu, slot_meta, st);
    if (mt & 32) {
      // ---- a unit's first tile: q fragments ---------------------------------
      unit = __shfl_sync(0xffffffffu, slot_unit, st);
      whole = mt & 128;
      const int grp = unit / B, b = unit - grp * B;
      const int kvh = grp / hgroups, h0 = (grp - kvh * hgroups) * kRows;
#pragma unroll
      for (int ht = 0; ht < HT; ++ht) {
        const int hh = h0 + ht * 8 + g;
        const bool live = hh < p.group;
        const T* src = reinterpret_cast<const T*>(p.q) + b * p.qsb + (kvh * p.group + (live ? hh : 0)) * p.qsh + t * (D / 4);
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < kWords; ++w) {
          uint4 x = make_uint4(0, 0, 0, 0);  // 8 elements: one code word's
          if (live) x = *reinterpret_cast<const uint4*>(src + 8 * w);
          const float2 a0 = unpack2<T>(x.x), a1 = unpack2<T>(x.y), a2 = unpack2<T>(x.z), a3 = unpack2<T>(x.w);
          sum += ((a0.x + a0.y) + (a1.x + a1.y)) + ((a2.x + a2.y) + (a3.x + a3.y));
          // elements (i, i + 4) of the word, for products 4 (w / 2) + i
          qb[ht][4 * (w >> 1) + 0][w & 1] = prmt(x.x, x.z, 0x5410);
          qb[ht][4 * (w >> 1) + 1][w & 1] = prmt(x.x, x.z, 0x7632);
          qb[ht][4 * (w >> 1) + 2][w & 1] = prmt(x.y, x.w, 0x5410);
          qb[ht][4 * (w >> 1) + 3][w & 1] = prmt(x.y, x.w, 0x7632);
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        qs[ht][0] = __shfl_sync(0xffffffffu, sum, 8 * t);      // head 2 t is lanes 8 t ..
        qs[ht][1] = __shfl_sync(0xffffffffu, sum, 8 * t + 4);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          m[ht][e] = -INFINITY;
          l[ht][e] = z[ht][e] = 0.f;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) sp[ht][e] = 0.f;
#pragma unroll
        for (int i = 0; i < kM; ++i) o[ht][i][0] = o[ht][i][1] = o[ht][i][2] = o[ht][i][3] = 0.f;
      }
    }
    // the oldest copy is complete once at most the newer ones are pending;
    // near the end of the run fewer are pending than that, so wait for all
    if (issued - consumed == kS) cp_async_wait<kS - 1>(); else cp_async_wait<0>();
    __syncwarp();
    if (mt & 512) {
      const int valid = mt & 31;
      const uint8_t* kt = ring + st * G::kStage;
      const uint8_t* vt = kt + G::kCodeBytes;
      const uint32_t* par = reinterpret_cast<const uint32_t*>(kt + 2 * G::kCodeBytes);
      // ---- S^T = K Q^T ---------------------------------------------------------
      uint32_t kw[2][kWords];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int row = row0 + 8 * r;
        if constexpr (D == 64) {
          const uint2 x = *reinterpret_cast<const uint2*>(kt + row * 32 + t * 8);
          kw[r][0] = x.x;
          kw[r][1] = x.y;
        } else {
          const uint4 x = *reinterpret_cast<const uint4*>(kt + row * 64 + ((t ^ swz(row)) << 4));
          kw[r][0] = x.x;
          kw[r][1] = x.y;
          kw[r][2] = x.z;
          kw[r][3] = x.w;
        }
      }
      float s[HT][4], s1[HT][4];
#pragma unroll
      for (int ht = 0; ht < HT; ++ht) {
        s[ht][0] = s[ht][2] = Nib<T>::kKStart * qs[ht][0];
        s[ht][1] = s[ht][3] = Nib<T>::kKStart * qs[ht][1];
        s1[ht][0] = s1[ht][1] = s1[ht][2] = s1[ht][3] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < kM; ++i) {
        const int w = 2 * (i >> 2), nb = i & 3;
        const uint32_t a0 = Nib<T>::k(kw[0][w], nb), a1 = Nib<T>::k(kw[1][w], nb);
        const uint32_t a2 = Nib<T>::k(kw[0][w + 1], nb), a3 = Nib<T>::k(kw[1][w + 1], nb);
#pragma unroll
        for (int ht = 0; ht < HT; ++ht)
          mma_16816<T>(Nib<T>::kSums && (i & 1) ? s1[ht] : s[ht], a0, a1, a2, a3, qb[ht][i][0], qb[ht][i][1]);
      }
      // ---- scores (log2 scale), probabilities ----------------------------------
      float2 kp[2], vp[2];  // (step, mid) of tokens row0 and 8 + row0
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        kp[r] = unpack2<T>(par[row0 + 8 * r]);
        vp[r] = unpack2<T>(par[16 + row0 + 8 * r]);
      }
      const bool ok0 = row0 < valid, ok1 = row0 + 8 < valid;
      if (valid < 16) {  // rows past the context may hold anything
        if (!ok0) kp[0] = vp[0] = make_float2(0.f, 0.f);
        if (!ok1) kp[1] = vp[1] = make_float2(0.f, 0.f);
      }
      float x[HT][4];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float ks = kp[r].x * sc, km = kp[r].y * sc;
        if (Nib<T>::kSums) {
          km = fmaf(-7.5f, ks, km);
          ks *= kTwo24;
        }
#pragma unroll
        for (int ht = 0; ht < HT; ++ht) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float a = s[ht][2 * r + e];
            if (Nib<T>::kSums) a = fmaf(s1[ht][2 * r + e], 0.0625f, a);
            x[ht][2 * r + e] = fmaf(ks, a, km * qs[ht][e]);
          }
        }
      }
      if (valid < 16) {
#pragma unroll
        for (int ht = 0; ht < HT; ++ht) {
          if (!ok0) x[ht][0] = x[ht][1] = -INFINITY;
          if (!ok1) x[ht][2] = x[ht][3] = -INFINITY;
        }
      }
      // The maximum the exponents refer to moves only when some score is above
      // it by more than the limit: most tiles touch no accumulator.
      bool grow = false;
#pragma unroll
      for (int ht = 0; ht < HT; ++ht) {
#pragma unroll
        for (int e = 0; e < 2; ++e) grow = grow || fmaxf(x[ht][e], x[ht][2 + e]) > m[ht][e] + growth_limit<T>();
      }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int ht = 0; ht < HT; ++ht) {
          float al[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float mx = fmaxf(x[ht][e], x[ht][2 + e]);
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            mx = fmaxf(mx, m[ht][e]);
            al[e] = m[ht][e] == -INFINITY ? 0.f : ex2_approx(m[ht][e] - mx);
            m[ht][e] = mx;
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
          if (Nib<T>::kSums) {
            sp[ht][0] *= al[0];
            sp[ht][1] *= al[1];
          }
        }
      }
      uint32_t pb[HT][2];  // B fragments of P^T
      const float vm0 = fmaf(Nib<T>::kVMid, vp[0].x, vp[0].y), vm1 = fmaf(Nib<T>::kVMid, vp[1].x, vp[1].y);
#pragma unroll
      for (int ht = 0; ht < HT; ++ht) {
        float pr[4];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float mu = m[ht][e] == -INFINITY ? 0.f : m[ht][e];
          pr[e] = ex2_approx(x[ht][e] - mu);
          pr[2 + e] = ex2_approx(x[ht][2 + e] - mu);
          l[ht][e] += pr[e] + pr[2 + e];
          z[ht][e] = fmaf(pr[e], vm0, fmaf(pr[2 + e], vm1, z[ht][e]));
        }
        pb[ht][0] = movmatrix_t(pack2<T>(pr[0] * vp[0].x, pr[1] * vp[0].x));
        pb[ht][1] = movmatrix_t(pack2<T>(pr[2] * vp[1].x, pr[3] * vp[1].x));
      }
      // ---- O^T += V^T P^T --------------------------------------------------------
      uint32_t vw[4][D / 64];  // tokens pi(2 t), pi(2 t + 1) and those plus 8
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = pi(2 * t + (r & 1)) + 8 * (r >> 1);
        if constexpr (D == 64) {
          vw[r][0] = *reinterpret_cast<const uint32_t*>(vt + row * 32 + g * 4);
        } else {
          const uint2 w = *reinterpret_cast<const uint2*>(vt + row * 64 + (((g >> 1) ^ swz(row)) << 4) + (g & 1) * 8);
          vw[r][0] = w.x;
          vw[r][1] = w.y;
        }
      }
#pragma unroll
      for (int q = 0; q < D / 64; ++q) {
        const uint32_t x01 = prmt(vw[0][q], vw[1][q], 0x5410), y01 = prmt(vw[0][q], vw[1][q], 0x7632);
        const uint32_t x23 = prmt(vw[2][q], vw[3][q], 0x5410), y23 = prmt(vw[2][q], vw[3][q], 0x7632);
#pragma unroll
        for (int nb = 0; nb < 4; ++nb) {
          const uint32_t a0 = Nib<T>::v(x01, nb), a1 = Nib<T>::v(y01, nb), a2 = Nib<T>::v(x23, nb),
                         a3 = Nib<T>::v(y23, nb);
#pragma unroll
          for (int ht = 0; ht < HT; ++ht) mma_16816<T>(o[ht][4 * q + nb], a0, a1, a2, a3, pb[ht][0], pb[ht][1]);
        }
      }
      if (Nib<T>::kSums) {
#pragma unroll
        for (int ht = 0; ht < HT; ++ht)
          mma_16816<T>(sp[ht], 0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u, pb[ht][0], pb[ht][1]);
      }
    }
    __syncwarp();
    ++consumed;
    if (c_ok) issue_one();  // refill the stage just freed

    if (mt & 64) {
      // ---- the warp's share of the unit is done --------------------------------
      const int grp = unit / B, b = unit - grp * B;
      const int kvh = grp / hgroups, h0 = (grp - kvh * hgroups) * kRows;
      whole = whole && (mt & 256);
      float* piece = nullptr;
      if (!whole) {
        // the first piece has its own place; the other one ends the run, when
        // the warp's ring is free
        const int k = pieces++;
        piece = k == 0 ? first_piece : reinterpret_cast<float*>(ring);
        if (lane == 0) s_unit[2 * warp + k] = unit;
        if (k == 1) __syncwarp();
      }
#pragma unroll
      for (int ht = 0; ht < HT; ++ht) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float ll = l[ht][e], zz = z[ht][e];
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) {
            ll += __shfl_xor_sync(0xffffffffu, ll, d);
            zz += __shfl_xor_sync(0xffffffffu, zz, d);
          }
          // elements (D / 8) g + 8 q + {0 .. 7}: nibbles 0-3 are row g, 4-7 row g + 8
          float r[D / 8];
#pragma unroll
          for (int q = 0; q < D / 64; ++q) {
#pragma unroll
            for (int nb = 0; nb < 4; ++nb) {
              float a = o[ht][4 * q + nb][e], c = o[ht][4 * q + nb][2 + e];
              if (Nib<T>::kSums) {
                const float w = nb & 1 ? kTwo24 / 16.f : kTwo24;
                a = fmaf(a, w, -7.5f * sp[ht][e]);
                c = fmaf(c, w, -7.5f * sp[ht][e]);
              }
              r[8 * q + nb] = a + zz;
              r[8 * q + 4 + nb] = c + zz;
            }
          }
          const int hr = ht * 8 + 2 * t + e, hh = h0 + hr;
          if (!whole) {
            float4* dst = reinterpret_cast<float4*>(piece + hr * D + g * (D / 8));
#pragma unroll
            for (int q = 0; q < D / 32; ++q) dst[q] = make_float4(r[4 * q], r[4 * q + 1], r[4 * q + 2], r[4 * q + 3]);
            if (g == 0) {
              piece[kRows * D + 2 * hr] = m[ht][e];
              piece[kRows * D + 2 * hr + 1] = ll;
            }
          } else if (hh < p.group) {
            const float inv = ll == 0.f ? 0.f : 1.f / ll;
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
  __syncthreads();
  const int mine = lane < 2 * kW ? s_unit[lane] : -1;
  const uint32_t peers = __match_any_sync(0xffffffffu, mine);
  uint32_t leaders = __ballot_sync(0xffffffffu, mine >= 0 && lane == __ffs(peers) - 1);
  const int cta_a = deal.start(blockIdx.x * kW), cta_e = deal.start((blockIdx.x + 1) * kW);
  for (int k = 0; leaders; ++k) {
    const int lead = __ffs(leaders) - 1;
    leaders &= leaders - 1;
    const uint32_t run = __shfl_sync(0xffffffffu, peers, lead);
    const int u = __shfl_sync(0xffffffffu, mine, lead);
    const int grp = u / B, b = u - grp * B;
    const int u_a = grp * n_seq + pre[b], u_e = grp * n_seq + pre[b + 1];
    const int kvh = grp / hgroups, h0 = (grp - kvh * hgroups) * kRows;
    for (int hr = (warp + kW - (k * kRows) % kW) % kW; hr < kRows; hr += kW) {  // rows over warps, run after run
      auto piece_of = [&](int s) -> const float* {
        return (s & 1) ? reinterpret_cast<const float*>(smem + (s >> 1) * G::kRing)
                       : reinterpret_cast<const float*>(smem + kW * G::kRing) + (s >> 1) * G::kPartFloats;
      };
      float mx = -INFINITY, ll = 0.f, acc[D / 32];
#pragma unroll
      for (int i = 0; i < D / 32; ++i) acc[i] = 0.f;
      for (uint32_t r = run; r; r &= r - 1) mx = fmaxf(mx, piece_of(__ffs(r) - 1)[kRows * D + 2 * hr]);
      const float mu = mx == -INFINITY ? 0.f : mx;
      for (uint32_t r = run; r; r &= r - 1) {
        const float* pc = piece_of(__ffs(r) - 1);
        const float w = ex2_approx(pc[kRows * D + 2 * hr] - mu);
        ll = fmaf(pc[kRows * D + 2 * hr + 1], w, ll);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) acc[i] = fmaf(pc[hr * D + lane + 32 * i], w, acc[i]);
      }
      if (u_a >= cta_a && u_e <= cta_e) {
        if (h0 + hr < p.group) {
          const float inv = ll == 0.f ? 0.f : 1.f / ll;
          T* dst = reinterpret_cast<T*>(p.out) + b * p.osb + (kvh * p.group + h0 + hr) * p.osh;
#pragma unroll
          for (int i = 0; i < D / 32; ++i) dst[lane + 32 * i] = Elem<T>::from_float(acc[i] * inv);
        }
      } else {
        // cut at the CTA's start (slot 0) or only at its end (slot 1)
        float* dst = p.part + static_cast<int64_t>(2 * blockIdx.x + (u_a < cta_a ? 0 : 1)) * G::kPartFloats;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) dst[hr * D + lane + 32 * i] = acc[i];
        if (lane == 0) {
          dst[kRows * D + 2 * hr] = mx;
          dst[kRows * D + 2 * hr + 1] = ll;
        }
      }
    }
  }
}

// Joins the partials of the unit cut by CTA boundary blockIdx.x (the first
// boundary that cuts it; other boundaries of the same unit have nothing to
// do): one warp per q head.  Starts while the decode runs and works out its
// unit from the lengths alone, as the decode dealt them.
template <typename T, int D, int HT>
__global__ void __launch_bounds__(8 * HT * 32) int4_combine_kernel(const Int4DecodeParams p, int decode_grid) {
  using G = Geo<D, HT>;
  extern __shared__ int32_t sm[];
  int32_t* pre = sm;
  int32_t* s_ctx = pre + p.batch + 1;
  const int lane = threadIdx.x & 31, hr = threadIdx.x >> 5, B = p.batch;
  const int hgroups = (p.group + G::kRows - 1) / G::kRows;
  const int n_seq = build_prefix(p, pre, s_ctx, false);
  const int n_items = n_seq * (p.hkv * hgroups);
  const int act = active_ctas(n_items, G::kWarps, decode_grid);
  const int c0 = blockIdx.x;
  pdl_wait();
  pdl_launch_dependents();
  if (c0 + 1 >= act) return;
  const Deal deal(n_items, act * G::kWarps);
  const int cut = deal.start((c0 + 1) * G::kWarps);
  if (cut >= n_items) return;
  const int grp = cut / n_seq, r = cut - grp * n_seq;
  const int b = find_seq(pre, B, r);
  const int u_a = grp * n_seq + pre[b], u_e = grp * n_seq + pre[b + 1];
  if (u_a >= cut || u_a < deal.start(c0 * G::kWarps)) return;  // not cut here, or cut before
  int c1 = c0 + 1;
  while (c1 + 1 < act && deal.start((c1 + 1) * G::kWarps) < u_e) ++c1;
  const int kvh = grp / hgroups, hh = (grp - kvh * hgroups) * G::kRows + hr;
  if (hh >= p.group) return;
  auto piece_of = [&](int c) { return p.part + static_cast<int64_t>(2 * c + (c == c0 ? 1 : 0)) * G::kPartFloats; };
  float mx = -INFINITY, ll = 0.f, acc[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i) acc[i] = 0.f;
  for (int c = c0 + lane; c <= c1; c += 32) mx = fmaxf(mx, __ldcg(piece_of(c) + G::kRows * D + 2 * hr));
#pragma unroll
  for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  const float mu = mx == -INFINITY ? 0.f : mx;
#pragma unroll 4
  for (int c = c0; c <= c1; ++c) {
    const float* pc = piece_of(c);
    const float w = ex2_approx(__ldcg(pc + G::kRows * D + 2 * hr) - mu);
    ll = fmaf(__ldcg(pc + G::kRows * D + 2 * hr + 1), w, ll);
#pragma unroll
    for (int i = 0; i < D / 32; ++i) acc[i] = fmaf(__ldcg(pc + hr * D + lane + 32 * i), w, acc[i]);
  }
  const float inv = ll == 0.f ? 0.f : 1.f / ll;
  T* dst = reinterpret_cast<T*>(p.out) + b * p.osb + (kvh * p.group + hh) * p.osh;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) dst[lane + 32 * i] = Elem<T>::from_float(acc[i] * inv);
}

// Upper bound of the items from the host-known longest context.
int64_t max_items(int batch, int hkv, int group, int rows, int max_context) {
  return static_cast<int64_t>(batch) * hkv * ((group + rows - 1) / rows) *
         std::max<int64_t>(1, (static_cast<int64_t>(max_context) + 15) / 16);
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
  const int64_t want = (items + G::kWarps * kMinTiles - 1) / (G::kWarps * kMinTiles);
  const int grid = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(want, std::min(sms, kMaxCtas))));
  discard_stale_error();
  cudaError_t e = launch_pdl(kern, dim3(static_cast<unsigned>(grid)), dim3(G::kThreads), smem, stream, p);
  if (e != cudaSuccess) return record_cuda_error(e);
  if (grid > 1) {
    if (!prefer_max_shared(reinterpret_cast<const void*>(comb))) return PSB_ERR_CUDA;
    const size_t csmem = sizeof(int32_t) * (2 * static_cast<size_t>(p.batch) + 1);
    e = launch_pdl(comb, dim3(static_cast<unsigned>(grid - 1)), dim3(8 * HT * 32), csmem, stream, p, grid);
    if (e != cudaSuccess) return record_cuda_error(e);
  }
  return check_launch();
}

int head_tiles(int group) { return group <= 8 ? 1 : 2; }

}  // namespace

bool int4_decode_fast_geometry(int dtype, int batch, int hkv, int group, int head_dim, int block_size,
                               int max_context) {
  const int rows = 8 * head_tiles(group);
  return (dtype == PSB_BF16 || dtype == PSB_F16) && (head_dim == 64 || head_dim == 128) && block_size % 16 == 0 &&
         batch <= kMaxBatch && max_items(batch, hkv, group, rows, max_context) < (int64_t(1) << 31) - 64;
}

size_t int4_decode_fast_workspace(int group, int head_dim) {
  return sizeof(float) * 2 * kMaxCtas * static_cast<size_t>(8 * head_tiles(group)) * (head_dim + 2);
}

int int4_decode_fast_launch(const Int4DecodeParams& p, int dtype, cudaStream_t s) {
  const int sms = device_sm_count();
  if (sms <= 0) return PSB_ERR_CUDA;
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
