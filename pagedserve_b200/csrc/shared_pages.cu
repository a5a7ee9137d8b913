// fork_tables / release_tables / copy_blocks: pages that several rows of the
// table store hold at once.
//
// ``shares`` int32 [2, N]: word x of its first row counts the holders of block x
// beyond the first (0 for a block that one row holds, or none), so blocks that
// are never shared need no bookkeeping and extend_step can hand them out as they
// are; the second row is scratch of release_tables, zero between calls.
//
// fork_tables lets child rows share their parents' whole blocks; of an unfinished
// one, which both will write to, the child gets its own from the free ring, and
// the pair to copy.  release_tables takes rows' blocks away, entry by entry in
// table order: a block that others hold loses one of them, any other goes to the
// ring's tail.  Of a block that one call releases for all its holders, the last
// of those in that order returns it: the order in which a host with a
// counter per block would return them, whatever order the threads come in.
//
// All of it is integers, a few hundred kilobytes at most, and bound by latency: one
// cluster of up to 16 CTAs, by the most that the call can have to do, works it off,
// its phases parted by cluster barriers (every id checked before the first word is
// changed; counts, then ranks).  A call that cannot be carried out whole changes
// nothing, as extend_step and trim_tables.
//
// The work is dealt over the warps in units of up to 256 blocks of one entry, in
// entry and table order, eight blocks a lane whose loads and atomics are in
// flight together; what a phase has read stays in shared memory for the next (where
// it fits; else it is read again).  (One block a thread and a search for its entry
// each time: 28 us for 255 forks of 250 blocks and 70 us for their release; so 14 and
// 21, with units of 128 14 and 28.)  4 forks of 50 blocks: 8 and 10, three or four dependent
// loads and as many barriers.
//
// release: first every item takes one off its block's counter and leaves its
// number, if it is the highest, in the scratch word.  Behind the barrier a counter
// below 0 says that all holders let go; the item whose number stands in the scratch
// word puts the block on the ring, at the tail plus the number of such items before it.
#include <cooperative_groups.h>

#include <algorithm>

#include "common.cuh"
#include "host_util.h"

namespace cg = cooperative_groups;

namespace psb {
namespace {

constexpr int kPageThreads = 512;
constexpr int kPageWarps = kPageThreads / 32;
constexpr int kPageCtas = 16;  // CTAs of the cluster, at most
constexpr int kUnit = 256, kLanes = kUnit / 32;  // blocks of a unit, and of each lane
constexpr size_t kPagesSmem = 200 * 1024;

struct PagesParams {
  int32_t* store;
  int64_t store_stride;
  int32_t store_rows, store_width;
  const int32_t* rows;    // fork: parents; release: rows
  const int32_t* first;   // fork: children; release: held lengths
  const int32_t* second;  // fork: lengths; release: kept lengths
  int32_t batch, block_size, shift;  // block_size is 2^shift, or shift is -1
  int32_t* shares;
  int32_t* ring;
  int32_t* state;
  int32_t ring_size;
  int32_t cache;  // blocks that a CTA has room for in shared memory
  int32_t* copy_src;
  int32_t* copy_dst;
  int32_t* err;
};

__device__ __forceinline__ uint32_t over(const PagesParams& p, uint32_t x) {
  return p.shift >= 0 ? x >> p.shift : x / static_cast<uint32_t>(p.block_size);
}
__device__ __forceinline__ uint32_t blocks_for(const PagesParams& p, uint32_t tokens) {
  return tokens == 0 ? 0 : over(p, tokens - 1) + 1;
}

// Exclusive scan of two counts per thread over the CTA, and their totals.
__device__ __forceinline__ void scan2(int64_t& a, int64_t& b, int64_t& a_total, int64_t& b_total) {
  __shared__ int64_t sums[2][kPageWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t a0 = a, b0 = b;
#pragma unroll 1
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t x = __shfl_up_sync(0xffffffffu, a, o), y = __shfl_up_sync(0xffffffffu, b, o);
    if (lane >= o) {
      a += x;
      b += y;
    }
  }
  if (lane == 31) {
    sums[0][warp] = a;
    sums[1][warp] = b;
  }
  __syncthreads();
  a -= a0;
  b -= b0;
  a_total = b_total = 0;
#pragma unroll 1
  for (int w = 0; w < kPageWarps; ++w) {
    const int64_t x = sums[0][w], y = sums[1][w];
    if (w < warp) {
      a += x;
      b += y;
    }
    a_total += x;
    b_total += y;
  }
}

__device__ __forceinline__ bool mark_row(uint32_t* seen, int32_t row) {
  const uint32_t bit = 1u << (row & 31);
  return (atomicOr(seen + (row >> 5), bit) & bit) != 0;
}
__device__ __forceinline__ bool row_marked(const uint32_t* seen, int32_t row) { return (seen[row >> 5] >> (row & 31)) & 1; }

// The units of a call, and those of a CTA and a warp.
struct Units {
  const int32_t* pre;  // [batch + 1] units before an entry
  const int32_t* len;  // [batch] its blocks
  int32_t batch;
  int32_t cta0, cta1, u0, u1;
  __device__ __forceinline__ void deal(int32_t total) {
    const int64_t n = gridDim.x * kPageWarps, w = blockIdx.x * kPageWarps + (threadIdx.x >> 5);
    cta0 = static_cast<int32_t>(total * static_cast<int64_t>(blockIdx.x) / gridDim.x);
    cta1 = static_cast<int32_t>(total * static_cast<int64_t>(blockIdx.x + 1) / gridDim.x);
    u0 = static_cast<int32_t>(total * w / n);
    u1 = static_cast<int32_t>(total * (w + 1) / n);
  }
  // f(unit, entry, its first block there, blocks) for each unit of the warp
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    if (u0 >= u1) return;
    int lo = 0, hi = batch - 1;  // the last entry with pre <= u0
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (pre[mid] <= u0) lo = mid; else hi = mid - 1;
    }
#pragma unroll 1
    for (int32_t u = u0; u < u1; ++u) {
      while (pre[lo + 1] <= u) ++lo;
      const int32_t j = (u - pre[lo]) * kUnit;
      f(u, lo, j, min(kUnit, len[lo] - j));
    }
  }
};

__device__ __forceinline__ bool refused_before(const PagesParams& p) {
  return p.err != nullptr && (*static_cast<volatile const int32_t*>(p.err) & PSB_DEVERR_REFUSED) != 0;
}

// The OR of the CTAs' words, for every CTA of the cluster; a barrier of all its
// threads, behind which each sees what the others wrote before it (the cluster's
// barrier releases and acquires).  ``words`` [kPageCtas] is not used again by another
// call before a further barrier.
__device__ __forceinline__ int32_t cluster_or(cg::cluster_group& cluster, int32_t* words, int32_t bits) {
  __shared__ int32_t mine;
  if (threadIdx.x == 0) mine = 0;
  __syncthreads();
  if (bits != 0) atomicOr(&mine, bits);
  __syncthreads();
  const int n = static_cast<int>(cluster.num_blocks()), me = static_cast<int>(cluster.block_rank());
  if (static_cast<int>(threadIdx.x) < n) cluster.map_shared_rank(words, threadIdx.x)[me] = mine;
  cluster.sync();
  int32_t all = 0;
  for (int i = 0; i < n; ++i) all |= words[i];
  return all;
}

__global__ void __launch_bounds__(kPageThreads) fork_tables_kernel(const PagesParams p) {
  extern __shared__ int32_t sm[];
  __shared__ int32_t words[kPageCtas];
  cg::cluster_group cluster = cg::this_cluster();
  int32_t* const s_pre = sm;                   // [batch + 1] units before an entry
  int32_t* const s_new = s_pre + p.batch + 1;  // [batch + 1] new blocks before an entry
  int32_t* const s_len = s_new + p.batch + 1;  // [batch] whole blocks of an entry
  uint32_t* const seen = reinterpret_cast<uint32_t*>(s_len + p.batch);  // rows named as children
  int32_t* const cache = reinterpret_cast<int32_t*>(seen + (p.store_rows + 31) / 32);  // the blocks of the CTA's units
  const int tid = threadIdx.x, lane = tid & 31, n_threads = gridDim.x * kPageThreads, at = blockIdx.x * kPageThreads + tid;
  for (int i = tid; i < (p.store_rows + 31) / 32; i += kPageThreads) seen[i] = 0;
  __syncthreads();
  cluster.barrier_arrive();  // (waited for before another CTA's shared memory is written: every CTA has begun)
  pdl_wait();
  pdl_launch_dependents();
  const int32_t head = p.state[0], count = p.state[1];
  int32_t bits = refused_before(p) ? PSB_DEVERR_REFUSED : 0;
  const int per = (p.batch + kPageThreads - 1) / kPageThreads;
  const int begin = min(tid * per, p.batch), end = min(begin + per, p.batch);
  int64_t units = 0, fresh = 0;
#pragma unroll 1
  for (int b = begin; b < end; ++b) {
    const int32_t child = p.first[b], n = p.second[b], parent = p.rows[b];
    int32_t w = 0, f = 0;
    if (child >= 0) {  // (a padding entry takes nothing)
      if (child >= p.store_rows || parent < 0 || parent >= p.store_rows || n < 0 ||
          blocks_for(p, n) > static_cast<uint32_t>(p.store_width)) {
        bits |= PSB_DEVERR_CONTEXT;
      } else {
        if (mark_row(seen, child)) bits |= PSB_DEVERR_ROWS;
        w = static_cast<int32_t>(over(p, n));
        f = static_cast<int32_t>(blocks_for(p, n)) - w;
      }
    }
    s_len[b] = w;
    s_new[b] = f;
    units += (static_cast<int64_t>(w) + kUnit - 1) / kUnit;
    fresh += f;
  }
  int64_t u_total, f_total;
  scan2(units, fresh, u_total, f_total);
#pragma unroll 1
  for (int b = begin; b < end; ++b) {
    const int32_t f = s_new[b], parent = p.rows[b];
    s_pre[b] = static_cast<int32_t>(units);
    s_new[b] = static_cast<int32_t>(fresh);
    units += (static_cast<int64_t>(s_len[b]) + kUnit - 1) / kUnit;
    fresh += f;
    // a row that is forked into in the same call has no pages to give yet
    if (p.first[b] >= 0 && parent >= 0 && parent < p.store_rows && row_marked(seen, parent)) bits |= PSB_DEVERR_ROWS;
  }
  if (tid == 0) {
    s_pre[p.batch] = static_cast<int32_t>(u_total);
    s_new[p.batch] = static_cast<int32_t>(f_total);
  }
  if (head < 0 || head >= p.ring_size || count < 0 || count > p.ring_size || f_total > count || u_total > INT32_MAX / kUnit) bits |= PSB_DEVERR_POOL;
  const bool planned = __syncthreads_or(bits != 0) == 0;
  cluster.barrier_wait();
  Units all_units{s_pre, s_len, p.batch};
  all_units.deal(planned ? static_cast<int32_t>(u_total) : 0);
  const bool cached = (all_units.cta1 - all_units.cta0) <= p.cache / kUnit;
  auto ring_at = [&](int i) -> int32_t {
    int64_t to = static_cast<int64_t>(head) + i;
    if (to >= p.ring_size) to -= p.ring_size;
    return p.ring[to];
  };
  auto outside = [&](int32_t v) { return v < 0 || v >= p.ring_size; };
  // every id that is shared, copied from or taken, before a word is changed
  all_units.each([&](int32_t u, int b, int32_t j, int32_t n) {
    const int32_t* const from = p.store + p.rows[b] * p.store_stride + j;
    int32_t* const keep = cache + (u - all_units.cta0) * kUnit;
    int32_t v[kLanes];
#pragma unroll
    for (int k = 0; k < kLanes; ++k) v[k] = lane + 32 * k < n ? from[lane + 32 * k] : 0;
#pragma unroll
    for (int k = 0; k < kLanes; ++k) {
      if (lane + 32 * k < n && outside(v[k])) bits |= PSB_DEVERR_BLOCK_RANGE;
      if (cached) keep[lane + 32 * k] = v[k];
    }
  });
  int32_t dst0 = -1;  // of the thread's first entry
  if (planned) {
#pragma unroll 1
    for (int b = at; b < p.batch; b += n_threads) {
      int32_t src = -1, dst = -1;
      if (s_new[b + 1] > s_new[b]) {
        src = p.store[p.rows[b] * p.store_stride + over(p, p.second[b])];
        dst = ring_at(s_new[b]);
        if (outside(src) || outside(dst)) bits |= PSB_DEVERR_BLOCK_RANGE;
      }
      p.copy_src[b] = src;
      p.copy_dst[b] = dst;
      if (b == at) dst0 = dst;
    }
  }
  const int32_t all = cluster_or(cluster, words, bits);
  if (all != 0) {
    if (at == 0 && (all & PSB_DEVERR_REFUSED) == 0) flag_error(p.err, all | PSB_DEVERR_REFUSED);
    for (int b = at; b < p.batch; b += n_threads) p.copy_src[b] = p.copy_dst[b] = -1;
    return;
  }
  all_units.each([&](int32_t u, int b, int32_t j, int32_t n) {
    int32_t* const to = p.store + p.first[b] * p.store_stride + j;
    const int32_t* const from = cached ? cache + (u - all_units.cta0) * kUnit : p.store + p.rows[b] * p.store_stride + j;
    int32_t v[kLanes];
#pragma unroll
    for (int k = 0; k < kLanes; ++k) v[k] = lane + 32 * k < n ? from[lane + 32 * k] : 0;
#pragma unroll
    for (int k = 0; k < kLanes; ++k) {
      if (lane + 32 * k >= n) continue;
      to[lane + 32 * k] = v[k];
      atomicAdd(p.shares + v[k], 1);
    }
  });
#pragma unroll 1
  for (int b = at; b < p.batch; b += n_threads)
    if (s_new[b + 1] > s_new[b])
      p.store[p.first[b] * p.store_stride + over(p, p.second[b])] = b == at ? dst0 : p.copy_dst[b];
  if (at == 0) {  // (every CTA read these before the barrier)
    int64_t to = static_cast<int64_t>(head) + f_total;
    if (to >= p.ring_size) to -= p.ring_size;
    p.state[0] = static_cast<int32_t>(to);
    p.state[1] = count - static_cast<int32_t>(f_total);
  }
}

__global__ void __launch_bounds__(kPageThreads) release_tables_kernel(const PagesParams p) {
  extern __shared__ int32_t sm[];
  __shared__ int32_t words[kPageCtas], late[kPageCtas], freed_of[kPageCtas];
  __shared__ int32_t warp_sums[kPageWarps];
  cg::cluster_group cluster = cg::this_cluster();
  int32_t* const s_pre = sm;                   // [batch + 1] units before an entry
  int32_t* const s_len = s_pre + p.batch + 1;  // [batch] blocks that it releases
  uint32_t* const seen = reinterpret_cast<uint32_t*>(s_len + p.batch);
  int32_t* const cache = reinterpret_cast<int32_t*>(seen + (p.store_rows + 31) / 32);  // the blocks of the CTA's units
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n_threads = gridDim.x * kPageThreads, at = blockIdx.x * kPageThreads + tid;
  for (int i = tid; i < (p.store_rows + 31) / 32; i += kPageThreads) seen[i] = 0;
  __syncthreads();
  cluster.barrier_arrive();  // (waited for before another CTA's shared memory is written: every CTA has begun)
  pdl_wait();
  pdl_launch_dependents();
  const int32_t head = p.state[0], count = p.state[1];
  int32_t bits = refused_before(p) ? PSB_DEVERR_REFUSED : 0;
  const int per = (p.batch + kPageThreads - 1) / kPageThreads;
  const int begin = min(tid * per, p.batch), end = min(begin + per, p.batch);
  int64_t units = 0, parts = 0;  // parts: entries that keep a part of a block
#pragma unroll 1
  for (int b = begin; b < end; ++b) {
    const int32_t row = p.rows[b], held = p.first[b], keep = p.second[b];
    int32_t less = 0;
    if (row >= 0) {
      const uint32_t have = blocks_for(p, max(held, 0));
      if (row >= p.store_rows || keep < 0 || keep > held || have > static_cast<uint32_t>(p.store_width)) {
        bits |= PSB_DEVERR_CONTEXT;
      } else {
        if (mark_row(seen, row)) bits |= PSB_DEVERR_ROWS;
        less = static_cast<int32_t>(have - blocks_for(p, keep));
        parts += keep < held && over(p, keep) * static_cast<uint32_t>(p.block_size) != static_cast<uint32_t>(keep);
      }
    }
    s_len[b] = less;
    units += (static_cast<int64_t>(less) + kUnit - 1) / kUnit;
  }
  int64_t u_total, parts_total;
  scan2(units, parts, u_total, parts_total);
#pragma unroll 1
  for (int b = begin; b < end; ++b) {
    s_pre[b] = static_cast<int32_t>(units);
    units += (static_cast<int64_t>(s_len[b]) + kUnit - 1) / kUnit;
  }
  if (tid == 0) s_pre[p.batch] = static_cast<int32_t>(u_total);
  if (head < 0 || head >= p.ring_size || count < 0 || count > p.ring_size || u_total > INT32_MAX / kUnit) bits |= PSB_DEVERR_POOL;
  const bool planned = __syncthreads_or(bits != 0) == 0;
  cluster.barrier_wait();
  Units all_units{s_pre, s_len, p.batch};
  all_units.deal(planned ? static_cast<int32_t>(u_total) : 0);
  const bool cached = (all_units.cta1 - all_units.cta0) <= p.cache / kUnit;
  int32_t* const last = p.shares + p.ring_size;
  auto entries = [&](int b, int32_t j) { return p.store + p.rows[b] * p.store_stride + blocks_for(p, p.second[b]) + j; };
  // where a unit's blocks are between the phases: in the tables themselves if not in shared memory
  auto kept = [&](int32_t u, int b, int32_t j) { return cached ? cache + (u - all_units.cta0) * kUnit : entries(b, j); };
  all_units.each([&](int32_t u, int b, int32_t j, int32_t n) {
    const int32_t* const from = entries(b, j);
    int32_t* const keep = cache + (u - all_units.cta0) * kUnit;
    int32_t v[kLanes];
#pragma unroll
    for (int k = 0; k < kLanes; ++k) v[k] = lane + 32 * k < n ? from[lane + 32 * k] : 0;
#pragma unroll
    for (int k = 0; k < kLanes; ++k) {
      if (lane + 32 * k >= n) continue;
      if (cached) keep[lane + 32 * k] = v[k];
      if (v[k] < 0 || v[k] >= p.ring_size) {
        bits |= PSB_DEVERR_BLOCK_RANGE;
      } else {
        atomicSub(p.shares + v[k], 1);
        atomicMax(last + v[k], u * kUnit + lane + 32 * k + 1);
      }
    }
  });
  int32_t all = cluster_or(cluster, words, bits);
  if (all == 0 && parts_total > 0) {
    // a block that is kept in part will be written to: nobody else may hold it then
    bits = 0;
#pragma unroll 1
    for (int b = at; b < p.batch; b += n_threads) {
      const int32_t keep = p.second[b];
      const uint32_t j = p.rows[b] < 0 ? 0 : over(p, keep);
      if (p.rows[b] >= 0 && keep < p.first[b] && j * static_cast<uint32_t>(p.block_size) != static_cast<uint32_t>(keep)) {
        const int32_t v = p.store[p.rows[b] * p.store_stride + j];
        if (v < 0 || v >= p.ring_size) bits |= PSB_DEVERR_BLOCK_RANGE;
        else if (__ldcg(p.shares + v) > 0) bits |= PSB_DEVERR_SHARED;
      }
    }
    all = cluster_or(cluster, late, bits);
  }
  // What was counted is put back; ``marked``: blocks that do not go to the ring stand as their complement.
  auto put_back = [&](bool marked) {
    all_units.each([&](int32_t u, int b, int32_t j, int32_t n) {
      const int32_t* const from = kept(u, b, j);
      int32_t* const entry = entries(b, j);
#pragma unroll 1
      for (int i = lane; i < n; i += 32) {
        int32_t v = from[i];
        if (marked && v < 0) v = ~v;
        if (marked && !cached) entry[i] = v;
        if (v >= 0 && v < p.ring_size) {
          atomicAdd(p.shares + v, 1);
          last[v] = 0;
        }
      }
    });
  };
  if (all != 0) {
    put_back(false);
    if (at == 0 && (all & PSB_DEVERR_REFUSED) == 0) flag_error(p.err, all);
    return;
  }
  // Which blocks go to the ring; the scratch words are zero again behind it (a block's
  // other items see their number there neither before nor after).
  int mine = 0;
  bool less = false;  // a block was released more often than it was held
  all_units.each([&](int32_t u, int b, int32_t j, int32_t n) {
    int32_t* const slot = kept(u, b, j);
    int32_t v[kLanes], top[kLanes], left[kLanes];
#pragma unroll
    for (int k = 0; k < kLanes; ++k) v[k] = lane + 32 * k < n ? slot[lane + 32 * k] : 0;
#pragma unroll
    for (int k = 0; k < kLanes; ++k) {
      top[k] = left[k] = 0;
      if (lane + 32 * k >= n) continue;
      top[k] = __ldcg(last + v[k]);
      left[k] = __ldcg(p.shares + v[k]);
    }
#pragma unroll
    for (int k = 0; k < kLanes; ++k) {
      if (lane + 32 * k >= n) continue;
      const bool newest = top[k] == u * kUnit + lane + 32 * k + 1;
      if (newest) last[v[k]] = 0;
      less = less || left[k] < -1;
      const bool out = newest && left[k] < 0;
      slot[lane + 32 * k] = out ? v[k] : ~v[k];
      mine += out;
    }
  });
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  if (lane == 0) warp_sums[warp] = mine;
  less = __syncthreads_or(less) != 0;
  if (tid < static_cast<int>(cluster.num_blocks())) {
    int sum = 0;
    for (int w = 0; w < kPageWarps; ++w) sum += warp_sums[w];
    cluster.map_shared_rank(freed_of, tid)[cluster.block_rank()] = less ? -1 : sum;
  }
  cluster.sync();
  int before = 0, freed = 0;
  for (int c = 0; c < static_cast<int>(cluster.num_blocks()); ++c) {
    less = less || freed_of[c] < 0;
    if (c < static_cast<int>(cluster.block_rank())) before += freed_of[c];
    freed += freed_of[c];
  }
  for (int w = 0; w < warp; ++w) before += warp_sums[w];
  if (less || count + freed > p.ring_size) {  // or more blocks than the pool has: the list, the counts or a table are not what they should be
    put_back(true);
    if (at == 0) flag_error(p.err, PSB_DEVERR_POOL);
    return;
  }
  all_units.each([&](int32_t u, int b, int32_t j, int32_t n) {
    const int32_t* const from = kept(u, b, j);
    int32_t* const entry = entries(b, j);
    int32_t v[kLanes];
#pragma unroll
    for (int k = 0; k < kLanes; ++k) v[k] = lane + 32 * k < n ? from[lane + 32 * k] : -1;
#pragma unroll
    for (int k = 0; k < kLanes; ++k) {
      const uint32_t mask = __ballot_sync(0xffffffffu, v[k] >= 0);
      if (lane + 32 * k < n) entry[lane + 32 * k] = 0;
      if (v[k] >= 0) {
        int64_t to = static_cast<int64_t>(head) + count + before + __popc(mask & ((1u << lane) - 1));  // below two rings
        if (to >= p.ring_size) to -= p.ring_size;
        p.ring[to] = v[k];
        p.shares[v[k]] = 0;
      }
      before += __popc(mask);
    }
  });
  if (at == 0) p.state[1] = count + freed;
}

// ---------------------------------------------------------------------------
// copies of blocks
// ---------------------------------------------------------------------------
// Pieces of V bytes, kFlight in flight a thread; blockIdx.y is a pool's layer.
constexpr int kCopyThreads = 256, kFlight = 4, kMaxPools = 4;

struct CopyParams {
  char* base[kMaxPools];
  uint32_t pieces[kMaxPools];  // of a block
  const int32_t* src;
  const int32_t* dst;
  int32_t pairs, layers;
  int64_t num_blocks;
  int32_t* err;
};

template <typename V>
__global__ void __launch_bounds__(kCopyThreads) copy_blocks_kernel(const CopyParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const int pool = blockIdx.y / p.layers, layer = blockIdx.y - pool * p.layers;
  const uint32_t pieces = pool == 0 ? p.pieces[0] : pool == 1 ? p.pieces[1] : pool == 2 ? p.pieces[2] : p.pieces[3];
  char* const base = pool == 0 ? p.base[0] : pool == 1 ? p.base[1] : pool == 2 ? p.base[2] : p.base[3];
  V* const rows = reinterpret_cast<V*>(base) + static_cast<int64_t>(layer) * p.num_blocks * pieces;
  const uint32_t total = p.pairs * pieces;  // below 2^31
  const uint32_t step = gridDim.x * kCopyThreads;
  for (uint32_t i0 = blockIdx.x * kCopyThreads + threadIdx.x; i0 < total; i0 += kFlight * step) {
    V v[kFlight];
    V* to[kFlight];
#pragma unroll
    for (int k = 0; k < kFlight; ++k) {
      const uint32_t i = i0 + k * step;
      to[k] = nullptr;
      if (i < total && i >= i0) {
        const uint32_t pair = i / pieces, off = i - pair * pieces;
        const int32_t a = __ldg(p.src + pair), b = __ldg(p.dst + pair);
        if (a >= 0 && b >= 0) {
          if (a >= p.num_blocks || b >= p.num_blocks) {
            if (off == 0) flag_error(p.err, PSB_DEVERR_BLOCK_RANGE);
          } else {
            v[k] = rows[static_cast<int64_t>(a) * pieces + off];
            to[k] = rows + static_cast<int64_t>(b) * pieces + off;
          }
        }
      }
    }
#pragma unroll
    for (int k = 0; k < kFlight; ++k)
      if (to[k] != nullptr) *to[k] = v[k];
  }
}

int32_t block_shift(int32_t block_size) {
  if ((block_size & (block_size - 1)) != 0) return -1;
  int32_t s = 0;
  while ((1 << s) < block_size) ++s;
  return s;
}

// ``arrays``: of the batch's length and one.
int launch_pages(void (*kern)(PagesParams), PagesParams p, int arrays, cudaStream_t s) {
  const size_t plan = sizeof(int32_t) * (arrays * (static_cast<size_t>(p.batch) + 1) + (static_cast<size_t>(p.store_rows) + 31) / 32);
  if (plan > kPagesSmem) return PSB_ERR_UNSUPPORTED;
  // a unit a warp and more: barriers of few CTAs are cheaper
  const int64_t most = static_cast<int64_t>(p.batch) * ((static_cast<int64_t>(p.store_width) + kUnit - 1) / kUnit);
  int ctas = 1;
  const int limit = plan < kPagesSmem / 2 ? kPageCtas : 8;  // (16 with an SM each is more than a GPC may have)
  while (ctas < limit && most > static_cast<int64_t>(ctas) * kPageWarps) ctas *= 2;
  const size_t want = static_cast<size_t>(most / ctas + 1) * kUnit * sizeof(int32_t);
  const size_t room = std::min((want + 4095) / 4096 * 4096, plan < kPagesSmem / 2 ? (kPagesSmem / 2 - plan) / 4096 * 4096 : 0);
  p.cache = static_cast<int32_t>(room / sizeof(int32_t));
  const size_t smem = plan + room;
  int occ = 0;
  if (!kernel_occupancy(reinterpret_cast<const void*>(kern), kPageThreads, smem, &occ)) return PSB_ERR_CUDA;
  if (ctas > 8) {  // beyond the portable limit
    const cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void*>(kern), cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return record_cuda_error(e);
  }
  discard_stale_error();
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ctas;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kPageThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
  if (e != cudaSuccess) return record_cuda_error(e);
  return check_launch();
}

bool bad_store(const int32_t* store, int64_t stride, int32_t rows, int32_t width, int32_t batch, int32_t block_size, int32_t num_blocks) {
  return batch < 0 || block_size <= 0 || rows <= 0 || width <= 0 || stride < width || num_blocks <= 0 || (batch > 0 && !store);
}

}  // namespace
}  // namespace psb

using namespace psb;

extern "C" int psb_fork_tables(int32_t* table_store, int64_t store_stride, int32_t store_rows, int32_t store_width,
                               const int32_t* parent_rows, const int32_t* child_rows, const int32_t* lens, int32_t batch,
                               int32_t* shares, int32_t* free_blocks, int32_t num_blocks, int32_t* free_state,
                               int32_t block_size, int32_t* copy_src, int32_t* copy_dst, int32_t* error_flag,
                               psb_stream_t stream) {
  if (bad_store(table_store, store_stride, store_rows, store_width, batch, block_size, num_blocks)) return PSB_ERR_INVALID;
  if (batch == 0) return PSB_OK;
  if (!parent_rows || !child_rows || !lens || !shares || !free_blocks || !free_state || !copy_src || !copy_dst) return PSB_ERR_INVALID;
  PagesParams p{};
  p.store = table_store;
  p.store_stride = store_stride;
  p.store_rows = store_rows;
  p.store_width = store_width;
  p.rows = parent_rows;
  p.first = child_rows;
  p.second = lens;
  p.batch = batch;
  p.block_size = block_size;
  p.shift = block_shift(block_size);
  p.shares = shares;
  p.ring = free_blocks;
  p.state = free_state;
  p.ring_size = num_blocks;
  p.copy_src = copy_src;
  p.copy_dst = copy_dst;
  p.err = error_flag;
  return launch_pages(fork_tables_kernel, p, 3, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int psb_release_tables(int32_t* table_store, int64_t store_stride, int32_t store_rows, int32_t store_width,
                                  const int32_t* req_rows, const int32_t* held_lens, const int32_t* keep_lens, int32_t batch,
                                  int32_t* shares, int32_t* free_blocks, int32_t num_blocks, int32_t* free_state,
                                  int32_t block_size, int32_t* error_flag, psb_stream_t stream) {
  if (bad_store(table_store, store_stride, store_rows, store_width, batch, block_size, num_blocks)) return PSB_ERR_INVALID;
  if (batch == 0) return PSB_OK;
  if (!req_rows || !held_lens || !keep_lens || !shares || !free_blocks || !free_state) return PSB_ERR_INVALID;
  PagesParams p{};
  p.store = table_store;
  p.store_stride = store_stride;
  p.store_rows = store_rows;
  p.store_width = store_width;
  p.rows = req_rows;
  p.first = held_lens;
  p.second = keep_lens;
  p.batch = batch;
  p.block_size = block_size;
  p.shift = block_shift(block_size);
  p.shares = shares;
  p.ring = free_blocks;
  p.state = free_state;
  p.ring_size = num_blocks;
  p.err = error_flag;
  return launch_pages(release_tables_kernel, p, 2, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int psb_copy_blocks(void* const* pools, const int64_t* block_bytes, int32_t num_pools, const int32_t* src,
                               const int32_t* dst, int32_t pairs, int32_t num_layers, int64_t num_blocks, int32_t* error_flag,
                               psb_stream_t stream) {
  if (num_pools < 0 || num_pools > kMaxPools || pairs < 0 || num_layers <= 0 || num_blocks <= 0 || num_blocks > INT32_MAX)
    return PSB_ERR_INVALID;
  if (pairs == 0 || num_pools == 0) return PSB_OK;
  if (!pools || !block_bytes || !src || !dst) return PSB_ERR_INVALID;
  uintptr_t align = 16;
  for (int i = 0; i < num_pools; ++i) {
    if (!pools[i] || block_bytes[i] <= 0) return PSB_ERR_INVALID;
    const uintptr_t x = reinterpret_cast<uintptr_t>(pools[i]) | static_cast<uintptr_t>(block_bytes[i]);
    while (x % align) align /= 2;
  }
  if (align == 8) align = 4;
  if (align == 2) align = 1;
  CopyParams p{};
  int64_t most = 0;
  for (int i = 0; i < num_pools; ++i) {
    p.base[i] = static_cast<char*>(pools[i]);
    const int64_t n = block_bytes[i] / static_cast<int64_t>(align);
    most = std::max(most, n);
    if (n > INT32_MAX) return PSB_ERR_UNSUPPORTED;
    p.pieces[i] = static_cast<uint32_t>(n);
  }
  // (i0 + kFlight steps stay below 2^32)
  if (most * pairs >= (int64_t(1) << 31) || static_cast<int64_t>(num_layers) * num_pools > 65535) return PSB_ERR_UNSUPPORTED;
  p.src = src;
  p.dst = dst;
  p.pairs = pairs;
  p.layers = num_layers;
  p.num_blocks = num_blocks;
  p.err = error_flag;
  const int sms = device_sm_count();
  if (sms <= 0) return PSB_ERR_CUDA;
  const int64_t planes = static_cast<int64_t>(num_layers) * num_pools;
  const int64_t want = (most * pairs + kCopyThreads * kFlight - 1) / (kCopyThreads * kFlight);
  const int64_t cap = std::max<int64_t>(1, 16 * static_cast<int64_t>(sms) / planes);
  const dim3 grid(static_cast<unsigned>(std::min(want, cap)), static_cast<unsigned>(planes));
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const auto kern = align == 16 ? copy_blocks_kernel<uint4> : align == 4 ? copy_blocks_kernel<uint32_t> : copy_blocks_kernel<uint8_t>;
  discard_stale_error();
  const cudaError_t e = launch_pdl(kern, grid, dim3(kCopyThreads), 0, s, p);
  if (e != cudaSuccess) return record_cuda_error(e);
  return check_launch();
}
