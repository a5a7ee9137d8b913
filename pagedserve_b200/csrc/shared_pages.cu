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
// cluster of eight CTAs works a call off, its phases parted by cluster barriers
// (every id checked before the first word is changed; counts, then ranks).  A
// call that cannot be carried out whole changes nothing, as extend_step and
// trim_tables.
//
// release: an item is one block of one entry.  First every item takes one off
// its block's counter and leaves its number, if it is the highest, in the
// scratch word.  Behind the barrier a counter of -1 says that all holders let go;
// the item whose number stands in the scratch word puts the block on the
// ring, at the tail plus the number of such items before it.
#include <cooperative_groups.h>

#include <algorithm>

#include "common.cuh"
#include "host_util.h"

namespace cg = cooperative_groups;

namespace psb {
namespace {

constexpr int kPageThreads = 512;
constexpr int kPageWarps = kPageThreads / 32;
constexpr int kPageCtas = 8;  // CTAs of the cluster (the portable limit)

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

// Last b with pre[b] <= i (pre ascending, pre[0] = 0).
__device__ __forceinline__ int entry_of(const int32_t* pre, int batch, int i) {
  int lo = 0, hi = batch - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (pre[mid] <= i) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ bool refused_before(const PagesParams& p) {
  return p.err != nullptr && (*static_cast<volatile const int32_t*>(p.err) & PSB_DEVERR_REFUSED) != 0;
}

// The OR of the CTAs' words, for every CTA of the cluster; a barrier of all its
// threads, behind which each sees what the others wrote before it.  ``words``
// [kPageCtas] is not used again by another call before a further barrier.
__device__ __forceinline__ int32_t cluster_or(cg::cluster_group& cluster, int32_t* words, int32_t bits) {
  __shared__ int32_t mine;
  if (threadIdx.x == 0) mine = 0;
  __syncthreads();
  if (bits != 0) atomicOr(&mine, bits);
  __threadfence();
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
  int32_t* const s_pre = sm;                   // [batch + 1] whole blocks before an entry
  int32_t* const s_new = s_pre + p.batch + 1;  // [batch + 1] new blocks before an entry
  uint32_t* const seen = reinterpret_cast<uint32_t*>(s_new + p.batch + 1);  // rows named as children
  const int tid = threadIdx.x, n_threads = gridDim.x * kPageThreads, at = blockIdx.x * kPageThreads + tid;
  for (int i = tid; i < (p.store_rows + 31) / 32; i += kPageThreads) seen[i] = 0;
  cluster.sync();  // every CTA has begun: its shared memory may be written
  pdl_wait();
  const int32_t head = p.state[0], count = p.state[1];
  int32_t bits = 0;
  __syncthreads();
  const int per = (p.batch + kPageThreads - 1) / kPageThreads;
  const int begin = min(tid * per, p.batch), end = min(begin + per, p.batch);
  int64_t whole = 0, fresh = 0;
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
    s_pre[b] = w;
    s_new[b] = f;
    whole += w;
    fresh += f;
  }
  int64_t w_total, f_total;
  scan2(whole, fresh, w_total, f_total);
#pragma unroll 1
  for (int b = begin; b < end; ++b) {
    const int32_t w = s_pre[b], f = s_new[b], parent = p.rows[b];
    s_pre[b] = static_cast<int32_t>(whole);
    s_new[b] = static_cast<int32_t>(fresh);
    whole += w;
    fresh += f;
    // a row that is forked into in the same call has no pages to give yet
    if (p.first[b] >= 0 && parent >= 0 && parent < p.store_rows && row_marked(seen, parent)) bits |= PSB_DEVERR_ROWS;
  }
  if (tid == 0) {
    s_pre[p.batch] = static_cast<int32_t>(w_total);
    s_new[p.batch] = static_cast<int32_t>(f_total);
  }
  if (head < 0 || head >= p.ring_size || count < 0 || count > p.ring_size || f_total > count || w_total > INT32_MAX) bits |= PSB_DEVERR_POOL;
  const bool planned = __syncthreads_or(bits != 0) == 0;
  const int items = planned ? static_cast<int>(w_total) : 0;
  auto ring_at = [&](int i) -> int32_t {
    int64_t to = static_cast<int64_t>(head) + i;
    if (to >= p.ring_size) to -= p.ring_size;
    return p.ring[to];
  };
  auto outside = [&](int32_t v) { return v < 0 || v >= p.ring_size; };
  // every id that is shared, copied from or taken, before a word is changed
#pragma unroll 1
  for (int i = at; i < items; i += n_threads) {
    const int b = entry_of(s_pre, p.batch, i);
    if (outside(p.store[p.rows[b] * p.store_stride + (i - s_pre[b])])) bits |= PSB_DEVERR_BLOCK_RANGE;
  }
  if (planned) {
#pragma unroll 1
    for (int b = at; b < p.batch; b += n_threads)
      if (s_new[b + 1] > s_new[b] &&
          (outside(p.store[p.rows[b] * p.store_stride + over(p, p.second[b])]) || outside(ring_at(s_new[b]))))
        bits |= PSB_DEVERR_BLOCK_RANGE;
  }
  if (refused_before(p)) bits |= PSB_DEVERR_REFUSED;
  const int32_t all = cluster_or(cluster, words, bits);
  if (all != 0) {
    if (at == 0 && (all & PSB_DEVERR_REFUSED) == 0) flag_error(p.err, all | PSB_DEVERR_REFUSED);
    for (int b = at; b < p.batch; b += n_threads) p.copy_src[b] = p.copy_dst[b] = -1;
    return;
  }
#pragma unroll 1
  for (int i = at; i < items; i += n_threads) {
    const int b = entry_of(s_pre, p.batch, i), j = i - s_pre[b];
    const int32_t v = p.store[p.rows[b] * p.store_stride + j];
    p.store[p.first[b] * p.store_stride + j] = v;
    atomicAdd(p.shares + v, 1);
  }
#pragma unroll 1
  for (int b = at; b < p.batch; b += n_threads) {
    int32_t src = -1, dst = -1;
    if (s_new[b + 1] > s_new[b]) {
      const uint32_t j = over(p, p.second[b]);
      src = p.store[p.rows[b] * p.store_stride + j];
      dst = ring_at(s_new[b]);
      p.store[p.first[b] * p.store_stride + j] = dst;
    }
    p.copy_src[b] = src;
    p.copy_dst[b] = dst;
  }
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
  int32_t* const s_pre = sm;  // [batch + 1] blocks released before an entry
  uint32_t* const seen = reinterpret_cast<uint32_t*>(s_pre + p.batch + 1);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n_threads = gridDim.x * kPageThreads, at = blockIdx.x * kPageThreads + tid;
  for (int i = tid; i < (p.store_rows + 31) / 32; i += kPageThreads) seen[i] = 0;
  cluster.sync();  // every CTA has begun: its shared memory may be written
  pdl_wait();
  const int32_t head = p.state[0], count = p.state[1];
  int32_t bits = 0;
  __syncthreads();
  const int per = (p.batch + kPageThreads - 1) / kPageThreads;
  const int begin = min(tid * per, p.batch), end = min(begin + per, p.batch);
  int64_t back = 0, parts = 0;  // parts: entries that keep a part of a block
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
    s_pre[b] = less;
    back += less;
  }
  int64_t back_total, parts_total;
  scan2(back, parts, back_total, parts_total);
#pragma unroll 1
  for (int b = begin; b < end; ++b) {
    const int32_t less = s_pre[b];
    s_pre[b] = static_cast<int32_t>(back);
    back += less;
  }
  if (head < 0 || head >= p.ring_size || count < 0 || count > p.ring_size || back_total > INT32_MAX) bits |= PSB_DEVERR_POOL;
  const bool planned = __syncthreads_or(bits != 0) == 0;
  const bool stopped = refused_before(p);
  const int items = planned ? static_cast<int>(back_total) : 0;
  int32_t* const last = p.shares + p.ring_size;
  auto place_of = [&](int i) -> int32_t* {  // the i-th entry to be released
    const int b = entry_of(s_pre, p.batch, i);
    return p.store + p.rows[b] * p.store_stride + blocks_for(p, p.second[b]) + (i - s_pre[b]);
  };
  // Consecutive items to each CTA, so that ranks are sums over the CTAs before.
  const int share = (items + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x);
  const int i0 = min(static_cast<int>(blockIdx.x) * share, items), i1 = min(i0 + share, items);
#pragma unroll 1
  for (int i = i0 + tid; i < i1; i += kPageThreads) {
    const int32_t v = *place_of(i);
    if (v < 0 || v >= p.ring_size) {
      bits |= PSB_DEVERR_BLOCK_RANGE;
    } else {
      if (atomicSub(p.shares + v, 1) < 0) bits |= PSB_DEVERR_POOL;  // more often than it is held
      atomicMax(last + v, i + 1);
    }
  }
  if (stopped) bits |= PSB_DEVERR_REFUSED;
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
  auto put_back = [&]() {  // what was counted
#pragma unroll 1
    for (int i = i0 + tid; i < i1; i += kPageThreads) {
      const int32_t v = *place_of(i);
      if (v >= 0 && v < p.ring_size) {
        atomicAdd(p.shares + v, 1);
        last[v] = 0;
      }
    }
  };
  if (all != 0) {
    put_back();
    if (at == 0 && (all & PSB_DEVERR_REFUSED) == 0) flag_error(p.err, all);
    return;
  }
  // whether item i returns its block
  auto returns = [&](int i, int32_t v) { return __ldcg(last + v) == i + 1 && __ldcg(p.shares + v) < 0; };
  int n = 0;
#pragma unroll 1
  for (int i = i0 + tid; i < i1; i += kPageThreads) n += returns(i, *place_of(i));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
  if (lane == 0) warp_sums[warp] = n;
  __syncthreads();
  if (tid < static_cast<int>(cluster.num_blocks())) {
    int sum = 0;
    for (int w = 0; w < kPageWarps; ++w) sum += warp_sums[w];
    cluster.map_shared_rank(freed_of, tid)[cluster.block_rank()] = sum;
  }
  cluster.sync();  // (from here on words of finished items are reset: those are nobody else's)
  int base = 0, freed = 0;
  for (int c = 0; c < static_cast<int>(cluster.num_blocks()); ++c) {
    if (c < static_cast<int>(cluster.block_rank())) base += freed_of[c];
    freed += freed_of[c];
  }
  if (count + freed > p.ring_size) {  // more blocks than the pool has: the list or a table is not what it should be
    put_back();
    if (at == 0) flag_error(p.err, PSB_DEVERR_POOL);
    return;
  }
#pragma unroll 1
  for (int c = i0; c < i1; c += kPageThreads) {
    const int i = c + tid;
    int32_t v = 0;
    bool out = false;
    if (i < i1) {
      int32_t* const entry = place_of(i);
      v = *entry;
      *entry = 0;
      out = returns(i, v);
      if (__ldcg(last + v) == i + 1) last[v] = 0;
      if (out) p.shares[v] = 0;
    }
    const uint32_t mask = __ballot_sync(0xffffffffu, out);
    __syncthreads();
    if (lane == 0) warp_sums[warp] = __popc(mask);
    __syncthreads();
    int before = base, sum = 0;
    for (int w = 0; w < kPageWarps; ++w) {
      if (w < warp) before += warp_sums[w];
      sum += warp_sums[w];
    }
    if (out) {
      int64_t to = static_cast<int64_t>(head) + count + before + __popc(mask & ((1u << lane) - 1));  // below two rings
      if (to >= p.ring_size) to -= p.ring_size;
      p.ring[to] = v;
    }
    base += sum;
  }
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

int launch_pages(void (*kern)(PagesParams), const PagesParams& p, int arrays, cudaStream_t s) {
  const size_t smem = sizeof(int32_t) * (arrays * (static_cast<size_t>(p.batch) + 1) + (static_cast<size_t>(p.store_rows) + 31) / 32);
  if (smem > 200 * 1024) return PSB_ERR_UNSUPPORTED;
  int occ = 0;
  if (!kernel_occupancy(reinterpret_cast<const void*>(kern), kPageThreads, smem, &occ)) return PSB_ERR_CUDA;
  discard_stale_error();
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = kPageCtas;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(kPageCtas);
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
  return launch_pages(fork_tables_kernel, p, 2, reinterpret_cast<cudaStream_t>(stream));
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
  return launch_pages(release_tables_kernel, p, 1, reinterpret_cast<cudaStream_t>(stream));
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
