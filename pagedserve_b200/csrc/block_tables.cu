// extend_step / trim_tables: block tables that grow and shrink on the GPU.
//
// The host-side BlockManager (a FIFO free list: blocks are taken from its head
// and come back at its tail) as device state: ``free_blocks`` int32 [N] is a
// ring of free block ids, ``free_state`` int32 [4] = {head, count, arrivals,
// 0}.  extend_step takes, in entry order, the blocks the step's new tokens
// need, appends them to the requests' rows of the table store and builds what
// pack_step builds (cu_seqlens, lengths, slots, positions, padded tables), so
// a captured step can admit tokens without a host round trip; trim_tables
// gives the blocks past each request's kept length back in entry order and
// zeroes their store entries.  Taken in the same order, the ids are the ones
// BlockManager hands out.
//
// Both are latency bound: integers only, a few hundred kilobytes at most.
// Every CTA scans the whole plan into shared memory itself (no second launch,
// no grid-wide wait), then the grid strides over table entries and tokens.
// The ring and the counters are only read in that phase; the last CTA to
// arrive (a ticket in free_state[2], reset by it) moves head and count, after
// every CTA has read them.  A step that cannot be carried out whole - not
// enough free blocks, a store row named twice or out of range, a negative
// start or count, more blocks than a row holds - changes neither the store
// nor the free list.
#include <algorithm>

#include "common.cuh"
#include "host_util.h"

namespace psb {
namespace {

constexpr int kTabThreads = 256;
constexpr int kTabWarps = kTabThreads / 32;

struct TablesParams {
  int32_t* store;
  int64_t store_stride;
  int32_t store_rows, store_width;
  const int32_t* rows;
  const int32_t* first;   // extend: starts; trim: held lengths
  const int32_t* second;  // extend: new tokens; trim: kept lengths
  int32_t batch, block_size;
  int32_t* ring;
  int32_t* state;
  int32_t ring_size;
  int32_t* err;
  // extend only
  int32_t total, out_width;
  int32_t* cu;
  int32_t* ctx;
  int64_t* slots;
  int64_t* positions;
  int32_t* tables;
};

__device__ __forceinline__ int64_t blocks_for(int64_t tokens, int block_size) {
  return (tokens + block_size - 1) / block_size;
}

// Exclusive scan over the CTA of one int64 per thread; also the total.
__device__ int64_t scan_threads(int64_t v, int64_t* warp_sums, int64_t& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t x = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += x;
  }
  if (lane == 31) warp_sums[warp] = incl;
  __syncthreads();
  int64_t run = incl - v;
  total = 0;
  for (int w = 0; w < kTabWarps; ++w) {
    if (w < warp) run += warp_sums[w];
    total += warp_sums[w];
  }
  __syncthreads();  // warp_sums may be used again
  return run;
}

// The last CTA to get here moves the ring; called by every thread once the
// CTA has read everything it needs of the ring and its counters.
__device__ __forceinline__ void finish_ring(const TablesParams& p, int32_t head, int32_t count) {
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    if (atomicAdd(p.state + 2, 1) == static_cast<int>(gridDim.x) - 1) {
      p.state[0] = head;
      p.state[1] = count;
      p.state[2] = 0;
    }
  }
}

// Marks entry b's row in the CTA's bitmap; true when it was marked before.
__device__ __forceinline__ bool mark_row(uint32_t* seen, int32_t row) {
  const uint32_t bit = 1u << (row & 31);
  return (atomicOr(seen + (row >> 5), bit) & bit) != 0;
}

// Last b with pre[b] <= i (pre ascending, pre[0] = 0).
__device__ __forceinline__ int entry_of(const int32_t* pre, int batch, int i) {
  int lo = 0, hi = batch - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (pre[mid] <= i) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__global__ void __launch_bounds__(kTabThreads) extend_step_kernel(const TablesParams p) {
  extern __shared__ int32_t sm[];
  int32_t* s_cu = sm;                        // [batch + 1] tokens before entry b
  int32_t* s_gr = s_cu + p.batch + 1;        // [batch + 1] new blocks before entry b
  uint32_t* seen = reinterpret_cast<uint32_t*>(s_gr + p.batch + 1);  // store rows named so far
  __shared__ int64_t warp_sums[kTabWarps];
  const int tid = threadIdx.x, BS = p.block_size;
  for (int i = tid; i < (p.store_rows + 31) / 32; i += kTabThreads) seen[i] = 0;
  __syncthreads();
  const int per = (p.batch + kTabThreads - 1) / kTabThreads;
  const int begin = min(tid * per, p.batch), end = min(begin + per, p.batch);
  int64_t tok = 0, grow = 0;
  int32_t bits = 0;
  for (int b = begin; b < end; ++b) {
    const int32_t row = p.rows[b], start = p.first[b], n = p.second[b];
    tok += max(n, 0);
    if (n < 0) bits |= PSB_DEVERR_CONTEXT;
    if (row < 0) continue;  // a padding entry holds and takes nothing
    const int64_t len = static_cast<int64_t>(start) + max(n, 0);
    if (row >= p.store_rows || start < 0 || blocks_for(len, BS) > static_cast<int64_t>(min(p.store_width, p.out_width))) {
      bits |= PSB_DEVERR_CONTEXT;
      continue;
    }
    if (mark_row(seen, row)) bits |= PSB_DEVERR_ROWS;
    grow += blocks_for(len, BS) - blocks_for(start, BS);
  }
  int64_t tok_total, grow_total;
  int64_t tok_at = scan_threads(tok, warp_sums, tok_total);
  int64_t grow_at = scan_threads(grow, warp_sums, grow_total);
  const int32_t head = p.state[0], count = p.state[1];
  if (tok_total != p.total) bits |= PSB_DEVERR_SEQLENS;
  if (head < 0 || head >= p.ring_size || count < 0 || count > p.ring_size || grow_total > count)
    bits |= PSB_DEVERR_POOL;
  const bool bad = __syncthreads_or(bits) != 0;
  if (bits != 0 && blockIdx.x == 0) flag_error(p.err, bits);
  for (int b = begin; b < end; ++b) {
    const int32_t row = p.rows[b], start = p.first[b], n = max(p.second[b], 0);
    // a refused step may hold counts that no int32 sum does: kept in range
    s_cu[b] = static_cast<int32_t>(min(tok_at, static_cast<int64_t>(p.total)));
    s_gr[b] = bad ? 0 : static_cast<int32_t>(grow_at);
    tok_at += n;
    if (!bad && row >= 0) grow_at += blocks_for(static_cast<int64_t>(start) + n, BS) - blocks_for(start, BS);
  }
  if (tid == 0) {
    s_cu[p.batch] = static_cast<int32_t>(min(tok_total, static_cast<int64_t>(p.total)));
    s_gr[p.batch] = bad ? 0 : static_cast<int32_t>(grow_total);
  }
  __syncthreads();

  const int64_t gtid = blockIdx.x * static_cast<int64_t>(kTabThreads) + tid;
  const int64_t gstride = static_cast<int64_t>(gridDim.x) * kTabThreads;
  // block ``j`` of entry b: one it holds, or its share of the ring
  auto block_of = [&](int b, int32_t row, int64_t held, int64_t j) -> int32_t {
    if (j < held) return p.store[row * p.store_stride + j];
    int64_t at = static_cast<int64_t>(head) + s_gr[b] + (j - held);
    if (at >= p.ring_size) at -= p.ring_size;
    return p.ring[at];
  };
  if (blockIdx.x == 0) {
    for (int b = tid; b <= p.batch; b += kTabThreads) p.cu[b] = s_cu[b];
    for (int b = tid; b < p.batch; b += kTabThreads)
      p.ctx[b] = bad || p.rows[b] < 0 ? 0 : p.first[b] + p.second[b];
  }
  // padded tables, and the new ids into the store
  for (int64_t i = gtid; i < static_cast<int64_t>(p.batch) * p.out_width; i += gstride) {
    const int b = static_cast<int>(i / p.out_width), j = static_cast<int>(i - static_cast<int64_t>(b) * p.out_width);
    const int32_t row = p.rows[b];
    int32_t v = 0;
    if (!bad && row >= 0) {
      const int64_t start = p.first[b], held = blocks_for(start, BS);
      if (j < blocks_for(start + p.second[b], BS)) {
        v = block_of(b, row, held, j);
        if (v < 0 || v >= p.ring_size) flag_error(p.err, PSB_DEVERR_BLOCK_RANGE);
        if (j >= held) p.store[row * p.store_stride + j] = v;
      }
    }
    p.tables[i] = v;
  }
  // slot and position of every new token
  for (int64_t i = gtid; i < p.total; i += gstride) {
    int64_t slot = -1, pos = 0;
    if (!bad) {
      const int b = entry_of(s_cu, p.batch, static_cast<int>(i));
      const int32_t row = p.rows[b];
      if (row >= 0) {
        const int32_t start = p.first[b];
        pos = static_cast<int64_t>(start) + (i - s_cu[b]);
        const int64_t j = pos / BS;
        const int32_t v = block_of(b, row, blocks_for(start, BS), j);
        if (v >= 0 && v < p.ring_size) slot = static_cast<int64_t>(v) * BS + (pos - j * BS);
      }
    }
    p.slots[i] = slot;
    p.positions[i] = pos;
  }
  int64_t new_head = static_cast<int64_t>(head) + s_gr[p.batch];
  if (new_head >= p.ring_size) new_head -= p.ring_size;
  finish_ring(p, bad ? head : static_cast<int32_t>(new_head), count - s_gr[p.batch]);
}

__global__ void __launch_bounds__(kTabThreads) trim_tables_kernel(const TablesParams p) {
  extern __shared__ int32_t sm[];
  int32_t* s_pre = sm;  // [batch + 1] blocks given back before entry b
  uint32_t* seen = reinterpret_cast<uint32_t*>(s_pre + p.batch + 1);
  __shared__ int64_t warp_sums[kTabWarps];
  const int tid = threadIdx.x, BS = p.block_size;
  for (int i = tid; i < (p.store_rows + 31) / 32; i += kTabThreads) seen[i] = 0;
  __syncthreads();
  const int per = (p.batch + kTabThreads - 1) / kTabThreads;
  const int begin = min(tid * per, p.batch), end = min(begin + per, p.batch);
  int64_t back = 0;
  int32_t bits = 0;
  for (int b = begin; b < end; ++b) {
    const int32_t row = p.rows[b], held = p.first[b], keep = p.second[b];
    if (row < 0) continue;
    if (row >= p.store_rows || keep < 0 || keep > held || blocks_for(held, BS) > p.store_width) {
      bits |= PSB_DEVERR_CONTEXT;
      continue;
    }
    if (mark_row(seen, row)) bits |= PSB_DEVERR_ROWS;
    back += blocks_for(held, BS) - blocks_for(keep, BS);
  }
  int64_t back_total;
  int64_t at = scan_threads(back, warp_sums, back_total);
  const int32_t head = p.state[0], count = p.state[1];
  if (head < 0 || head >= p.ring_size || count < 0 || count + back_total > p.ring_size) bits |= PSB_DEVERR_POOL;
  const bool bad = __syncthreads_or(bits) != 0;
  if (bits != 0 && blockIdx.x == 0) flag_error(p.err, bits);
  if (!bad) {  // the same for every thread of every CTA
    for (int b = begin; b < end; ++b) {
      s_pre[b] = static_cast<int32_t>(at);
      if (p.rows[b] >= 0) at += blocks_for(p.first[b], BS) - blocks_for(p.second[b], BS);
    }
    __syncthreads();
    const int64_t gstride = static_cast<int64_t>(gridDim.x) * kTabThreads;
    for (int64_t i = blockIdx.x * static_cast<int64_t>(kTabThreads) + tid; i < back_total; i += gstride) {
      const int b = entry_of(s_pre, p.batch, static_cast<int>(i));
      const int64_t j = blocks_for(p.second[b], BS) + (i - s_pre[b]);
      int32_t* entry = p.store + p.rows[b] * p.store_stride + j;
      const int32_t v = *entry;
      if (v < 0 || v >= p.ring_size) flag_error(p.err, PSB_DEVERR_BLOCK_RANGE);
      int64_t to = static_cast<int64_t>(head) + count + i;
      if (to >= p.ring_size) to -= p.ring_size;
      p.ring[to] = v;
      *entry = 0;
    }
  }
  finish_ring(p, head, bad ? count : count + static_cast<int32_t>(back_total));
}

// Shared bytes of a launch: ``arrays`` prefixes over the batch and the bitmap.
size_t tables_smem(int arrays, int32_t batch, int32_t store_rows) {
  return sizeof(int32_t) * (arrays * (static_cast<size_t>(batch) + 1) + (static_cast<size_t>(store_rows) + 31) / 32);
}

int launch_tables(void (*kern)(TablesParams), const TablesParams& p, int arrays, int64_t work, cudaStream_t s) {
  const size_t smem = tables_smem(arrays, p.batch, p.store_rows);
  if (smem > 200 * 1024) return PSB_ERR_UNSUPPORTED;
  const int sms = device_sm_count();
  if (sms <= 0) return PSB_ERR_CUDA;
  int occ = 0;
  if (!kernel_occupancy(reinterpret_cast<const void*>(kern), kTabThreads, smem, &occ)) return PSB_ERR_CUDA;
  const int64_t grid = std::max<int64_t>(1, std::min<int64_t>((work + kTabThreads - 1) / kTabThreads, sms));
  discard_stale_error();
  kern<<<static_cast<unsigned>(grid), kTabThreads, smem, s>>>(p);
  return check_launch();
}

}  // namespace
}  // namespace psb

using namespace psb;

extern "C" int psb_extend_step(int32_t* table_store, int64_t store_stride, int32_t store_rows, int32_t store_width,
                               const int32_t* req_rows, const int32_t* starts, const int32_t* query_lens,
                               int32_t batch, int32_t* free_blocks, int32_t num_blocks, int32_t* free_state,
                               int32_t total, int32_t block_size, int32_t* cu_seqlens, int32_t* context_lens,
                               int64_t* slot_mapping, int64_t* positions, int32_t* block_tables, int32_t out_width,
                               int32_t* error_flag, psb_stream_t stream) {
  if (batch < 0 || total < 0 || block_size <= 0 || store_rows <= 0 || store_width <= 0 || store_stride < store_width ||
      num_blocks <= 0 || out_width <= 0)
    return PSB_ERR_INVALID;
  if (batch == 0) return total == 0 ? PSB_OK : PSB_ERR_INVALID;
  if (!table_store || !req_rows || !starts || !query_lens || !free_blocks || !free_state || !cu_seqlens ||
      !context_lens || !block_tables || (total > 0 && (!slot_mapping || !positions)))
    return PSB_ERR_INVALID;
  TablesParams p{};
  p.store = table_store;
  p.store_stride = store_stride;
  p.store_rows = store_rows;
  p.store_width = store_width;
  p.rows = req_rows;
  p.first = starts;
  p.second = query_lens;
  p.batch = batch;
  p.block_size = block_size;
  p.ring = free_blocks;
  p.state = free_state;
  p.ring_size = num_blocks;
  p.err = error_flag;
  p.total = total;
  p.out_width = out_width;
  p.cu = cu_seqlens;
  p.ctx = context_lens;
  p.slots = slot_mapping;
  p.positions = positions;
  p.tables = block_tables;
  return launch_tables(extend_step_kernel, p, 2, std::max<int64_t>(total, static_cast<int64_t>(batch) * out_width),
                       reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int psb_trim_tables(int32_t* table_store, int64_t store_stride, int32_t store_rows, int32_t store_width,
                               const int32_t* req_rows, const int32_t* held_lens, const int32_t* keep_lens,
                               int32_t batch, int32_t* free_blocks, int32_t num_blocks, int32_t* free_state,
                               int32_t block_size, int32_t* error_flag, psb_stream_t stream) {
  if (batch < 0 || block_size <= 0 || store_rows <= 0 || store_width <= 0 || store_stride < store_width ||
      num_blocks <= 0)
    return PSB_ERR_INVALID;
  if (batch == 0) return PSB_OK;
  if (!table_store || !req_rows || !held_lens || !keep_lens || !free_blocks || !free_state) return PSB_ERR_INVALID;
  TablesParams p{};
  p.store = table_store;
  p.store_stride = store_stride;
  p.store_rows = store_rows;
  p.store_width = store_width;
  p.rows = req_rows;
  p.first = held_lens;
  p.second = keep_lens;
  p.batch = batch;
  p.block_size = block_size;
  p.ring = free_blocks;
  p.state = free_state;
  p.ring_size = num_blocks;
  p.err = error_flag;
  // what comes back is known on the device only: a few blocks per request is
  // the common case, a whole store the largest
  return launch_tables(trim_tables_kernel, p, 1, std::min<int64_t>(static_cast<int64_t>(batch) * store_width, 32 * kTabThreads),
                       reinterpret_cast<cudaStream_t>(stream));
}
