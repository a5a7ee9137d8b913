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
// Both are latency bound: integers only, a few hundred kilobytes at most, and
// short code (a cold instruction cache costs a kernel of this size more than
// its loads: the same work with 64-bit divisions, 40 KB of code, took 12.6 +
// 8.2 us where this takes 10.4 + 6.1 us for 256 requests, by the profiler; 10.0 us
// for both in a replayed graph).  So positions and
// counts are 32 bits (what is added to them is checked first), a division by
// block_size is a shift where it is a power of two, and the grid walks rows of
// the table instead of elements.
// Every CTA scans the whole plan into shared memory itself (no second launch,
// no grid-wide wait), then the grid strides over table rows and tokens.
// The list and the counters are only read in that phase; the last CTA to
// arrive (a ticket in free_state[2], reset by it) moves head and count, after
// every CTA has read them.  A step that cannot be carried out whole - not
// enough free blocks, a store row named twice or out of range, a negative
// start or count, more blocks than a row holds, an id outside the pool among
// those taken or given back - changes neither the store nor the free list
// (words of the ring that are not on the list are scratch).
// What was planned behind a refused step (the trim of the same captured step,
// the next step) counts on blocks the requests never got, and the host cannot
// take it back in time: a refused extend_step also leaves PSB_DEVERR_REFUSED in
// error_flag, and while that is set both kernels refuse.
#include <algorithm>

#include "common.cuh"
#include "host_util.h"

namespace psb {
namespace {

constexpr int kTabThreads = 256;
constexpr int kTabWarps = kTabThreads / 32;
constexpr int kPiece = 128;  // table columns a warp writes at a time
constexpr int32_t kOutside = 1 << 16;  // added to trim's ticket by a CTA that found an id outside the pool (CTAs: <= kTrimCtas)
constexpr int kTrimCtas = 32;

struct TablesParams {
  int32_t* store;
  int64_t store_stride;
  int32_t store_rows, store_width;
  const int32_t* rows;
  const int32_t* first;   // extend: starts; trim: held lengths
  const int32_t* second;  // extend: new tokens; trim: kept lengths
  int32_t batch, block_size, shift;  // block_size is 2^shift, or shift is -1
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

// Blocks of ``tokens`` (below 2^32) tokens.
__device__ __forceinline__ uint32_t over(const TablesParams& p, uint32_t x) {
  return p.shift >= 0 ? x >> p.shift : x / static_cast<uint32_t>(p.block_size);
}
__device__ __forceinline__ uint32_t blocks_for(const TablesParams& p, uint32_t tokens) {
  return tokens == 0 ? 0 : over(p, tokens - 1) + 1;
}

// Exclusive scan over the CTA of two values per thread (``a`` up to 2^40, ``b``
// up to 2^40), and their totals.
__device__ __forceinline__ void scan_threads(int64_t& a, int64_t& b, int64_t& a_total, int64_t& b_total) {
  __shared__ int64_t sums[2][kTabWarps];
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
  for (int w = 0; w < kTabWarps; ++w) {
    const int64_t x = sums[0][w], y = sums[1][w];
    if (w < warp) {
      a += x;
      b += y;
    }
    a_total += x;
    b_total += y;
  }
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

// Whether an earlier step was refused and the host has not cleared the flag.
// (A CTA of the step that is being refused may see its own: the same answer.)
__device__ __forceinline__ bool refused_before(const TablesParams& p) {
  return p.err != nullptr && (*static_cast<volatile const int32_t*>(p.err) & PSB_DEVERR_REFUSED) != 0;
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
  const int tid = threadIdx.x, lane = tid & 31;
  for (int i = tid; i < (p.store_rows + 31) / 32; i += kTabThreads) seen[i] = 0;
  pdl_wait();
  const int32_t head = p.state[0], count = p.state[1];
  const bool stopped = refused_before(p);
  __syncthreads();
  const int per = (p.batch + kTabThreads - 1) / kTabThreads;
  const int begin = min(tid * per, p.batch), end = min(begin + per, p.batch);
  const uint32_t width = min(p.store_width, p.out_width);
  int64_t tok = 0, grow = 0;
  int32_t bits = 0;
#pragma unroll 1
  for (int b = begin; b < end; ++b) {
    const int32_t row = p.rows[b], start = p.first[b], n = p.second[b];
    tok += max(n, 0);
    if (n < 0) bits |= PSB_DEVERR_CONTEXT;
    int32_t more = 0;
    if (row >= 0) {  // (a padding entry holds and takes nothing)
      const uint32_t tokens = static_cast<uint32_t>(max(start, 0)) + static_cast<uint32_t>(max(n, 0)), need = blocks_for(p, tokens);
      if (row >= p.store_rows || start < 0 || need > width || tokens > INT32_MAX) {
        bits |= PSB_DEVERR_CONTEXT;
      } else {
        if (mark_row(seen, row)) bits |= PSB_DEVERR_ROWS;
        more = static_cast<int32_t>(need - blocks_for(p, start));
      }
    }
    s_gr[b] = more;
    grow += more;
  }
  int64_t tok_total, grow_total;
  scan_threads(tok, grow, tok_total, grow_total);
  if (tok_total != p.total) bits |= PSB_DEVERR_SEQLENS;
  if (head < 0 || head >= p.ring_size || count < 0 || count > p.ring_size || grow_total > count) {
    bits |= PSB_DEVERR_POOL;
  } else {
    // every id the step takes, before any is handed out, eight loads in flight
    // (what is read again below comes from L1): 0.6 us for 16 ids, 1.2 us for 3000
    const uint32_t want = static_cast<uint32_t>(grow_total), size = p.ring_size;
#pragma unroll 1
    for (uint32_t i0 = tid; i0 < want; i0 += 8 * kTabThreads) {
#pragma unroll
      for (uint32_t k = 0; k < 8; ++k) {
        const uint32_t i = i0 + k * kTabThreads;
        uint32_t at = static_cast<uint32_t>(head) + min(i, want - 1);
        if (at >= size) at -= size;
        if (static_cast<uint32_t>(p.ring[at]) >= size) bits |= PSB_DEVERR_BLOCK_RANGE;
      }
    }
  }
  const bool bad = __syncthreads_or(stopped || bits != 0) != 0;
  if (bits != 0 && !stopped && blockIdx.x == 0) flag_error(p.err, bits | PSB_DEVERR_REFUSED);
#pragma unroll 1
  for (int b = begin; b < end; ++b) {
    // a refused step may hold counts that no int32 sum does: kept in range
    s_cu[b] = static_cast<int32_t>(min(tok, static_cast<int64_t>(p.total)));
    tok += max(p.second[b], 0);
    const int32_t more = s_gr[b];
    s_gr[b] = bad ? 0 : static_cast<int32_t>(grow);
    grow += more;
  }
  const int32_t taken = bad ? 0 : static_cast<int32_t>(grow_total);
  if (tid == 0) {
    s_cu[p.batch] = static_cast<int32_t>(min(tok_total, static_cast<int64_t>(p.total)));
    s_gr[p.batch] = taken;
  }
  __syncthreads();

  // block ``j`` of entry b, which holds ``held``: one of those, or its share of the ring
  auto block_of = [&](int b, int32_t row, uint32_t held, uint32_t j) -> int32_t {
    if (j < held) return p.store[row * p.store_stride + j];
    uint32_t at = static_cast<uint32_t>(head) + static_cast<uint32_t>(s_gr[b]) + (j - held);  // below 2^32: two counts
    if (at >= static_cast<uint32_t>(p.ring_size)) at -= p.ring_size;
    return p.ring[at];
  };
  if (blockIdx.x == 0) {
    for (int b = tid; b <= p.batch; b += kTabThreads) {
      p.cu[b] = s_cu[b];
      if (b < p.batch) p.ctx[b] = bad || p.rows[b] < 0 ? 0 : p.first[b] + p.second[b];
    }
  }
  // padded tables, and the new ids into the store: a warp per piece of a row
  const int pieces = (p.out_width + kPiece - 1) / kPiece;
  const int64_t tasks = static_cast<int64_t>(p.batch) * pieces;
#pragma unroll 1
  for (int64_t t = blockIdx.x * kTabWarps + (tid >> 5); t < tasks; t += static_cast<int64_t>(gridDim.x) * kTabWarps) {
    const int b = pieces == 1 ? static_cast<int>(t) : static_cast<int>(t / pieces);
    const int j0 = static_cast<int>(t - static_cast<int64_t>(b) * pieces) * kPiece;
    const int32_t row = bad ? -1 : p.rows[b];
    uint32_t held = 0, need = 0;
    if (row >= 0) {
      const uint32_t start = p.first[b];
      held = blocks_for(p, start);
      need = blocks_for(p, start + static_cast<uint32_t>(p.second[b]));
    }
    int32_t* const out = p.tables + static_cast<int64_t>(b) * p.out_width;
#pragma unroll 1
    for (int j = j0 + lane; j < min(j0 + kPiece, p.out_width); j += 32) {
      int32_t v = 0;
      if (static_cast<uint32_t>(j) < need) {
        v = block_of(b, row, held, j);
        if (v < 0 || v >= p.ring_size) flag_error(p.err, PSB_DEVERR_BLOCK_RANGE);
        if (static_cast<uint32_t>(j) >= held) p.store[row * p.store_stride + j] = v;
      }
      out[j] = v;
    }
  }
  // slot and position of every new token
#pragma unroll 1
  for (uint32_t i = blockIdx.x * kTabThreads + tid; i < static_cast<uint32_t>(p.total); i += gridDim.x * kTabThreads) {
    int64_t slot = -1;
    uint32_t pos = 0;
    if (!bad) {
      const int b = entry_of(s_cu, p.batch, static_cast<int>(i));
      const int32_t row = p.rows[b];
      if (row >= 0) {
        const uint32_t start = p.first[b];
        pos = start + (i - static_cast<uint32_t>(s_cu[b]));
        const uint32_t j = over(p, pos);
        const int32_t v = block_of(b, row, blocks_for(p, start), j);
        if (v >= 0 && v < p.ring_size)
          slot = static_cast<int64_t>(v) * p.block_size + (pos - j * static_cast<uint32_t>(p.block_size));
      }
    }
    p.slots[i] = slot;
    p.positions[i] = pos;
  }
  uint32_t new_head = static_cast<uint32_t>(head) + static_cast<uint32_t>(taken);
  if (!bad && new_head >= static_cast<uint32_t>(p.ring_size)) new_head -= p.ring_size;
  finish_ring(p, static_cast<int32_t>(new_head), count - taken);
}

__global__ void __launch_bounds__(kTabThreads) trim_tables_kernel(const TablesParams p) {
  extern __shared__ int32_t sm[];
  int32_t* s_pre = sm;  // [batch + 1] blocks given back before entry b
  uint32_t* seen = reinterpret_cast<uint32_t*>(s_pre + p.batch + 1);
  const int tid = threadIdx.x;
  for (int i = tid; i < (p.store_rows + 31) / 32; i += kTabThreads) seen[i] = 0;
  pdl_wait();
  const int32_t head = p.state[0], count = p.state[1];
  const bool stopped = refused_before(p);
  __syncthreads();
  const int per = (p.batch + kTabThreads - 1) / kTabThreads;
  const int begin = min(tid * per, p.batch), end = min(begin + per, p.batch);
  int64_t back = 0, unused = 0;
  int32_t bits = 0;
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
      }
    }
    s_pre[b] = less;
    back += less;
  }
  int64_t back_total, unused_total;
  scan_threads(back, unused, back_total, unused_total);
  if (head < 0 || head >= p.ring_size || count < 0 || count + back_total > p.ring_size) bits |= PSB_DEVERR_POOL;
  const bool bad = __syncthreads_or(stopped || bits != 0) != 0;
  if (bits != 0 && !stopped && blockIdx.x == 0) flag_error(p.err, bits);
  bool outside = false;  // an id of this CTA's share is outside the pool
  auto place_of = [&](uint32_t i) -> int32_t* {  // the i-th entry to come back
    const int b = entry_of(s_pre, p.batch, static_cast<int>(i));
    return p.store + p.rows[b] * p.store_stride + blocks_for(p, p.second[b]) + (i - static_cast<uint32_t>(s_pre[b]));
  };
  auto ring_of = [&](uint32_t i) -> int32_t* {  // where it goes: behind the list's end
    int64_t to = static_cast<int64_t>(head) + count + i;  // below two rings
    if (to >= p.ring_size) to -= p.ring_size;
    return p.ring + to;
  };
  if (!bad) {  // the same for every thread of every CTA
#pragma unroll 1
    for (int b = begin; b < end; ++b) {
      const int32_t less = s_pre[b];
      s_pre[b] = static_cast<int32_t>(back);
      back += less;
    }
    __syncthreads();
#pragma unroll 1
    for (uint32_t i = blockIdx.x * kTabThreads + tid; i < static_cast<uint32_t>(back_total); i += gridDim.x * kTabThreads) {
      int32_t* entry = place_of(i);
      const int32_t v = *entry;
      outside = outside || v < 0 || v >= p.ring_size;
      *ring_of(i) = v;
      *entry = 0;
    }
  }
  // The ids are on the ring, but behind its end: the last CTA to arrive moves
  // the end if all of them are in range, and else puts them back where they
  // were.  (Looking at all of them first, in every CTA, took 2 us more for 3000.)
  __shared__ int32_t s_found;
  outside = __syncthreads_or(outside) != 0;
  if (tid == 0) {
    __threadfence();
    s_found = atomicAdd(p.state + 2, outside ? kOutside + 1 : 1) + (outside ? kOutside : 0);
  }
  __syncthreads();
  const int32_t found = s_found;
  if ((found & (kOutside - 1)) != static_cast<int32_t>(gridDim.x) - 1) return;
  const bool undo = found >= kOutside;
  if (undo) {
    __threadfence();
#pragma unroll 1
    for (uint32_t i = tid; i < static_cast<uint32_t>(back_total); i += kTabThreads) *place_of(i) = __ldcg(ring_of(i));
  }
  if (tid == 0) {
    if (undo) flag_error(p.err, PSB_DEVERR_BLOCK_RANGE);
    if (!bad && !undo) p.state[1] = count + static_cast<int32_t>(back_total);
    p.state[2] = 0;
  }
}

int32_t block_shift(int32_t block_size) {
  if ((block_size & (block_size - 1)) != 0) return -1;
  int32_t s = 0;
  while ((1 << s) < block_size) ++s;
  return s;
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
  const cudaError_t e = launch_pdl(kern, dim3(static_cast<unsigned>(grid)), dim3(kTabThreads), smem, s, p);
  if (e != cudaSuccess) return record_cuda_error(e);
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
  p.shift = block_shift(block_size);
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
  p.shift = block_shift(block_size);
  p.ring = free_blocks;
  p.state = free_state;
  p.ring_size = num_blocks;
  p.err = error_flag;
  // what comes back is known on the device only: a few blocks per request is
  // the common case, a whole store the largest
  return launch_tables(trim_tables_kernel, p, 1, std::min<int64_t>(static_cast<int64_t>(batch) * store_width, kTrimCtas * kTabThreads),
                       reinterpret_cast<cudaStream_t>(stream));
}
