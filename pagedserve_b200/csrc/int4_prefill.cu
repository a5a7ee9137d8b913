// Prefix-aware (chunked) causal prefill over the 4-bit KV pool (format:
// int4_cache.cuh).
//
// Generic path (fp32, or a geometry the tensor-core path does not cover): one
// warp per (query row, q head), 32 keys per step (one key per lane for Q.K,
// lanes over head_dim for P.V), values decoded to fp32 as they are read,
// online softmax in fp32.  Bound by its arithmetic and by decoding every key
// again for every row: 512 tokens on 8 K take 11.4 ms in fp32 where the
// tensor-core path takes 55 us, and 28.9 ms with 32 / 8 heads of 128 (105 us with
// as many of 64).  16-bit types come here for head_dim other than 64, rows of q
// off 16 bytes, more than 2048 sequences or 128 q heads per kv head.
#include <algorithm>

#include "common.cuh"
#include "host_util.h"
#include "int4_attention.h"
#include "int4_cache.cuh"

namespace psb {
namespace {

constexpr int kGenThreads = 128;
constexpr int kMaxPairsPerLane = kInt4MaxDim / 64;

template <typename T>
__global__ void __launch_bounds__(kGenThreads) int4_prefill_generic_kernel(const Int4PrefillParams p) {
  extern __shared__ float s_q[];  // [warps][D]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int D = p.head_dim, pairs = D / 2, BS = p.block_size;
  const int64_t task = blockIdx.x * static_cast<int64_t>(kGenThreads / 32) + warp;
  if (task >= static_cast<int64_t>(p.total) * p.hq) return;
  const int row = static_cast<int>(task / p.hq), qh = static_cast<int>(task - static_cast<int64_t>(row) * p.hq);
  const int kh = qh / (p.hq / p.hkv);
  int lo = 0, hi = p.num_seqs - 1;  // the sequence of this row
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (p.cu[mid] <= row) lo = mid; else hi = mid - 1;
  }
  const int c0 = p.cu[lo], c1 = p.cu[lo + 1];
  if (row < c0 || row >= c1) return;  // a row behind the last sequence
  const int n = c1 - c0;
  int ctx = p.ctx[lo];
  if (ctx < n || ctx > p.max_context) {
    if (lane == 0) flag_error(p.err, PSB_DEVERR_CONTEXT);
    ctx = min(max(ctx, n), p.max_context);
  }
  const int last = ctx - n + (row - c0);
  const int32_t* table = p.tables + static_cast<int64_t>(lo) * p.table_stride;
  auto row_of = [&](int pos, int kv) -> int64_t {
    const int32_t blk = table[pos / BS];
    if (blk < 0 || blk >= p.num_blocks) return -1;
    return int4_row(p.layer_tiles + static_cast<int64_t>(blk) * p.hkv + kh, kv, pos % BS, BS);
  };
  float* q = s_q + warp * D;
  const T* qp = reinterpret_cast<const T*>(p.q) + row * p.qst + qh * p.qsh;
  for (int d = lane; d < D; d += 32) q[d] = Elem<T>::to_float(qp[d]);
  __syncwarp();
  float m = -INFINITY, l = 0.f, acc[kMaxPairsPerLane][2];
#pragma unroll
  for (int i = 0; i < kMaxPairsPerLane; ++i) acc[i][0] = acc[i][1] = 0.f;
  for (int k0 = 0; k0 <= last; k0 += 32) {
    const int key = k0 + lane;
    float s = -INFINITY;
    if (key <= last) {
      const int64_t r = row_of(key, 0);
      if (r < 0) {
        flag_error(p.err, PSB_DEVERR_BLOCK_RANGE);
      } else {
        const T* pr = reinterpret_cast<const T*>(p.params) + r * 2;
        const float st = Elem<T>::to_float(pr[0]), md = Elem<T>::to_float(pr[1]);
        float dot = 0.f;
        for (int j = 0; j < pairs; ++j) {
          const uint32_t c = p.codes[r * pairs + j];
          dot = fmaf(q[2 * j], int4_value(c & 15u, st, md), dot);
          dot = fmaf(q[2 * j + 1], int4_value(c >> 4, st, md), dot);
        }
        s = dot * p.scale_log2;
      }
    }
    float mx = s;
#pragma unroll
    for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    const float m_new = fmaxf(m, mx), mu = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = m == -INFINITY ? 0.f : exp2f(m - mu);
    const float pr = exp2f(s - mu);  // 0 at -inf
    float psum = pr;
#pragma unroll
    for (int o = 16; o; o >>= 1) psum += __shfl_xor_sync(0xffffffffu, psum, o);
    l = l * alpha + psum;
#pragma unroll
    for (int i = 0; i < kMaxPairsPerLane; ++i) {
      acc[i][0] *= alpha;
      acc[i][1] *= alpha;
    }
    const int nk = min(32, last - k0 + 1);
    for (int j = 0; j < nk; ++j) {
      const float pj = __shfl_sync(0xffffffffu, pr, j);
      const int64_t r = row_of(k0 + j, 1);
      if (r < 0) continue;  // flagged above
      const T* par = reinterpret_cast<const T*>(p.params) + r * 2;
      const float st = Elem<T>::to_float(par[0]), md = Elem<T>::to_float(par[1]);
#pragma unroll
      for (int i = 0; i < kMaxPairsPerLane; ++i) {
        const int d2 = lane + 32 * i;
        if (d2 < pairs) {
          const uint32_t c = p.codes[r * pairs + d2];
          acc[i][0] = fmaf(pj, int4_value(c & 15u, st, md), acc[i][0]);
          acc[i][1] = fmaf(pj, int4_value(c >> 4, st, md), acc[i][1]);
        }
      }
    }
    m = m_new;
  }
  T* op = reinterpret_cast<T*>(p.out) + row * p.ost + qh * p.osh;
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int i = 0; i < kMaxPairsPerLane; ++i) {
    const int d2 = lane + 32 * i;
    if (d2 < pairs) {
      op[2 * d2] = Elem<T>::from_float(acc[i][0] * inv);
      op[2 * d2 + 1] = Elem<T>::from_float(acc[i][1] * inv);
    }
  }
}

template <typename T>
int launch_generic(const Int4PrefillParams& p, cudaStream_t s) {
  const int64_t tasks = static_cast<int64_t>(p.total) * p.hq;
  const int64_t blocks = (tasks + kGenThreads / 32 - 1) / (kGenThreads / 32);
  if (blocks >= (int64_t(1) << 31)) return PSB_ERR_UNSUPPORTED;
  const size_t smem = sizeof(float) * (kGenThreads / 32) * p.head_dim;
  discard_stale_error();
  int4_prefill_generic_kernel<T><<<static_cast<unsigned>(blocks), kGenThreads, smem, s>>>(p);
  return check_launch();
}

// cu_seqlens sanity, so a malformed batch is reported.
__global__ void check_seqlens_kernel(const int32_t* cu, int32_t n, int32_t total, int32_t max_seqlen, int32_t* err) {
  for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < n; i += gridDim.x * blockDim.x) {
    const int a = cu[i], b = cu[i + 1];
    if (a < 0 || b < a || b > total || (i == 0 && a != 0) || b - a > max_seqlen) flag_error(err, PSB_DEVERR_SEQLENS);
  }
}

}  // namespace
}  // namespace psb

using namespace psb;

extern "C" size_t psb_paged_prefill_int4_workspace_size(int32_t total_tokens, int32_t num_seqs, int32_t q_heads,
                                                        int32_t num_kv_heads, int32_t head_dim, int32_t block_size,
                                                        int32_t max_context, int32_t dtype) {
  if (total_tokens < 0 || num_seqs < 0 || num_kv_heads <= 0 || q_heads <= 0 || q_heads % num_kv_heads ||
      head_dim <= 0 || head_dim % 2 || head_dim > kInt4MaxDim || block_size <= 0 || max_context < 0 ||
      (dtype != PSB_F32 && dtype != PSB_F16 && dtype != PSB_BF16))
    return 0;
  return int4_prefill_tc_geometry(dtype, total_tokens, num_seqs, q_heads, num_kv_heads, head_dim, block_size, max_context)
             ? int4_prefill_tc_workspace(total_tokens, num_seqs, q_heads, num_kv_heads, max_context)
             : 256;
}

extern "C" int psb_paged_prefill_int4(const void* q, int64_t q_stride_t, int64_t q_stride_h, const void* kv_codes,
                                      const void* kv_params, const int32_t* block_tables, int64_t table_stride,
                                      const int32_t* context_lens, void* out, int64_t o_stride_t, int64_t o_stride_h,
                                      const int32_t* cu_seqlens, int32_t num_seqs, int32_t total_tokens,
                                      int32_t max_seqlen, int32_t max_context, int32_t q_heads, int32_t layer,
                                      int32_t num_layers, int64_t num_blocks, int32_t num_kv_heads,
                                      int32_t block_size, int32_t head_dim, int32_t dtype, float scale,
                                      void* workspace, size_t workspace_bytes, int32_t* error_flag,
                                      psb_stream_t stream) {
  if (num_seqs < 0 || total_tokens < 0 || max_seqlen < 0 || max_context < max_seqlen || q_heads <= 0 ||
      num_kv_heads <= 0 || q_heads % num_kv_heads || head_dim <= 0 || head_dim % 2 || head_dim > kInt4MaxDim ||
      num_layers <= 0 || layer < 0 || layer >= num_layers || num_blocks <= 0 || block_size <= 0 ||
      table_stride < (static_cast<int64_t>(max_context) + block_size - 1) / block_size)
    return PSB_ERR_INVALID;
  if (dtype != PSB_F32 && dtype != PSB_F16 && dtype != PSB_BF16) return PSB_ERR_INVALID;
  if (num_seqs == 0 || total_tokens == 0) return PSB_OK;
  if (!q || !kv_codes || !kv_params || !out || !cu_seqlens || !block_tables || !context_lens) return PSB_ERR_INVALID;
  if (reinterpret_cast<uintptr_t>(kv_codes) % 16 || reinterpret_cast<uintptr_t>(kv_params) % 16 ||
      reinterpret_cast<uintptr_t>(workspace) % 16)
    return PSB_ERR_INVALID;
  if (workspace == nullptr ||
      workspace_bytes < psb_paged_prefill_int4_workspace_size(total_tokens, num_seqs, q_heads, num_kv_heads, head_dim,
                                                              block_size, max_context, dtype))
    return PSB_ERR_WORKSPACE;
  Int4PrefillParams p;
  p.q = q;
  p.qst = q_stride_t;
  p.qsh = q_stride_h;
  p.out = out;
  p.ost = o_stride_t;
  p.osh = o_stride_h;
  p.codes = static_cast<const uint8_t*>(kv_codes);
  p.params = kv_params;
  p.tables = block_tables;
  p.table_stride = table_stride;
  p.ctx = context_lens;
  p.cu = cu_seqlens;
  p.num_seqs = num_seqs;
  p.total = total_tokens;
  p.max_seqlen = max_seqlen;
  p.max_context = max_context;
  p.hq = q_heads;
  p.hkv = num_kv_heads;
  p.block_size = block_size;
  p.head_dim = head_dim;
  p.num_blocks = num_blocks;
  p.layer_tiles = static_cast<int64_t>(layer) * num_blocks * num_kv_heads;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.err = error_flag;
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (error_flag != nullptr) {
    discard_stale_error();
    check_seqlens_kernel<<<1, 256, 0, s>>>(cu_seqlens, num_seqs, total_tokens, max_seqlen, error_flag);
  }
  // the tensor-core path reads q by TMA: 16-byte bases and strides
  const bool aligned = q_stride_t % 8 == 0 && q_stride_h % 8 == 0 && q_stride_t > 0 && q_stride_h > 0 &&
                       reinterpret_cast<uintptr_t>(q) % 16 == 0;
  if (aligned && int4_prefill_tc_geometry(dtype, total_tokens, num_seqs, q_heads, num_kv_heads, head_dim, block_size,
                                          max_context))
    return int4_prefill_tc_launch(p, dtype, static_cast<float*>(workspace), s);
  switch (dtype) {
    case PSB_BF16: return launch_generic<__nv_bfloat16>(p, s);
    case PSB_F16: return launch_generic<__half>(p, s);
    default: return launch_generic<float>(p, s);
  }
}
