// Paged GQA decode attention over the 4-bit KV pool (format: int4_cache.cuh).
//
// Generic path (fp32, or a geometry the fast path does not cover): CUDA
// cores.  A CTA takes one (sequence, kv head, chunk of the context): K and V
// rows of 64 tokens at a time are decoded to fp32 in shared memory, every q
// head of the kv head keeps an online softmax in fp32.  Chunks are sized so
// that about eight CTAs per SM exist; a sequence of several chunks leaves
// (max, sum, output) partials that int4_merge_kernel, launched next on the
// same stream, joins in chunk order.  It is bound by its arithmetic (every code
// becomes an fp32 product per q head): 256 sequences of 62 MB in blocks of 8 take
// 1546 us where the tensor-core path takes 26 in blocks of 16, so 16-bit types
// come here only for what that path does not take: head_dim other than 64 and
// 128, block_size no multiple of 16, rows of q or out off 16 bytes, more than
// 2560 sequences.
#include <algorithm>

#include "common.cuh"
#include "host_util.h"
#include "int4_attention.h"
#include "int4_cache.cuh"

namespace psb {
namespace {

constexpr int kGenThreads = 128;
constexpr int kGenStep = 64;  // tokens decoded to shared memory at a time

__device__ __forceinline__ int clamp_ctx(const Int4DecodeParams& p, int b, bool flag) {
  int n = p.ctx[b];
  if (n < 0 || n > p.max_context) {
    if (flag) flag_error(p.err, PSB_DEVERR_CONTEXT);
    n = n < 0 ? 0 : p.max_context;
  }
  return n;
}

// Shared memory of the generic kernel, in floats.
struct GenLayout {
  int q, kv, sc, m, l, a, o, total;
  __host__ __device__ GenLayout(int G, int D) {
    q = 0;
    kv = q + G * D;
    sc = kv + kGenStep * (D + 1);
    m = sc + G * kGenStep;
    l = m + G;
    a = l + G;
    o = a + G;
    total = o + G * D;
  }
};

// One partial: [G] max (scaled by log2 e), [G] sum, [G][D] unnormalised output.
__host__ __device__ inline int64_t gen_part_floats(int group, int head_dim) {
  return static_cast<int64_t>(group) * (head_dim + 2);
}

template <typename T>
__global__ void __launch_bounds__(kGenThreads) int4_decode_generic_kernel(const Int4DecodeParams p, int chunk,
                                                                          int max_split) {
  extern __shared__ float gsm[];
  const int G = p.group, D = p.head_dim, BS = p.block_size, tid = threadIdx.x, ldk = D + 1, pairs = D / 2;
  const GenLayout lay(G, D);
  float* q_s = gsm + lay.q;
  float* kv_s = gsm + lay.kv;
  float* sc_s = gsm + lay.sc;
  float* m_s = gsm + lay.m;
  float* l_s = gsm + lay.l;
  float* a_s = gsm + lay.a;
  float* o_s = gsm + lay.o;
  const int64_t u = blockIdx.x;
  const int c = static_cast<int>(u % max_split);
  const int64_t bh = u / max_split;
  const int h = static_cast<int>(bh % p.hkv), b = static_cast<int>(bh / p.hkv);
  const int ctx = clamp_ctx(p, b, c == 0 && h == 0 && tid == 0);
  const int nsplit = max(1, (ctx + chunk - 1) / chunk);
  if (c >= nsplit) return;
  const int begin = c * chunk, end = min(ctx, begin + chunk);
  for (int i = tid; i < G * D; i += kGenThreads) {
    const int g = i / D, d = i - g * D;
    q_s[i] = Elem<T>::to_float(reinterpret_cast<const T*>(p.q)[b * p.qsb + (h * G + g) * p.qsh + d]);
    o_s[i] = 0.f;
  }
  for (int g = tid; g < G; g += kGenThreads) {
    m_s[g] = -INFINITY;
    l_s[g] = 0.f;
  }
  const int32_t* table = p.tables + static_cast<int64_t>(b) * p.table_stride;
  // pool row of position pos, -1 when its block id is outside the pool
  auto row_of = [&](int pos, int kv) -> int64_t {
    const int32_t blk = table[pos / BS];
    if (blk < 0 || blk >= p.num_blocks) return -1;
    return int4_row(p.layer_tiles + static_cast<int64_t>(blk) * p.hkv + h, kv, pos % BS, BS);
  };
  auto load_rows = [&](int kv, int t0, int n) {
    for (int i = tid; i < n * pairs; i += kGenThreads) {
      const int r = i / pairs, j = i - r * pairs;
      const int64_t row = row_of(t0 + r, kv);
      float x = 0.f, y = 0.f;
      if (row >= 0) {
        const uint32_t code = p.codes[row * pairs + j];
        const T* pr = reinterpret_cast<const T*>(p.params) + row * 2;
        const float st = Elem<T>::to_float(pr[0]), md = Elem<T>::to_float(pr[1]);
        x = int4_value(code & 15u, st, md);
        y = int4_value(code >> 4, st, md);
      } else if (j == 0) {
        flag_error(p.err, PSB_DEVERR_BLOCK_RANGE);
      }
      kv_s[r * ldk + 2 * j] = x;
      kv_s[r * ldk + 2 * j + 1] = y;
    }
  };
  for (int t0 = begin; t0 < end; t0 += kGenStep) {
    const int n = min(kGenStep, end - t0);
    __syncthreads();
    load_rows(0, t0, n);
    __syncthreads();
    for (int i = tid; i < G * kGenStep; i += kGenThreads) {
      const int g = i / kGenStep, r = i - g * kGenStep;
      float acc = -INFINITY;
      if (r < n && row_of(t0 + r, 0) >= 0) {
        acc = 0.f;
        for (int d = 0; d < D; ++d) acc = fmaf(q_s[g * D + d], kv_s[r * ldk + d], acc);
        acc *= p.scale_log2;
      }
      sc_s[i] = acc;
    }
    __syncthreads();
    load_rows(1, t0, n);
    for (int g = tid >> 5; g < G; g += kGenThreads / 32) {
      const int lane = tid & 31;
      float mx = m_s[g];
      for (int r = lane; r < kGenStep; r += 32) mx = fmaxf(mx, sc_s[g * kGenStep + r]);
#pragma unroll
      for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      const float mu = mx == -INFINITY ? 0.f : mx;
      float sum = 0.f;
      for (int r = lane; r < kGenStep; r += 32) {
        const float pr = exp2f(sc_s[g * kGenStep + r] - mu);  // 0 at -inf
        sum += pr;
        sc_s[g * kGenStep + r] = pr;
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      __syncwarp();
      if (lane == 0) {
        const float a = m_s[g] == -INFINITY ? 0.f : exp2f(m_s[g] - mu);
        a_s[g] = a;
        m_s[g] = mx;
        l_s[g] = l_s[g] * a + sum;
      }
    }
    __syncthreads();
    for (int i = tid; i < G * D; i += kGenThreads) {
      const int g = i / D, d = i - g * D;
      float acc = o_s[i] * a_s[g];
      for (int r = 0; r < n; ++r) acc = fmaf(sc_s[g * kGenStep + r], kv_s[r * ldk + d], acc);
      o_s[i] = acc;
    }
  }
  __syncthreads();
  if (nsplit == 1) {
    for (int i = tid; i < G * D; i += kGenThreads) {
      const int g = i / D, d = i - g * D;
      const float l = l_s[g];
      reinterpret_cast<T*>(p.out)[b * p.osb + (h * G + g) * p.osh + d] = Elem<T>::from_float(l == 0.f ? 0.f : o_s[i] / l);
    }
    return;
  }
  float* part = p.part + u * gen_part_floats(G, D);
  for (int g = tid; g < G; g += kGenThreads) {
    part[g] = m_s[g];
    part[G + g] = l_s[g];
  }
  for (int i = tid; i < G * D; i += kGenThreads) part[2 * G + i] = o_s[i];
}

// Joins the partials of one (sequence, kv head, q head) in chunk order.
template <typename T>
__global__ void __launch_bounds__(kGenThreads) int4_merge_kernel(const Int4DecodeParams p, int chunk, int max_split) {
  const int G = p.group, D = p.head_dim;
  const int64_t bh = blockIdx.x / G;
  const int g = static_cast<int>(blockIdx.x - bh * G);
  const int h = static_cast<int>(bh % p.hkv), b = static_cast<int>(bh / p.hkv);
  const int nsplit = (clamp_ctx(p, b, false) + chunk - 1) / chunk;
  if (nsplit <= 1) return;
  const int64_t stride = gen_part_floats(G, D);
  const float* part = p.part + bh * max_split * stride;
  float m = -INFINITY;
  for (int c = 0; c < nsplit; ++c) m = fmaxf(m, part[c * stride + g]);
  const float mu = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  for (int c = 0; c < nsplit; ++c) l = fmaf(part[c * stride + G + g], exp2f(part[c * stride + g] - mu), l);
  for (int d = threadIdx.x; d < D; d += kGenThreads) {
    float acc = 0.f;
    for (int c = 0; c < nsplit; ++c)
      acc = fmaf(part[c * stride + 2 * G + g * D + d], exp2f(part[c * stride + g] - mu), acc);
    reinterpret_cast<T*>(p.out)[b * p.osb + (h * G + g) * p.osh + d] = Elem<T>::from_float(l == 0.f ? 0.f : acc / l);
  }
}

// Context split of the generic path: chunks of a multiple of 64 tokens, long
// enough that the units stay near eight per SM of a full-size GPU.
constexpr int64_t kGenUnits = 1184;

struct GenSplit {
  int chunk, max_split;
};

GenSplit gen_split(int batch, int hkv, int max_context) {
  const int64_t bh = static_cast<int64_t>(batch) * hkv;
  const int64_t per = std::max<int64_t>(1, kGenUnits / bh);
  int64_t chunk = (std::max(1, max_context) + per - 1) / per;
  chunk = (chunk + kGenStep - 1) / kGenStep * kGenStep;
  return {static_cast<int>(chunk), static_cast<int>(std::max<int64_t>(1, (max_context + chunk - 1) / chunk))};
}

size_t gen_workspace(int batch, int hkv, int group, int head_dim, int max_context) {
  const GenSplit s = gen_split(batch, hkv, max_context);
  if (s.max_split == 1) return 0;
  return sizeof(float) * static_cast<size_t>(batch) * hkv * s.max_split * gen_part_floats(group, head_dim);
}

template <typename T>
int launch_generic(const Int4DecodeParams& p, cudaStream_t s) {
  const GenSplit sp = gen_split(p.batch, p.hkv, p.max_context);
  const size_t smem = sizeof(float) * GenLayout(p.group, p.head_dim).total;
  if (smem > 227 * 1024) return PSB_ERR_UNSUPPORTED;
  int occ = 0;
  if (!kernel_occupancy(reinterpret_cast<const void*>(int4_decode_generic_kernel<T>), kGenThreads, smem, &occ))
    return PSB_ERR_CUDA;
  const int64_t units = static_cast<int64_t>(p.batch) * p.hkv * sp.max_split;
  const int64_t merges = static_cast<int64_t>(p.batch) * p.hq;
  if (units >= (int64_t(1) << 31) || merges >= (int64_t(1) << 31)) return PSB_ERR_UNSUPPORTED;
  discard_stale_error();
  int4_decode_generic_kernel<T><<<static_cast<unsigned>(units), kGenThreads, smem, s>>>(p, sp.chunk, sp.max_split);
  if (sp.max_split > 1)
    int4_merge_kernel<T><<<static_cast<unsigned>(merges), kGenThreads, 0, s>>>(p, sp.chunk, sp.max_split);
  return check_launch();
}

}  // namespace
}  // namespace psb

using namespace psb;

extern "C" size_t psb_paged_decode_int4_workspace_size(int32_t batch, int32_t q_heads, int32_t num_kv_heads,
                                                       int32_t head_dim, int32_t block_size, int32_t max_context,
                                                       int32_t dtype) {
  if (batch <= 0 || num_kv_heads <= 0 || q_heads <= 0 || q_heads % num_kv_heads || head_dim <= 0 || head_dim % 2 ||
      head_dim > kInt4MaxDim || block_size <= 0 || max_context < 0 ||
      (dtype != PSB_F32 && dtype != PSB_F16 && dtype != PSB_BF16))
    return 0;
  // for whichever path the geometry allows (the fast path also needs aligned
  // rows, known only at the call)
  const int group = q_heads / num_kv_heads;
  const size_t fast = int4_decode_fast_geometry(dtype, batch, num_kv_heads, group, head_dim, block_size, max_context, 1, 1)
                          ? int4_decode_fast_workspace(group, head_dim) : 0;
  return std::max({size_t(256), fast, gen_workspace(batch, num_kv_heads, group, head_dim, max_context)});
}

extern "C" int psb_paged_decode_int4(const void* query, int64_t q_stride_b, int64_t q_stride_h, void* out,
                                     int64_t o_stride_b, int64_t o_stride_h, const void* kv_codes,
                                     const void* kv_params, const int32_t* block_tables, int64_t table_stride,
                                     const int32_t* context_lens, int32_t batch, int32_t q_heads, int32_t layer,
                                     int32_t num_layers, int64_t num_blocks, int32_t num_kv_heads,
                                     int32_t block_size, int32_t head_dim, int32_t dtype, int32_t max_context,
                                     float scale, void* workspace, size_t workspace_bytes, int32_t* error_flag,
                                     psb_stream_t stream) {
  if (!query || !out || !kv_codes || !kv_params || !block_tables || !context_lens) return PSB_ERR_INVALID;
  if (batch <= 0 || q_heads <= 0 || num_kv_heads <= 0 || q_heads % num_kv_heads || head_dim <= 0 || head_dim % 2 ||
      head_dim > kInt4MaxDim || block_size <= 0 || num_blocks <= 0 || num_layers <= 0 || layer < 0 ||
      layer >= num_layers || max_context < 0 ||
      table_stride < (static_cast<int64_t>(max_context) + block_size - 1) / block_size)
    return PSB_ERR_INVALID;
  if (dtype != PSB_F32 && dtype != PSB_F16 && dtype != PSB_BF16) return PSB_ERR_INVALID;
  if (reinterpret_cast<uintptr_t>(kv_codes) % 16 || reinterpret_cast<uintptr_t>(kv_params) % 16 ||
      reinterpret_cast<uintptr_t>(workspace) % 16)
    return PSB_ERR_INVALID;
  if (workspace == nullptr ||
      workspace_bytes < psb_paged_decode_int4_workspace_size(batch, q_heads, num_kv_heads, head_dim, block_size,
                                                             max_context, dtype))
    return PSB_ERR_WORKSPACE;
  Int4DecodeParams p;
  p.q = query;
  p.qsb = q_stride_b;
  p.qsh = q_stride_h;
  p.out = out;
  p.osb = o_stride_b;
  p.osh = o_stride_h;
  p.codes = static_cast<const uint8_t*>(kv_codes);
  p.params = kv_params;
  p.tables = block_tables;
  p.table_stride = table_stride;
  p.ctx = context_lens;
  p.batch = batch;
  p.hq = q_heads;
  p.hkv = num_kv_heads;
  p.group = q_heads / num_kv_heads;
  p.block_size = block_size;
  p.head_dim = head_dim;
  p.max_context = max_context;
  p.num_blocks = num_blocks;
  p.layer_tiles = static_cast<int64_t>(layer) * num_blocks * num_kv_heads;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.part = static_cast<float*>(workspace);
  p.err = error_flag;
  p.tile_div = 0;
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const bool aligned = q_stride_b % 8 == 0 && q_stride_h % 8 == 0 && o_stride_b % 8 == 0 && o_stride_h % 8 == 0 &&
                       reinterpret_cast<uintptr_t>(query) % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0;
  if (aligned && int4_decode_fast_geometry(dtype, batch, num_kv_heads, p.group, head_dim, block_size, max_context,
                                            num_layers, num_blocks))
    return int4_decode_fast_launch(p, dtype, s);
  switch (dtype) {
    case PSB_BF16: return launch_generic<__nv_bfloat16>(p, s);
    case PSB_F16: return launch_generic<__half>(p, s);
    default: return launch_generic<float>(p, s);
  }
}
