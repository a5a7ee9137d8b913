// Writes into the 4-bit KV pool and the read-back of its rows.
//
// reshape_and_cache_int4 quantises each new token's K and V rows and scatters
// codes and parameters through the int64 slot mapping;
// rope_reshape_and_cache_int4 rotates q and k first (the products and the sum
// rounded to the storage type, as rope_reshape_and_cache rounds them) and
// quantises the rounded key; gather_cache_int4 returns the values stored at
// given slots.  The format is in int4_cache.cuh.
//
// One warp takes one row (q, k or v of one head of one token): lane l holds
// the element pairs l, l + 32, ... and a pair is one byte of codes.
#include <algorithm>

#include "common.cuh"
#include "host_util.h"
#include "int4_cache.cuh"

namespace psb {
namespace {

struct Int4WriteParams {
  const char* q;  // null without RoPE
  int64_t qst, qsh;
  char* qo;
  int64_t qost, qosh;
  const char* k;
  int64_t kst, ksh;
  char* ko;  // may be null
  int64_t kost, kosh;
  const char* v;
  int64_t vst, vsh;  // all strides in elements
  const char* cos;
  const char* sin;
  int64_t cst;
  uint8_t* codes;
  char* params;
  const int64_t* slots;
  int32_t tokens, hq, hkv, block_size, head_dim;
  int64_t layer_tiles, pool_slots;
  int32_t* err;
};

constexpr int kWriteThreads = 256;
constexpr int kPairs = kInt4MaxDim / 64;  // element pairs per lane at most

template <typename T>
__device__ __forceinline__ float rnd(float x) {
  return Elem<T>::to_float(Elem<T>::from_float(x));
}

template <typename T, bool ROPE>
__global__ void __launch_bounds__(kWriteThreads) int4_write_kernel(const Int4WriteParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int D = p.head_dim, half = D / 2, pairs = D / 2;
  const int heads = (ROPE ? p.hq : 0) + 2 * p.hkv;
  const int64_t units = static_cast<int64_t>(p.tokens) * heads;
  const int64_t warps = static_cast<int64_t>(gridDim.x) * (kWriteThreads / 32);
  for (int64_t u = blockIdx.x * static_cast<int64_t>(kWriteThreads / 32) + (threadIdx.x >> 5); u < units; u += warps) {
    const int64_t t = u / heads;
    int h = static_cast<int>(u - t * heads);
    int role = 0;  // 0 q, 1 k, 2 v
    if (ROPE && h >= p.hq) {
      h -= p.hq;
      role = 1;
    } else if (!ROPE) {
      role = 1;
    }
    if (role == 1 && h >= p.hkv) {
      h -= p.hkv;
      role = 2;
    }
    const T* src = reinterpret_cast<const T*>(role == 0 ? p.q : role == 1 ? p.k : p.v) +
                   t * (role == 0 ? p.qst : role == 1 ? p.kst : p.vst) +
                   h * (role == 0 ? p.qsh : role == 1 ? p.ksh : p.vsh);
    float x[kPairs][2];
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      const int j = lane + 32 * i;
      if (j >= pairs) continue;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int d = 2 * j + e;
        float a = Elem<T>::to_float(src[d]);
        if (ROPE && role < 2) {
          const float b = d < half ? -Elem<T>::to_float(src[d + half]) : Elem<T>::to_float(src[d - half]);
          const float c = Elem<T>::to_float(reinterpret_cast<const T*>(p.cos)[t * p.cst + d]);
          const float s = Elem<T>::to_float(reinterpret_cast<const T*>(p.sin)[t * p.cst + d]);
          a = rnd<T>(__fadd_rn(rnd<T>(__fmul_rn(a, c)), rnd<T>(__fmul_rn(b, s))));
        }
        x[i][e] = a;
      }
    }
    if (ROPE && role < 2) {
      __syncwarp();  // query_out may be query itself: every lane has read the row before any writes it
      T* dst = role == 0 ? reinterpret_cast<T*>(p.qo) + t * p.qost + h * p.qosh
                         : p.ko ? reinterpret_cast<T*>(p.ko) + t * p.kost + h * p.kosh : nullptr;
      if (dst != nullptr) {
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
          const int j = lane + 32 * i;
          if (j >= pairs) continue;
          dst[2 * j] = Elem<T>::from_float(x[i][0]);
          dst[2 * j + 1] = Elem<T>::from_float(x[i][1]);
        }
      }
      if (role == 0) continue;
    }
    const int64_t slot = __ldg(p.slots + t);
    if (slot < 0) continue;
    if (slot >= p.pool_slots) {
      if (lane == 0 && h == 0 && role == 1) flag_error(p.err, PSB_DEVERR_SLOT_RANGE);
      continue;
    }
    float lo = INFINITY, hi = -INFINITY;
    bool finite = true;
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      if (lane + 32 * i >= pairs) continue;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        lo = fminf(lo, x[i][e]);
        hi = fmaxf(hi, x[i][e]);
        finite = finite && finite_f32(x[i][e]);
      }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
      hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    finite = __all_sync(0xffffffffu, finite);
    T step, mid;
    int4_row_params<T>(lo, hi, finite, step, mid);
    const float st = Elem<T>::to_float(step), md = Elem<T>::to_float(mid);
    const int64_t blk = slot / p.block_size;
    const int64_t row = int4_row(p.layer_tiles + blk * p.hkv + h, role - 1, static_cast<int>(slot - blk * p.block_size),
                                 p.block_size);
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      const int j = lane + 32 * i;
      if (j >= pairs) continue;
      p.codes[row * pairs + j] =
          static_cast<uint8_t>(int4_code(x[i][0], st, md) | (int4_code(x[i][1], st, md) << 4));
    }
    if (lane == 0) {
      T* pr = reinterpret_cast<T*>(p.params) + row * 2;
      pr[0] = step;
      pr[1] = mid;
    }
  }
}

struct Int4GatherParams {
  const uint8_t* codes;
  const char* params;
  char* k;
  int64_t kst, ksh;
  char* v;
  int64_t vst, vsh;  // elements
  const int64_t* slots;
  int32_t tokens, hkv, block_size, head_dim;
  int64_t layer_tiles, pool_slots;
  int32_t* err;
};

template <typename T>
__global__ void __launch_bounds__(kWriteThreads) int4_gather_kernel(const Int4GatherParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int pairs = p.head_dim / 2;
  const int64_t per_tok = static_cast<int64_t>(2) * p.hkv * pairs;
  const int64_t total = per_tok * p.tokens;
  for (int64_t i = blockIdx.x * static_cast<int64_t>(kWriteThreads) + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * kWriteThreads) {
    const int64_t t = i / per_tok;
    int r = static_cast<int>(i - t * per_tok);
    const int j = r % pairs;
    r /= pairs;
    const int kv = r / p.hkv, h = r - kv * p.hkv;
    const int64_t slot = __ldg(p.slots + t);
    float a = 0.f, b = 0.f;
    if (slot >= p.pool_slots) {
      if (r == 0 && j == 0) flag_error(p.err, PSB_DEVERR_SLOT_RANGE);
    } else if (slot >= 0) {
      const int64_t blk = slot / p.block_size;
      const int64_t row = int4_row(p.layer_tiles + blk * p.hkv + h, kv, static_cast<int>(slot - blk * p.block_size),
                                   p.block_size);
      const uint32_t c = p.codes[row * pairs + j];
      const T* pr = reinterpret_cast<const T*>(p.params) + row * 2;
      const float st = Elem<T>::to_float(pr[0]), md = Elem<T>::to_float(pr[1]);
      a = int4_value(c & 15u, st, md);
      b = int4_value(c >> 4, st, md);
    }
    T* dst = kv ? reinterpret_cast<T*>(p.v) + t * p.vst + h * p.vsh : reinterpret_cast<T*>(p.k) + t * p.kst + h * p.ksh;
    dst[2 * j] = Elem<T>::from_float(a);
    dst[2 * j + 1] = Elem<T>::from_float(b);
  }
}

template <typename T, bool ROPE>
int launch_write(const Int4WriteParams& p, cudaStream_t s, int sms) {
  const int64_t units = static_cast<int64_t>(p.tokens) * ((ROPE ? p.hq : 0) + 2 * p.hkv);
  const int64_t blocks = std::max<int64_t>(1, std::min<int64_t>((units + 7) / 8, static_cast<int64_t>(sms) * 8));
  const auto kern = int4_write_kernel<T, ROPE>;
  if (!prefer_max_l1(reinterpret_cast<const void*>(kern))) return PSB_ERR_CUDA;
  discard_stale_error();
  const cudaError_t e = launch_pdl(kern, dim3(static_cast<unsigned>(blocks)), dim3(kWriteThreads), 0, s, p);
  if (e != cudaSuccess) return record_cuda_error(e);
  return check_launch();
}

template <typename T>
int launch_gather(const Int4GatherParams& p, cudaStream_t s, int sms) {
  const int64_t total = static_cast<int64_t>(p.tokens) * p.hkv * p.head_dim;
  const int64_t blocks = std::max<int64_t>(
      1, std::min<int64_t>((total + kWriteThreads - 1) / kWriteThreads, static_cast<int64_t>(sms) * 8));
  const auto kern = int4_gather_kernel<T>;
  if (!prefer_max_l1(reinterpret_cast<const void*>(kern))) return PSB_ERR_CUDA;
  discard_stale_error();
  const cudaError_t e = launch_pdl(kern, dim3(static_cast<unsigned>(blocks)), dim3(kWriteThreads), 0, s, p);
  if (e != cudaSuccess) return record_cuda_error(e);
  return check_launch();
}

bool geometry_ok(int32_t num_tokens, int32_t layer, int32_t num_layers, int64_t num_blocks, int32_t num_kv_heads,
                 int32_t block_size, int32_t head_dim, int32_t dtype) {
  return num_tokens >= 0 && num_layers > 0 && layer >= 0 && layer < num_layers && num_blocks > 0 && num_kv_heads > 0 &&
         block_size > 0 && head_dim > 0 && head_dim % 2 == 0 && head_dim <= kInt4MaxDim &&
         (dtype == PSB_F32 || dtype == PSB_F16 || dtype == PSB_BF16);
}

// Parameter pairs are read and written as pairs, code rows in words where
// their length allows: the pools start on 16 bytes.
bool pools_aligned(const void* codes, const void* params) {
  return reinterpret_cast<uintptr_t>(codes) % 16 == 0 && reinterpret_cast<uintptr_t>(params) % 16 == 0;
}

}  // namespace
}  // namespace psb

using namespace psb;

extern "C" int psb_reshape_and_cache_int4(const void* key, int64_t key_stride_t, int64_t key_stride_h,
                                          const void* value, int64_t value_stride_t, int64_t value_stride_h,
                                          void* kv_codes, void* kv_params, const int64_t* slot_mapping,
                                          int32_t num_tokens, int32_t layer, int32_t num_layers, int64_t num_blocks,
                                          int32_t num_kv_heads, int32_t block_size, int32_t head_dim, int32_t dtype,
                                          int32_t* error_flag, psb_stream_t stream) {
  if (!geometry_ok(num_tokens, layer, num_layers, num_blocks, num_kv_heads, block_size, head_dim, dtype))
    return PSB_ERR_INVALID;
  if (num_tokens == 0) return PSB_OK;
  if (!key || !value || !kv_codes || !kv_params || !slot_mapping || !pools_aligned(kv_codes, kv_params))
    return PSB_ERR_INVALID;
  const int sms = device_sm_count();
  if (sms <= 0) return PSB_ERR_CUDA;
  Int4WriteParams p{};
  p.k = static_cast<const char*>(key);
  p.kst = key_stride_t;
  p.ksh = key_stride_h;
  p.v = static_cast<const char*>(value);
  p.vst = value_stride_t;
  p.vsh = value_stride_h;
  p.codes = static_cast<uint8_t*>(kv_codes);
  p.params = static_cast<char*>(kv_params);
  p.slots = slot_mapping;
  p.tokens = num_tokens;
  p.hkv = num_kv_heads;
  p.block_size = block_size;
  p.head_dim = head_dim;
  p.layer_tiles = static_cast<int64_t>(layer) * num_blocks * num_kv_heads;
  p.pool_slots = num_blocks * block_size;
  p.err = error_flag;
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  switch (dtype) {
    case PSB_BF16: return launch_write<__nv_bfloat16, false>(p, s, sms);
    case PSB_F16: return launch_write<__half, false>(p, s, sms);
    default: return launch_write<float, false>(p, s, sms);
  }
}

extern "C" int psb_rope_reshape_and_cache_int4(
    const void* query, int64_t q_stride_t, int64_t q_stride_h, void* query_out, int64_t qo_stride_t,
    int64_t qo_stride_h, const void* key, int64_t k_stride_t, int64_t k_stride_h, void* key_out, int64_t ko_stride_t,
    int64_t ko_stride_h, const void* value, int64_t v_stride_t, int64_t v_stride_h, const void* cos, const void* sin,
    int64_t cs_stride_t, void* kv_codes, void* kv_params, const int64_t* slot_mapping, int32_t num_tokens,
    int32_t num_q_heads, int32_t layer, int32_t num_layers, int64_t num_blocks, int32_t num_kv_heads,
    int32_t block_size, int32_t head_dim, int32_t dtype, int32_t* error_flag, psb_stream_t stream) {
  if (!geometry_ok(num_tokens, layer, num_layers, num_blocks, num_kv_heads, block_size, head_dim, dtype) ||
      num_q_heads < 0)
    return PSB_ERR_INVALID;
  if (num_tokens == 0) return PSB_OK;
  if (!key || !value || !cos || !sin || !kv_codes || !kv_params || !slot_mapping ||
      !pools_aligned(kv_codes, kv_params) || (num_q_heads > 0 && (!query || !query_out)))
    return PSB_ERR_INVALID;
  const int sms = device_sm_count();
  if (sms <= 0) return PSB_ERR_CUDA;
  Int4WriteParams p{};
  p.q = static_cast<const char*>(query);
  p.qst = q_stride_t;
  p.qsh = q_stride_h;
  p.qo = static_cast<char*>(query_out);
  p.qost = qo_stride_t;
  p.qosh = qo_stride_h;
  p.k = static_cast<const char*>(key);
  p.kst = k_stride_t;
  p.ksh = k_stride_h;
  p.ko = static_cast<char*>(key_out);
  p.kost = ko_stride_t;
  p.kosh = ko_stride_h;
  p.v = static_cast<const char*>(value);
  p.vst = v_stride_t;
  p.vsh = v_stride_h;
  p.cos = static_cast<const char*>(cos);
  p.sin = static_cast<const char*>(sin);
  p.cst = cs_stride_t;
  p.codes = static_cast<uint8_t*>(kv_codes);
  p.params = static_cast<char*>(kv_params);
  p.slots = slot_mapping;
  p.tokens = num_tokens;
  p.hq = num_q_heads;
  p.hkv = num_kv_heads;
  p.block_size = block_size;
  p.head_dim = head_dim;
  p.layer_tiles = static_cast<int64_t>(layer) * num_blocks * num_kv_heads;
  p.pool_slots = num_blocks * block_size;
  p.err = error_flag;
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  switch (dtype) {
    case PSB_BF16: return launch_write<__nv_bfloat16, true>(p, s, sms);
    case PSB_F16: return launch_write<__half, true>(p, s, sms);
    default: return launch_write<float, true>(p, s, sms);
  }
}

extern "C" int psb_gather_cache_int4(const void* kv_codes, const void* kv_params, const int64_t* slot_mapping,
                                     void* key_out, int64_t key_stride_t, int64_t key_stride_h, void* value_out,
                                     int64_t value_stride_t, int64_t value_stride_h, int32_t num_tokens,
                                     int32_t layer, int32_t num_layers, int64_t num_blocks, int32_t num_kv_heads,
                                     int32_t block_size, int32_t head_dim, int32_t dtype, int32_t* error_flag,
                                     psb_stream_t stream) {
  if (!geometry_ok(num_tokens, layer, num_layers, num_blocks, num_kv_heads, block_size, head_dim, dtype))
    return PSB_ERR_INVALID;
  if (num_tokens == 0) return PSB_OK;
  if (!key_out || !value_out || !kv_codes || !kv_params || !slot_mapping || !pools_aligned(kv_codes, kv_params))
    return PSB_ERR_INVALID;
  const int sms = device_sm_count();
  if (sms <= 0) return PSB_ERR_CUDA;
  Int4GatherParams p{};
  p.codes = static_cast<const uint8_t*>(kv_codes);
  p.params = static_cast<const char*>(kv_params);
  p.k = static_cast<char*>(key_out);
  p.kst = key_stride_t;
  p.ksh = key_stride_h;
  p.v = static_cast<char*>(value_out);
  p.vst = value_stride_t;
  p.vsh = value_stride_h;
  p.slots = slot_mapping;
  p.tokens = num_tokens;
  p.hkv = num_kv_heads;
  p.block_size = block_size;
  p.head_dim = head_dim;
  p.layer_tiles = static_cast<int64_t>(layer) * num_blocks * num_kv_heads;
  p.pool_slots = num_blocks * block_size;
  p.err = error_flag;
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  switch (dtype) {
    case PSB_BF16: return launch_gather<__nv_bfloat16>(p, s, sms);
    case PSB_F16: return launch_gather<__half>(p, s, sms);
    default: return launch_gather<float>(p, s, sms);
  }
}
