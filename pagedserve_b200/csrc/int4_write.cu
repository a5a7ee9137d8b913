// Writes into the 4-bit KV pool and the read-back of its rows.
//
// reshape_and_cache_int4 quantises each new token's K and V rows and scatters
// codes and parameters through the int64 slot mapping;
// rope_reshape_and_cache_int4 rotates q and k first (the products and the sum
// rounded to the storage type, as rope_reshape_and_cache rounds them) and
// quantises the rounded key; gather_cache_int4 returns the values stored at
// given slots.  The format is in int4_cache.cuh.
//
// All three are bound by HBM (a 16 K-token pack of 14 + 2 heads moves 80 MB,
// three quarters of it q in and out), so a thread moves 16-byte pieces: one of
// each half of a row, which the rotation pairs, and the rows' extremes meet in
// two to five shuffles between the row's threads.  A thread's eight codes of a
// piece are one word.  Rows that are not 16-byte aligned, or whose pieces are
// not a power of two, take a warp per row instead: lane l holds the element
// pairs l, l + 32, ... and a pair is one byte of codes.
//
// Measured, write and read-back together: a 16 K-token pack of 14 + 2 heads of
// head_dim 64 22.2 us (86 MB: 3.9 TB/s, 60% of the copy rate; a warp per row
// took 131 us, a division per code 42 us, index divisions and conversions of
// codes by instructions of their own 25.5 us), 1333 plain tokens of 8 heads of
// 128 in f16 8.8 us, 256 tokens 4.4 us.  Instructions, not HBM, are what is
// left: 290 per 16 elements written, 170 per 8 read back.
#include <algorithm>

#include "common.cuh"
#include "host_util.h"
#include "int4_cache.cuh"

namespace psb {
namespace {

// Division by a divisor of the launch: n / d = (mulhi(n, mul) + n) >> shift for
// 0 <= n < 2^31, with shift = ceil(log2 d) and mul = floor(2^32 (2^shift - d) / d) + 1
// (Granlund and Montgomery, Division by invariant integers using multiplication,
// 1994); 64-bit indices divide.
struct Divisor {
  uint32_t d, mul, shift;
};

Divisor divisor(int64_t d) {
  Divisor v{static_cast<uint32_t>(d), 0, 0};
  while ((int64_t(1) << v.shift) < d) ++v.shift;
  v.mul = static_cast<uint32_t>((((uint64_t(1) << v.shift) - static_cast<uint64_t>(d)) << 32) / static_cast<uint64_t>(d) + 1);
  return v;
}

__device__ __forceinline__ int32_t divide(int32_t n, const Divisor& v) {
  return static_cast<int32_t>((__umulhi(static_cast<uint32_t>(n), v.mul) + static_cast<uint32_t>(n)) >> v.shift);
}
__device__ __forceinline__ int64_t divide(int64_t n, const Divisor& v) { return n / v.d; }

// log2 of a power of two, -1 for the rest.
int log2_exact(int64_t n) {
  if (n & (n - 1)) return -1;
  int s = 0;
  while ((int64_t(1) << s) < n) ++s;
  return s;
}

// Pool row of kv (0 K, 1 V) of a slot for head h.
template <typename P>
__device__ __forceinline__ int64_t slot_row(const P& p, int64_t slot, int h, int kv) {
  const int64_t blk = p.block_shift >= 0 ? slot >> p.block_shift : slot / p.block_size;
  return int4_row(p.layer_tiles + blk * p.hkv + h, kv, static_cast<int>(slot - blk * p.block_size), p.block_size);
}

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
  int32_t tokens, hq, hkv, block_size, block_shift, head_dim;
  Divisor q_div, kv_div;  // pieces of a token's q rows, of its k and v rows (vector kernel)
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
    const int64_t row = slot_row(p, slot, h, role - 1);
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

// VEC consecutive elements, moved as one 16-byte access.
template <typename T>
struct Piece16 {
  static constexpr int kVec = 16 / sizeof(T);
  alignas(16) T e[kVec];
  __device__ __forceinline__ void load(const T* src) { *reinterpret_cast<uint4*>(e) = *reinterpret_cast<const uint4*>(src); }
  __device__ __forceinline__ void store(T* dst) const { *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(e); }
};

// Codes of a piece: 8 a word (16-bit types) or 4 in its low half (fp32).
template <typename T>
__device__ __forceinline__ uint32_t piece_codes(const Piece16<T>& x, float step, float mid) {
  uint32_t w = 0;
  if constexpr (sizeof(T) == 2) {
    if (step > 1e-30f) {
      const float inv = __frcp_rn(step);
#pragma unroll
      for (int i = 0; i < Piece16<T>::kVec; ++i) w |= int4_code16(Elem<T>::to_float(x.e[i]), step, mid, inv) << (4 * i);
      return w;
    }
  }
#pragma unroll
  for (int i = 0; i < Piece16<T>::kVec; ++i) w |= int4_code(Elem<T>::to_float(x.e[i]), step, mid) << (4 * i);
  return w;
}

// a b and a + b of packed 16-bit pairs, rounded as PyTorch rounds the two
// operations (an explicit .rn is never contracted into a multiply-add).
template <typename T> struct Pair;
template <> struct Pair<__nv_bfloat16> {
  __device__ static uint32_t mul(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
  }
  __device__ static uint32_t add(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
  }
};
template <> struct Pair<__half> {
  __device__ static uint32_t mul(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
  }
  __device__ static uint32_t add(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("add.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
  }
};

// (a, b) -> (a cos - b sin, b cos + a sin), each product and sum rounded to T.
template <typename T>
__device__ __forceinline__ void rotate(Piece16<T>& a, Piece16<T>& b, const Piece16<T>& c1, const Piece16<T>& c2,
                                       const Piece16<T>& s1, const Piece16<T>& s2) {
  if constexpr (sizeof(T) == 2) {
    uint32_t* x = reinterpret_cast<uint32_t*>(a.e);
    uint32_t* y = reinterpret_cast<uint32_t*>(b.e);
    const uint32_t* p1 = reinterpret_cast<const uint32_t*>(c1.e);
    const uint32_t* p2 = reinterpret_cast<const uint32_t*>(c2.e);
    const uint32_t* q1 = reinterpret_cast<const uint32_t*>(s1.e);
    const uint32_t* q2 = reinterpret_cast<const uint32_t*>(s2.e);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t u = x[j], v = y[j];
      x[j] = Pair<T>::add(Pair<T>::mul(u, p1[j]), Pair<T>::mul(v ^ 0x80008000u, q1[j]));
      y[j] = Pair<T>::add(Pair<T>::mul(v, p2[j]), Pair<T>::mul(u, q2[j]));
    }
  } else {
#pragma unroll
    for (int j = 0; j < Piece16<T>::kVec; ++j) {
      const float x = a.e[j], y = b.e[j];
      a.e[j] = __fadd_rn(__fmul_rn(x, c1.e[j]), __fmul_rn(-y, s1.e[j]));
      b.e[j] = __fadd_rn(__fmul_rn(y, c2.e[j]), __fmul_rn(x, s2.e[j]));
    }
  }
}

// One thread per (token, head, piece of a half row); ``pieces`` consecutive
// lanes hold one row.  The q rows of all tokens come first, then the k and v
// rows, so that a warp's lanes share a path.  (Idx: int32 while every index fits.)
template <typename T, bool ROPE, typename Idx>
__global__ void __launch_bounds__(kWriteThreads) int4_write_vec_kernel(const Int4WriteParams p, int log_pieces) {
  constexpr int VEC = Piece16<T>::kVec;
  pdl_launch_dependents();
  pdl_wait();
  const int half = p.head_dim / 2, pieces = 1 << log_pieces;
  const Idx q_tok = static_cast<Idx>(ROPE ? p.hq : 0) * pieces, kv_tok = static_cast<Idx>(2 * p.hkv) * pieces;
  const Idx q_total = q_tok * p.tokens, total = q_total + kv_tok * p.tokens;
  const int lane = threadIdx.x & 31;
  for (Idx base = (blockIdx.x * static_cast<Idx>(kWriteThreads) + threadIdx.x) & ~static_cast<Idx>(31); base < total;
       base += static_cast<Idx>(gridDim.x) * kWriteThreads) {
    // Lanes past the end take part in the warp's shuffles and votes only: each of
    // them holds the last piece, not a row, so its extremes are not the row's and
    // it stores nothing.
    const bool live = base + lane < total;
    const Idx i = min(base + lane, total - 1);
    const bool is_q = ROPE && i < q_total;
    const Idx u = is_q ? i : i - q_total, per = is_q ? q_tok : kv_tok;
    const Idx t = divide(u, is_q ? p.q_div : p.kv_div);
    const int r = static_cast<int>(u - t * per);
    int h = r >> log_pieces;
    const int e0 = (r & (pieces - 1)) * VEC;
    int role = is_q ? 0 : 1;  // 0 q, 1 k, 2 v
    if (!is_q && h >= p.hkv) {
      role = 2;
      h -= p.hkv;
    }
    const T* src = reinterpret_cast<const T*>(role == 0 ? p.q : role == 1 ? p.k : p.v) +
                   t * (role == 0 ? p.qst : role == 1 ? p.kst : p.vst) +
                   h * (role == 0 ? p.qsh : role == 1 ? p.ksh : p.vsh) + e0;
    Piece16<T> a, b;
    a.load(src);
    b.load(src + half);
    int64_t slot = -1;
    if (role && live) slot = __ldg(p.slots + t);
    if (ROPE && role < 2) {
      const T* cs = reinterpret_cast<const T*>(p.cos) + t * p.cst + e0;
      const T* sn = reinterpret_cast<const T*>(p.sin) + t * p.cst + e0;
      Piece16<T> c1, c2, s1, s2;
      c1.load(cs);
      c2.load(cs + half);
      s1.load(sn);
      s2.load(sn + half);
      rotate(a, b, c1, c2, s1, s2);
    }
    if (ROPE) {
      __syncwarp();  // in place: the lanes past the end have read the last piece before its own lane writes it
      T* dst = role == 0 ? reinterpret_cast<T*>(p.qo) + t * p.qost + h * p.qosh + e0
                         : role == 1 && p.ko ? reinterpret_cast<T*>(p.ko) + t * p.kost + h * p.kosh + e0 : nullptr;
      if (dst != nullptr && live) {
        a.store(dst);
        b.store(dst + half);
      }
    }
    if (!__any_sync(0xffffffffu, slot >= 0)) continue;
    float lo = INFINITY, hi = -INFINITY, bad = 0.f;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const float x = Elem<T>::to_float(a.e[j]), y = Elem<T>::to_float(b.e[j]);
      lo = fminf(lo, fminf(x, y));
      hi = fmaxf(hi, fmaxf(x, y));
      if (!finite_f32(x) || !finite_f32(y)) bad = 1.f;
    }
    for (int o = 1; o < pieces; o <<= 1) {
      lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
      hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
      bad = fmaxf(bad, __shfl_xor_sync(0xffffffffu, bad, o));
    }
    if (slot < 0) continue;
    if (slot >= p.pool_slots) {
      if (e0 == 0 && h == 0 && role == 1) flag_error(p.err, PSB_DEVERR_SLOT_RANGE);
      continue;
    }
    T step, mid;
    int4_row_params<T>(lo, hi, bad == 0.f, step, mid);
    const float st = Elem<T>::to_float(step), md = Elem<T>::to_float(mid);
    const int64_t row = slot_row(p, slot, h, role - 1);
    uint8_t* dst = p.codes + row * half + e0 / 2;
    const uint32_t ca = piece_codes(a, st, md), cb = piece_codes(b, st, md);
    if constexpr (VEC == 8) {
      *reinterpret_cast<uint32_t*>(dst) = ca;
      *reinterpret_cast<uint32_t*>(dst + half / 2) = cb;
    } else {
      *reinterpret_cast<uint16_t*>(dst) = static_cast<uint16_t>(ca);
      *reinterpret_cast<uint16_t*>(dst + half / 2) = static_cast<uint16_t>(cb);
    }
    if (e0 == 0) {
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
  int32_t tokens, hkv, block_size, block_shift, head_dim;
  Divisor tok_div, row_div;  // pieces of a token, of a row (vector kernel)
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
      const int64_t row = slot_row(p, slot, h, kv);
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

// One thread per VEC elements of a row.  (Idx: int32 while every index fits.)
template <typename T, typename Idx>
__global__ void __launch_bounds__(kWriteThreads) int4_gather_vec_kernel(const Int4GatherParams p) {
  constexpr int VEC = Piece16<T>::kVec;
  pdl_launch_dependents();
  pdl_wait();
  const int pieces = p.head_dim / VEC;
  const Idx per_tok = static_cast<Idx>(2) * p.hkv * pieces, total = per_tok * p.tokens;
  for (Idx i = blockIdx.x * static_cast<Idx>(kWriteThreads) + threadIdx.x; i < total;
       i += static_cast<Idx>(gridDim.x) * kWriteThreads) {
    const Idx t = divide(i, p.tok_div);
    const int r = static_cast<int>(i - t * per_tok);
    const int hv = divide(r, p.row_div), e0 = (r - hv * pieces) * VEC;
    const int kv = hv >= p.hkv ? 1 : 0, h = hv - kv * p.hkv;
    const int64_t slot = __ldg(p.slots + t);
    Piece16<T> x;
    *reinterpret_cast<uint4*>(x.e) = make_uint4(0, 0, 0, 0);
    if (slot >= p.pool_slots) {
      if (r == 0) flag_error(p.err, PSB_DEVERR_SLOT_RANGE);
    } else if (slot >= 0) {
      const int64_t row = slot_row(p, slot, h, kv);
      const uint8_t* src = p.codes + row * (p.head_dim / 2) + e0 / 2;
      const uint32_t w = VEC == 8 ? *reinterpret_cast<const uint32_t*>(src) : *reinterpret_cast<const uint16_t*>(src);
      const T* pr = reinterpret_cast<const T*>(p.params) + row * 2;
      const float st = Elem<T>::to_float(pr[0]), md = Elem<T>::to_float(pr[1]);
#pragma unroll
      for (int j = 0; j < VEC; ++j) x.e[j] = Elem<T>::from_float(fmaf(st, int4_centered(w, j), md));
    }
    x.store((kv ? reinterpret_cast<T*>(p.v) + t * p.vst + h * p.vsh : reinterpret_cast<T*>(p.k) + t * p.kst + h * p.ksh) + e0);
  }
}

bool aligned16(const void* ptr) { return reinterpret_cast<uintptr_t>(ptr) % 16 == 0; }

// Whether rows of these strides (elements of ``esz`` bytes) start on 16 bytes.
bool rows16(const void* ptr, int64_t st, int64_t sh, int esz) {
  return aligned16(ptr) && st * esz % 16 == 0 && sh * esz % 16 == 0;
}

// Lanes per row of the vector kernel, 0 when it does not apply.
template <typename T, bool ROPE>
int write_pieces(const Int4WriteParams& p) {
  constexpr int esz = sizeof(T), VEC = Piece16<T>::kVec;
  const int half = p.head_dim / 2, pieces = half / VEC;
  if (half % VEC || pieces > 32 || (pieces & (pieces - 1))) return 0;
  bool ok = rows16(p.k, p.kst, p.ksh, esz) && rows16(p.v, p.vst, p.vsh, esz);
  if (ROPE) {
    ok = ok && rows16(p.cos, p.cst, 0, esz) && rows16(p.sin, p.cst, 0, esz);
    if (p.hq > 0) ok = ok && rows16(p.q, p.qst, p.qsh, esz) && rows16(p.qo, p.qost, p.qosh, esz);
    if (p.ko != nullptr) ok = ok && rows16(p.ko, p.kost, p.kosh, esz);
  }
  return ok ? pieces : 0;
}

// One wave of resident CTAs striding over ``threads`` threads' work.
int64_t wave(const void* kern, int64_t threads, int sms) {
  const int occ = std::max(1, std::min(resident_ctas(kern, kWriteThreads, 0), 8));
  return std::max<int64_t>(1, std::min<int64_t>((threads + kWriteThreads - 1) / kWriteThreads,
                                                static_cast<int64_t>(sms) * occ));
}

template <typename... K, typename... A>
int launch_stream(void (*kern)(K...), int64_t blocks, cudaStream_t s, A... args) {
  if (!prefer_max_l1(reinterpret_cast<const void*>(kern))) return PSB_ERR_CUDA;
  discard_stale_error();
  const cudaError_t e = launch_pdl(kern, dim3(static_cast<unsigned>(blocks)), dim3(kWriteThreads), 0, s, args...);
  if (e != cudaSuccess) return record_cuda_error(e);
  return check_launch();
}

template <typename T, bool ROPE>
int launch_write(const Int4WriteParams& p, cudaStream_t s, int sms) {
  const int64_t rows = static_cast<int64_t>(p.tokens) * ((ROPE ? p.hq : 0) + 2 * p.hkv);
  if (const int pieces = write_pieces<T, ROPE>(p)) {
    const int64_t units = rows * pieces;
    // int32 indices while the last one and a grid stride past it fit
    const auto kern = units + static_cast<int64_t>(sms) * 8 * kWriteThreads < (int64_t(1) << 31)
                          ? int4_write_vec_kernel<T, ROPE, int32_t> : int4_write_vec_kernel<T, ROPE, int64_t>;
    Int4WriteParams v = p;
    v.q_div = divisor(static_cast<int64_t>(std::max(p.hq, 1)) * pieces);
    v.kv_div = divisor(static_cast<int64_t>(2) * p.hkv * pieces);
    return launch_stream(kern, wave(reinterpret_cast<const void*>(kern), units, sms), s, v, log2_exact(pieces));
  }
  const auto kern = int4_write_kernel<T, ROPE>;
  return launch_stream(kern, wave(reinterpret_cast<const void*>(kern), rows * 32, sms), s, p);
}

template <typename T>
int launch_gather(const Int4GatherParams& p, cudaStream_t s, int sms) {
  constexpr int esz = sizeof(T), VEC = Piece16<T>::kVec;
  const int64_t elems = static_cast<int64_t>(p.tokens) * 2 * p.hkv * p.head_dim;
  if (p.head_dim % VEC == 0 && rows16(p.k, p.kst, p.ksh, esz) && rows16(p.v, p.vst, p.vsh, esz)) {
    const int64_t units = elems / VEC;
    const auto kern = units + static_cast<int64_t>(sms) * 8 * kWriteThreads < (int64_t(1) << 31)
                          ? int4_gather_vec_kernel<T, int32_t> : int4_gather_vec_kernel<T, int64_t>;
    Int4GatherParams v = p;
    v.row_div = divisor(p.head_dim / VEC);
    v.tok_div = divisor(static_cast<int64_t>(2) * p.hkv * (p.head_dim / VEC));
    return launch_stream(kern, wave(reinterpret_cast<const void*>(kern), units, sms), s, v);
  }
  const auto kern = int4_gather_kernel<T>;
  return launch_stream(kern, wave(reinterpret_cast<const void*>(kern), elems / 2, sms), s, p);
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
  p.block_shift = log2_exact(block_size);
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
  p.block_shift = log2_exact(block_size);
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
  p.block_shift = log2_exact(block_size);
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
