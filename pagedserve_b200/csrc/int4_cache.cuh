// The 4-bit KV pool: format and element helpers shared by its kernels.
//
// One row x of head_dim values (one token, one kv head, K or V) of element
// type T is kept as one code per value and one (step, mid) pair of type T:
//     lo, hi = min x, max x
//     mid  = T(lo / 2 + hi / 2)
//     step = T(max(hi - mid, mid - lo) / 7.5)
//     code = clamp(floor((x - mid) / step) + 8, 0, 15), 8 where step is 0
//     x^   = mid + step (code - 7.5)
// with every operation before a rounding to T in fp32, so the codes are the
// same wherever fp32 arithmetic is IEEE.  A constant row (step 0) is exact;
// otherwise |x - x^| <= step / 2 plus what rounding step and mid to T moves
// (both ends of the row stay within a 7.5 step reach of mid up to one part
// in 2^(bits of T)).  A row that holds an infinity or a NaN gets mid = NaN:
// what it stands for is NaN throughout, never a finite guess.
//
// Pools (contiguous):
//     kv_codes  uint8 [num_layers, num_blocks, num_kv_heads, 2, block_size, head_dim / 2]
//     kv_params T     [num_layers, num_blocks, num_kv_heads, 2, block_size, 2]
// with K at index 0 and V at index 1 of the fourth axis, byte j of a code row
// holding elements 2 j (low half) and 2 j + 1 (high half), and a parameter
// pair (step, mid).  K and V of one (layer, block, kv head) are adjacent, so
// a 16-token block is one contiguous run of codes and one of parameters.
#pragma once

#include "common.cuh"

namespace psb {

constexpr float kInt4Mid = 7.5f;      // the code a row's mid corresponds to
constexpr int kInt4MaxDim = 256;      // head_dim limit of the 4-bit kernels

// Index of row ``tok`` of (tile = (layer * num_blocks + block) * num_kv_heads
// + head, kv): the row's codes start at byte index * head_dim / 2, its
// parameters at element index * 2.
__device__ __forceinline__ int64_t int4_row(int64_t tile, int kv, int tok, int block_size) {
  return (tile * 2 + kv) * block_size + tok;
}

// (step, mid) of a row from its extremes; finite is false when the row holds
// an infinity or a NaN.
template <typename T>
__device__ __forceinline__ void int4_row_params(float lo, float hi, bool finite, T& step, T& mid) {
  if (!finite) {
    step = Elem<T>::from_float(0.f);
    mid = Elem<T>::from_float(__int_as_float(0x7fffffff));
    return;
  }
  mid = Elem<T>::from_float(__fadd_rn(0.5f * lo, 0.5f * hi));
  const float m = Elem<T>::to_float(mid);
  step = Elem<T>::from_float(__fdiv_rn(fmaxf(__fsub_rn(hi, m), __fsub_rn(m, lo)), kInt4Mid));
}

__device__ __forceinline__ uint32_t int4_code(float x, float step, float mid) {
  if (!(step > 0.f)) return 8u;
  const float c = floorf(__fdiv_rn(__fsub_rn(x, mid), step)) + 8.f;
  return static_cast<uint32_t>(fminf(fmaxf(c, 0.f), 15.f));
}

// The same code for a step of a 16-bit type, without the division: the
// quotient's floor is estimated with inv ~ 1 / step (a finite normal number)
// and put right by the signs of two exact remainders.  That is the floor of
// the exact quotient, and of the rounded one too: d = fl(x - mid) and n step
// (at most 15 bits) are multiples of d's last place, so a quotient that is not
// the integer n is further from it than half a last place of n, and rounding
// never reaches n.
__device__ __forceinline__ uint32_t int4_code16(float x, float step, float mid, float inv) {
  constexpr float kMagic = 12582912.f;  // 1.5 2^23: adding it rounds to an integer
  const float d = __fsub_rn(x, mid);
  float f = __fadd_rn(__fmul_rn(d, inv), kMagic) - kMagic;
  if (fmaf(-f, step, d) < 0.f) f -= 1.f;
  else if (fmaf(-(f + 1.f), step, d) >= 0.f) f += 1.f;
  const int c = __float_as_int(f + kMagic) - __float_as_int(kMagic) + 8;
  return static_cast<uint32_t>(min(max(c, 0), 15));
}

__device__ __forceinline__ float int4_value(uint32_t code, float step, float mid) {
  return fmaf(step, static_cast<float>(code) - kInt4Mid, mid);
}

// Code j of a word minus 7.5, exactly, without a conversion: c in bits 4-7 of
// 2^19's mantissa is 2^19 + c.
__device__ __forceinline__ float int4_centered(uint32_t w, int j) {
  const uint32_t c = (j == 0 ? w << 4 : w >> (4 * j - 4)) & 0xf0u;
  return __uint_as_float(c | 0x49000000u) - 524295.5f;
}

__device__ __forceinline__ bool finite_f32(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

// Packed fp32 pairs (sm_100 f32x2 instructions).
__device__ __forceinline__ uint64_t f2_pack(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 f2_unpack(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t f2_mul(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// Two values of type T in a word, as fp32.
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

// 2^e for -126 <= e <= 127, and floor(log2 |x|) of a normal x.
__device__ __forceinline__ float exp2_int(int e) { return __int_as_float((e + 127) << 23); }
__device__ __forceinline__ int ilogb_f32(float x) { return ((__float_as_int(x) >> 23) & 255) - 127; }

}  // namespace psb
