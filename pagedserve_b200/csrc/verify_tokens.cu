// verify_tokens: drafted tokens against the target's probabilities, with given
// random numbers, and the token behind the last one taken.
//
// Row r of the logits, at its sequence's temperature t, stands for
// p = softmax(logits[r] / t) (t = 0: all of it on the first maximum).  The draft d
// behind row r was drawn from q = draft_probs[r] (none given: all of q on d).  It is
// taken if u0 q(d) < p(d); at the first row whose draft is not taken, the new
// token is drawn from max(p - q, 0) (from p where that is nothing), at the last
// row, or one without a draft, from p: the first token whose cumulative weight is
// above u1 times the weights' sum.  Tokens so emitted are distributed as if each
// had been drawn from p.  Without drafts it is sampling at a temperature.
//
// One cluster of CTAs per sequence.  It reads the sequence's rows in batches (of
// four; few sequences, bound by latency: of eight), each warp a consecutive part of one row: the maximum, its place at temperature 0,
// and the sum of exponentials in one pass, joined through distributed shared memory.
// Rows behind the first rejection are not read by later batches.  The sample is
// then found in the part that the random number falls in, cut once more for all of
// the CTA's warps.
//
// Precision.  A border between two of V tokens is missed with a probability of V
// times the cumulative weight's error, so weights good to 24 bits would misplace one
// sample in a hundred at V = 152 K.  Weights in 64 bits for every row cost a multiple
// of the read, so they are used where fp32 leaves the answer open.  An fp32 weight
// 2^(x c - octave) (c = log2(e) / t, the octave an integer near the maximum's, so that
// parts are joined exactly), up to 31 octaves below the maximum's, is off by 1.08e-6 +
// 21.5 dc of itself at most: rounding the exponent, below 32, 2^-20 ln 2; c, which is off by
// dc of itself (2^-24 at most, known for each temperature), 31 dc ln 2 next to the
// maximum's; the exponential 2^-22; the sum of a piece's eight three times 2^-24.
// Those further below are off by more (4.3e-6 down to 62 octaves; what is left is nothing)
// but they are few: of V, 2^-31 V next to the maximum's.  fp32 is asked only about sums
// of 2^-26 V and more of it (of the whole row, V up to 2^25; of a sample, by its target),
// where these are 2^-5 at most of what is compared, and cost it another 2e-7 with the octave's
// rounding.  All further sums are in 64 bits.  A draft's test or a sample closer to its
// border than twice all that is done again in 64 bits, as is what is drawn from
// max(p - q, 0), where little may be left of much.
#include <cooperative_groups.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <type_traits>

#include "common.cuh"
#include "host_util.h"
#include "packed_f32.cuh"

namespace cg = cooperative_groups;

namespace psb {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCtas = 16;      // CTAs of a cluster
constexpr int kMaxRows = 8;       // rows read before the drafts among them are looked at, at most
constexpr int kOwnElems = 96;     // of the vocabulary per thread of a sequence up to which it does its 64-bit work itself
constexpr double kErr = 1.3e-6, kErrOfC = 21.5;  // of a sum of fp32 weights, relative: kErr + kErrOfC times c's
constexpr double kLeast = 1.0 / (1 << 26);       // of the largest weight, times the vocabulary: sums that this holds for
constexpr int kMostFast = 1 << 25;               // vocabulary
constexpr float kLargest = 1 << 20;  // octaves that logits may span for fp32

struct VerifyParams {
  const void* logits;
  int64_t row_stride;
  const int64_t* tokens;
  const int32_t* cu;
  const float* uniforms;  // [T, 2]
  const float* temperature;
  const void* probs;
  int64_t probs_stride;
  int64_t* out;
  int32_t* counts;
  int32_t batch, total, vocab;
  int4* todo;  // [batch], where 64-bit work is left for the second launch: row (-1: none), mode, the maximum's bits, the sum's
  int32_t* err;
};

// What a part of a row amounts to: its maximum (NaN above all), the maximum's
// first place (temperature 0), the sum of 2^(x c - octave).
struct Part {
  double sum;
  float max;
  int32_t octave, at;
};

__device__ __forceinline__ bool above(float a, float b) { return a > b || (a != a && b == b); }

// 2^n for n above -1023; 0 below
__device__ __forceinline__ double power(int n) { return n < -1000 ? 0.0 : __hiloint2double((n + 1023) << 20, 0); }

// A float's place among all floats, NaN above them, as an integer; and back
__device__ __forceinline__ int rank_of(float x) {
  const int b = __float_as_int(x == 0.f ? 0.f : x);  // (-0 as 0)
  return x != x ? INT_MAX : b ^ ((b >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float ranked(int k) { return k == INT_MAX ? __int_as_float(0x7fffffff) : __int_as_float(k ^ ((k >> 31) & 0x7fffffff)); }

// The parts of a warp's lanes joined, in every lane; ``sum`` stays the lane's own, in
// units of the joined octave.
__device__ __forceinline__ Part join_lanes(Part p, double& own) {
  const int k = rank_of(p.max), top = __reduce_max_sync(0xffffffffu, k);
  const int octave = __reduce_max_sync(0xffffffffu, p.octave);
  own = p.sum * power(p.octave - octave);
  p.at = __reduce_min_sync(0xffffffffu, k == top ? p.at : INT_MAX);
  p.max = ranked(top);
  p.octave = octave;
  p.sum = own;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) p.sum += __shfl_xor_sync(0xffffffffu, p.sum, o);
  return p;
}

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// 16 bytes of a row
template <typename T>
struct Piece {
  static constexpr int n = 16 / sizeof(T);
  uint32_t w[4];
  __device__ __forceinline__ float2 pair(int i) const {  // elements 2 i, 2 i + 1
    if constexpr (sizeof(T) == 4) {
      return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
    } else if constexpr (Elem<T>::code == PSB_BF16) {
      return make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
    } else {
      return __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    }
  }
  // NaN if there is one
  __device__ __forceinline__ float max() const {
    if constexpr (sizeof(T) == 4) {
      float a, b;
      asm("max.NaN.f32 %0, %1, %2;" : "=f"(a) : "f"(__uint_as_float(w[0])), "f"(__uint_as_float(w[1])));
      asm("max.NaN.f32 %0, %1, %2;" : "=f"(b) : "f"(__uint_as_float(w[2])), "f"(__uint_as_float(w[3])));
      asm("max.NaN.f32 %0, %0, %1;" : "+f"(a) : "f"(b));
      return a;
    } else {
      uint32_t a, b;
      Piece<T> r;
      if constexpr (Elem<T>::code == PSB_BF16) {
        asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(a) : "r"(w[0]), "r"(w[1]));
        asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(b) : "r"(w[2]), "r"(w[3]));
        asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(a) : "r"(b));
      } else {
        asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(a) : "r"(w[0]), "r"(w[1]));
        asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(b) : "r"(w[2]), "r"(w[3]));
        asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(a) : "r"(b));
      }
      r.w[0] = a;
      const float2 f = r.pair(0);
      float m;
      asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(f.x), "f"(f.y));
      return m;
    }
  }
};

// A row in 16-byte pieces: piece c holds elements c n - skip .. of it (the first
// and the last one perhaps in part: -infinity beside the row).
template <typename T>
struct Row {
  static constexpr int n = Piece<T>::n;
  const T* x;
  int vocab, skip, pieces;
  __device__ Row(const T* row, int v) : x(row), vocab(v) {
    skip = static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    pieces = (v + skip + n - 1) / n;
  }
  __device__ __forceinline__ int first(int c) const { return c * n - skip; }
  __device__ __forceinline__ Piece<T> load(int c) const {
    const int e0 = first(c);
    Piece<T> p;
    if (e0 >= 0 && e0 + n <= vocab) {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(x + e0));
      p.w[0] = v.x;
      p.w[1] = v.y;
      p.w[2] = v.z;
      p.w[3] = v.w;
    } else {
      T e[n];
#pragma unroll
      for (int i = 0; i < n; ++i) e[i] = e0 + i >= 0 && e0 + i < vocab ? x[e0 + i] : Elem<T>::from_float(-INFINITY);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) p.w[i] = __float_as_uint(e[i]);
        else p.w[i] = static_cast<uint32_t>(reinterpret_cast<const uint16_t&>(e[2 * i])) | static_cast<uint32_t>(reinterpret_cast<const uint16_t&>(e[2 * i + 1])) << 16;
      }
    }
    return p;
  }
  __device__ __forceinline__ Piece<T> whole(int c) const {  // a piece that lies in the row
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(x + first(c)));
    return Piece<T>{{v.x, v.y, v.z, v.w}};
  }
  // Calls f(piece, its number) for this lane's share of pieces c0 .. c1 - 1, in
  // ascending order but for the row's first piece where it is a part: F loads in
  // flight (one at a time, a row of 152 K took 30 us of latency).
  template <int F, typename Fn>
  __device__ __forceinline__ void each(int c0, int c1, Fn&& f) const {
    const int lane = threadIdx.x & 31;
    const bool head = c0 < c1 && first(c0) < 0;
    const int begin = c0 + (head ? 1 : 0), end = first(c1) > vocab ? c1 - 1 : c1;  // the whole pieces
#pragma unroll 1
    for (int k0 = begin + lane; k0 < end; k0 += 32 * F) {
      Piece<T> v[F];
#pragma unroll
      for (int u = 0; u < F; ++u) v[u] = whole(min(k0 + 32 * u, end - 1));
#pragma unroll
      for (int u = 0; u < F; ++u)
        if (k0 + 32 * u < end) f(v[u], k0 + 32 * u);
    }
    if (head || end < c1) {  // the row's ends, one lane each
      const int k = lane == 0 && head ? c0 : lane == 1 && end < c1 && end >= begin ? end : -1;
      if (k >= 0) f(load(k), k);
    }
  }
  // Its pieces from ``before`` of ``all`` equal parts on.
  __device__ __forceinline__ int cut(int before, int all) const { return static_cast<int>(static_cast<int64_t>(pieces) * before / all); }
};

// fp32 weights 2^(x c - octave).
struct Fast {
  float c, minus, limit;  // minus the octave; a logit times c above which the octave moves
  int octave;
  __device__ __forceinline__ Fast(double c64) : c(static_cast<float>(c64)) { unit(0); }
  __device__ __forceinline__ void unit(int o) {
    octave = o;
    minus = -static_cast<float>(o);
    limit = static_cast<float>(o) + 16.f;
  }
  __device__ __forceinline__ void set(float max) {  // the octave of a maximum (of -infinity and beyond the span: the span's end)
    unit(__float2int_rn(fminf(fmaxf(max * c, -kLargest), kLargest)));
  }
  __device__ __forceinline__ uint64_t weigh(float2 x) const {
    const float2 y = unpair2(fma2(pair2(x.x, x.y), pair2(c, c), pair2(minus, minus)));
    return pair2(ex2_approx(y.x), ex2_approx(y.y));
  }
};

// Elements of the draft's probabilities; what is none (NaN, below 0) counts as 0.
template <typename Q>
__device__ __forceinline__ double prob_at(const void* probs, int64_t at) {
  const float f = Elem<Q>::to_float(reinterpret_cast<const Q*>(probs)[at]);
  return f > 0.f ? static_cast<double>(f) : 0.0;
}

struct NoProbs {};

// ---------------------------------------------------------------------------
// a row's weights in 64 bits
// ---------------------------------------------------------------------------
struct Sums {  // in shared memory
  double warp[kWarps];
  double ctas[2][kMaxCtas];  // the CTAs' sums, two exchanges in turn
  double table[16];          // 2^(i / 16)
  int open[kWarps][4], n_open[kWarps];  // elements of a warp's part that wait for the row's sum
};

__device__ __forceinline__ void fill_table(Sums& s) {
  if (threadIdx.x < 16) s.table[threadIdx.x] = exp2(threadIdx.x / 16.0);
}

// A warp's inclusive scan of ``count`` sums, one a lane (zeros behind them).
__device__ __forceinline__ double scan_sums(const double* sums, int count) {
  const int lane = threadIdx.x & 31;
  double v = lane < count ? sums[lane] : 0.0;
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) {
    const double x = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += x;
  }
  return v;  // (up to sixteen sums)
}
// The sum of up to sixteen.
__device__ __forceinline__ double all_of(const double* sums, int count) { return __shfl_sync(0xffffffffu, scan_sums(sums, count), 15); }
// The first of ``count`` sums with a cumulative one, on top of ``run``, above ``target``,
// -1 if there is none; ``run``: the cumulative sum before it.  By whole warps.
__device__ __forceinline__ int first_above(const double* sums, int count, double target, double& run) {
  const int lane = threadIdx.x & 31;
  const double incl = run + scan_sums(sums, count);
  const uint32_t mask = __ballot_sync(0xffffffffu, lane < count && incl > target);
  const int at = __ffs(mask) - 1;
  const double before = __shfl_sync(0xffffffffu, incl, max(at - 1, 0));
  if (at > 0) run = before;
  return at;
}
__device__ __forceinline__ int last_above_0(const double* sums, int count) {
  const int lane = threadIdx.x & 31;
  return max(0, 31 - __clz(__ballot_sync(0xffffffffu, lane < count && sums[min(lane, count - 1)] > 0)));
}

// What the cluster's CTAs know of each other: their sums, from the sums per warp.
struct Cluster {
  cg::cluster_group group;
  Sums* sums;
  int ctas, me, passes;
  __device__ explicit Cluster(Sums* s) : group(cg::this_cluster()), sums(s), passes(0) {
    ctas = static_cast<int>(group.num_blocks());
    me = static_cast<int>(group.block_rank());
  }
  // Behind a write of sums->warp: a sum for every CTA.
  __device__ const double* exchange() {
    double* const to = sums->ctas[passes & 1];
    ++passes;
    __syncthreads();
    if (threadIdx.x < 32) {
      const double t = all_of(sums->warp, kWarps);
      if (static_cast<int>(threadIdx.x) < ctas) group.map_shared_rank(to, threadIdx.x)[me] = t;
    }
    group.sync();
    return to;
  }
  __device__ const double* exchange(double of_warp) {
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sums->warp[threadIdx.x >> 5] = of_warp;
    return exchange();
  }
};

// The sum of weights(piece, its number, w[n]) over pieces a0 .. a1 - 1, by one warp.
template <typename T, typename W>
__device__ __forceinline__ double sum_of(const Row<T>& row, W&& weights, int a0, int a1) {
  constexpr int n = Row<T>::n;
  double sum = 0;
  row.template each<2>(a0, a1, [&](const Piece<T>& x, int k) {
    double w[n];
    weights(x, k, w);
#pragma unroll
    for (int i = 0; i < n; ++i) sum += w[i];
  });
  return warp_sum(sum);
}

// The token among pieces a0 .. a1 - 1 with the first cumulative weight above ``target``
// (-1: none), by one warp; the cumulative weights before and after it; ``latest``: the
// last token with any weight.
template <typename T, typename W>
__device__ int search(const Row<T>& row, W&& weights, int a0, int a1, double base, double target, double& before, double& after, int& latest) {
  constexpr int n = Row<T>::n;
  const int lane = threadIdx.x & 31;
  latest = 0;
#pragma unroll 1
  for (int k0 = a0; k0 < a1; k0 += 32) {
    double w[n], own = 0;
#pragma unroll
    for (int i = 0; i < n; ++i) w[i] = 0;
    if (k0 + lane < a1) weights(row.load(k0 + lane), k0 + lane, w);
#pragma unroll
    for (int i = 0; i < n; ++i) own += w[i];
    double incl = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double x = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += x;
    }
    const int e0 = row.first(k0 + lane);
    int hit = -1, weighty = -1;
    double at = base + (incl - own), lo = 0, hi = 0;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const double next = at + w[i];
      if (w[i] > 0) {
        weighty = e0 + i;
        if (hit < 0 && next > target) {
          hit = e0 + i;
          lo = at;
          hi = next;
        }
      }
      at = next;
    }
    const uint32_t hits = __ballot_sync(0xffffffffu, hit >= 0), some = __ballot_sync(0xffffffffu, weighty >= 0);
    if (some) latest = __shfl_sync(0xffffffffu, weighty, 31 - __clz(some));
    if (hits) {
      const int at_lane = __ffs(hits) - 1;
      before = __shfl_sync(0xffffffffu, lo, at_lane);
      after = __shfl_sync(0xffffffffu, hi, at_lane);
      return __shfl_sync(0xffffffffu, hit, at_lane);
    }
    base += __shfl_sync(0xffffffffu, incl, 31);
  }
  return -1;
}

// Pieces a0 .. a1 - 1 cut for the CTA's warps: cut i's first, and the cuts' sums to sums->warp.
__device__ __forceinline__ int cut_of(int a0, int a1, int i) { return a0 + static_cast<int>(static_cast<int64_t>(a1 - a0) * i / kWarps); }
template <typename T, typename W>
__device__ __forceinline__ void cut_sums(const Row<T>& row, W&& weights, int a0, int a1, Sums* sums) {
  const int warp = threadIdx.x >> 5;
  const double sum = sum_of(row, weights, cut_of(a0, a1, warp), cut_of(a0, a1, warp + 1));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sums->warp[warp] = sum;
  __syncthreads();
}

// Weights in 64 bits, to 3e-12, in units of 2^(m / 16), m the integer nearest to the
// maximum's exponent in sixteenths of an octave; below 2^-900 there are none.  Of a
// logit's exponent in sixteenths the nearest integer n is found by an addition of
// 1.5 2^52, 2^((n - m) / 16) from a table of sixteen and an exponent, a polynomial of
// degree 4 (interpolation at Chebyshev's points of [-1/2, 1/2]) gives the rest: ten
// operations in 64 bits.
struct Exact {
  double c16;    // sixteenths of an octave per logit
  double magic;  // 1.5 2^52 - m
  double bias;   // taken from the logits first where their exponents are beyond 2^40 (m is 0 then)
  float low;     // logits up to it have none (no logit lies between it and the exact border)
  bool far;
  const double* table;
  __device__ Exact(double c, float top, const double* t) : c16(16.0 * c), table(t) {
    const double m = static_cast<double>(top) * c16;
    far = !(fabs(m) < 1099511627776.0);
    bias = far ? static_cast<double>(top) : 0.0;
    magic = 6755399441055744.0 - (far ? 0.0 : rint(m));
    // rounded down twice, so that it is below the maximum however small 900 / c is beside it
    low = __double2float_rd(__dsub_rd(static_cast<double>(top), 900.0 / c));
  }
  __device__ __forceinline__ double weight(float x) const {
    double xd = static_cast<double>(x);
    if (far) xd -= bias;
    const double t = fma(xd, c16, magic);
    const double f = fma(xd, c16, magic - t);
    const int i = __double2loint(t);
    double r = 1.4676387238435006e-07;
    r = fma(r, f, 1.3551205154935067e-05);
    r = fma(r, f, 0.0009383847926296646);
    r = fma(r, f, 0.043321698760160544);
    r = fma(r, f, 1.0);
    r *= table[i & 15];
    r = __hiloint2double(__double2hiint(r) + ((i >> 4) << 20), __double2loint(r));
    return x > low ? r : 0.0;
  }
  template <typename T>
  __device__ __forceinline__ void piece(const Piece<T>& x, double* w) const {
#pragma unroll
    for (int j = 0; j < Piece<T>::n / 2; ++j) {
      const float2 f = x.pair(j);
      w[2 * j] = weight(f.x);
      w[2 * j + 1] = weight(f.y);
    }
  }
  // A sum of fp32 weights (in units of ``octave``) in these units: next to the
  // maximum's weight, whose fp32 exponent is max times the rounded factor.
  __device__ double from_fast(double sum, int octave, float top, float c32) const {
    const double top64 = static_cast<double>(top);
    const double shift = static_cast<double>(octave) - top64 * static_cast<double>(c32);
    return sum * exp2(shift) * weight(top);
  }
  // the sum over a row, by the cluster
  template <typename T>
  __device__ double row_sum(const Row<T>& row, Cluster& cl) const {
    const int parts = cl.ctas * kWarps, part_of = cl.me * kWarps + (threadIdx.x >> 5);
    auto weights = [&](const Piece<T>& x, int, double* w) { piece(x, w); };
    return all_of(cl.exchange(sum_of(row, weights, row.cut(part_of, parts), row.cut(part_of + 1, parts))), cl.ctas);
  }
};

template <typename T>
__device__ __forceinline__ Row<T> row_of(const VerifyParams& p, int r) {
  return Row<T>(reinterpret_cast<const T*>(p.logits) + static_cast<int64_t>(r) * p.row_stride, p.vocab);
}

// What the new token is drawn from: p; p without the draft; max(p - q, 0).
enum Mode { kWhole = 0, kWithout = 1, kRest = 2 };

// The new token of row ``r`` in 64 bits, by a cluster.  ``z``: the row's sum in 64 bits,
// or in fp32.  max(e - q z, 0) needs it before the first weight; summed are e and
// q apart where e > q z by the fp32 z, so one pass gives z and, with it, the sum.  Elements
// that z's error (2.7e-6) leaves open, within 2^-18 of e (one in a row of 152 K, or all of them
// where q is next to p), wait until z is known, four a warp; where one meets a fifth the sum is
// taken again.  (Counted by the fp32 z, they misplaced what is drawn where little is left: 1.5 us of 36.)
template <typename T, typename Q>
__device__ void draw(const VerifyParams& p, Cluster& cl, int r, int d, int mode, float top, double c, double z) {
  constexpr bool kProbs = !std::is_same<Q, NoProbs>::value;
  constexpr int n = Row<T>::n;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int parts = cl.ctas * kWarps, part_of = cl.me * kWarps + warp;
  const Row<T> row = row_of<T>(p, r);
  const Exact ex(c, top, cl.sums->table);
  const double u = static_cast<double>(__ldg(p.uniforms + 2 * static_cast<int64_t>(r) + 1));
  const int c0 = row.cut(part_of, parts), c1 = row.cut(part_of + 1, parts);
  auto probs = [&](int k, double* q) {  // of piece k
    if constexpr (kProbs) {
      const int e0 = row.first(k);
      const Q* const x = reinterpret_cast<const Q*>(p.probs) + static_cast<int64_t>(r) * p.probs_stride + e0;
      const bool inside = e0 >= 0 && e0 + n <= p.vocab;
#pragma unroll
      for (int i = 0; i < n; ++i) {
        const float f = inside || (e0 + i >= 0 && e0 + i < p.vocab) ? Elem<Q>::to_float(x[i]) : 0.f;
        q[i] = static_cast<double>(f > 0.f ? f : 0.f);
      }
    }
  };
  const int of_d = (d + row.skip) / n;
  auto weights = [&](const Piece<T>& x, int k, double* w) {
    ex.piece(x, w);
    if (mode == kWithout && k == of_d) {
#pragma unroll
      for (int i = 0; i < n; ++i)
        if (row.first(k) + i == d) w[i] = 0;
    }
    if constexpr (kProbs) {
      if (mode == kRest) {
        double q[n];
        probs(k, q);
#pragma unroll
        for (int i = 0; i < n; ++i) w[i] = fmax(fma(-q[i], z, w[i]), 0.0);
      }
    }
  };
  const double* sums;
  double all;
#pragma unroll 1
  while (true) {
    if (kProbs && mode == kRest) {
      double e = 0, q = 0, whole = 0;
      if (lane == 0) cl.sums->n_open[warp] = 0;
      __syncwarp();
      row.template each<1>(c0, c1, [&](const Piece<T>& x, int k) {
        double w[n], v[n];
        ex.piece(x, w);
        probs(k, v);
#pragma unroll
        for (int i = 0; i < n; ++i) {
          whole += w[i];
          const int left = __double2hiint(fma(-v[i], z, w[i]));  // (sign and exponent are enough)
          if ((left & 0x7fffffff) + (18 << 20) <= __double2hiint(w[i])) {
            const int at = atomicAdd(&cl.sums->n_open[warp], 1);
            if (at < 4) cl.sums->open[warp][at] = row.first(k) + i;
          } else if (left >= 0) {
            e += w[i];
            q += v[i];
          }
        }
      });
      z = all_of(cl.exchange(warp_sum(whole)), cl.ctas);
      double rest = fma(-z, q, e);
      const int n_open = cl.sums->n_open[warp];
      if constexpr (kProbs) {
        if (n_open <= 4 && lane < n_open) {  // lane i the i-th of them, in whatever order they came: the sum is always the same
          const int* const all_open = cl.sums->open[warp];
          int d0 = 0;
          for (int j = 0; j < n_open; ++j) {
            int smaller = 0;
            for (int i = 0; i < n_open; ++i) smaller += all_open[i] < all_open[j];
            if (smaller == lane) d0 = all_open[j];
          }
          rest += fmax(fma(-z, prob_at<Q>(p.probs, static_cast<int64_t>(r) * p.probs_stride + d0), ex.weight(Elem<T>::to_float(row.x[d0]))), 0.0);
        }
      }
      if (n_open > 4) rest = __longlong_as_double(0x7ff8000000000000ll);  // (no number: what every CTA sees of it)
      sums = cl.exchange(warp_sum(rest));
      all = all_of(sums, cl.ctas);
      if (all != all) {
        sums = cl.exchange(sum_of(row, weights, c0, c1));
        all = all_of(sums, cl.ctas);
      }
    } else {
      sums = cl.exchange(sum_of(row, weights, c0, c1));
      all = all_of(sums, cl.ctas);
    }
    if (all > 0 || mode == kWhole) break;
    mode = kWhole;  // nothing is left of p: from p itself
  }
  // where rounding leaves no part above the target, the last with any weight
  const double target = u * all;
  double run = 0;
  int owner = first_above(sums, cl.ctas, target, run);
  bool none = owner < 0;
  if (none) owner = last_above_0(sums, cl.ctas);
  if (owner != cl.me) return;
  int w = none ? -1 : first_above(cl.sums->warp, kWarps, target, run);
  none = w < 0;
  if (none) w = last_above_0(cl.sums->warp, kWarps);
  const int a0 = row.cut(cl.me * kWarps + w, parts), a1 = row.cut(cl.me * kWarps + w + 1, parts);
  cut_sums(row, weights, a0, a1, cl.sums);
  int i = none ? -1 : first_above(cl.sums->warp, kWarps, target, run);
  none = i < 0;
  if (none) i = last_above_0(cl.sums->warp, kWarps);
  if (warp == i) {
    double before, after;
    int latest;
    const int hit = search(row, weights, cut_of(a0, a1, i), cut_of(a0, a1, i + 1), none ? -INFINITY : run, target, before, after, latest);
    if (lane == 0) p.out[r] = hit >= 0 ? hit : latest;
  }
}

// log2(e) / temperature; 0 for temperature 0 and what is taken for it: no temperature
// (NaN, negative, infinite).
__device__ __forceinline__ double exponent_of(float temperature) {
  return temperature > 0.f && temperature < INFINITY ? 1.4426950408889634 / static_cast<double>(temperature) : 0.0;
}

__device__ __forceinline__ bool finite(float m) { return m > -INFINITY && m < INFINITY; }

// kLater: 64-bit draws are left for verify_rest_kernel (p.todo).
template <typename T, typename Q, bool kLater>
__global__ void __launch_bounds__(kThreads, 2) verify_kernel(const VerifyParams p) {
  constexpr bool kProbs = !std::is_same<Q, NoProbs>::value;
  constexpr int n = Row<T>::n;
  __shared__ Sums s_sums;
  __shared__ Part s_part[kMaxRows][kWarps];  // this CTA's parts of a batch's rows
  __shared__ Part s_cta[2][kMaxRows];        // joined; two batches in turn
  __shared__ Part s_row[kMaxRows];
  __shared__ double s_ctasum[kMaxRows][kMaxCtas];  // the CTAs' sums of a batch's rows, in units of the rows' octaves
  __shared__ double s_of_part[kWarps];
  __shared__ int s_stop, s_open, s_found;
  Cluster cl(&s_sums);
  const int ctas = cl.ctas, me = cl.me;
  const int seq = blockIdx.x / ctas;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  fill_table(s_sums);
  if (tid == 0) s_found = 0;
  cl.group.sync();  // every CTA has begun: its shared memory may be read and written
  pdl_wait();
  if (kLater) pdl_launch_dependents();
  const int r0 = __ldg(p.cu + seq), r1 = __ldg(p.cu + seq + 1);
  if (kLater && me == 0 && tid == 0) p.todo[seq] = make_int4(-1, 0, 0, 0);
  if (seq == 0 && p.total > 0) {  // rows that belong to no sequence
    const int first = __ldg(p.cu), end = __ldg(p.cu + p.batch);
    for (int r = me * kThreads + tid; r < p.total; r += ctas * kThreads)
      if (r < first || r >= end) p.out[r] = -1;
  }
  if (r0 < 0 || r1 < r0 || r1 > p.total) {
    if (me == 0 && tid == 0) {
      flag_error(p.err, PSB_DEVERR_SEQLENS);
      p.counts[seq] = 0;
    }
    return;
  }
  if (r1 == r0) {
    if (me == 0 && tid == 0) p.counts[seq] = 0;
    return;
  }
  const float temp = __ldg(p.temperature + seq);
  if (!(temp >= 0.f && temp < INFINITY) && me == 0 && tid == 0) flag_error(p.err, PSB_DEVERR_LOGITS);
  const double c = exponent_of(temp);
  const bool hot = c > 0;
  Fast fast(c);
  // whether fp32 weights of a row with this maximum are good to error()
  auto in_fp32 = [&](float m) { return c > 1e-30 && c < 1e30 && fabsf(m * fast.c) < kLargest && p.vocab <= kMostFast; };
  auto error = [&]() {  // (c is log2(e) / temp: no division)
    return kErr + kErrOfC * 0.6931471805599453 * fabs(fma(static_cast<double>(fast.c), static_cast<double>(temp), -1.4426950408889634));
  };

  // ---- the rows, until a draft is not taken ---------------------------------------
  // rows behind a rejection are read for nothing, but a batch takes 5 us however few its rows
  const int most = ctas == kMaxCtas ? kMaxRows : kMaxRows / 2;
  int stop = r1 - 1, in_batch = 0, wpr = kWarps;
#pragma unroll 1
  for (int b0 = r0, batch = 0; b0 < r1; b0 += most, ++batch) {
    const int rows = min(most, r1 - b0);
    if (batch > 0) __syncthreads();  // s_part and s_row are read no more
    // what the drafts' tests need, on its way
    int d = -1;
    float at_d = 0.f, u0 = 0.f;
    double q = 1.0;
    if (warp == 0 && lane < rows) {
      const int r = b0 + lane;
      const int64_t next = r + 1 < r1 ? __ldg(p.tokens + r + 1) : -1;
      if (next >= 0 && next < p.vocab) d = static_cast<int>(next);
      u0 = __ldg(p.uniforms + 2 * static_cast<int64_t>(r));
      if (d >= 0) {
        at_d = Elem<T>::to_float(row_of<T>(p, r).x[d]);
        if constexpr (kProbs) q = prob_at<Q>(p.probs, static_cast<int64_t>(r) * p.probs_stride + d);
      }
    }
    // wpr warps of every CTA to a row, each a part of it
    wpr = rows == 1 ? kWarps : rows == 2 ? kWarps / 2 : rows <= 4 ? kWarps / 4 : kWarps / 8;
    const int i = warp / wpr;
    if (i < rows) {
      const Row<T> row = row_of<T>(p, b0 + i);
      const int part_of = me * wpr + (warp - i * wpr), parts = ctas * wpr;
      const int c0 = row.cut(part_of, parts), c1 = row.cut(part_of + 1, parts);
      Part part{0.0, -INFINITY, INT_MIN / 2, INT_MAX};
      if (hot) {
        float m = -INFINITY;
        double sum = 0;
        bool begun = false;
        row.template each<4>(c0, c1, [&](const Piece<T>& x, int) {
          const float pm = x.max();
          m = above(pm, m) ? pm : m;
          if (!begun || pm * fast.c > fast.limit) {  // (rare: the weights' unit moves)
            const int before = fast.octave;
            fast.set(pm);
            sum = begun ? sum * power(before - fast.octave) : 0.0;
            begun = true;
          }
          uint64_t s0 = fast.weigh(x.pair(0)), s1 = fast.weigh(x.pair(1));
          if constexpr (n == 8) {
            s0 = add2(s0, fast.weigh(x.pair(2)));
            s1 = add2(s1, fast.weigh(x.pair(3)));
          }
          const float2 s = unpair2(add2(s0, s1));
          sum += static_cast<double>(s.x + s.y);
        });
        part.max = m;
        part.sum = sum;
        if (begun) part.octave = fast.octave;
      } else {
        int best = INT_MAX;
        row.template each<4>(c0, c1, [&](const Piece<T>& x, int k) {
          const float pm = x.max();
          if (above(pm, part.max) || best == INT_MAX || (k < best && !above(part.max, pm))) {
            part.max = pm;
            best = k;
          }
        });
        if (best < INT_MAX) {  // the first place of the maximum in its piece
          const Piece<T> x = row.load(best);
#pragma unroll
          for (int j = n - 1; j >= 0; --j) {
            const float2 f2 = x.pair(j / 2);
            const float f = j & 1 ? f2.y : f2.x;
            const int e = row.first(best) + j;
            if (e >= 0 && e < p.vocab && (f == part.max || (f != f && part.max != part.max))) part.at = e;
          }
        }
      }
      double own;
      part = join_lanes(part, own);
      if (lane == 0) s_part[i][warp - i * wpr] = part;
    }
    __syncthreads();
    if (warp < rows) {
      Part part{0.0, -INFINITY, INT_MIN / 2, INT_MAX};
      double own;
      if (lane < wpr) part = s_part[warp][lane];
      part = join_lanes(part, own);
      if (lane == 0) s_cta[batch & 1][warp] = part;
    }
    cl.group.sync();
    if (warp < rows) {
      Part part{0.0, -INFINITY, INT_MIN / 2, INT_MAX};
      double own;
      if (lane < ctas) part = cl.group.map_shared_rank(s_cta[batch & 1], lane)[warp];
      part = join_lanes(part, own);
      if (lane < ctas) s_ctasum[warp][lane] = own;
      if (lane == 0) s_row[warp] = part;
    }
    __syncthreads();
    // every CTA decides alike: from the same numbers
    int from = 0;       // rows of the batch before it have their drafts taken
    double exact = -1;  // the sum of row ``from`` in 64 bits, once it is known
#pragma unroll 1
    while (true) {
      if (warp == 0) {
        int state = 0;  // 1: taken, 0: not (or there is no draft), 2: open
        if (lane >= from && lane < rows && d >= 0) {
          const Part part = s_row[lane];
          const double uq = static_cast<double>(u0) * q;
          if (!hot) {
            state = uq < (d == part.at ? 1.0 : 0.0) ? 1 : 0;
          } else if (finite(part.max)) {
            const Exact ex(c, part.max, s_sums.table);
            const double e = ex.weight(at_d);
            const bool sure = exact >= 0 && lane == from;
            const double sum = sure ? exact : ex.from_fast(part.sum, part.octave, part.max, fast.c);
            state = uq * sum < e ? 1 : 0;
            if (!sure && (!in_fp32(part.max) || fabs(uq * sum - e) <= 2.0 * error() * e)) state = 2;
          }
        }
        const uint32_t other = __ballot_sync(0xffffffffu, lane >= from && lane < rows && state != 1);
        const uint32_t open = __ballot_sync(0xffffffffu, state == 2);
        if (lane == 0) {
          s_stop = other ? __ffs(other) - 1 : rows;
          s_open = other ? (open >> (__ffs(other) - 1)) & 1 : 0;
        }
      }
      __syncthreads();
      from = s_stop;
      const bool open = s_open != 0;
      __syncthreads();
      exact = -1;
      if (from == rows || !open) break;  // all drafts of the batch are taken, or one is not
      exact = Exact(c, s_row[from].max, s_sums.table).row_sum(row_of<T>(p, b0 + from), cl);
    }
    if (from < rows) {
      stop = b0 + from;
      in_batch = from;
      break;
    }
  }
  // (the last row has no draft: the loop always stops at a row)

  // ---- the new token ------------------------------------------------------------------
  const Part at_stop = s_row[in_batch];
  const float top = at_stop.max;
  if (me == 0) {
    for (int r = r0 + tid; r < r1; r += kThreads)
      if (r != stop) p.out[r] = r < stop ? __ldg(p.tokens + r + 1) : -1;
    if (tid == 0) {
      p.counts[seq] = stop - r0 + 1;
      if (!hot) p.out[stop] = at_stop.at;
    }
  }
  const Row<T> row = row_of<T>(p, stop);
  if (!hot || !finite(top)) {
    // all of p on the first maximum: so is what is left of it
    if (hot && me == 0) {  // a row without probabilities: one CTA looks for its maximum's place
      int best = INT_MAX;
      for (int k = tid; k < row.pieces && best == INT_MAX; k += kThreads) {
        const Piece<T> x = row.load(k);
#pragma unroll
        for (int j = n - 1; j >= 0; --j) {
          const float2 f2 = x.pair(j / 2);
          const float f = j & 1 ? f2.y : f2.x;
          const int e = row.first(k) + j;
          if (e >= 0 && e < p.vocab && (f == top || (f != f && top != top))) best = e;
        }
      }
      best = __reduce_min_sync(0xffffffffu, best);
      if (lane == 0) s_part[0][warp].at = best;
      __syncthreads();
      if (tid == 0) {
        for (int w = 0; w < kWarps; ++w) best = min(best, s_part[0][w].at);
        p.out[stop] = best;
        flag_error(p.err, PSB_DEVERR_LOGITS);
      }
    }
    cl.group.sync();  // no CTA leaves while its shared memory may still be read
    return;
  }
  const int64_t next = stop + 1 < r1 ? __ldg(p.tokens + stop + 1) : -1;
  const int d = next >= 0 && next < p.vocab ? static_cast<int>(next) : -1;
  const int mode = d < 0 ? kWhole : kProbs ? kRest : kWithout;
  const double u = static_cast<double>(__ldg(p.uniforms + 2 * static_cast<int64_t>(stop) + 1));
  if (mode != kRest && in_fp32(top)) {
    // from the sums that are there
    if (tid < wpr) s_of_part[tid] = s_part[in_batch][tid].sum * power(s_part[in_batch][tid].octave - at_stop.octave);
    fast.unit(at_stop.octave);
    const int of_d = mode == kWithout ? (d + row.skip) / n : -1;
    auto weights = [&](const Piece<T>& x, int k, double* w) {
#pragma unroll
      for (int j = 0; j < n / 2; ++j) {
        const float2 v = unpair2(fast.weigh(x.pair(j)));
        w[2 * j] = static_cast<double>(v.x);
        w[2 * j + 1] = static_cast<double>(v.y);
      }
      if (k == of_d) {
#pragma unroll
        for (int j = 0; j < n; ++j)
          if (row.first(k) + j == d) w[j] = 0;
      }
    };
    auto part_at = [&](int w) { return row.cut(me * wpr + w, ctas * wpr); };
    __syncthreads();
    const double* sums = s_ctasum[in_batch];
    if (mode == kWithout) {  // the sums without the draft: its part's is taken again
      for (int w = 0; w < wpr; ++w)
        if (of_d >= part_at(w) && of_d < part_at(w + 1)) {  // (the same for the whole CTA)
          cut_sums(row, weights, part_at(w), part_at(w + 1), &s_sums);
          const double sum = all_of(s_sums.warp, kWarps);
          if (tid == 0) s_of_part[w] = sum;
        }
      __syncthreads();
      if (tid < kWarps) s_sums.warp[tid] = tid < wpr ? s_of_part[tid] : 0.0;
      sums = cl.exchange();
    }
    const double target = u * all_of(sums, ctas), room = 2.0 * error() * target;
    double run = 0;
    if (target >= kLeast * p.vocab && first_above(sums, ctas, target, run) == me) {
      const int w = first_above(s_of_part, wpr, target, run);
      if (w >= 0) {
        const int a0 = part_at(w), a1 = part_at(w + 1);
        cut_sums(row, weights, a0, a1, &s_sums);
        const int i = first_above(s_sums.warp, kWarps, target, run);
        if (warp == i) {
          double before = 0, after = 0;
          int latest;
          const int hit = search(row, weights, cut_of(a0, a1, i), cut_of(a0, a1, i + 1), run, target, before, after, latest);
          if (hit >= 0 && target - before >= room && after - target > room) {
            if (lane == 0) p.out[stop] = hit;
            if (lane < ctas) *cl.group.map_shared_rank(&s_found, lane) = 1;
          }
        }
      }
    }
    cl.group.sync();
    if (s_found != 0) return;  // (nobody reads this CTA's shared memory any more)
  }
  // (the sum by which max(p - q, 0) is first told from 0: in 64 bits where fp32 does not hold it)
  double z = 0;
  if (mode == kRest) {
    const Exact ex(c, top, s_sums.table);
    z = in_fp32(top) ? ex.from_fast(at_stop.sum, at_stop.octave, top, fast.c) : ex.row_sum(row, cl);
  }
  if constexpr (kLater) {
    if (me == 0 && tid == 0) p.todo[seq] = make_int4(stop, mode, __float_as_int(top), __float_as_int(static_cast<float>(z)));
  } else {
    draw<T, Q>(p, cl, stop, d, mode, top, c, z);
  }
  cl.group.sync();  // no CTA leaves while its shared memory may still be read
}

// The 64-bit draws of a batch of many sequences, one cluster each in turn.  In
// verify_kernel, with few CTAs a sequence, they would be its longest part by far (one
// of 256 sequences over V = 152 K: 51 us; this launch costs 5 us, and 10 us a draw).
template <typename T, typename Q>
__global__ void __launch_bounds__(kThreads, 2) verify_rest_kernel(const VerifyParams p) {
  __shared__ Sums s_sums;
  __shared__ int s_list[kThreads], s_count[kWarps];
  Cluster cl(&s_sums);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n = gridDim.x / cl.ctas, j = blockIdx.x / cl.ctas;  // clusters, this one
  fill_table(s_sums);
  cl.group.sync();
  pdl_wait();
  int before = 0;  // such sequences so far: this cluster takes the j-th of every n
#pragma unroll 1
  for (int b0 = 0; b0 < p.batch; b0 += kThreads) {
    const bool some = b0 + tid < p.batch && __ldcg(&p.todo[b0 + tid].x) >= 0;
    const uint32_t mask = __ballot_sync(0xffffffffu, some);
    __syncthreads();
    if (lane == 0) s_count[warp] = __popc(mask);
    __syncthreads();
    int rank = before + __popc(mask & ((1u << lane) - 1)), here = 0;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) rank += s_count[w];
      here += s_count[w];
    }
    const int skip = (before + n - 1 - j) / n;  // of those before, this cluster's
    if (some && rank % n == j) s_list[rank / n - skip] = b0 + tid;
    before += here;
    const int count = (before + n - 1 - j) / n - skip;
    __syncthreads();
#pragma unroll 1
    for (int i = 0; i < count; ++i) {
      const int seq = s_list[i];
      const int4 t = __ldcg(p.todo + seq);
      const int d = t.y == kWhole ? -1 : static_cast<int>(__ldg(p.tokens + t.x + 1));
      draw<T, Q>(p, cl, t.x, d, t.y, __int_as_float(t.z), exponent_of(__ldg(p.temperature + seq)), static_cast<double>(__int_as_float(t.w)));
      __syncthreads();
    }
  }
  cl.group.sync();  // no CTA leaves while its shared memory may still be written
}

// Two CTAs fit an SM: the largest power of two that keeps a batch's clusters all resident.
int ctas_for(int batch, int sms) {
  int c = 1;
  while (c < kMaxCtas && static_cast<int64_t>(batch) * c * 2 <= 2 * static_cast<int64_t>(sms)) c *= 2;
  return c;
}

template <typename K>
cudaError_t launch_clusters(K kern, int clusters, int ctas, const VerifyParams& p, cudaStream_t s) {
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ctas;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(clusters * ctas));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kern, p);
}

template <typename T, typename Q>
int launch(const VerifyParams& p, cudaStream_t s) {
  const int sms = device_sm_count();
  if (sms <= 0) return PSB_ERR_CUDA;
  const int ctas = ctas_for(p.batch, sms);
  const bool later = p.vocab > kOwnElems * ctas * kThreads;
  const auto kern = later ? verify_kernel<T, Q, true> : verify_kernel<T, Q, false>;
  const auto rest = verify_rest_kernel<T, Q>;
  // 22 KB: two CTAs' shared memory, the rest for loads in flight
  if (!prefer_shared_percent(reinterpret_cast<const void*>(kern), 10) || !prefer_shared_percent(reinterpret_cast<const void*>(rest), 10))
    return PSB_ERR_CUDA;
  if (ctas > 8) {  // beyond the portable limit
    const cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void*>(kern), cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return record_cuda_error(e);
  }
  discard_stale_error();
  cudaError_t e = launch_clusters(kern, p.batch, ctas, p, s);
  // Small clusters for many draws, larger ones for few: drafts with probabilities are
  // mostly drawn for, samples one in ten (of 256: eight CTAs 48 us, four 53; all of
  // 256: 172 and 127).
  const int more = p.probs != nullptr || p.batch > 2 * sms ? 4 : 8;
  if (e == cudaSuccess && later) e = launch_clusters(rest, std::min(p.batch, std::max(1, 2 * sms / more)), more, p, s);
  if (e != cudaSuccess) return record_cuda_error(e);
  return check_launch();
}

template <typename T>
int launch_for(const VerifyParams& p, int probs_dtype, cudaStream_t s) {
  if (p.probs == nullptr) return launch<T, NoProbs>(p, s);
  if (probs_dtype == PSB_F32) return launch<T, float>(p, s);
  if (probs_dtype == PSB_F16) return launch<T, __half>(p, s);
  return launch<T, __nv_bfloat16>(p, s);
}

bool known(int dtype) { return dtype == PSB_F32 || dtype == PSB_F16 || dtype == PSB_BF16; }

}  // namespace
}  // namespace psb

using namespace psb;

extern "C" size_t psb_verify_tokens_workspace_size(int32_t batch) { return batch > 0 ? sizeof(int4) * static_cast<size_t>(batch) : 0; }

extern "C" int psb_verify_tokens(const void* logits, int64_t row_stride, int32_t total, int32_t vocab, int32_t dtype,
                                 const int64_t* tokens, const int32_t* cu_seqlens, int32_t batch, const float* uniforms,
                                 const float* temperature, const void* draft_probs, int64_t probs_stride, int32_t probs_dtype,
                                 int64_t* new_tokens, int32_t* counts, void* workspace, size_t workspace_bytes, int32_t* error_flag,
                                 psb_stream_t stream) {
  if (total < 0 || vocab <= 0 || batch < 0 || row_stride < 0 || probs_stride < 0 || !known(dtype) ||
      (draft_probs != nullptr && !known(probs_dtype)) || (total > 1 && row_stride < vocab) || (draft_probs != nullptr && total > 1 && probs_stride < vocab))
    return PSB_ERR_INVALID;
  if (batch == 0) return total == 0 ? PSB_OK : PSB_ERR_INVALID;
  if (!cu_seqlens || !temperature || !counts || (total > 0 && (!logits || !tokens || !uniforms || !new_tokens))) return PSB_ERR_INVALID;
  const int elem = dtype == PSB_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(logits) % elem) return PSB_ERR_INVALID;
  if (batch > (1 << 26)) return PSB_ERR_UNSUPPORTED;
  if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16 || workspace_bytes < psb_verify_tokens_workspace_size(batch)) return PSB_ERR_WORKSPACE;
  VerifyParams p{logits, row_stride, tokens, cu_seqlens, uniforms, temperature, draft_probs, probs_stride, new_tokens, counts, batch, total, vocab,
                 static_cast<int4*>(workspace), error_flag};
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == PSB_F32) return launch_for<float>(p, probs_dtype, s);
  if (dtype == PSB_F16) return launch_for<__half>(p, probs_dtype, s);
  return launch_for<__nv_bfloat16>(p, probs_dtype, s);
}