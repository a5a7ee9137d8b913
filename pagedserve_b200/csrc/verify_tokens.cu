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
// One cluster of CTAs per sequence.  It reads the sequence's rows in batches of
// kBatchRows, each CTA a slice of the vocabulary: a running maximum, its place
// and the sum of exponentials in one pass, in fp32, joined through distributed
// shared memory.  Whether a draft is taken needs one logit and that sum; where
// fp32 leaves it open (within 2^-12 of the border) the sum is taken again in 64
// bits.  Rows behind the first rejection are not read by later batches.  The row
// that the new token is drawn from is read again (from L2) for sums per warp in 64
// bits, and the warp whose part the random number falls in goes over its part once
// more.  64 bits because a border between two of V tokens is missed with a
// probability of V times the cumulative weight's error: in fp32 one sample in a
// hundred at V = 152 K, here one in 10^9.
#include <cooperative_groups.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <type_traits>

#include "common.cuh"
#include "host_util.h"

namespace cg = cooperative_groups;

namespace psb {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCtas = 16;     // CTAs of a cluster
constexpr int kBatchRows = 8;    // rows read before the drafts among them are looked at
constexpr double kOpen = 1.0 / 4096;  // relative distance below which an fp32 decision is taken again

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
  int32_t* err;
};

// What a part of a row amounts to.
struct Part {
  float max, sum;  // the maximum (NaN above all), the sum of 2^((x - max) k)
  int32_t at;      // its first place
};

__device__ __forceinline__ bool above(float a, float b) { return a > b || (a != a && b == b); }

__device__ __forceinline__ Part join(const Part& a, const Part& b, float k) {
  const bool second = above(b.max, a.max) || (!above(a.max, b.max) && b.at < a.at);
  Part r;
  r.max = second ? b.max : a.max;
  r.at = second ? b.at : a.at;
  const float m = r.max == -INFINITY ? 0.f : r.max;
  // (a maximum that is not finite leaves a sum that is not a number: such a row is treated on its own)
  r.sum = a.sum * ex2_approx((a.max - m) * k) + b.sum * ex2_approx((b.max - m) * k);
  return r;
}

template <typename T>
struct Vec {
  static constexpr int n = 16 / sizeof(T);
  T v[n];
};

// A row in 16-byte pieces: piece c holds elements c n - skip .. of it (the first
// and the last one perhaps in part).
template <typename T>
struct Row {
  static constexpr int n = 16 / sizeof(T);
  const T* x;
  int vocab, skip, pieces;
  __device__ Row(const T* row, int v) : x(row), vocab(v) {
    skip = static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    pieces = (v + skip + n - 1) / n;
  }
  // elements of piece c as floats; those outside the row are ``fill``
  __device__ __forceinline__ void load(int c, float fill, float* f) const {
    const int e0 = c * n - skip;
    if (e0 >= 0 && e0 + n <= vocab) {
      Vec<T> v;
      *reinterpret_cast<uint4*>(&v) = __ldg(reinterpret_cast<const uint4*>(x + e0));
#pragma unroll
      for (int i = 0; i < n; ++i) f[i] = Elem<T>::to_float(v.v[i]);
    } else {
#pragma unroll
      for (int i = 0; i < n; ++i) f[i] = e0 + i >= 0 && e0 + i < vocab ? Elem<T>::to_float(x[e0 + i]) : fill;
    }
  }
};

// Elements of the draft's probabilities beside a piece of the logits; what is no
// probability (NaN, below 0) counts as 0.
template <typename Q>
__device__ __forceinline__ double prob_at(const void* probs, int64_t at) {
  const float f = Elem<Q>::to_float(reinterpret_cast<const Q*>(probs)[at]);
  return f > 0.f ? static_cast<double>(f) : 0.0;
}

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

struct NoProbs {};

template <typename T, typename Q>
__global__ void __launch_bounds__(kThreads) verify_kernel(const VerifyParams p) {
  constexpr bool kProbs = !std::is_same<Q, NoProbs>::value;
  constexpr int n = Row<T>::n;
  __shared__ Part s_warp[kBatchRows][kWarps];
  __shared__ Part s_cta[2][kBatchRows];  // this CTA's part of a batch's rows, two batches in turn
  __shared__ Part s_row[kBatchRows];
  __shared__ double s_wsum[kWarps];
  __shared__ double s_ctas[2][kMaxCtas];  // the CTAs' sums, two passes in turn
  __shared__ int s_stop, s_open;
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = static_cast<int>(cluster.num_blocks()), me = static_cast<int>(cluster.block_rank());
  const int seq = blockIdx.x / ctas;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  cluster.sync();  // every CTA has begun: its shared memory may be read and written
  pdl_wait();
  int r0 = __ldg(p.cu + seq), r1 = __ldg(p.cu + seq + 1);
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
  // one that is no temperature (NaN, negative, infinite) is flagged and taken for 0, as is one whose inverse fp32 does not hold
  if (!(temp >= 0.f && temp < INFINITY) && me == 0 && tid == 0) flag_error(p.err, PSB_DEVERR_LOGITS);
  const bool hot = temp >= 1e-37f && temp < INFINITY;
  const double inv_t = hot ? 1.0 / static_cast<double>(temp) : 1.0;
  const float k = static_cast<float>(inv_t * 1.4426950408889634);
  const T* const logits = reinterpret_cast<const T*>(p.logits);
  int passes = 0;  // sums over the cluster so far

  // The sum of a value per thread over the cluster; ``before``: over the CTAs before this one.
  auto cluster_sum = [&](double v, double& before) -> double {
    v = warp_sum(v);
    __syncthreads();
    if (lane == 0) s_wsum[warp] = v;
    __syncthreads();
    double* const sums = s_ctas[passes & 1];
    ++passes;
    if (tid < ctas) {
      double t = 0;
      for (int w = 0; w < kWarps; ++w) t += s_wsum[w];
      cluster.map_shared_rank(sums, tid)[me] = t;
    }
    cluster.sync();
    double all = 0;
    before = 0;
    for (int c = 0; c < ctas; ++c) {
      if (c < me) before += sums[c];
      all += sums[c];
    }
    return all;
  };
  // exp((x - max) / t) in 64 bits
  auto weight = [&](float x, float max) -> double { return exp((static_cast<double>(x) - static_cast<double>(max)) * inv_t); };
  // This warp's pieces of a row: consecutive ones for every warp of the cluster, in order.
  auto my_pieces = [&](const Row<T>& row, int& c0, int& c1) {
    const int64_t all = static_cast<int64_t>(ctas) * kWarps, w = me * kWarps + warp;
    c0 = static_cast<int>(row.pieces * w / all);
    c1 = static_cast<int>(row.pieces * (w + 1) / all);
  };
  auto row_sum = [&](int r, float max) -> double {
    const Row<T> row(logits + static_cast<int64_t>(r) * p.row_stride, p.vocab);
    int c0, c1;
    my_pieces(row, c0, c1);
    double sum = 0, unused;
#pragma unroll 1
    for (int c = c0 + lane; c < c1; c += 32) {
      float f[n];
      row.load(c, -INFINITY, f);
#pragma unroll
      for (int i = 0; i < n; ++i) sum += weight(f[i], max);
    }
    return cluster_sum(sum, unused);
  };

  // ---- the rows, until a draft is not taken ---------------------------------------
  int stop = r1 - 1;
  Part at_stop{};
#pragma unroll 1
  for (int b0 = r0, batch = 0; b0 < r1; b0 += kBatchRows, ++batch) {
    const int rows = min(kBatchRows, r1 - b0);
#pragma unroll 1
    for (int i = 0; i < rows; ++i) {
      const Row<T> row(logits + static_cast<int64_t>(b0 + i) * p.row_stride, p.vocab);
      const int c0 = static_cast<int>(static_cast<int64_t>(row.pieces) * me / ctas), c1 = static_cast<int>(static_cast<int64_t>(row.pieces) * (me + 1) / ctas);
      float m = -INFINITY, s = 0.f;
      int best = c0 + tid;
#pragma unroll 1
      for (int c = c0 + tid; c < c1; c += kThreads) {
        float f[n];
        row.load(c, -INFINITY, f);
        float cm = f[0];
#pragma unroll
        for (int j = 1; j < n; ++j) cm = above(f[j], cm) ? f[j] : cm;
        if (above(cm, m)) {
          const float mu = cm == -INFINITY ? 0.f : cm;
          s *= ex2_approx((m - mu) * k);
          m = cm;
          best = c;
        }
        const float mu = m == -INFINITY ? 0.f : m;
        float t = 0.f;
#pragma unroll
        for (int j = 0; j < n; ++j) t += ex2_approx((f[j] - mu) * k);
        s += t;
      }
      Part part{m, s, INT_MAX};
      if (best < c1) {  // the first place of the maximum in its piece
        float f[n];
        row.load(best, -INFINITY, f);
#pragma unroll
        for (int j = n - 1; j >= 0; --j) {
          const int e = best * n - row.skip + j;
          if (e >= 0 && e < p.vocab && (f[j] == m || (m != m && f[j] != f[j]))) part.at = e;
        }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        Part other;
        other.max = __shfl_xor_sync(0xffffffffu, part.max, o);
        other.sum = __shfl_xor_sync(0xffffffffu, part.sum, o);
        other.at = __shfl_xor_sync(0xffffffffu, part.at, o);
        part = join(part, other, k);
      }
      if (lane == 0) s_warp[i][warp] = part;
    }
    __syncthreads();
    if (tid < rows) {
      Part part = s_warp[tid][0];
      for (int w = 1; w < kWarps; ++w) part = join(part, s_warp[tid][w], k);
      s_cta[batch & 1][tid] = part;
    }
    cluster.sync();
    if (tid < rows) {
      Part part = cluster.map_shared_rank(s_cta[batch & 1], 0)[tid];
      for (int c = 1; c < ctas; ++c) part = join(part, cluster.map_shared_rank(s_cta[batch & 1], c)[tid], k);
      s_row[tid] = part;
    }
    __syncthreads();
    // every CTA decides alike: from the same numbers
    int from = 0;  // rows of the batch before it have their drafts taken
    bool over = false;
    double forced = 0;  // row ``from`` has this sum in 64 bits
    bool has_forced = false;
#pragma unroll 1
    while (true) {
      if (warp == 0) {
        int state = 0;  // 1: taken, 0: not (or there is no draft), 2: open
        if (lane >= from && lane < rows) {
          const int r = b0 + lane;
          const Part part = s_row[lane];
          const int64_t d = r + 1 < r1 ? __ldg(p.tokens + r + 1) : -1;
          if (d >= 0 && d < p.vocab) {
            double q = 1.0;
            if constexpr (kProbs) q = prob_at<Q>(p.probs, static_cast<int64_t>(r) * p.probs_stride + d);
            const double uq = static_cast<double>(__ldg(p.uniforms + 2 * static_cast<int64_t>(r))) * q;
            const bool plain = hot && part.max > -INFINITY && part.max < INFINITY;
            if (!plain) {
              state = uq < (d == part.at ? 1.0 : 0.0) ? 1 : 0;
            } else {
              const double e = weight(Elem<T>::to_float(logits[static_cast<int64_t>(r) * p.row_stride + d]), part.max);
              const bool sure = has_forced && lane == from;
              const double lhs = uq * (sure ? forced : static_cast<double>(part.sum));
              state = lhs < e ? 1 : 0;
              if (!sure && fabs(lhs - e) <= kOpen * e) state = 2;
            }
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
      const int at = s_stop;
      const bool open = s_open != 0;
      __syncthreads();
      from = at;
      has_forced = false;
      if (at == rows) break;  // all drafts of the batch are taken
      if (open) {
        forced = row_sum(b0 + at, s_row[at].max);
        has_forced = true;
        continue;
      }
      over = true;
      break;
    }
    if (over) {
      stop = b0 + from;
      at_stop = s_row[from];
      break;
    }
  }
  // (the last row has no draft: the loop always stops at a row)

  // ---- the new token ------------------------------------------------------------------
  const bool plain = hot && at_stop.max > -INFINITY && at_stop.max < INFINITY;
  if (hot && !plain && me == 0 && tid == 0) flag_error(p.err, PSB_DEVERR_LOGITS);
  if (me == 0) {
    for (int r = r0 + tid; r < r1; r += kThreads)
      if (r != stop) p.out[r] = r < stop ? __ldg(p.tokens + r + 1) : -1;
    if (tid == 0) {
      p.counts[seq] = stop - r0 + 1;
      if (!plain) p.out[stop] = at_stop.at;
    }
  }
  if (!plain) {  // all of p on the first maximum: so is what is left of it
    cluster.sync();  // no CTA leaves while its shared memory may still be read
    return;
  }
  const Row<T> row(logits + static_cast<int64_t>(stop) * p.row_stride, p.vocab);
  const float max = at_stop.max;
  int64_t d = stop + 1 < r1 ? __ldg(p.tokens + stop + 1) : -1;
  if (d >= p.vocab) d = -1;
  const double u = static_cast<double>(__ldg(p.uniforms + 2 * static_cast<int64_t>(stop) + 1));
  int c0, c1;
  my_pieces(row, c0, c1);
  int mode = d < 0 ? 0 : kProbs ? 2 : 1;  // weights: p; p without d; max(p - q, 0)
  double z = 0;
  if (mode == 2) z = row_sum(stop, max);
  // the weights of piece c
  auto weights = [&](int c, double* w) {
    float f[n];
    row.load(c, -INFINITY, f);
    const int e0 = c * n - row.skip;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      w[i] = weight(f[i], max);
      if (mode == 1 && e0 + i == d) w[i] = 0;
      if constexpr (kProbs) {
        if (mode == 2 && e0 + i >= 0 && e0 + i < p.vocab)
          w[i] = fmax(w[i] - prob_at<Q>(p.probs, static_cast<int64_t>(stop) * p.probs_stride + e0 + i) * z, 0.0);
      }
    }
  };
  double before, all;
#pragma unroll 1
  while (true) {
    double sum = 0;
#pragma unroll 1
    for (int c = c0 + lane; c < c1; c += 32) {
      double w[n];
      weights(c, w);
#pragma unroll
      for (int i = 0; i < n; ++i) sum += w[i];
    }
    all = cluster_sum(sum, before);
    if (all > 0 || mode == 0) break;
    mode = 0;  // nothing is left of p: from p itself
  }
  // The first warp whose cumulative weight is above the target, or, where rounding
  // leaves none, the last one with any weight; every thread finds the same.
  const double target = u * all;
  const double* const sums = s_ctas[(passes - 1) & 1];
  int owner = -1, last = 0;
  {
    double run = 0;
    for (int c = 0; c < ctas; ++c) {
      if (sums[c] > 0) last = c;
      if (owner < 0 && run + sums[c] > target) owner = c;
      run += sums[c];
    }
  }
  if (owner < 0) owner = last;
  if (owner == me) {
    int w_owner = -1, w_last = 0;
    double run = before, w_before = 0;
    for (int w = 0; w < kWarps; ++w) {
      if (s_wsum[w] > 0) w_last = w;
      if (w_owner < 0 && run + s_wsum[w] > target) {
        w_owner = w;
        w_before = run;
      }
      run += s_wsum[w];
    }
    const bool w_none = w_owner < 0;
    if (w_none) w_owner = w_last;
    if (warp == w_owner) {
      double base = w_none ? -INFINITY : w_before;  // (none: no weight passes the target, the last token with any is taken)
      int64_t found = -1, latest = 0;
#pragma unroll 1
      for (int c = c0; c < c1 && found < 0; c += 32) {
        double w[n], own = 0;
#pragma unroll
        for (int i = 0; i < n; ++i) w[i] = 0;
        if (c + lane < c1) weights(c + lane, w);
#pragma unroll
        for (int i = 0; i < n; ++i) own += w[i];
        double incl = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double x = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += x;
        }
        const int e0 = (c + lane) * n - row.skip;
        int hit = -1, weighty = -1;
        double at = base + (incl - own);
#pragma unroll
        for (int i = 0; i < n; ++i) {
          at += w[i];
          if (w[i] > 0) {
            weighty = e0 + i;
            if (hit < 0 && at > target) hit = e0 + i;
          }
        }
        const uint32_t hits = __ballot_sync(0xffffffffu, hit >= 0), some = __ballot_sync(0xffffffffu, weighty >= 0);
        if (hits) found = __shfl_sync(0xffffffffu, hit, __ffs(hits) - 1);
        if (some) latest = __shfl_sync(0xffffffffu, weighty, 31 - __clz(some));
        base += __shfl_sync(0xffffffffu, incl, 31);
      }
      if (lane == 0) p.out[stop] = found >= 0 ? found : latest;
    }
  }
  cluster.sync();  // no CTA leaves while its shared memory may still be read
}

int ctas_for(int batch, int sms) {
  // enough CTAs for two or more on every SM, up to 16 a sequence
  int c = 1;
  while (c < kMaxCtas && static_cast<int64_t>(batch) * c * 2 <= 4 * static_cast<int64_t>(sms)) c *= 2;
  return c;
}

template <typename T, typename Q>
int launch(const VerifyParams& p, cudaStream_t s) {
  const auto kern = verify_kernel<T, Q>;
  const void* f = reinterpret_cast<const void*>(kern);
  const int sms = device_sm_count();
  if (sms <= 0 || !prefer_max_l1(f)) return PSB_ERR_CUDA;
  const int ctas = ctas_for(p.batch, sms);
  if (ctas > 8) {  // beyond the portable limit: asked for once per kernel and device, which costs little
    const cudaError_t e = cudaFuncSetAttribute(f, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
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
  cfg.gridDim = dim3(static_cast<unsigned>(p.batch * ctas));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
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

extern "C" int psb_verify_tokens(const void* logits, int64_t row_stride, int32_t total, int32_t vocab, int32_t dtype,
                                 const int64_t* tokens, const int32_t* cu_seqlens, int32_t batch, const float* uniforms,
                                 const float* temperature, const void* draft_probs, int64_t probs_stride, int32_t probs_dtype,
                                 int64_t* new_tokens, int32_t* counts, int32_t* error_flag, psb_stream_t stream) {
  if (total < 0 || vocab <= 0 || batch < 0 || row_stride < 0 || probs_stride < 0 || !known(dtype) ||
      (draft_probs != nullptr && !known(probs_dtype)) || (total > 1 && row_stride < vocab) || (draft_probs != nullptr && total > 1 && probs_stride < vocab))
    return PSB_ERR_INVALID;
  if (batch == 0) return total == 0 ? PSB_OK : PSB_ERR_INVALID;
  if (!cu_seqlens || !temperature || !counts || (total > 0 && (!logits || !tokens || !uniforms || !new_tokens))) return PSB_ERR_INVALID;
  const int elem = dtype == PSB_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(logits) % elem) return PSB_ERR_INVALID;
  if (batch > (1 << 26)) return PSB_ERR_UNSUPPORTED;
  VerifyParams p{logits, row_stride, tokens, cu_seqlens, uniforms, temperature, draft_probs, probs_stride, new_tokens, counts, batch, total, vocab, error_flag};
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == PSB_F32) return launch_for<float>(p, probs_dtype, s);
  if (dtype == PSB_F16) return launch_for<__half>(p, probs_dtype, s);
  return launch_for<__nv_bfloat16>(p, probs_dtype, s);
}
