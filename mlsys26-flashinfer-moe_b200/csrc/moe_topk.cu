// Routing to experts for layers that do not use the fused DeepSeek-V3 router:
// softmax or sigmoid scores over any number of experts up to 1024, an optional
// bias that only takes part in the choice, groups of experts ranked by their
// best or their two best scores, top-k, renormalised weights.
//
//   s = softmax(x) or sigmoid(x)           c = s + bias
//   keep the topk_group groups with the largest group score (ties: lowest group)
//   idx = the top_k experts of the kept groups by c, largest first (ties: lowest id)
//   w = s[idx] (/ (sum of them + 1e-20) when renormalised) * routed_scaling_factor
//
// The order is that of the scores in 64 bits.  Without a bias (and without
// top-2 group sums) the scores grow with the logits, so the logits themselves
// are compared and only the chosen ones are exponentiated.
//
// A NaN logit or bias counts as -inf.  A -inf logit has the score 0: its expert weighs
// 0 and ranks last, but with a bias where the bias puts it (a row without a single
// finite logit has zero weights).  A -inf bias ranks last.  +inf logits share a softmax
// row's weight equally.
//
// One warp per token.  Lane l holds experts l, l+32, ..., so loads are
// coalesced and an expert's lane is its id modulo 32.
#include "moe_kernels.cuh"

#include <cuda_fp16.h>

namespace moe {

namespace {

constexpr int kTopkWarps = 4;
// Resident blocks an SM that the registers are held to: a grid of that size keeps
// a warp busy with token after token, the next one's loads in flight.
constexpr int topk_blocks_per_sm(int nv) { return nv <= 8 ? 8 : nv == 16 ? 5 : 3; }
constexpr float kScoreSlack = 28.f * 0x1p-24f;
constexpr float kSigmoidSlack = 5.f * 0x1p-24f;
constexpr unsigned kFull = 0xffffffffu;

__device__ __forceinline__ float load_elem(const void* p, int dtype, int64_t i) {
  if (dtype == MOE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  if (dtype == MOE_F16) return __half2float(static_cast<const __half*>(p)[i]);
  return static_cast<const float*>(p)[i];
}

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }

__device__ __forceinline__ float no_nan(float v) { return fmaxf(v, -INFINITY); }   // NaN -> -inf

// Unsigned key with the order of the float (-inf is 0x007fffff, above 0).
__device__ __forceinline__ unsigned order_key(float v) {
  const int b = __float_as_int(v + 0.f);   // -0 and 0 are the same score
  return static_cast<unsigned>(b ^ ((b >> 31) | static_cast<int>(0x80000000u)));
}
__device__ __forceinline__ float key_value(unsigned key) {
  return __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key);
}

// e / group_size: exact for e < 1024 (the reciprocal is off by less than one unit
// of 2^-20, so the product by less than 2^-20 e < 1 / group_size).
__device__ __forceinline__ unsigned group_of(const TopkParams& p, unsigned e) {
  return (e * p.group_inv) >> 20;
}

__device__ __forceinline__ double warp_max(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmax(v, __shfl_xor_sync(kFull, v, o));
  return v;
}

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}

// exp(x - m) of a softmax row with maximum m: equal infinities count as equal,
// a row of -inf has no weight.
__device__ __forceinline__ float shifted_exp(float x, float m) {
  return m == -INFINITY ? 0.f : x == m ? 1.f : expf(x - m);
}
__device__ __forceinline__ double shifted_exp64(float x, float m) {
  return m == -INFINITY ? 0.0 : x == m ? 1.0 : exp(static_cast<double>(x) - static_cast<double>(m));
}

}  // namespace

// Stores the weight of expert `e`, the token's choice number `rank`, on the lanes
// whose rank is below top_k; s: its score, or with a renormalised softmax any
// multiple of it (0 on the other lanes).
__device__ __forceinline__ void store_choice(const TopkParams& p, int64_t t, int rank, int e, float s) {
  if (p.renormalize) s = __fdividef(s, warp_sum(s) + 1e-20f);
  if (rank < p.top_k) {
    p.topk_idx[t * p.top_k + rank] = e;
    p.topk_weights[t * p.top_k + rank] = s * p.factor;
  }
}
__device__ __forceinline__ float sigmoid(float x) { return __fdividef(1.f, 1.f + expf(-x)); }

// Bit g * lanes_per_group: group g is kept.  c: the token's scores in shared
// memory.  gap: smallest kept score minus largest dropped one.
template <typename C>
__device__ __forceinline__ unsigned kept_groups(const TopkParams& p, const C* c, int lane, C* gap) {
  const C ninf = -static_cast<C>(INFINITY);
  const int lpg = p.lanes_per_group, g = lane / lpg, size = p.group_size;
  C m1 = ninf, m2 = ninf;
  if (g < p.n_group) {
    for (int i = lane % lpg; i < size; i += lpg) {
      const C v = c[g * size + i];
      m2 = v > m1 ? m1 : v > m2 ? v : m2;
      m1 = v > m1 ? v : m1;
    }
  }
  for (int o = 1; o < lpg; o <<= 1) {
    const C o1 = __shfl_xor_sync(kFull, m1, o), o2 = __shfl_xor_sync(kFull, m2, o);
    const C lo = m1 < o1 ? m1 : o1;
    m1 = m1 < o1 ? o1 : m1;
    m2 = m2 < o2 ? o2 : m2;
    m2 = m2 < lo ? lo : m2;
  }
  const C score = !p.top2 || m1 == -ninf ? m1 : m1 + m2;
  int better = 0;
  for (int o = 0; o < p.n_group; ++o) {
    const C v = __shfl_sync(kFull, score, o * lpg);
    better += v > score || (v == score && o < g);
  }
  const bool keep = g < p.n_group && better < p.topk_group;
  C lo = keep ? score : -ninf, hi = keep || g >= p.n_group ? ninf : score;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const C a = __shfl_xor_sync(kFull, lo, o), b = __shfl_xor_sync(kFull, hi, o);
    lo = a < lo ? a : lo;
    hi = b > hi ? b : hi;
  }
  *gap = lo - hi;
  return __ballot_sync(kFull, keep);
}

// One token in 64 bits, NV experts a lane; `scores`: the scores with their bias
// are compared, else the logits.
template <int NV>
__device__ __noinline__ void route_exact(const TopkParams& p, int64_t t, int lane, double* stage,
                                         bool scores) {
  const double ninf = -static_cast<double>(INFINITY);
  const int64_t row = t * p.ld;
  float x[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int e = j * 32 + lane;
    x[j] = e < p.E ? no_nan(load_elem(p.logits, p.dtype, row + e)) : -INFINITY;
  }
  float m = x[0];
#pragma unroll
  for (int j = 1; j < NV; ++j) m = fmaxf(m, x[j]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kFull, m, o));
  double c[NV];
  float sum = 0.f;   // of a softmax row's exponentials
  if (p.sigmoid) {
#pragma unroll
    for (int j = 0; j < NV; ++j) c[j] = 1.0 / (1.0 + exp(-static_cast<double>(x[j])));
  } else {
    double total = 0.0;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      c[j] = j * 32 + lane < p.E ? shifted_exp64(x[j], m) : 0.0;
      total += c[j];
    }
    total = warp_sum(total);
    const double inv = total > 0.0 ? 1.0 / total : 0.0;
#pragma unroll
    for (int j = 0; j < NV; ++j) c[j] *= inv;
    sum = static_cast<float>(total);
  }
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int e = j * 32 + lane;
    if (!scores) c[j] = static_cast<double>(x[j]);
    if (p.bias && e < p.E) c[j] += static_cast<double>(load_elem(p.bias, p.bias_dtype, e));
    if (isnan(c[j])) c[j] = ninf;
  }
  // experts that may still be chosen, one bit per j
  unsigned open = 0u;
#pragma unroll
  for (int j = 0; j < NV; ++j) open |= (j * 32 + lane < p.E ? 1u : 0u) << j;
  if (p.topk_group < p.n_group) {
    __syncwarp();
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (j * 32 + lane < p.E) stage[j * 32 + lane] = c[j];
    __syncwarp();
    double gap;
    const unsigned kept = kept_groups(p, stage, lane, &gap);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int e = j * 32 + lane;
      if (e < p.E && !((kept >> (group_of(p, e) * p.lanes_per_group)) & 1u)) open &= ~(1u << j);
    }
  }
  // the lane's best open expert (the first of equals: its lowest id)
  double bv = ninf;
  int bj = -1;
  auto scan = [&] {
    bv = ninf;
    bj = -1;
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (((open >> j) & 1u) && (bj < 0 || c[j] > bv)) {
        bv = c[j];
        bj = j;
      }
  };
  scan();
  int my_idx = 0;
  for (int k = 0; k < p.top_k; ++k) {
    // a 64-bit score rounded to 32 bits keeps the order except for equal keys
    const unsigned key = bj < 0 ? 0u : order_key(static_cast<float>(bv));
    bool best = key == __reduce_max_sync(kFull, key);
    if (__popc(__ballot_sync(kFull, best)) > 1) {
      const double top = warp_max(best && bj >= 0 ? bv : ninf);
      best = best && bj >= 0 && bv == top;
    }
    const unsigned e = __reduce_min_sync(kFull, best && bj >= 0 ? bj * 32u + lane : kFull);
    if (lane == k) my_idx = static_cast<int>(e);
    if (lane == static_cast<int>(e & 31u)) {
      open &= ~(1u << (e >> 5));
      scan();
    }
  }
  float s = 0.f;
  if (lane < p.top_k) {
    const float mx = no_nan(load_elem(p.logits, p.dtype, row + my_idx));
    s = p.sigmoid ? sigmoid(mx) : sum > 0.f ? shifted_exp(mx, m) / sum : 0.f;
  }
  store_choice(p, t, lane, my_idx, s);
}

// 1 / (sum of a softmax row's exponentials) in 64 bits; finite m.
__device__ __forceinline__ double exact_inverse(const TopkParams& p, int64_t row, int lane, float m) {
  if (p.sigmoid) return 1.0;
  double total = 0.0;
#pragma unroll 1
  for (int e = lane; e < p.E; e += 32)
    total += shifted_exp64(no_nan(load_elem(p.logits, p.dtype, row + e)), m);
  return 1.0 / warp_sum(total);
}
// Score with bias of expert e in 64 bits.
__device__ __forceinline__ double exact_score(const TopkParams& p, int64_t row, int e, float m, double inv) {
  const float x = no_nan(load_elem(p.logits, p.dtype, row + e));
  double c = p.sigmoid ? 1.0 / (1.0 + exp(-static_cast<double>(x))) : shifted_exp64(x, m) * inv;
  if (p.bias) c += static_cast<double>(load_elem(p.bias, p.bias_dtype, e));
  return isnan(c) ? -static_cast<double>(INFINITY) : c;
}

// X: type of the logits.  kScores: scores with a bias or summed over groups are
// compared, not logits.
//
// Scores are compared as 32-bit integers of the same order.  The top_k-th largest
// of the 32 lanes' best scores is a threshold that the chosen experts reach: the
// experts that do, about top_k of them, are moved to one lane each, and their
// ranks are counted by comparing all of them with all.  Logits are compared
// exactly.  A score in fp32 is off by kScoreSlack of the row's largest: where one
// of the chosen is no further than that from another candidate, the candidates'
// scores are computed in 64 bits and ranked again, and where a kept group is no
// further from a dropped one, those of all experts (normal logits: one token in
// thousands).  Tokens with more than 32 candidates (rows of equal scores), NaN or
// infinite maxima or masked experts among the chosen go through route_exact.
//
// kScoreSlack: expf is within 2 ulps (2^-22) and its argument within half an ulp
// (2^-24 |d|, and e^-|d| |d| < 0.37); the sum is off by the mean of that over its
// weights (|d| below log 1024 on average) and by a tree of ten additions; two
// products round: less than 28 * 2^-24.  kSigmoidSlack: a sigmoid moves by s (1 - s)
// <= 1/4 of its exponential's 2^-22, its sum rounds (2^-24) and its quotient is
// within two ulps (2 * 2^-24 below 1): 4 * 2^-24.
//
// About 650 instructions a token of 512 experts without a bias, 1000 with one (fp32,
// T = 16384, logits in L2: 14 and 21 us; from DRAM they take 5).  Bound by the latency of
// a token's chain of reductions (maximum, sum, threshold, scan, ranks) at 20 warps an
// SM: 58% of the issue slots are used.
template <int NV, bool kScores, bool kGrouped, typename X>
__global__ void __launch_bounds__(kTopkWarps * 32, topk_blocks_per_sm(NV))
    moe_topk_kernel(const __grid_constant__ TopkParams p) {
  extern __shared__ double stage_s[];            // grouped: a token's scores for each warp
  __shared__ unsigned long long found[kTopkWarps][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t warps = static_cast<int64_t>(gridDim.x) * kTopkWarps;
  double* const stage = stage_s + warp * (NV * 32);
  float bias[kScores ? NV : 1];
  if constexpr (kScores) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int e = j * 32 + lane;
      bias[j] = p.bias && e < p.E ? load_elem(p.bias, p.bias_dtype, e) : 0.f;
    }
  }
  // The next token's logits are on their way while one is routed.
  const X* const logits = static_cast<const X*>(p.logits) + lane;
  X next[NV];
  auto load = [&](int64_t t) {
    const X* const r = logits + t * p.ld;
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (j * 32 + lane < p.E) next[j] = r[j * 32];
  };
  int64_t t = static_cast<int64_t>(blockIdx.x) * kTopkWarps + warp;
  if (t < p.T) load(t);
  // Tokens to route again wait for the end of a run of 32, so that the call's
  // registers are not the loop's.
  while (t < p.T) {
    const int64_t run = t;
    unsigned again = 0u;
    for (int it = 0; it < 32 && t < p.T; ++it, t += warps) {
      const int64_t row = t * p.ld;
      float c[NV];
#pragma unroll
      for (int j = 0; j < NV; ++j) c[j] = j * 32 + lane < p.E ? to_float(next[j]) : -INFINITY;
      if (t + warps < p.T) load(t + warps);
      float m = c[0], slack = 0.f;   // a NaN does not become the maximum
#pragma unroll
      for (int j = 1; j < NV; ++j) m = fmaxf(m, c[j]);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kFull, m, o));
      bool sure = m < INFINITY && m > -INFINITY;
      float inv = 0.f;
      if constexpr (kScores) {
        if (p.sigmoid) {   // a NaN logit takes part with its bias, also in its group
#pragma unroll
          for (int j = 0; j < NV; ++j) c[j] = sigmoid(no_nan(c[j])) + bias[j];
          slack = kSigmoidSlack;
        } else {
          float part[NV];
#pragma unroll
          for (int j = 0; j < NV; ++j) part[j] = c[j] = expf(c[j] - m);
#pragma unroll
          for (int w = NV / 2; w > 0; w >>= 1)
#pragma unroll
            for (int j = 0; j < w; ++j) part[j] += part[j + w];
          inv = 1.f / warp_sum(part[0]);
#pragma unroll
          for (int j = 0; j < NV; ++j) c[j] = fmaf(c[j], inv, bias[j]);
          slack = kScoreSlack * inv;
        }
      }
      unsigned kept = kFull;
      if constexpr (kGrouped) {
        float* st = reinterpret_cast<float*>(stage);
        __syncwarp();
#pragma unroll
        for (int j = 0; j < NV; ++j)
          if (j * 32 + lane < p.E) st[j * 32 + lane] = no_nan(c[j]);
        __syncwarp();
        float gap;
        kept = kept_groups(p, st, lane, &gap);
        if constexpr (kScores) {
          unsigned top = 0u;   // bits of the largest finite |c|
#pragma unroll
          for (int j = 0; j < NV; ++j)
            if (fabsf(c[j]) < INFINITY) top = max(top, __float_as_uint(fabsf(c[j])));
          top = __reduce_max_sync(kFull, top);
          if (sure && !(gap > 4.f * slack + 4.f * 0x1p-23f * __uint_as_float(top))) {
            const double inv64 = exact_inverse(p, row, lane, m);
            __syncwarp();
#pragma unroll 1
            for (int e = lane; e < p.E; e += 32) stage[e] = exact_score(p, row, e, m, inv64);
            __syncwarp();
            double gap64;
            kept = kept_groups(p, stage, lane, &gap64);
          }
        }
      }
      unsigned key[NV];   // 0: not open to choice
      unsigned best = 0u;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int e = j * 32 + lane;
        bool open = e < p.E;
        if constexpr (kGrouped) open = open && ((kept >> (group_of(p, e) * p.lanes_per_group)) & 1u);
        key[j] = open ? order_key(c[j]) : 0u;
        best = max(best, key[j]);
      }
      // the top_k-th largest of the lanes' best, or less where some are equal
      unsigned threshold = 0u, largest = 0u;
      for (int k = 0; k < p.top_k; ++k) {
        threshold = __reduce_max_sync(kFull, best);
        if (best == threshold) best = 0u;
        if (k == 0) largest = threshold;
      }
      // no masked expert or NaN (keys below and above the infinities') takes part
      constexpr unsigned kNegInf = 0x007fffffu, kPosInf = 0xff800000u;
      sure = sure && largest < kPosInf && (threshold > kNegInf || threshold == 0u);
      float tol = 0.f;
      if constexpr (kScores) {
        // candidates within the scores' error below the threshold come along
        const float v = threshold ? key_value(threshold) : 0.f;
        tol = 2.f * slack + 0x1p-22f * fabsf(v);   // two scores' errors and roundings
        if (threshold != 0u) threshold = order_key(v - tol);
      }
      threshold = max(threshold, 1u);
      // one candidate a lane: key and complement of the id, larger first
      int count = 0;
#pragma unroll
      for (int j = 0; j < NV; ++j) count += key[j] >= threshold ? 1 : 0;
      int at = count;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(kFull, at, o);
        if (lane >= o) at += v;
      }
      const int n = __shfl_sync(kFull, at, 31);
      sure = sure && n <= 32;
      if (!sure) {   // the same on all lanes
        again |= 1u << it;
        continue;
      }
      at -= count;
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (key[j] >= threshold) {
          found[warp][at] = (static_cast<unsigned long long>(key[j]) << 32) | ~(j * 32u + lane);
          ++at;
        }
      __syncwarp();
      const unsigned long long mine = lane < n ? found[warp][lane] : 0ull;
      const float value = key_value(static_cast<unsigned>(mine >> 32));
      int rank = 0;
      for (int i = 0; i < n; ++i) rank += found[warp][i] > mine;
      if (lane >= n) rank = 32;
      __syncwarp();   // `found` is read
      const int e = static_cast<int>(~static_cast<unsigned>(mine));
      // with fewer candidates than top_k, or among logits -inf chosen, masked
      // experts take part
      if (n < p.top_k ||
          (!kScores && __any_sync(kFull, rank < p.top_k && static_cast<unsigned>(mine >> 32) <= kNegInf))) {
        again |= 1u << it;
        continue;
      }
      if constexpr (kScores) {
        // in the order of the ranks: is each of the chosen far enough from the next?
        float* const order = reinterpret_cast<float*>(found[warp]);
        if (lane < n) order[rank] = value;
        __syncwarp();
        const float next = rank + 1 < n ? order[rank + 1] : -INFINITY;
        const bool close = rank < p.top_k && rank + 1 < n && !(value - next > tol + 0x1p-22f * fabsf(value));
        __syncwarp();
        if (__any_sync(kFull, close)) {
          const double inv64 = exact_inverse(p, row, lane, m);
          const double c64 = lane < n ? exact_score(p, row, e, m, inv64) : 0.0;
          rank = 0;
#pragma unroll 1
          for (int i = 0; i < n; ++i) {
            const double o = __shfl_sync(kFull, c64, i);
            const int oe = __shfl_sync(kFull, e, i);
            rank += o > c64 || (o == c64 && oe < e);
          }
          if (lane >= n) rank = 32;
        }
      }
      const bool chosen = rank < p.top_k;
      float x = value;
      if constexpr (kScores) x = chosen ? no_nan(load_elem(p.logits, p.dtype, row + e)) : 0.f;
      float s = 0.f;
      if (p.sigmoid) {
        s = chosen ? sigmoid(x) : 0.f;
      } else {
        s = chosen ? expf(x - m) : 0.f;
        if constexpr (kScores) {
          s *= inv;
        } else if (!p.renormalize || !(warp_sum(s) > 1e-10f)) {
          // The row's sum cancels when renormalising, unless the chosen weights
          // vanish beside the row's maximum (a dropped group's).
          float sum = 0.f;
#pragma unroll
          for (int j = 0; j < NV; ++j) sum += expf(no_nan(c[j] - m));
          s = __fdividef(s, warp_sum(sum));
        }
      }
      store_choice(p, t, rank, e, s);
    }
    for (; again; again &= again - 1u)
      route_exact<NV>(p, run + (__ffs(again) - 1) * warps, lane, stage, kScores);
  }
}

namespace {

template <int NV, typename X>
int launch_topk_x(const TopkParams& p, bool scores, int blocks, cudaStream_t s) {
  const bool grouped = p.topk_group < p.n_group;
  const size_t smem = grouped ? sizeof(double) * kTopkWarps * NV * 32 : 0;
  if (scores && grouped)
    moe_topk_kernel<NV, true, true, X><<<blocks, kTopkWarps * 32, smem, s>>>(p);
  else if (scores)
    moe_topk_kernel<NV, true, false, X><<<blocks, kTopkWarps * 32, 0, s>>>(p);
  else if (grouped)
    moe_topk_kernel<NV, false, true, X><<<blocks, kTopkWarps * 32, smem, s>>>(p);
  else
    moe_topk_kernel<NV, false, false, X><<<blocks, kTopkWarps * 32, 0, s>>>(p);
  return cudaGetLastError() == cudaSuccess ? MOE_OK : MOE_ERR_CUDA;
}

template <int NV>
int launch_topk(const TopkParams& p, bool scores, int sms, cudaStream_t s) {
  int64_t want = (p.T + kTopkWarps - 1) / kTopkWarps;
  if (want > static_cast<int64_t>(sms) * topk_blocks_per_sm(NV)) want = sms * topk_blocks_per_sm(NV);
  const int blocks = static_cast<int>(want);
  if (p.dtype == MOE_BF16) return launch_topk_x<NV, __nv_bfloat16>(p, scores, blocks, s);
  if (p.dtype == MOE_F16) return launch_topk_x<NV, __half>(p, scores, blocks, s);
  return launch_topk_x<NV, float>(p, scores, blocks, s);
}

}  // namespace

}  // namespace moe

extern "C" int moe_route_topk(const void* logits, int32_t dtype, int64_t ld, const void* bias,
                              int32_t bias_dtype, int64_t T, int64_t E, int64_t top_k,
                              int32_t score, int64_t n_group, int64_t topk_group,
                              int32_t group_score, int32_t renormalize,
                              float routed_scaling_factor, int32_t* topk_idx, float* topk_weights,
                              void* stream) {
  using namespace moe;
  if (T < 0 || T > (int64_t(1) << 24) || E < 1 || E > kTopkMaxExperts) return MOE_ERR_SHAPE;
  if (n_group < 1 || n_group > 32 || E % n_group != 0) return MOE_ERR_SHAPE;
  if (topk_group < 1 || topk_group > n_group) return MOE_ERR_SHAPE;
  if (top_k < 1 || top_k > 32 || top_k > topk_group * (E / n_group)) return MOE_ERR_SHAPE;
  if (ld < E) return MOE_ERR_SHAPE;
  auto dtype_ok = [](int32_t d) { return d == MOE_F32 || d == MOE_BF16 || d == MOE_F16; };
  if (!dtype_ok(dtype) || (bias && !dtype_ok(bias_dtype))) return MOE_ERR_INVALID_ARG;
  if (score != MOE_SCORE_SOFTMAX && score != MOE_SCORE_SIGMOID) return MOE_ERR_INVALID_ARG;
  if (group_score != MOE_GROUP_TOP2 && group_score != MOE_GROUP_MAX) return MOE_ERR_INVALID_ARG;
  const bool grouped = topk_group < n_group;
  if (grouped && group_score == MOE_GROUP_TOP2 && E / n_group < 2) return MOE_ERR_SHAPE;
  if (T == 0) return MOE_OK;
  if (!logits || !topk_idx || !topk_weights) return MOE_ERR_INVALID_ARG;
  const uintptr_t elem = dtype == MOE_F32 ? 3u : 1u, belem = bias_dtype == MOE_F32 ? 3u : 1u;
  if ((reinterpret_cast<uintptr_t>(logits) & elem) || (bias && (reinterpret_cast<uintptr_t>(bias) & belem)) ||
      (reinterpret_cast<uintptr_t>(topk_idx) & 3u) || (reinterpret_cast<uintptr_t>(topk_weights) & 3u))
    return MOE_ERR_ALIGNMENT;
  int sms = 0;
  const int st = num_sms(&sms);
  if (st) return st;
  TopkParams p{};
  p.logits = logits;
  p.dtype = dtype;
  p.ld = ld;
  p.bias = bias;
  p.bias_dtype = bias_dtype;
  p.T = T;
  p.E = static_cast<int>(E);
  p.top_k = static_cast<int>(top_k);
  p.sigmoid = score == MOE_SCORE_SIGMOID;
  p.n_group = static_cast<int>(n_group);
  p.topk_group = static_cast<int>(topk_group);
  p.group_size = static_cast<int>(E / n_group);
  p.group_inv = static_cast<unsigned>(((1 << 20) + p.group_size - 1) / p.group_size);
  p.lanes_per_group = 32;
  while (p.lanes_per_group * p.n_group > 32) p.lanes_per_group /= 2;
  p.top2 = group_score == MOE_GROUP_TOP2;
  p.renormalize = renormalize != 0;
  p.factor = routed_scaling_factor;
  p.topk_idx = topk_idx;
  p.topk_weights = topk_weights;
  const bool scores = bias != nullptr || (grouped && p.top2);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (E <= 32) return launch_topk<1>(p, scores, sms, s);
  if (E <= 64) return launch_topk<2>(p, scores, sms, s);
  if (E <= 128) return launch_topk<4>(p, scores, sms, s);
  if (E <= 256) return launch_topk<8>(p, scores, sms, s);
  if (E <= 512) return launch_topk<16>(p, scores, sms, s);
  return launch_topk<32>(p, scores, sms, s);
}
