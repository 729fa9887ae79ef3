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
// A NaN logit or bias counts as -inf: such an expert ranks last, and a -inf
// logit weighs 0 (a row without a single finite logit has zero weights).
// +inf logits share a softmax row's weight equally.
//
// One warp per token.  Lane l holds experts l, l+32, ..., so loads are
// coalesced and an expert's lane is its id modulo 32.  A round of the top-k is
// one warp maximum of an order-preserving 32-bit key (redux) and one warp
// minimum of the ids that hold it; 64-bit scores are rounded to 32 bits for the
// key, which keeps their order except for equal keys, and only those are
// compared in full.
#include "moe_kernels.cuh"

#include <cuda_fp16.h>

namespace moe {

namespace {

constexpr int kTopkWarps = 4;
constexpr unsigned kFull = 0xffffffffu;

__device__ __forceinline__ float load_elem(const void* p, int dtype, int64_t i) {
  if (dtype == MOE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  if (dtype == MOE_F16) return __half2float(static_cast<const __half*>(p)[i]);
  return static_cast<const float*>(p)[i];
}

__device__ __forceinline__ float no_nan(float v) { return isnan(v) ? -INFINITY : v; }

// Unsigned key with the order of the float (-inf is 0x007fffff, above 0).
__device__ __forceinline__ unsigned order_key(float v) {
  v = v == 0.f ? 0.f : v;   // -0 and 0 are the same score
  const unsigned b = __float_as_uint(v);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
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

// NV experts a lane.  C = float: the logits are compared; C = double: the
// scores with their bias are.
template <int NV, typename C>
__global__ void __launch_bounds__(kTopkWarps * 32) moe_topk_kernel(TopkParams p) {
  constexpr bool k64 = std::is_same<C, double>::value;
  __shared__ C stage[kTopkWarps][NV * 32];   // one token's scores, for the groups
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t warps = static_cast<int64_t>(gridDim.x) * kTopkWarps;
  const C ninf = -static_cast<C>(INFINITY);
  float bias[k64 ? NV : 1];
  if constexpr (k64) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int e = j * 32 + lane;
      bias[j] = p.bias && e < p.E ? load_elem(p.bias, p.bias_dtype, e) : 0.f;
    }
  }
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * kTopkWarps + warp; t < p.T; t += warps) {
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
    C c[NV];
    double total = 0.0;   // sum of a softmax row's exponentials
    if constexpr (k64) {
      if (p.sigmoid) {
#pragma unroll
        for (int j = 0; j < NV; ++j) c[j] = 1.0 / (1.0 + exp(-static_cast<double>(x[j])));
      } else {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          c[j] = j * 32 + lane < p.E ? shifted_exp64(x[j], m) : 0.0;
          total += c[j];
        }
        total = warp_sum(total);
        const double inv = total > 0.0 ? 1.0 / total : 0.0;
#pragma unroll
        for (int j = 0; j < NV; ++j) c[j] *= inv;
      }
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        c[j] += static_cast<double>(bias[j]);
        if (isnan(c[j])) c[j] = ninf;
      }
    } else {
#pragma unroll
      for (int j = 0; j < NV; ++j) c[j] = x[j];
    }
    // experts that may still be chosen, one bit per j
    unsigned open = 0u;
#pragma unroll
    for (int j = 0; j < NV; ++j) open |= (j * 32 + lane < p.E ? 1u : 0u) << j;
    if (p.topk_group < p.n_group) {
      // lanes_per_group lanes share a group: its two best scores, then its rank
      __syncwarp();
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (j * 32 + lane < p.E) stage[warp][j * 32 + lane] = c[j];
      __syncwarp();
      const int lpg = p.lanes_per_group, g = lane / lpg, size = p.group_size;
      C m1 = ninf, m2 = ninf;
      if (g < p.n_group) {
        for (int i = lane % lpg; i < size; i += lpg) {
          const C v = stage[warp][g * size + i];
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
      const unsigned kept = __ballot_sync(kFull, g < p.n_group && better < p.topk_group);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int e = j * 32 + lane;
        if (e < p.E && !((kept >> ((e / size) * lpg)) & 1u)) open &= ~(1u << j);
      }
    }
    // the lane's best open expert (the first of equals: its lowest id)
    C bv = ninf;
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
      const unsigned key = bj < 0 ? 0u : order_key(static_cast<float>(bv));
      const unsigned kmax = __reduce_max_sync(kFull, key);
      bool best = key == kmax;
      if constexpr (k64) {
        if (__popc(__ballot_sync(kFull, best)) > 1) {   // equal in 32 bits: compare in 64
          const double top = warp_max(best && bj >= 0 ? bv : ninf);
          best = best && bj >= 0 && bv == top;
        }
      }
      const unsigned e = __reduce_min_sync(kFull, best && bj >= 0 ? bj * 32u + lane : kFull);
      if (lane == k) my_idx = static_cast<int>(e);
      if (lane == static_cast<int>(e & 31u)) {
        open &= ~(1u << (e >> 5));
        scan();
      }
    }
    // weights of the chosen experts, one per lane
    float s = 0.f;
    const bool mine = lane < p.top_k;
    const float xs = mine ? no_nan(load_elem(p.logits, p.dtype, row + my_idx)) : -INFINITY;
    if (p.sigmoid) {
      s = mine ? 1.f / (1.f + expf(-xs)) : 0.f;
    } else {
      s = mine ? shifted_exp(xs, m) : 0.f;
      float sum;
      if constexpr (k64) {
        sum = static_cast<float>(total);
      } else if (p.renormalize && warp_sum(s) > 1e-10f) {
        sum = 1.f;   // cancels (1e-20 adds less than a rounding)
      } else {
        sum = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j)
          if (j * 32 + lane < p.E) sum += shifted_exp(x[j], m);
        sum = warp_sum(sum);
      }
      s = sum > 0.f ? s / sum : 0.f;
    }
    if (p.renormalize) s = s / (warp_sum(s) + 1e-20f);
    if (mine) {
      p.topk_idx[t * p.top_k + lane] = my_idx;
      p.topk_weights[t * p.top_k + lane] = s * p.factor;
    }
  }
}

namespace {

template <int NV>
int launch_topk(const TopkParams& p, bool wide, int blocks, cudaStream_t s) {
  if (wide)
    moe_topk_kernel<NV, double><<<blocks, kTopkWarps * 32, 0, s>>>(p);
  else
    moe_topk_kernel<NV, float><<<blocks, kTopkWarps * 32, 0, s>>>(p);
  return cudaGetLastError() == cudaSuccess ? MOE_OK : MOE_ERR_CUDA;
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
  p.lanes_per_group = 32;
  while (p.lanes_per_group * p.n_group > 32) p.lanes_per_group /= 2;
  p.top2 = group_score == MOE_GROUP_TOP2;
  p.renormalize = renormalize != 0;
  p.factor = routed_scaling_factor;
  p.topk_idx = topk_idx;
  p.topk_weights = topk_weights;
  const bool wide = bias != nullptr || (grouped && p.top2);
  int64_t blocks = (T + kTopkWarps - 1) / kTopkWarps;
  if (blocks > static_cast<int64_t>(sms) * 16) blocks = static_cast<int64_t>(sms) * 16;
  const int b = static_cast<int>(blocks);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (E <= 32) return launch_topk<1>(p, wide, b, s);
  if (E <= 64) return launch_topk<2>(p, wide, b, s);
  if (E <= 128) return launch_topk<4>(p, wide, b, s);
  if (E <= 256) return launch_topk<8>(p, wide, b, s);
  if (E <= 512) return launch_topk<16>(p, wide, b, s);
  return launch_topk<32>(p, wide, b, s);
}
