// Residual addition, RMS norm and FP8 quantisation in one pass: the producer of
// the layer's hidden_states / hidden_states_scale (and of the router GEMM's
// 16-bit input) from the output of the block before it.
//
//   h = x + residual                      (fp32; stored back in the residual's type)
//   y = h * rsqrt(mean(h^2) + eps) * w    (fp32; stored in x's type when asked for)
//   scale[b, t] = max(amax |y| over the 128 columns of block b * fp32(1/448), 1e-12)
//   q = e4m3(y / scale)
//
// One block per row, the row in registers: every input is read once and every
// output written once.  A thread owns vectors of 8 columns, so the 16 lanes of
// a half warp hold one 128-column scale block and its maximum takes four
// shuffles.  The norm and the codes are computed from the unrounded fp32 sum h and
// the fp32 product y.  The squares are added in trees in a warp and in 64 bits
// across the row (no slower than one fp32 chain), and the quotient by the scale is
// a multiplication by its reciprocal with one correction step, as exact as a
// division at a third of its instructions.  Carrying the rounding errors of the two
// products of y into the codes as well was measured and left out: 88 -> 95 us at
// T = 8192, H = 7168, for about one code in a million (errors of 1e-7 against codes
// a tenth apart).  Of 58.7 M codes some 2,100 are not the exact ones (the formula in fp32
// has as many), all but a handful of them values that lie exactly between two codes.
//
// Bound by memory: 9 bytes an element with a 16-bit residual and the normed
// output.
#include "moe_kernels.cuh"

#include <cuda_fp16.h>

namespace moe {

namespace {

__device__ __forceinline__ float2 unpack2(uint32_t v, __nv_bfloat16) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
}
__device__ __forceinline__ float2 unpack2(uint32_t v, __half) {
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&p);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
  const __half2 p = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&p);
}

// The larger one, NaN if either is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Eight consecutive elements as they lie in memory, 16 bytes or 32.  32 move at once if
// they are aligned to their size (`wide`): half sectors of L2 cost more (fp32 residual
// and weight at T = 901, H = 2048: 5.3 us in halves, 4.7 us; T = 1024, H = 7168: 19.7, 17.9).
template <typename E>
struct Vec8 {
  uint4 v;
  __device__ __forceinline__ void load(const E* p, bool) { v = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 a = unpack2(w[i], E{});
      f[2 * i] = a.x;
      f[2 * i + 1] = a.y;
    }
  }
  static __device__ __forceinline__ void store(E* p, const float (&f)[8], bool) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack2(f[0], f[1], E{}), pack2(f[2], f[3], E{}),
                                              pack2(f[4], f[5], E{}), pack2(f[6], f[7], E{}));
  }
};
template <>
struct Vec8<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p, bool wide) {
    if (wide) {
      asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                   : "=f"(a.x), "=f"(a.y), "=f"(a.z), "=f"(a.w), "=f"(b.x), "=f"(b.y), "=f"(b.z), "=f"(b.w)
                   : "l"(p)
                   : "memory");
    } else {
      a = *reinterpret_cast<const float4*>(p);
      b = *reinterpret_cast<const float4*>(p + 4);
    }
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  }
  static __device__ __forceinline__ void store(float* p, const float (&f)[8], bool wide) {
    if (wide) {
      asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(f[0]), "f"(f[1]),
                   "f"(f[2]), "f"(f[3]), "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7])
                   : "memory");
    } else {
      *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
      *reinterpret_cast<float4*>(p + 4) = make_float4(f[4], f[5], f[6], f[7]);
    }
  }
};

struct NoResidual {};

// Threads a row may have with P vectors each: 8192 columns with one and 16384 with
// up to four stay in registers.
constexpr int max_threads(int p) { return p == 1 || p == 8 ? 1024 : 512; }

}  // namespace

// R = NoResidual: no residual.  P vectors of 8 columns a thread.  The residual
// may be updated in place: a thread reads its elements before it writes them.
template <typename X, typename R, typename W, int P>
__global__ void __launch_bounds__(max_threads(P)) moe_rms_norm_1x128_kernel(NormParams p) {
  constexpr bool kRes = !std::is_same<R, NoResidual>::value;
  using RV = typename std::conditional<kRes, R, float>::type;
  __shared__ float part[32];
  const int64_t t = blockIdx.x;
  const int nvec = p.H / 8;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nwarps = blockDim.x >> 5;
  const X* xr = static_cast<const X*>(p.x) + t * p.ld_x;
  Vec8<X> xv[P];
  Vec8<RV> rv[P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int v = tid + i * blockDim.x;
    if (v < nvec) {
      xv[i].load(xr + 8 * v, false);
      if constexpr (kRes) rv[i].load(static_cast<const R*>(p.residual) + t * p.ld_res + 8 * v, p.wide);
    }
  }
  Vec8<W> wv[P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int v = tid + i * blockDim.x;
    if (v < nvec) wv[i].load(static_cast<const W*>(p.weight) + 8 * v, p.wide);
  }
  float h[P][8];
  float sums[P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int v = tid + i * blockDim.x;
    sums[i] = 0.f;
    if (v < nvec) {
      xv[i].get(h[i]);
      if constexpr (kRes) {
        float r[8];
        rv[i].get(r);
#pragma unroll
        for (int j = 0; j < 8; ++j) h[i][j] += r[j];
        Vec8<RV>::store(static_cast<RV*>(p.residual_out) + t * p.ld_res_out + 8 * v, h[i], p.wide);
      }
      float two[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) two[j] = fmaf(h[i][j], h[i][j], h[i][j + 4] * h[i][j + 4]);
      sums[i] = (two[0] + two[1]) + (two[2] + two[3]);
    }
  }
#pragma unroll
  for (int w = P / 2; w > 0; w >>= 1)
#pragma unroll
    for (int i = 0; i < w; ++i) sums[i] += sums[i + w];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sums[0] += __shfl_xor_sync(0xffffffffu, sums[0], o);
  if (lane == 0) part[warp] = sums[0];
  __syncthreads();
  double sum = lane < nwarps ? part[lane] : 0.0;
  for (int o = 1; o < nwarps; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  sum = __shfl_sync(0xffffffffu, sum, 0);
  const double var = fma(sum, p.inv_h, static_cast<double>(p.eps));
  float rstd = rsqrtf(static_cast<float>(var));
  // one step in 64 bits rounds it to nearest (not of zero, infinity and NaN)
  const double rest = 1.0 - static_cast<double>(rstd) * rstd * var;
  if (fabs(rest) < 1e-5) rstd = static_cast<float>(rstd + 0.5 * rstd * rest);
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int v = tid + i * blockDim.x;
    // H is a multiple of 128: the 16 lanes of a scale block are all inside or
    // all outside the row.  A NaN reaches the scale.
    float w[8];
    float m = 0.f;
    if (v < nvec) {
      wv[i].get(w);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float n = h[i][j] * rstd, y = n * w[j];
        h[i][j] = y;
        m = max_nan(m, fabsf(y));
      }
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (v < nvec) {
      const float top = m * (1.0f / 448.0f);
      const float s = top < 1e-12f ? 1e-12f : top;
      const float inv = __frcp_rn(s);
      float d[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float d0 = h[i][j] * inv;   // inv = 0: s is infinite
        d[j] = inv > 0.f ? fmaf(fmaf(-d0, s, h[i][j]), inv, d0) : d0;
      }
      const uint32_t q0 = pack_e4m3x2(d[0], d[1]), q1 = pack_e4m3x2(d[2], d[3]);
      const uint32_t q2 = pack_e4m3x2(d[4], d[5]), q3 = pack_e4m3x2(d[6], d[7]);
      *reinterpret_cast<uint2*>(p.q + t * p.H + 8 * v) =
          make_uint2(q0 | (q1 << 16), q2 | (q3 << 16));
      if ((lane & 15) == 0) p.scale[static_cast<int64_t>(v / 16) * p.T + t] = s;
      if (p.normed) Vec8<X>::store(static_cast<X*>(p.normed) + t * p.ld_normed + 8 * v, h[i], false);
    }
  }
}

namespace {

template <typename X, typename R, typename W>
int launch_p(const NormParams& p, int vecs, int threads, cudaStream_t s) {
  const unsigned grid = static_cast<unsigned>(p.T);
  switch (vecs) {
    case 1: moe_rms_norm_1x128_kernel<X, R, W, 1><<<grid, threads, 0, s>>>(p); break;
    case 2: moe_rms_norm_1x128_kernel<X, R, W, 2><<<grid, threads, 0, s>>>(p); break;
    case 4: moe_rms_norm_1x128_kernel<X, R, W, 4><<<grid, threads, 0, s>>>(p); break;
    default: moe_rms_norm_1x128_kernel<X, R, W, 8><<<grid, threads, 0, s>>>(p); break;
  }
  return cudaGetLastError() == cudaSuccess ? MOE_OK : MOE_ERR_CUDA;
}

template <typename X, typename R>
int launch_w(const NormParams& p, int w_dtype, int vecs, int threads, cudaStream_t s) {
  return w_dtype == MOE_F32 ? launch_p<X, R, float>(p, vecs, threads, s)
                            : launch_p<X, R, X>(p, vecs, threads, s);
}

template <typename X>
int launch_r(const NormParams& p, int r_dtype, int w_dtype, int vecs, int threads, cudaStream_t s) {
  if (!p.residual) return launch_w<X, NoResidual>(p, w_dtype, vecs, threads, s);
  return r_dtype == MOE_F32 ? launch_w<X, float>(p, w_dtype, vecs, threads, s)
                            : launch_w<X, X>(p, w_dtype, vecs, threads, s);
}

}  // namespace

int launch_rms_norm_1x128(const NormParams& p, int x_dtype, int r_dtype, int w_dtype, int sms,
                          cudaStream_t s) {
  // Vectors a thread holds: one when there are too few rows to fill the SMs
  // (the shortest chain of loads), more when rows queue up.
  const int nvec = p.H / 8;
  int vecs = p.T <= 2 * sms ? 1 : nvec >= 512 ? 4 : nvec >= 256 ? 2 : 1;
  while ((nvec + vecs - 1) / vecs > max_threads(vecs)) vecs *= 2;
  const int threads = ((nvec + vecs - 1) / vecs + 31) / 32 * 32;
  return x_dtype == MOE_BF16 ? launch_r<__nv_bfloat16>(p, r_dtype, w_dtype, vecs, threads, s)
                             : launch_r<__half>(p, r_dtype, w_dtype, vecs, threads, s);
}

}  // namespace moe

extern "C" int moe_rms_norm_1x128(const void* x, int32_t x_dtype, int64_t ld_x, const void* residual,
                                  int32_t residual_dtype, int64_t ld_residual, const void* weight,
                                  int32_t weight_dtype, float eps, int64_t T, int64_t H,
                                  void* residual_out, int64_t ld_residual_out, void* normed,
                                  int64_t ld_normed, void* q, float* scale, void* stream) {
  using namespace moe;
  if (T < 0 || T > (int64_t(1) << 24) || H < 128 || H % 128 != 0 || H > 65536) return MOE_ERR_SHAPE;
  if (x_dtype != MOE_BF16 && x_dtype != MOE_F16) return MOE_ERR_INVALID_ARG;
  if (weight_dtype != x_dtype && weight_dtype != MOE_F32) return MOE_ERR_INVALID_ARG;
  if (residual && residual_dtype != x_dtype && residual_dtype != MOE_F32) return MOE_ERR_INVALID_ARG;
  if ((residual == nullptr) != (residual_out == nullptr)) return MOE_ERR_INVALID_ARG;
  if (!(eps >= 0.f)) return MOE_ERR_INVALID_ARG;
  if (T == 0) return MOE_OK;
  if (!x || !weight || !q || !scale) return MOE_ERR_INVALID_ARG;
  const int64_t r_unit = residual_dtype == MOE_F32 ? 4 : 8;   // elements of 16 bytes
  auto rows_ok = [H](int64_t ld, int64_t unit) { return ld >= H && ld % unit == 0; };
  if (!rows_ok(ld_x, 8) || (normed && !rows_ok(ld_normed, 8)) ||
      (residual && (!rows_ok(ld_residual, r_unit) || !rows_ok(ld_residual_out, r_unit))))
    return MOE_ERR_SHAPE;
  auto off16 = [](const void* a) { return (reinterpret_cast<uintptr_t>(a) & 15u) != 0; };
  if (off16(x) || off16(residual) || off16(weight) || off16(residual_out) || off16(normed) ||
      off16(q) || (reinterpret_cast<uintptr_t>(scale) & 3u) != 0)
    return MOE_ERR_ALIGNMENT;
  int sms = 0;
  const int st = num_sms(&sms);
  if (st) return st;
  NormParams p{};
  p.x = x;
  p.residual = residual;
  p.weight = weight;
  p.residual_out = residual_out;
  p.normed = normed;
  p.q = static_cast<uint8_t*>(q);
  p.scale = scale;
  p.T = T;
  p.H = static_cast<int>(H);
  p.ld_x = ld_x;
  p.ld_res = ld_residual;
  p.ld_res_out = ld_residual_out;
  p.ld_normed = ld_normed;
  p.eps = eps;
  p.inv_h = 1.0 / static_cast<double>(H);
  auto off32 = [](const void* a) { return (reinterpret_cast<uintptr_t>(a) & 31u) != 0; };
  p.wide = !off32(weight) && !off32(residual) && !off32(residual_out) && ld_residual % 8 == 0 &&
           ld_residual_out % 8 == 0;
  return launch_rms_norm_1x128(p, x_dtype, residual_dtype, weight_dtype, sms,
                               static_cast<cudaStream_t>(stream));
}
