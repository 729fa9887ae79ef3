// Microscaled 4-bit floating point: quantisation to e2m1 codes with a scale per
// run of columns, and back.
//
//   mxfp4: runs of 32, e8m0 scale s = 2^(floor(log2(amax)) - 2) (at least 2^-127)
//   nvfp4: runs of 16, e4m3 scale s = rne(amax / (6 g)), at most 448 and, unless
//          amax is 0, at least 2^-9; g: one fp32 scale of the whole tensor
//   code = e2m1_rne(x / (s g)), saturating at 6;   value = code * s * g
//
// Both roundings are those of the exact quotients.  With a power of two that is
// a multiplication.  With an e4m3 scale it takes more, because tensor scales are
// ratios (amax / 2688), which put whole classes of 16-bit values exactly on, or
// one rounding beside, the border of two codes.  The borders of a run are 1, 3, 5
// and 7 times powers of two times s g, 32 mantissas for all e4m3 scales, so a block
// finds out beforehand which of them 16-bit values can be near at all (their
// mantissa is that of a 16-bit number but for its last bits) and on which side of
// it those are, by a comparison in 64 bits, which is exact.  They are moved there
// by 2^-18 before the conversion.  An fp32 value is converted a little below and a little above its
// quotient, and compared with the borders in 64 bits where the two codes differ.
// (Converting 16-bit values twice as well took 50 us at 8192 x 7168: a conversion
// to e2m1 keeps its unit busy for many cycles.  Doing half of the conversions in
// fp32 arithmetic instead, as the minimum of three straight lines, was no faster.)
//
// A run with a NaN or an infinity, and every run when g is not a positive
// number, gets the scale's NaN code (0xff, 0x7f), so that it stays NaN through
// a product.
//
// The scales go to the layout that the tensor core's scale copy reads: blocks of
// 128 rows x 4 scales, in which row r of the block and scale b are byte
// (r % 32) * 16 + (r / 32) * 4 + b; the threads of one block's four scales
// gather them with shuffles and store one word.  Rows and columns that fill up
// the last blocks have scale 0.  Bound by memory: 2.56 bytes an element.
#include "moe_kernels.cuh"

#include <cuda_fp16.h>
#include <cuda_fp4.h>

namespace moe {

namespace {

// 16 consecutive elements as they lie in memory.
template <typename X>
struct Raw16 {
  uint4 v[sizeof(X)];   // 32 or 64 bytes
  __device__ __forceinline__ void load(const X* p) {
#pragma unroll
    for (int h = 0; h < static_cast<int>(sizeof(X)); ++h) v[h] = reinterpret_cast<const uint4*>(p)[h];
  }
  __device__ __forceinline__ void get(float (&f)[16]) const {
#pragma unroll
    for (int h = 0; h < static_cast<int>(sizeof(X)); ++h) {
      const uint32_t w[4] = {v[h].x, v[h].y, v[h].z, v[h].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(X) == 4) {
          f[4 * h + i] = __uint_as_float(w[i]);
        } else {
          float2 two;
          if constexpr (std::is_same<X, __half>::value)
            two = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
          else
            two = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]));
          f[8 * h + 2 * i] = two.x;
          f[8 * h + 2 * i + 1] = two.y;
        }
      }
    }
  }
};

// Bits of the largest |f|; a NaN is above every number.
__device__ __forceinline__ uint32_t amax_bits(const float (&f)[16]) {
  uint32_t m = 0u;
#pragma unroll
  for (int j = 0; j < 16; ++j) m = max(m, __float_as_uint(f[j]) & 0x7fffffffu);
  return m;
}

// Eight e2m1 codes of f[0..7] times `scale`, the first in the lowest four bits.
__device__ __forceinline__ uint32_t pack_e2m1x8(const float* f, float scale) {
  uint32_t r = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    r |= static_cast<uint32_t>(__nv_cvt_float2_to_fp4x2(
             make_float2(f[2 * i] * scale, f[2 * i + 1] * scale), __NV_E2M1, cudaRoundNearest))
         << (8 * i);
  return r;
}

// The borders of a tensor's runs: with i = 1, 3, 5, 7 and a scale whose mantissa is
// m = 8..15, powers of two times m i g.  Entry 4 (m - 8) + i / 2 tells of one
// whether 16-bit values (kBits fraction bits) can be within 2^-20 of it, their
// mantissa, and the factor that moves them to their side of it; a value on the
// border goes to the even code, below the borders with i = 1 and 5 and above those
// with 3 and 7.  Values with a border's mantissa that are no border's are codes
// themselves, or beyond the largest, and can be moved as well.
struct Borders {
  uint32_t near;   // a bit per entry
  uint32_t mantissa[32];
  float move[32];
};
constexpr uint32_t kFraction = 0x7fffffu;

template <int kBits>
__device__ __forceinline__ void find_borders(Borders* b, float g, int lane) {
  constexpr uint32_t kRest = (1u << (23 - kBits)) - 1u, kNear = 16u;
  const int mi = (8 + lane / 4) * (2 * (lane & 3) + 1);
  const uint32_t t = __float_as_uint(static_cast<float>(mi) * g) + kNear;
  const double value = __uint_as_float(t & ~kRest);
  const double border = static_cast<double>(mi) * static_cast<double>(g);
  const bool up = value > border || (value == border && (lane & 1));
  b->mantissa[lane] = t & kFraction & ~kRest;
  b->move[lane] = up ? 1.f + 0x1p-18f : 1.f - 0x1p-18f;
  const uint32_t near = __ballot_sync(0xffffffffu, (t & kRest) <= 2u * kNear);
  if (lane == 0) b->near = near;
}

// Moves the values of f that are near a border of a run with scale s.
__device__ __forceinline__ void leave_borders(float (&f)[16], float s, uint32_t near, const Borders* b) {
  const uint32_t first = ((__float_as_uint(s) >> 20) & 7u) * 4u;
  for (uint32_t left = (near >> first) & 15u; left; left &= left - 1u) {
    const uint32_t k = first + __ffs(left) - 1u;
    const uint32_t mantissa = b->mantissa[k];
    const float move = b->move[k];
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if ((__float_as_uint(f[j]) & kFraction) == mantissa) f[j] *= move;
  }
}

// The code of v against the exact borders; den = s * g, exact.
__device__ __forceinline__ uint32_t e2m1_exact(float v, double den) {
  const double a = fabs(static_cast<double>(v));
  const uint32_t i = (a > 0.25 * den) + (a >= 0.75 * den) + (a > 1.25 * den) + (a >= 1.75 * den) +
                     (a > 2.5 * den) + (a >= 3.5 * den) + (a > 5.0 * den);
  return i | (signbit(v) ? 8u : 0u);
}

// Nearest e4m3 code (ties to even) of a non-negative double up to 448: the
// conversion to fp32 keeps the sticky bit, so the second rounding is exact.
__device__ __forceinline__ uint32_t e4m3_of_double(double t) {
  float f = __double2float_rz(t);
  if (static_cast<double>(f) != t) f = __uint_as_float(__float_as_uint(f) | 1u);
  return pack_e4m3x2(f, 0.f) & 0xffu;
}

__device__ __forceinline__ float e4m3_value(uint32_t code) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(code), __NV_E4M3)));
}
__device__ __forceinline__ float e8m0_value(uint32_t code) {
  return code == 0xffu ? NAN : __uint_as_float(code == 0u ? 0x00400000u : code << 23);
}

}  // namespace

namespace {

// What every run of one tensor shares (nvfp4).
struct TensorScale {
  float g, inv6g;
  bool ok, inv6g_ok;
  __device__ __forceinline__ explicit TensorScale(const float* p) {
    g = p ? __ldg(p) : 1.f;
    ok = g > 0.f && g < INFINITY;
    inv6g = 1.f / (6.f * g);   // within 3 * 2^-24
    inv6g_ok = g > 1e-36f && g < 1e36f;
  }
};

// One run of 16 values at x: codes in q0, q1; returns the scale's code.
template <typename X>
__device__ __forceinline__ uint32_t quantize_nv(float (&f)[16], const X* x, const TensorScale& ts,
                                                uint32_t near, const Borders* borders, uint32_t& q0,
                                                uint32_t& q1) {
  const uint32_t m = amax_bits(f);
  if (m >= 0x7f800000u || !ts.ok) {
    q0 = q1 = 0u;
    return 0x7fu;
  }
  if (m == 0u) {
    q0 = pack_e2m1x8(f, 1.f);   // the zeros' signs
    q1 = pack_e2m1x8(f + 8, 1.f);
    return 0u;
  }
  // e4m3 of amax / (6 g): three fraction bits, ties to even, of the fp32 quotient,
  // and of the exact one if that is too close to a border to tell, below the
  // normal e4m3 values (2^-6) or next to the end of the fp32 range
  const uint32_t t = __float_as_uint(fminf(__uint_as_float(m) * ts.inv6g, 448.f));
  uint32_t rounded = (t + 0x7ffffu + ((t >> 20) & 1u)) & ~0xfffffu;
  uint32_t code = (rounded >> 20) - (120u << 3);
  if (t < 0x3c800000u || ((t + 16u) & 0xfffffu) - 0x80000u <= 32u || !ts.inv6g_ok) {
    code = max(1u, e4m3_of_double(fmin(
                       static_cast<double>(__uint_as_float(m)) / (6.0 * static_cast<double>(ts.g)), 448.0)));
    rounded = __float_as_uint(e4m3_value(code));
  }
  const float s = __uint_as_float(rounded);
  const float d = s * ts.g;
  const float inv = __fdividef(1.f, d);   // within 2^-22
  unsigned long long differ = 0ull;   // values to be looked at, four bits each
  if constexpr (sizeof(X) == 2) {
    leave_borders(f, s, near, borders);
    q0 = pack_e2m1x8(f, inv);
    q1 = pack_e2m1x8(f + 8, inv);
  } else {
    const float below = inv * (1.f - 0x1p-20f), above = inv * (1.f + 0x1p-20f);
    q0 = pack_e2m1x8(f, below);
    q1 = pack_e2m1x8(f + 8, below);
    differ = (static_cast<unsigned long long>(q1 ^ pack_e2m1x8(f + 8, above)) << 32) |
             (q0 ^ pack_e2m1x8(f, above));
  }
  if (!(d > 1e-35f && d < 1e35f)) differ = ~0ull;   // subnormals: outside the bounds
  if (differ) {
    const double den = static_cast<double>(s) * static_cast<double>(ts.g);
    do {
      const int j = (__ffsll(differ) - 1) / 4;
      const uint32_t v = e2m1_exact(static_cast<float>(x[j]), den);
      const int at = 4 * (j & 7);
      if (j < 8)
        q0 = (q0 & ~(15u << at)) | (v << at);
      else
        q1 = (q1 & ~(15u << at)) | (v << at);
      differ &= ~(15ull << (4 * j));
    } while (differ);
  }
  return code;
}

}  // namespace

// A thread takes 64 bytes of input: 32 columns of a 16-bit type, 16 of fp32.
template <typename X, bool kNv>
__global__ void __launch_bounds__(256, kNv ? 4 : 5) moe_fp4_quantize_kernel(Fp4QuantParams p) {
  griddep_launch_dependents();   // a product that follows streams its weights meanwhile
  constexpr int kCols = 64 / static_cast<int>(sizeof(X)), kRun = kNv ? 16 : 32, kParts = kCols / 16;
  constexpr int kThreadsPerWord = 4 * kRun / kCols;   // threads whose scales share a word
  const int lane = threadIdx.x & 31;
  const int64_t units = static_cast<int64_t>(p.chunks) * kThreadsPerWord;   // per padded row
  const int64_t total = (p.R + 127) / 128 * 128 * units;   // a multiple of 32
  const int64_t stride = static_cast<int64_t>(gridDim.x) * blockDim.x;
  const TensorScale ts(p.global_scale);
  __shared__ Borders borders;
  uint32_t near = 0u;
  if constexpr (kNv && sizeof(X) == 2) {
    if (threadIdx.x < 32) find_borders<std::is_same<X, __half>::value ? 10 : 7>(&borders, ts.g, lane);
    __syncthreads();
    near = borders.near;
  }
  // row and column step by the grid's size (below 2^31) without divisions
  const uint32_t start = blockIdx.x * blockDim.x + threadIdx.x;
  int64_t i = start;
  int64_t r = start / static_cast<uint32_t>(units);
  int u = static_cast<int>(start % static_cast<uint32_t>(units));
  const int r_step = static_cast<int>(static_cast<uint32_t>(stride) / static_cast<uint32_t>(units));
  const int u_step = static_cast<int>(static_cast<uint32_t>(stride) % static_cast<uint32_t>(units));
  for (; i < total; i += stride) {
    const bool live = r < p.R && kCols * u < p.K;
    const X* const x = static_cast<const X*>(p.x) + r * p.ld + kCols * u;
    Raw16<X> raw[kParts];
    if (live) {
#pragma unroll
      for (int h = 0; h < kParts; ++h) raw[h].load(x + 16 * h);
    }
    uint32_t code = 0u;   // of the thread's scales
    uint32_t q[2 * kParts];
    if constexpr (kNv) {
      if (live) {
#pragma unroll
        for (int h = 0; h < kParts; ++h) {
          float f[16];
          raw[h].get(f);
          code |= quantize_nv<X>(f, x + 16 * h, ts, near, &borders, q[2 * h], q[2 * h + 1]) << (8 * h);
        }
      }
    } else {
      float f[kParts][16];
      uint32_t m = 0u;
      if (live) {
#pragma unroll
        for (int h = 0; h < kParts; ++h) {
          raw[h].get(f[h]);
          m = max(m, amax_bits(f[h]));
        }
      }
      if constexpr (kCols < kRun) m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
      if (live) {
        const bool bad = m >= 0x7f800000u;
        const int e = max(static_cast<int>(m >> 23) - 129, -127);
        code = bad ? 0xffu : static_cast<uint32_t>(e + 127);
        const float inv = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
#pragma unroll
        for (int h = 0; h < kParts; ++h) {
          q[2 * h] = bad ? 0u : pack_e2m1x8(f[h], inv);
          q[2 * h + 1] = bad ? 0u : pack_e2m1x8(f[h] + 8, inv);
        }
      }
    }
    if (live) {
      uint8_t* const c = p.codes + r * (p.K / 2) + kCols / 2 * u;
      if constexpr (kParts == 2)
        *reinterpret_cast<uint4*>(c) = make_uint4(q[0], q[1], q[2], q[3]);
      else
        *reinterpret_cast<uint2*>(c) = make_uint2(q[0], q[1]);
    }
    // one word of four scales: two or one a thread, or one for two threads
    uint32_t word = code;
    if constexpr (kThreadsPerWord == 2) {
      word |= __shfl_down_sync(0xffffffffu, word, 1) << 16;
    } else {
      constexpr int kStep = kThreadsPerWord / 4;
      word |= __shfl_down_sync(0xffffffffu, word, kStep) << 8;
      word |= __shfl_down_sync(0xffffffffu, word, 2 * kStep) << 16;
    }
    if (lane % kThreadsPerWord == 0) {
      const int64_t block = r / 128 * p.chunks + u / kThreadsPerWord;
      const int rr = static_cast<int>(r % 128);
      *reinterpret_cast<uint32_t*>(p.scales + block * 512 + (rr % 32) * 16 + (rr / 32) * 4) = word;
    }
    r += r_step;
    u += u_step;
    if (u >= units) {
      u -= static_cast<int>(units);
      ++r;
    }
  }
}

template <typename O>
__device__ __forceinline__ void store16(O* p, const float (&f)[16]);
template <>
__device__ __forceinline__ void store16(float* p, const float (&f)[16]) {
#pragma unroll
  for (int h = 0; h < 4; ++h)
    reinterpret_cast<float4*>(p)[h] = make_float4(f[4 * h], f[4 * h + 1], f[4 * h + 2], f[4 * h + 3]);
}
template <>
__device__ __forceinline__ void store16(__nv_bfloat16* p, const float (&f)[16]) {
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&b);
  }
  reinterpret_cast<uint4*>(p)[0] = make_uint4(w[0], w[1], w[2], w[3]);
  reinterpret_cast<uint4*>(p)[1] = make_uint4(w[4], w[5], w[6], w[7]);
}
template <>
__device__ __forceinline__ void store16(__half* p, const float (&f)[16]) {
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const __half2 b = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&b);
  }
  reinterpret_cast<uint4*>(p)[0] = make_uint4(w[0], w[1], w[2], w[3]);
  reinterpret_cast<uint4*>(p)[1] = make_uint4(w[4], w[5], w[6], w[7]);
}

// code * s is exact in fp32 (2 and 4 significant bits); the tensor scale and
// the output type each round once.  A thread takes 16 columns.
template <typename O, bool kNv>
__global__ void __launch_bounds__(256) moe_fp4_dequantize_kernel(Fp4QuantParams p) {
  const int64_t units = p.K / 16;
  const int64_t total = p.R * units;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * blockDim.x;
  const float g = kNv && p.global_scale ? __ldg(p.global_scale) : 1.f;
  // row and column step by the grid's size (below 2^31) without divisions
  const uint32_t start = blockIdx.x * blockDim.x + threadIdx.x;
  int64_t i = start;
  int64_t r = start / static_cast<uint32_t>(units);
  int u = static_cast<int>(start % static_cast<uint32_t>(units));
  const int r_step = static_cast<int>(static_cast<uint32_t>(stride) / static_cast<uint32_t>(units));
  const int u_step = static_cast<int>(static_cast<uint32_t>(stride) % static_cast<uint32_t>(units));
  for (; i < total; i += stride) {
    const int b = kNv ? u : u / 2;
    const int rr = static_cast<int>(r % 128);
    const uint2 q = __ldcs(reinterpret_cast<const uint2*>(p.codes + r * p.ld + 8 * u));
    const uint32_t sc =
        p.scales[(r / 128 * p.chunks + b / 4) * 512 + (rr % 32) * 16 + (rr / 32) * 4 + b % 4];
    const float s = kNv ? e4m3_value(sc) : e8m0_value(sc);
    float f[16];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t two = ((j < 4 ? q.x : q.y) >> (8 * (j & 3))) & 0xffu;
      const float2 v = __half22float2(
          __half2(__nv_cvt_fp4x2_to_halfraw2(static_cast<__nv_fp4x2_storage_t>(two), __NV_E2M1)));
      f[2 * j] = kNv ? v.x * s * g : v.x * s;
      f[2 * j + 1] = kNv ? v.y * s * g : v.y * s;
    }
    store16(static_cast<O*>(p.out) + r * p.K + 16 * u, f);
    r += r_step;
    u += u_step;
    if (u >= units) {
      u -= static_cast<int>(units);
      ++r;
    }
  }
}

namespace {

int blocks_for(int64_t threads, int sms) {
  int64_t b = (threads + 255) / 256;
  if (b > static_cast<int64_t>(sms) * 32) b = static_cast<int64_t>(sms) * 32;
  return static_cast<int>(b < 1 ? 1 : b);
}

template <bool kNv>
int quantize_dtype(const Fp4QuantParams& p, int dtype, int blocks, cudaStream_t s) {
  if (dtype == MOE_BF16)
    moe_fp4_quantize_kernel<__nv_bfloat16, kNv><<<blocks, 256, 0, s>>>(p);
  else if (dtype == MOE_F16)
    moe_fp4_quantize_kernel<__half, kNv><<<blocks, 256, 0, s>>>(p);
  else
    moe_fp4_quantize_kernel<float, kNv><<<blocks, 256, 0, s>>>(p);
  return cudaGetLastError() == cudaSuccess ? MOE_OK : MOE_ERR_CUDA;
}

template <bool kNv>
int dequantize_dtype(const Fp4QuantParams& p, int dtype, int blocks, cudaStream_t s) {
  if (dtype == MOE_BF16)
    moe_fp4_dequantize_kernel<__nv_bfloat16, kNv><<<blocks, 256, 0, s>>>(p);
  else if (dtype == MOE_F16)
    moe_fp4_dequantize_kernel<__half, kNv><<<blocks, 256, 0, s>>>(p);
  else
    moe_fp4_dequantize_kernel<float, kNv><<<blocks, 256, 0, s>>>(p);
  return cudaGetLastError() == cudaSuccess ? MOE_OK : MOE_ERR_CUDA;
}

}  // namespace

int launch_fp4_quantize(const Fp4QuantParams& p, int dtype, int format, int sms, cudaStream_t s) {
  const bool nv = format == MOE_NVFP4;
  const int64_t threads = (p.R + 127) / 128 * 128 * p.chunks * (nv ? 2 : 4) * (dtype == MOE_F32 ? 2 : 1);
  const int blocks = blocks_for(threads, sms);
  return nv ? quantize_dtype<true>(p, dtype, blocks, s) : quantize_dtype<false>(p, dtype, blocks, s);
}

int fp4_check(int32_t format, int64_t R, int64_t K) {
  if (format != MOE_MXFP4 && format != MOE_NVFP4) return MOE_ERR_INVALID_ARG;
  // K a multiple of 32: 16-byte rows of codes for the TMA, whole runs of both formats
  if (R < 0 || R > (int64_t(1) << 24) || K < 32 || K % 32 != 0 || K > 65536) return MOE_ERR_SHAPE;
  return MOE_OK;
}

int fp4_chunks(int32_t format, int64_t K) {
  return static_cast<int>(format == MOE_NVFP4 ? (K + 63) / 64 : (K + 127) / 128);
}

}  // namespace moe

using namespace moe;

namespace {
bool off(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) != 0; }
}  // namespace

extern "C" {

int moe_fp4_scales_size(int32_t format, int64_t R, int64_t K, size_t* bytes) {
  if (!bytes) return MOE_ERR_INVALID_ARG;
  const int st = fp4_check(format, R, K);
  if (st) return st;
  *bytes = static_cast<size_t>((R + 127) / 128) * fp4_chunks(format, K) * 512;
  return MOE_OK;
}

int moe_fp4_quantize(const void* x, int32_t x_dtype, int64_t ld, int64_t R, int64_t K,
                     int32_t format, const float* global_scale, void* codes, void* scales,
                     void* stream) {
  int st = fp4_check(format, R, K);
  if (st) return st;
  if (x_dtype != MOE_BF16 && x_dtype != MOE_F16 && x_dtype != MOE_F32) return MOE_ERR_INVALID_ARG;
  if (format == MOE_MXFP4 && global_scale) return MOE_ERR_INVALID_ARG;
  if (ld < K || ld % (x_dtype == MOE_F32 ? 4 : 8) != 0) return MOE_ERR_SHAPE;
  if (R == 0) return MOE_OK;
  if (!x || !codes || !scales) return MOE_ERR_INVALID_ARG;
  if (off(x, 16) || off(codes, 16) || off(scales, 16) || off(global_scale, 4)) return MOE_ERR_ALIGNMENT;
  int sms = 0;
  if ((st = num_sms(&sms))) return st;
  Fp4QuantParams p{};
  p.x = x;
  p.ld = ld;
  p.R = R;
  p.K = static_cast<int>(K);
  p.chunks = fp4_chunks(format, K);
  p.global_scale = global_scale;
  p.codes = static_cast<uint8_t*>(codes);
  p.scales = static_cast<uint8_t*>(scales);
  return launch_fp4_quantize(p, x_dtype, format, sms, static_cast<cudaStream_t>(stream));
}

int moe_fp4_dequantize(const void* codes, int64_t ld, const void* scales, int64_t R, int64_t K,
                       int32_t format, const float* global_scale, void* out, int32_t out_dtype,
                       void* stream) {
  int st = fp4_check(format, R, K);
  if (st) return st;
  if (out_dtype != MOE_BF16 && out_dtype != MOE_F16 && out_dtype != MOE_F32) return MOE_ERR_INVALID_ARG;
  if (format == MOE_MXFP4 && global_scale) return MOE_ERR_INVALID_ARG;
  if (ld < K / 2 || ld % 16 != 0) return MOE_ERR_SHAPE;
  if (R == 0) return MOE_OK;
  if (!codes || !scales || !out) return MOE_ERR_INVALID_ARG;
  if (off(codes, 16) || off(scales, 16) || off(out, 16) || off(global_scale, 4)) return MOE_ERR_ALIGNMENT;
  int sms = 0;
  if ((st = num_sms(&sms))) return st;
  Fp4QuantParams p{};
  p.codes = static_cast<uint8_t*>(const_cast<void*>(codes));
  p.scales = static_cast<uint8_t*>(const_cast<void*>(scales));
  p.ld = ld;
  p.R = R;
  p.K = static_cast<int>(K);
  p.chunks = fp4_chunks(format, K);
  p.global_scale = global_scale;
  p.out = out;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int blocks = blocks_for(R * (K / 16), sms);
  return format == MOE_NVFP4 ? dequantize_dtype<true>(p, out_dtype, blocks, s)
                             : dequantize_dtype<false>(p, out_dtype, blocks, s);
}

}  // extern "C"
