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
// and 7 times powers of two times s g, so a 16-bit value can be near one only if
// one of four numbers has the mantissa of a 16-bit number but for its last bits.
// Then the values with that mantissa are all on the same side, which one
// comparison in 64 bits (exact) tells, and are moved there by 2^-18 before the
// conversion.  An fp32 value is converted a little below and a little above its
// quotient, and compared with the borders in 64 bits where the two codes differ.
// (Converting 16-bit values twice as well took 50 us at 8192 x 7168: a conversion
// to e2m1 keeps its unit busy for many cycles.  Doing half of the conversions in
// fp32 arithmetic instead, as the minimum of three straight lines, was no faster.)
//
// A run with a NaN or an infinity, and every run when g is not a positive
// number, gets the scale's NaN code (0xff, 0x7f), so that it stays NaN through
// a product.
//
// A thread takes 16 columns: 32 bytes of 16-bit input, 8 bytes of codes.  The
// scales go to the layout that the tensor core's scale copy reads: blocks of
// 128 rows x 4 scales, in which row r of the block and scale b are byte
// (r % 32) * 16 + (r / 32) * 4 + b; the threads of one block's four scales
// gather them with shuffles and store one word.  Rows and columns that fill up
// the last blocks have scale 0.  Bound by memory: 2.56 bytes an element.
#include "moe_kernels.cuh"

#include <cuda_fp16.h>
#include <cuda_fp4.h>

namespace moe {

namespace {

__device__ __forceinline__ void load16(const __nv_bfloat16* p, float (&f)[16]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint4 u = reinterpret_cast<const uint4*>(p)[h];
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]));
      f[8 * h + 2 * i] = v.x;
      f[8 * h + 2 * i + 1] = v.y;
    }
  }
}
__device__ __forceinline__ void load16(const __half* p, float (&f)[16]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint4 u = reinterpret_cast<const uint4*>(p)[h];
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[8 * h + 2 * i] = v.x;
      f[8 * h + 2 * i + 1] = v.y;
    }
  }
}
__device__ __forceinline__ void load16(const float* p, float (&f)[16]) {
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    const float4 v = reinterpret_cast<const float4*>(p)[h];
    f[4 * h] = v.x;
    f[4 * h + 1] = v.y;
    f[4 * h + 2] = v.z;
    f[4 * h + 3] = v.w;
  }
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

// Moves the values of f (16-bit numbers with kBits fraction bits) that are within
// 2^-20 of a border of a run with scale s, d = fp32(s * g), to their side of it; a
// value on the border goes to the even code, below odd multiples 1 and 5 of the
// smallest border and above 3 and 7.  Values with a border's mantissa that are no
// border's are codes themselves, or beyond the largest, and can be moved as well.
template <int kBits>
__device__ __forceinline__ void leave_borders(float (&f)[16], float d, float s, float g) {
  constexpr uint32_t kRest = (1u << (23 - kBits)) - 1u, kNear = 16u, kMantissa = 0x7fffffu & ~kRest;
#pragma unroll
  for (int i = 1; i < 8; i += 2) {
    const uint32_t t = __float_as_uint(d * static_cast<float>(i)) + kNear;
    if ((t & kRest) <= 2u * kNear) {
      const double value = __uint_as_float(t & ~kRest);
      const double border = static_cast<double>(s) * i * static_cast<double>(g);
      const bool up = value > border || (value == border && (i & 2));
      const float move = up ? 1.f + 0x1p-18f : 1.f - 0x1p-18f;
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (((__float_as_uint(f[j]) ^ t) & kMantissa) == 0u) f[j] *= move;
    }
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

template <typename X, bool kNv>
__global__ void __launch_bounds__(256) moe_fp4_quantize_kernel(Fp4QuantParams p) {
  griddep_launch_dependents();   // a product that follows streams its weights meanwhile
  constexpr int kThreadsPerWord = kNv ? 4 : 8;   // threads whose scales share a word
  const int lane = threadIdx.x & 31;
  const int64_t units = static_cast<int64_t>(p.chunks) * kThreadsPerWord;   // per padded row
  const int64_t total = (p.R + 127) / 128 * 128 * units;   // a multiple of 32
  const bool small = total < (int64_t(1) << 32);
  const int64_t stride = static_cast<int64_t>(gridDim.x) * blockDim.x;
  float g = 1.f;
  bool g_ok = true;
  if (kNv && p.global_scale) {
    g = __ldg(p.global_scale);
    g_ok = g > 0.f && g < INFINITY;
  }
  const float inv6g = 1.f / (6.f * g);   // within 3 * 2^-24
  const bool inv6g_ok = g > 1e-36f && g < 1e36f;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total; i += stride) {
    const int64_t r = small ? static_cast<uint32_t>(i) / static_cast<uint32_t>(units) : i / units;
    const int u = static_cast<int>(i - r * units);
    const bool live = r < p.R && 16 * u < p.K;
    float f[16];
    uint32_t m = 0u;
    if (live) {
      load16(static_cast<const X*>(p.x) + r * p.ld + 16 * u, f);
#pragma unroll
      for (int j = 0; j < 16; ++j) m = max(m, __float_as_uint(fabsf(f[j])));
    }
    if constexpr (!kNv) m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    uint32_t code = 0u, q0 = 0u, q1 = 0u;
    const bool bad = m >= 0x7f800000u || !g_ok;
    if (live) {
      if constexpr (kNv) {
        if (bad) {
          code = 0x7fu;
        } else if (m == 0u) {
          q0 = pack_e2m1x8(f, 1.f);   // the zeros' signs
          q1 = pack_e2m1x8(f + 8, 1.f);
        } else {
          // the scale likewise: amax / (6 g) once in fp32, and exactly if that
          // is too close to a border (or to the fp32 range) to tell
          const uint32_t t = __float_as_uint(fminf(__uint_as_float(m) * inv6g, 448.f));
          // three fraction bits, ties to even, of a normal e4m3 value
          uint32_t rounded = (t + 0x7ffffu + ((t >> 20) & 1u)) & ~0xfffffu;
          if (t < 0x3c800000u || ((t + 16u) & 0xfffffu) - 0x80000u <= 32u || !inv6g_ok) {
            code = e4m3_of_double(
                fmin(static_cast<double>(__uint_as_float(m)) / (6.0 * static_cast<double>(g)), 448.0));
            rounded = __float_as_uint(e4m3_value(max(1u, code)));
          }
          const float s = __uint_as_float(rounded);
          code = rounded >= 0x3c800000u ? (rounded >> 20) - (120u << 3)      // normal, from 2^-6 on
                                        : static_cast<uint32_t>(s * 512.f);  // a multiple of 2^-9
          const float d = s * g;
          const float inv = __frcp_rn(d);
          unsigned long long differ = 0ull;   // values to be looked at, four bits each
          if constexpr (sizeof(X) == 2) {
            leave_borders<std::is_same<X, __half>::value ? 10 : 7>(f, d, s, g);
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
            const double den = static_cast<double>(s) * static_cast<double>(g);
            const X* const x = static_cast<const X*>(p.x) + r * p.ld + 16 * u;
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
        }
      } else {
        if (bad) {
          code = 0xffu;
        } else {
          const int e = max(static_cast<int>(m >> 23) - 129, -127);
          code = static_cast<uint32_t>(e + 127);
          const float inv = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
          q0 = pack_e2m1x8(f, inv);
          q1 = pack_e2m1x8(f + 8, inv);
        }
      }
      *reinterpret_cast<uint2*>(p.codes + r * (p.K / 2) + 8 * u) = make_uint2(q0, q1);
    }
    // one word of four scales
    constexpr int kStep = kThreadsPerWord / 4;
    const int first = lane / kThreadsPerWord * kThreadsPerWord;
    uint32_t word = 0u;
#pragma unroll
    for (int j = 0; j < 4; ++j) word |= __shfl_sync(0xffffffffu, code, first + j * kStep) << (8 * j);
    if (lane == first) {
      const int64_t block = r / 128 * p.chunks + u / kThreadsPerWord;
      const int rr = static_cast<int>(r % 128);
      *reinterpret_cast<uint32_t*>(p.scales + block * 512 + (rr % 32) * 16 + (rr / 32) * 4) = word;
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
// the output type each round once.
template <typename O, bool kNv>
__global__ void __launch_bounds__(256) moe_fp4_dequantize_kernel(Fp4QuantParams p) {
  const int64_t units = p.K / 16;
  const int64_t total = p.R * units;
  const bool small = total < (int64_t(1) << 32);
  const int64_t stride = static_cast<int64_t>(gridDim.x) * blockDim.x;
  const float g = kNv && p.global_scale ? __ldg(p.global_scale) : 1.f;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total; i += stride) {
    const int64_t r = small ? static_cast<uint32_t>(i) / static_cast<uint32_t>(units) : i / units;
    const int u = static_cast<int>(i - r * units);
    const int b = kNv ? u : u / 2;
    const int rr = static_cast<int>(r % 128);
    const uint32_t sc =
        p.scales[(r / 128 * p.chunks + b / 4) * 512 + (rr % 32) * 16 + (rr / 32) * 4 + b % 4];
    const float s = kNv ? e4m3_value(sc) : e8m0_value(sc);
    const uint2 q = *reinterpret_cast<const uint2*>(p.codes + r * p.ld + 8 * u);
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
  const int64_t threads = (p.R + 127) / 128 * 128 * p.chunks * (nv ? 4 : 8);
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
