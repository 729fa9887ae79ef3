// Device side of the 4-bit quantisation: one run of columns to e2m1 codes and the
// code of its scale.  See moe_fp4.cu for the formats.
//
// Both roundings are those of the exact quotients.  With a power of two that is
// a multiplication.  With an e4m3 scale it takes more, because tensor scales are
// ratios (amax / 2688), which put whole classes of 16-bit values exactly on, or
// one rounding beside, the border of two codes.  The borders of a run are 1, 3, 5
// and 7 times powers of two times s g, 32 mantissas for all e4m3 scales, so a block
// finds out beforehand which of them 16-bit values can be near at all (their
// mantissa is that of a 16-bit number but for its last bits) and on which side of
// it those are, by a comparison in 64 bits, which is exact.  For most scales the
// reciprocal of s g then only has to be moved by 2^-19 to that side, which cannot
// take another value across a border; where values are exactly on borders the
// quotient is rounded correctly, which leaves it on the border; what remains is
// moved value by value.  An fp32 value is converted a little below and a little
// above its quotient, and compared with the borders in 64 bits where the two codes
// differ.  (At 8192 x 7168 in bf16: 26 us, 39 with g = 1, where values on borders are
// common.  Converting 16-bit values twice as well cost 4 us more when it was tried, and
// moving every value near a border by itself 15 us more with g = 1.)
//
// A run with a NaN or an infinity, and every run when g is not a positive
// number, gets the scale's NaN code (0xff, 0x7f), so that it stays NaN through
// a product.
#pragma once

#include "moe_kernels.cuh"

#include <cuda_fp16.h>
#include <cuda_fp4.h>

namespace moe {

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
  // fp32 bits of the largest magnitude; a NaN is above every number.
  __device__ __forceinline__ uint32_t amax_bits() const {
    uint32_t m = 0u;
    if constexpr (sizeof(X) == 4) {
#pragma unroll
      for (int h = 0; h < 4; ++h)
        m = max(max(m, max(v[h].x & 0x7fffffffu, v[h].y & 0x7fffffffu)),
                max(v[h].z & 0x7fffffffu, v[h].w & 0x7fffffffu));
    } else {
      using X2 = typename std::conditional<std::is_same<X, __half>::value, __half2, __nv_bfloat162>::type;
      const uint32_t w[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w};
      X2 top = __habs2(*reinterpret_cast<const X2*>(&w[0]));
#pragma unroll
      for (int i = 1; i < 8; ++i) top = __hmax2_nan(top, __habs2(*reinterpret_cast<const X2*>(&w[i])));
      m = max(__float_as_uint(__low2float(top)), __float_as_uint(__high2float(top)));
    }
    return m;
  }
};

// (a.x * b, a.y * b) in one instruction.
__device__ __forceinline__ float2 mul2(float x, float y, float b) {
  float2 r;
  asm("{\n\t.reg .b64 v, w;\n\tmov.b64 v, {%2, %3};\n\tmov.b64 w, {%4, %4};\n\t"
      "mul.rn.f32x2 v, v, w;\n\tmov.b64 {%0, %1}, v;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(x), "f"(y), "f"(b));
  return r;
}

// Eight e2m1 codes of f[0..7] times `scale`, the first in the lowest four bits.
__device__ __forceinline__ uint32_t pack_e2m1x8(const float* f, float scale) {
  const float2 a = mul2(f[0], f[1], scale), b = mul2(f[2], f[3], scale);
  const float2 c = mul2(f[4], f[5], scale), d = mul2(f[6], f[7], scale);
  uint32_t r;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(r)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y), "f"(d.x), "f"(d.y));
  return r;
}

// The borders of a tensor's runs: with i = 1, 3, 5, 7 and a scale whose mantissa is
// m = 8..15, powers of two times m i g.  Entry 4 (m - 8) + i / 2 tells of one
// whether 16-bit values (kBits fraction bits) can be within 2^-18 of it, their
// mantissa, and the factor that moves them to their side of it; a value on the
// border goes to the even code, below the borders with i = 1 and 5 and above those
// with 3 and 7.  Values with a border's mantissa that are no border's are codes
// themselves, or beyond the largest, and can be moved as well.
struct Borders {
  float shift[8];      // of m: what all values of a run are moved by
  uint32_t on;         // a bit per m: quotients have to be rounded correctly
  uint32_t single;     // a bit per entry: the values near it are moved by themselves
  uint32_t mantissa[32];
  float move[32];
};
constexpr uint32_t kFraction = 0x7fffffu;

// Powers of two make no difference to any of it: g is taken into [1, 2), where the
// products stay finite.  (A subnormal g has other mantissas, but with one every value is
// compared with the borders itself, as its s g is below 1e-35.)
template <int kBits>
__device__ __forceinline__ void find_borders(Borders* b, float tensor_scale, int lane) {
  const float g = __uint_as_float((__float_as_uint(tensor_scale) & kFraction) | 0x3f800000u);
  constexpr uint32_t kRest = (1u << (23 - kBits)) - 1u, kNear = 64u, kAll = 0xffffffffu;
  const int mi = (8 + lane / 4) * (2 * (lane & 3) + 1);
  const uint32_t t = __float_as_uint(static_cast<float>(mi) * g) + kNear;
  const bool near = (t & kRest) <= 2u * kNear;
  const double value = __uint_as_float(t & ~kRest);
  const double border = static_cast<double>(mi) * static_cast<double>(g);
  const uint32_t above = __ballot_sync(kAll, near && value > border);
  const uint32_t below = __ballot_sync(kAll, near && value < border);
  const uint32_t equal = __ballot_sync(kAll, near && value == border);
  const bool up = value > border || (value == border && (lane & 1));
  b->mantissa[lane] = t & kFraction & ~kRest;
  b->move[lane] = up ? 1.f + 0x1p-19f : 1.f - 0x1p-19f;
  const uint32_t m4 = 15u << (lane / 4 * 4);   // the entries of this lane's m
  const bool one_side = !(equal & m4) && !((above & m4) && (below & m4));
  const bool exact = (equal & m4) && !((above | below) & m4);
  if ((lane & 3) == 0)
    b->shift[lane / 4] = !one_side ? 1.f : (above & m4) ? 1.f + 0x1p-19f : (below & m4) ? 1.f - 0x1p-19f : 1.f;
  const uint32_t single = __ballot_sync(kAll, near && !one_side && !exact);
  const uint32_t on = __ballot_sync(kAll, lane < 8 && (equal >> (4 * (lane & 7)) & 15u) &&
                                              !((above | below) >> (4 * (lane & 7)) & 15u));
  if (lane == 0) {
    b->single = single;
    b->on = on;
  }
}

// Moves the values of f that are near the entries `left` of mantissa index m.
__device__ __forceinline__ void leave_borders(float (&f)[16], uint32_t m, uint32_t left, const Borders* b) {
  for (; left; left &= left - 1u) {
    const uint32_t k = 4u * m + __ffs(left) - 1u;
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

// 16 values of an mxfp4 run whose largest magnitude has the bits m: codes in q0,
// q1; returns the scale's code.
__device__ __forceinline__ uint32_t quantize_mx(const float (&f)[16], uint32_t m, uint32_t& q0, uint32_t& q1) {
  if (m >= 0x7f800000u) {
    q0 = q1 = 0u;
    return 0xffu;
  }
  const int e = max(static_cast<int>(m >> 23) - 129, -127);
  const float inv = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
  q0 = pack_e2m1x8(f, inv);
  q1 = pack_e2m1x8(f + 8, inv);
  return static_cast<uint32_t>(e + 127);
}

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

// One run of 16 values at x whose largest magnitude has the bits m: codes in q0,
// q1; returns the scale's code.
template <typename X>
__device__ __forceinline__ uint32_t quantize_nv(float (&f)[16], uint32_t m, const X* x, const TensorScale& ts,
                                                const Borders* borders, uint32_t& q0, uint32_t& q1) {
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
  float inv = __fdividef(1.f, d);   // within 2^-22
  unsigned long long differ = 0ull;   // values to be looked at, four bits each
  if constexpr (sizeof(X) == 2) {
    const uint32_t mi = (rounded >> 20) & 7u;
    if ((borders->on >> mi) & 1u) {
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float q = f[j] * inv;
        // not what saturates (it may be infinite); a zero keeps its sign
        f[j] = fabsf(q) < 8.f ? copysignf(fmaf(fmaf(-q, d, f[j]), inv, q), q) : q;
      }
      inv = 1.f;
    } else {
      inv *= borders->shift[mi];
      const uint32_t single = (borders->single >> (4u * mi)) & 15u;
      if (single) leave_borders(f, mi, single, borders);
    }
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

}  // namespace moe
