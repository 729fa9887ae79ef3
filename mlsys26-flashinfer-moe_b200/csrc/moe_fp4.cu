// Microscaled 4-bit floating point: quantisation to e2m1 codes with a scale per
// run of columns, and back.
//
//   mxfp4: runs of 32, e8m0 scale s = 2^(floor(log2(amax)) - 2) (at least 2^-127)
//   nvfp4: runs of 16, e4m3 scale s = rne(amax / (6 g)), at most 448 and, unless
//          amax is 0, at least 2^-9; g: one fp32 scale of the whole tensor
//   code = e2m1_rne(x / (s g)), saturating at 6;   value = code * s * g
//
// The scales go to the layout that the tensor core's scale copy reads: blocks of
// 128 rows x 4 scales, in which row r of the block and scale b are byte
// (r % 32) * 16 + (r / 32) * 4 + b; the threads of one block's four scales
// gather them with shuffles and store one word.  Rows and columns that fill up
// the last blocks have scale 0.  Bound by memory: 2.56 bytes an element.
#include "moe_fp4.cuh"

namespace moe {

constexpr int kQuantThreads = 128;
// Resident blocks an SM, which are the whole grid: a block's setup (divisions, the
// borders) then counts little, and a thread's next 64 bytes are on their way while it
// works on some.  nvfp4 bf16 at 8192 x 7168, where bytes alone take 23 us: 26.4 us; seven
// blocks an SM spill registers (33), without the loads ahead 39, mxfp4 24.
constexpr int quant_blocks_per_sm(bool nv) { return nv ? 6 : 8; }
// The way back (23 us of bytes): 25.6 us to bf16 with 12 blocks, 28.5 with 8, 29 with 16.
constexpr int kDequantBlocksPerSm = 12;

// A thread takes 64 bytes of input: 32 columns of a 16-bit type, 16 of fp32.
template <typename X, bool kNv>
__global__ void __launch_bounds__(kQuantThreads, quant_blocks_per_sm(kNv)) moe_fp4_quantize_kernel(Fp4QuantParams p) {
  // A product of linear_fp4 that follows sets itself up meanwhile; the one for few tokens
  // also loads its first weights.
  griddep_launch_dependents();
  constexpr int kCols = 64 / static_cast<int>(sizeof(X)), kRun = kNv ? 16 : 32, kParts = kCols / 16;
  constexpr int kThreadsPerWord = 4 * kRun / kCols;   // threads whose scales share a word
  const int lane = threadIdx.x & 31;
  const uint32_t units = p.chunks * kThreadsPerWord;   // per padded row
  const TensorScale ts(p.global_scale);
  __shared__ Borders borders;
  if constexpr (kNv && sizeof(X) == 2) {
    if (threadIdx.x < 32) find_borders<std::is_same<X, __half>::value ? 10 : 7>(&borders, ts.g, lane);
    __syncthreads();
  }
  // row and column step by the grid's size without divisions
  const uint32_t start = blockIdx.x * blockDim.x + threadIdx.x;
  const uint32_t R = static_cast<uint32_t>(p.R), R128 = (R + 127u) / 128u * 128u;
  uint32_t r = start / units, u = start % units;
  auto inside = [&] { return r < R && kCols * u < static_cast<uint32_t>(p.K); };
  auto advance = [&] {
    r += p.r_step;
    u += p.u_step;
    if (u >= units) {
      u -= units;
      ++r;
    }
  };
  auto input = [&](uint32_t row, uint32_t part) { return static_cast<const X*>(p.x) + row * p.ld + kCols * part; };
  Raw16<X> next[kParts];
  auto load = [&] {
    const X* const x = input(r, u);
#pragma unroll
    for (int h = 0; h < kParts; ++h) next[h].load(x + 16 * h);
  };
  bool live_next = inside();
  if (live_next) load();
  while (r < R128) {   // the same for a whole warp: 128 units are a multiple of 32
    const uint32_t row = r, part = u;
    const bool live = live_next;
    Raw16<X> raw[kParts];
#pragma unroll
    for (int h = 0; h < kParts; ++h) raw[h] = next[h];
    advance();
    live_next = inside();
    if (live_next) load();
    uint32_t code = 0u;   // of the thread's scales
    uint32_t q[2 * kParts];
    if constexpr (kNv) {
      if (live) {
#pragma unroll
        for (int h = 0; h < kParts; ++h) {
          float f[16];
          raw[h].get(f);
          code |= quantize_nv<X>(f, raw[h].amax_bits(), input(row, part) + 16 * h, ts, &borders, q[2 * h], q[2 * h + 1]) << (8 * h);
        }
      }
    } else {
      float f[kParts][16];
      uint32_t m = 0u;
      if (live) {
#pragma unroll
        for (int h = 0; h < kParts; ++h) {
          raw[h].get(f[h]);
          m = max(m, raw[h].amax_bits());
        }
      }
      if constexpr (kCols < kRun) m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
      if (live) {
#pragma unroll
        for (int h = 0; h < kParts; ++h) code = quantize_mx(f[h], m, q[2 * h], q[2 * h + 1]);
      }
    }
    if (live) {
      uint8_t* const c = p.codes + static_cast<int64_t>(row) * (p.K / 2) + kCols / 2 * part;
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
      const uint32_t block = row / 128 * p.chunks + part / kThreadsPerWord;
      *reinterpret_cast<uint32_t*>(p.scales + static_cast<int64_t>(block) * 512 + (row % 32) * 16 +
                                   row % 128 / 32 * 4) = word;
    }
  }
}

// 32 bytes; in one store if they are aligned to their size (`wide`), which writes whole
// sectors of L2 (8192 x 7168 to fp32: 48 us, 74 in halves).
__device__ __forceinline__ void store32(void* p, const uint32_t (&w)[8], bool wide) {
  if (wide) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]),
                 "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
  } else {
    static_cast<uint4*>(p)[0] = make_uint4(w[0], w[1], w[2], w[3]);
    static_cast<uint4*>(p)[1] = make_uint4(w[4], w[5], w[6], w[7]);
  }
}
__device__ __forceinline__ uint32_t pack2(float2 v, __nv_bfloat16) {
  const __nv_bfloat162 b = __floats2bfloat162_rn(v.x, v.y);
  return *reinterpret_cast<const uint32_t*>(&b);
}
__device__ __forceinline__ uint32_t pack2(float2 v, __half) {
  const __half2 b = __floats2half2_rn(v.x, v.y);
  return *reinterpret_cast<const uint32_t*>(&b);
}

// Eight e2m1 codes as pairs of halves.
__device__ __forceinline__ void unpack_e2m1x8(uint32_t q, __half2 (&h)[4]) {
  uint32_t w[4];
  asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
      : "r"(q));
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = *reinterpret_cast<const __half2*>(&w[i]);
}

// code * s is exact (2 and 4 significant bits; with an e4m3 scale, 2^-10 to 2688,
// also in halves); the tensor scale and the output type each round once.  A thread
// takes 16 columns, its next ones on their way.
template <typename O, bool kNv>
__global__ void __launch_bounds__(kQuantThreads, kDequantBlocksPerSm) moe_fp4_dequantize_kernel(Fp4QuantParams p) {
  const uint32_t units = p.K / 16, R = static_cast<uint32_t>(p.R);
  const float g = kNv && p.global_scale ? __ldg(p.global_scale) : 1.f;
  const bool wide = (reinterpret_cast<uintptr_t>(p.out) & 31u) == 0;
  // row and column step by the grid's size without divisions
  const uint32_t start = blockIdx.x * blockDim.x + threadIdx.x;
  uint32_t r = start / units, u = start % units;
  uint2 q_next;
  uint32_t s_next;
  auto load = [&] {
    const uint32_t b = kNv ? u : u / 2;
    q_next = __ldcs(reinterpret_cast<const uint2*>(p.codes + r * p.ld + 8 * u));
    s_next = p.scales[static_cast<int64_t>(r / 128 * p.chunks + b / 4) * 512 + (r % 32) * 16 + r % 128 / 32 * 4 + b % 4];
  };
  if (r < R) load();
  while (r < R) {
    const uint2 q = q_next;
    const uint32_t sc = s_next;
    O* const o = static_cast<O*>(p.out) + static_cast<int64_t>(r) * p.K + 16 * u;
    r += p.r_step;
    u += p.u_step;
    if (u >= units) {
      u -= units;
      ++r;
    }
    if (r < R) load();
    __half2 h[8];
    unpack_e2m1x8(q.x, reinterpret_cast<__half2(&)[4]>(h[0]));
    unpack_e2m1x8(q.y, reinterpret_cast<__half2(&)[4]>(h[4]));
    float2 f[8];
    if constexpr (kNv) {
      const __half2 s = __half2half2(__half(__nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(sc), __NV_E4M3)));
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float2 v = __half22float2(__hmul2(h[j], s));
        f[j] = mul2(v.x, v.y, g);
      }
    } else {
      const float s = e8m0_value(sc);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float2 v = __half22float2(h[j]);
        f[j] = mul2(v.x, v.y, s);
      }
    }
    uint32_t w[8];
    if constexpr (sizeof(O) == 2) {
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = pack2(f[j], O{});
      store32(o, w, wide);
    } else {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          w[2 * j] = __float_as_uint(f[4 * half + j].x);
          w[2 * j + 1] = __float_as_uint(f[4 * half + j].y);
        }
        store32(o + 8 * half, w, wide);
      }
    }
  }
}

namespace {

int blocks_for(int64_t threads, int block, int most) {
  int64_t b = (threads + block - 1) / block;
  if (b > most) b = most;
  return static_cast<int>(b < 1 ? 1 : b);
}

template <bool kNv>
int quantize_dtype(const Fp4QuantParams& p, int dtype, int blocks, cudaStream_t s) {
  if (dtype == MOE_BF16)
    moe_fp4_quantize_kernel<__nv_bfloat16, kNv><<<blocks, kQuantThreads, 0, s>>>(p);
  else if (dtype == MOE_F16)
    moe_fp4_quantize_kernel<__half, kNv><<<blocks, kQuantThreads, 0, s>>>(p);
  else
    moe_fp4_quantize_kernel<float, kNv><<<blocks, kQuantThreads, 0, s>>>(p);
  return cudaGetLastError() == cudaSuccess ? MOE_OK : MOE_ERR_CUDA;
}

template <bool kNv>
int dequantize_dtype(const Fp4QuantParams& p, int dtype, int blocks, cudaStream_t s) {
  if (dtype == MOE_BF16)
    moe_fp4_dequantize_kernel<__nv_bfloat16, kNv><<<blocks, kQuantThreads, 0, s>>>(p);
  else if (dtype == MOE_F16)
    moe_fp4_dequantize_kernel<__half, kNv><<<blocks, kQuantThreads, 0, s>>>(p);
  else
    moe_fp4_dequantize_kernel<float, kNv><<<blocks, kQuantThreads, 0, s>>>(p);
  return cudaGetLastError() == cudaSuccess ? MOE_OK : MOE_ERR_CUDA;
}

}  // namespace

int launch_fp4_quantize(Fp4QuantParams p, int dtype, int format, int sms, cudaStream_t s) {
  const bool nv = format == MOE_NVFP4;
  const int units = p.chunks * (nv ? 2 : 4) * (dtype == MOE_F32 ? 2 : 1);   // threads' shares of a row
  const int blocks =
      blocks_for((p.R + 127) / 128 * 128 * units, kQuantThreads, sms * quant_blocks_per_sm(nv));
  p.r_step = blocks * kQuantThreads / units;
  p.u_step = blocks * kQuantThreads % units;
  return nv ? quantize_dtype<true>(p, dtype, blocks, s) : quantize_dtype<false>(p, dtype, blocks, s);
}

int fp4_check(int32_t format, int64_t R, int64_t K) {
  if (format != MOE_MXFP4 && format != MOE_NVFP4) return MOE_ERR_INVALID_ARG;
  // K a multiple of 32: 16-byte rows of codes for the TMA, whole runs of both formats
  if (R < 0 || R > (int64_t(1) << 24) || K < 32 || K % 32 != 0 || K > 65536) return MOE_ERR_SHAPE;
  return MOE_OK;
}

int fp4_check_input(const void* x, int32_t x_dtype, int64_t ld, int64_t R, int64_t K, int32_t format,
                    const float* global_scale) {
  if (x_dtype != MOE_BF16 && x_dtype != MOE_F16 && x_dtype != MOE_F32) return MOE_ERR_INVALID_ARG;
  if (format == MOE_MXFP4 && global_scale) return MOE_ERR_INVALID_ARG;
  if (ld < K || ld % (x_dtype == MOE_F32 ? 4 : 8) != 0) return MOE_ERR_SHAPE;
  if (R == 0) return MOE_OK;
  if (!x) return MOE_ERR_INVALID_ARG;
  if ((reinterpret_cast<uintptr_t>(x) & 15u) || (reinterpret_cast<uintptr_t>(global_scale) & 3u))
    return MOE_ERR_ALIGNMENT;
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
  if (!st) st = fp4_check_input(x, x_dtype, ld, R, K, format, global_scale);
  if (st) return st;
  if (R == 0) return MOE_OK;
  if (!codes || !scales) return MOE_ERR_INVALID_ARG;
  if (off(codes, 16) || off(scales, 16)) return MOE_ERR_ALIGNMENT;
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
  const int units = p.K / 16, blocks = blocks_for(R * units, kQuantThreads, sms * kDequantBlocksPerSm);
  p.r_step = blocks * kQuantThreads / units;
  p.u_step = blocks * kQuantThreads % units;
  return format == MOE_NVFP4 ? dequantize_dtype<true>(p, out_dtype, blocks, s)
                             : dequantize_dtype<false>(p, out_dtype, blocks, s);
}

}  // extern "C"
