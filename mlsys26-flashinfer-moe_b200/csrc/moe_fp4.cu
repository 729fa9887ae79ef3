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

// A thread takes 64 bytes of input: 32 columns of a 16-bit type, 16 of fp32.
template <typename X, bool kNv>
__global__ void __launch_bounds__(kQuantThreads, quant_blocks_per_sm(kNv)) moe_fp4_quantize_kernel(Fp4QuantParams p) {
  griddep_launch_dependents();   // a product that follows streams its weights meanwhile
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
    moe_fp4_dequantize_kernel<__nv_bfloat16, kNv><<<blocks, 256, 0, s>>>(p);
  else if (dtype == MOE_F16)
    moe_fp4_dequantize_kernel<__half, kNv><<<blocks, 256, 0, s>>>(p);
  else
    moe_fp4_dequantize_kernel<float, kNv><<<blocks, 256, 0, s>>>(p);
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
  const int blocks = blocks_for(R * (K / 16), 256, sms * 32);
  return format == MOE_NVFP4 ? dequantize_dtype<true>(p, out_dtype, blocks, s)
                             : dequantize_dtype<false>(p, out_dtype, blocks, s);
}

}  // extern "C"
