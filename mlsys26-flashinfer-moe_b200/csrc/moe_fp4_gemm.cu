// Product of two microscaled 4-bit matrices on the tensor core:
//   out[t, n] = ga * gb * sum_k a[t, k] sa[t, k/run] * w[n, k] sw[n, k/run]
// with tcgen05.mma's block-scaled kinds (kind::mxf4 with e8m0 scales for runs of
// 32, kind::mxf4nvf4 with e4m3 scales for runs of 16), fp32 accumulators in TMEM.
//
// The weight rows are the M = 128 operand and the tokens the N operand, so few
// tokens waste no tensor-core rows and the weights, most of the traffic, stream
// once.  A K block is 256 columns: 128-byte rows of codes, loaded by TMA with
// the 128-byte swizzle that the K-major descriptors expect, and 512-byte blocks
// of scales (128 rows x 4 scales), which are contiguous in memory and go to
// TMEM with tcgen05.cp (32 lanes x 128 bits, repeated for the four lane
// quarters).  A stage of the shared-memory ring has its own scale columns in
// TMEM, so a copy never overwrites scales that an MMA may still read.
//
// A tile's K blocks are cut among the CTAs of a cluster when there are fewer
// tiles than SMs; the partial sums meet through distributed shared memory and
// are added in rank order, so the result does not depend on timing.
//
// A few tokens (kFp4FusedTokens) are quantised by the product's own CTAs straight
// into the ring, each the columns of its K blocks, instead of by a kernel before.
#include <cudaTypedefs.h>

#include <mutex>

#include "moe_fp4.cuh"

namespace moe {

namespace {

constexpr int kFp4K = 256;            // columns of a K block: 128 bytes of codes
constexpr int kFp4M = 128;            // weight rows of a tile
constexpr int kFp4Threads = 192;      // warp 0: loads, warp 1: MMA, warps 2-5: accumulator
constexpr int kFp4ScaleChunk = 512;   // 128 rows x 4 scales
constexpr int kFp4ScaleBytes = 4 * kFp4ScaleChunk;   // per K block, at most
constexpr int kFp4TmemCols = 512;
constexpr int kStallLimitUs = 50;     // of a wait under MOE_FP4_TEST_STALL
// Up to this many tokens a product quantises them itself, in one launch instead of
// two and the same time on the GPU (nvfp4, K = 7168, N = 4096: 8.8 us; at 8 tokens
// 10.3, and 8.8 with the kernel before).
constexpr int64_t kFp4FusedTokens = 4;

// Error word of the products of this device: the first device-side wait that
// ran out since it was last read.  The tiles concerned are filled with NaN.
__device__ CtrlBlock g_fp4_ctrl;

template <int NT>
struct Fp4Cfg {
  static constexpr int kABytes = kFp4M * 128;
  static constexpr int kBBytes = NT * 128;
  static constexpr int kStageBytes = kABytes + kBBytes + 2 * kFp4ScaleBytes;
  static constexpr int kStages = NT <= 64 ? 7 : 6;
  static constexpr int kSmem = 1024 + kStages * kStageBytes + 256;
  static constexpr int kScaleCol = 128;   // TMEM: accumulator, then 32 columns a stage
  static_assert(kSmem <= kMaxDynSmemBytes, "ring exceeds shared memory");
  static_assert(kScaleCol + kStages * 32 <= kFp4TmemCols, "scales exceed TMEM");
  static_assert(NT * kFp4M * 4 <= kStages * kStageBytes, "partial sums reuse the ring");
};

// Block-scaled e2m1 x e2m1 -> fp32, both operands K-major.  The scale format
// is 0 for e4m3 and 1 for e8m0; scale ids select the first or second pair of
// bytes of a scale word (runs of 32: two scales per K = 64 step).
__host__ __device__ constexpr uint32_t umma_idesc_fp4(int n, bool e8m0) {
  return (1u << 7) | (1u << 10)                     // A, B = e2m1
         | (static_cast<uint32_t>(n >> 3) << 17)    // N / 8
         | (e8m0 ? 1u << 23 : 0u)                   // scale format
         | (1u << 27);                              // M / 128
}
__device__ __forceinline__ uint32_t umma_scale_ids(uint32_t id) { return (id << 4) | (id << 29); }

// The MMA warp runs its loop with all lanes, so that descriptors and addresses
// stay in uniform registers, and each tcgen05 instruction is issued by the lane
// whose `lead` is set.  (One lane in a divergent branch spent 60 cycles an
// instruction on moving its operands.)
#define MOE_FP4_MMA(name, group, kind, vec)                                                   \
  __device__ __forceinline__ void name(uint32_t lead, uint32_t d, uint64_t a, uint64_t b,     \
                                       uint32_t idesc, uint32_t sa, uint32_t sb,              \
                                       uint32_t accumulate) {                                 \
    asm volatile(                                                                             \
        "{\n\t.reg .pred p, l;\n\t"                                                           \
        "setp.ne.b32 p, %6, 0;\n\t"                                                           \
        "setp.ne.b32 l, %7, 0;\n\t"                                                           \
        "@l tcgen05.mma.cta_group::" group ".kind::" kind ".block_scale.scale_vec::" vec      \
        " [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),                                    \
        "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate), "r"(lead)              \
        : "memory");                                                                          \
  }
MOE_FP4_MMA(umma_nvf4, "1", "mxf4nvf4", "4X")
MOE_FP4_MMA(umma_mxf4, "1", "mxf4", "2X")
MOE_FP4_MMA(umma_nvf4_pair, "2", "mxf4nvf4", "4X")
MOE_FP4_MMA(umma_mxf4_pair, "2", "mxf4", "2X")
#undef MOE_FP4_MMA

__device__ __forceinline__ uint32_t elect_lane() {
  uint32_t lead;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(lead));
  return lead;
}

// 32 lanes x 128 bits from shared memory, repeated for the four lane quarters:
// a 512-byte scale block becomes four TMEM columns (rows r, r+32, r+64, r+96).
__device__ __forceinline__ uint64_t scale_desc(uint32_t smem_addr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((smem_addr >> 4) & 0x3FFFu);
  d |= static_cast<uint64_t>(128u >> 4) << 32;   // 8 rows of 16 bytes
  d |= static_cast<uint64_t>(1u) << 46;          // descriptor version, no swizzle
  return d;
}
// In cta_group::2 each CTA's copy is from its own shared memory to its own TMEM.
template <int kGroup>
__device__ __forceinline__ void tmem_copy_scales(uint32_t lead, uint32_t taddr, uint64_t desc) {
  if constexpr (kGroup == 1)
    asm volatile(
        "{\n\t.reg .pred l;\n\tsetp.ne.b32 l, %2, 0;\n\t"
        "@l tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;\n\t}" ::"r"(taddr),
        "l"(desc), "r"(lead)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred l;\n\tsetp.ne.b32 l, %2, 0;\n\t"
        "@l tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;\n\t}" ::"r"(taddr),
        "l"(desc), "r"(lead)
        : "memory");
}

// Arrives on the barrier once all tcgen05 operations issued so far by the lead lane
// have completed.
__device__ __forceinline__ void umma_commit_lead(uint32_t lead, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred l;\n\tsetp.ne.b32 l, %1, 0;\n\t"
      "@l tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(
          smem_u32(bar)),
      "r"(lead)
      : "memory");
}

// Contiguous bytes (a multiple of 16, both addresses 16-byte aligned) into shared memory.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr, uint32_t rank) {
  float4 v;
  asm volatile(
      "{\n\t.reg .b32 a;\n\t"
      "mapa.shared::cluster.u32 a, %4, %5;\n\t"
      "ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [a];\n\t}"
      : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
      : "r"(addr), "r"(rank)
      : "memory");
  return v;
}

// mbar_wait by a warp whose lanes go on or give up together.  Whether a lane's wait
// ran out depends on when it looked, so without the vote some would meet the others' next
// synchronisation of the warp somewhere else.  The MMA loops have no such
// synchronisation in them and do without it (a vote a K block cost 3 us of 106 at nvfp4
// T = 8192, K = 7168, N = 4096): there the lanes leave one by one.
__device__ __forceinline__ bool mbar_wait_warp(uint64_t* bar, uint32_t parity, volatile int* abort,
                                               CtrlBlock* ctrl, int where) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort, ctrl, where));
}

// Waits for what is in flight, until kWaitLimitNs after `since`.
__device__ __forceinline__ void drain_fp4(uint64_t* bar, uint32_t parity, unsigned long long since) {
  while (!mbar_try_wait(bar, parity)) {
    if (globaltimer() - since > kWaitLimitNs) return;
  }
}

// Four consecutive outputs of one token; `left` of them exist.
__device__ __forceinline__ void store_out4(const Fp4GemmParams& p, int64_t t, int n, const float (&v)[4]) {
  const int64_t at = t * p.ldo + n;
  const bool whole = p.vec_out && n + 4 <= p.N;
  if (p.out_dtype == MOE_F32) {
    float* o = static_cast<float*>(p.out) + at;
    if (whole) {
      *reinterpret_cast<float4*>(o) = make_float4(v[0], v[1], v[2], v[3]);
      return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (n + j < p.N) o[j] = v[j];
  } else {
    uint32_t w[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if (p.out_dtype == MOE_BF16) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
        w[j] = *reinterpret_cast<const uint32_t*>(&b);
      } else {
        const __half2 b = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
        w[j] = *reinterpret_cast<const uint32_t*>(&b);
      }
    }
    uint16_t* o = static_cast<uint16_t*>(p.out) + at;
    if (whole) {
      *reinterpret_cast<uint2*>(o) = make_uint2(w[0], w[1]);
      return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (n + j < p.N) o[j] = static_cast<uint16_t>(w[j / 2] >> (16 * (j & 1)));
  }
}

// What the sums are multiplied with: the product of the tensor scales where that is a
// normal number (or nothing else would help: a 0, a NaN).  Otherwise the scales one after
// the other, `before` first: below fp32's normal numbers the larger one, beyond its end
// the smaller one, so that what lies between is no further out than the output.
struct OutScale {
  float before, scale;   // before: 1 if there is one factor only
  __device__ __forceinline__ explicit OutScale(const Fp4GemmParams& p) {
    const float a = p.ga ? __ldg(p.ga) : 1.f, b = p.gb ? __ldg(p.gb) : 1.f;
    scale = a * b;
    before = 1.f;
    const bool low = fabsf(scale) < 0x1p-126f && a != 0.f && b != 0.f;
    if (low || isinf(scale)) {
      const bool a_before = (fabsf(a) > fabsf(b)) == low;
      before = a_before ? a : b;
      scale = a_before ? b : a;
    }
  }
};

// Adds the cluster's partial sums [nt, 128] in rank order and stores them: token j
// goes to CTA j % kSplit, there to warp j / kSplit % 6, each lane four weight
// rows.  Eight reads of the peers' shared memory are in flight at a time.
template <int kSplit>
__device__ __forceinline__ void add_partials(const Fp4GemmParams& p, const float* part, int rank, int warp,
                                             int lane, int nt, int t0, int n0, OutScale alpha) {
  constexpr int kWarps = kFp4Threads / 32, kTokens = 8 / kSplit;
  for (int j0 = rank + kSplit * warp; j0 < nt; j0 += kTokens * kSplit * kWarps) {
    float4 o[kTokens][kSplit];
#pragma unroll
    for (int i = 0; i < kTokens; ++i) {
      const int j = j0 + i * kSplit * kWarps;
      const float* at = part + j * kFp4M + 4 * lane;
      if (j < nt) {
#pragma unroll
        for (int r = 0; r < kSplit; ++r)
          o[i][r] = kSplit > 1 ? ld_cluster4(smem_u32(at), r) : *reinterpret_cast<const float4*>(at);
      }
    }
#pragma unroll
    for (int i = 0; i < kTokens; ++i) {
      const int j = j0 + i * kSplit * kWarps;
      if (j < nt) {
        float v[4] = {o[i][0].x, o[i][0].y, o[i][0].z, o[i][0].w};
#pragma unroll
        for (int r = 1; r < kSplit; ++r) {
          v[0] += o[i][r].x;
          v[1] += o[i][r].y;
          v[2] += o[i][r].z;
          v[3] += o[i][r].w;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = v[k] * alpha.before * alpha.scale;
        store_out4(p, t0 + j, n0 + 4 * lane, v);
      }
    }
  }
}

}  // namespace

// One tile of 128 weight rows x NT tokens per cluster (blockIdx.x / cluster,
// blockIdx.y), its K blocks cut evenly among the cluster's CTAs.  X: void, or the
// type of tokens that are quantised here.
template <int NT, bool kNv, typename X = void>
__global__ void __launch_bounds__(kFp4Threads, 1)
    moe_fp4_gemm_kernel(const __grid_constant__ CUtensorMap tm_w,
                        const __grid_constant__ CUtensorMap tm_t, Fp4GemmParams p) {
  using Cfg = Fp4Cfg<NT>;
  constexpr int S = Cfg::kStages;
  constexpr bool kQuantize = !std::is_same<X, void>::value;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* sA = smem;                               // S x 16 KB
  uint8_t* sB = sA + S * Cfg::kABytes;              // S x NT * 128
  uint8_t* sSA = sB + S * Cfg::kBBytes;             // S x 2 KB scales of the weights
  uint8_t* sSB = sSA + S * kFp4ScaleBytes;          // S x 2 KB scales of the tokens
  uint64_t* full = reinterpret_cast<uint64_t*>(sSB + S * kFp4ScaleBytes);
  uint64_t* empty = full + S;
  uint64_t* done = empty + S;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);   // [1]: wait limit

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = p.split;
  const int rank = split > 1 ? static_cast<int>(blockIdx.x) % split : 0;
  const int n0 = static_cast<int>(blockIdx.x) / split * kFp4M;
  const int t0 = static_cast<int>(blockIdx.y) * NT;
  const int KB = (p.K + kFp4K - 1) / kFp4K;
  const int kb0 = static_cast<int>(static_cast<int64_t>(KB) * rank / split);
  const int kb1 = static_cast<int>(static_cast<int64_t>(KB) * (rank + 1) / split);
  CtrlBlock* ctrl = &g_fp4_ctrl;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], kQuantize ? 1 + 4 : 1);   // the quantising warps
      mbar_init(&empty[s], 1);
    }
    mbar_init(done, 1);
    abort_flag[0] = 0;
    abort_flag[1] = p.stall ? kStallLimitUs : static_cast<int>(kWaitLimitNs / 1000);
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, kFp4TmemCols);
    tmem_relinquish();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tm_w);
    if constexpr (!kQuantize) tma_prefetch_desc(&tm_t);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    // ------------------------------------------------------------ loads
    if (lane == 0) {
      const uint8_t* sw = p.w_scales + static_cast<int64_t>(n0 / 128) * p.chunks * kFp4ScaleChunk;
      const uint8_t* st = p.t_scales + static_cast<int64_t>(t0 / 128) * p.chunks * kFp4ScaleChunk;
      auto scale_bytes = [&](int kb) {
        return static_cast<uint32_t>(min(p.chunks_per_block, p.chunks - kb * p.chunks_per_block)) *
               kFp4ScaleChunk;
      };
      auto load_weights = [&](int kb, int s) {
        const uint32_t sb = scale_bytes(kb);
        mbar_arrive_expect_tx(&full[s], Cfg::kABytes + sb + (kQuantize ? 0 : Cfg::kBBytes + sb));
        tma_load_2d(sA + s * Cfg::kABytes, &tm_w, &full[s], kb * 128, n0);
        bulk_load(sSA + s * kFp4ScaleBytes,
                  sw + static_cast<int64_t>(kb) * p.chunks_per_block * kFp4ScaleChunk, sb, &full[s]);
      };
      // The weights of the first ring pass go out before the wait for the
      // kernel that writes the tokens' codes (programmatic dependent launch).
      const int early = min(S, kb1 - kb0);
      for (int i = 0; i < early; ++i) load_weights(kb0 + i, i);
      griddep_wait();
      int stage = 0, issued = early;
      uint32_t phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (kb - kb0 >= early) {
          if (!mbar_wait(&empty[stage], phase ^ 1u, abort_flag, ctrl, 40)) break;
          load_weights(kb, stage);
          ++issued;
        }
        if constexpr (!kQuantize) {
          tma_load_2d(sB + stage * Cfg::kBBytes, &tm_t, &full[stage], kb * 128, t0);
          bulk_load(sSB + stage * kFp4ScaleBytes,
                    st + static_cast<int64_t>(kb) * p.chunks_per_block * kFp4ScaleChunk, scale_bytes(kb),
                    &full[stage]);
        }
        if (++stage == S) {
          stage = 0;
          phase ^= 1u;
        }
      }
      // Every load lands before the CTA can exit, also after an abort.
      const unsigned long long since = globaltimer();
      for (int i = max(0, issued - S); i < issued; ++i) drain_fp4(&full[i % S], (i / S) & 1u, since);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA
    const uint32_t lead = elect_lane();
    const uint32_t idesc = umma_idesc_fp4(NT, !kNv);
    const uint64_t da0 = umma_desc_sw128(smem_u32(sA)), db0 = umma_desc_sw128(smem_u32(sB));
    const uint64_t dsa0 = scale_desc(smem_u32(sSA)), dsb0 = scale_desc(smem_u32(sSB));
    int stage = 0;
    uint32_t phase = 0;
    uint32_t acc = 0;
    const bool go = !p.stall || mbar_wait(done, 0, abort_flag, ctrl, 43);
    for (int kb = kb0; go && kb < kb1; ++kb) {
      if (!mbar_wait(&full[stage], phase, abort_flag, ctrl, 41)) break;
      const int steps = min(4, (p.K - kb * kFp4K + 63) / 64);
      const uint32_t sa = tmem + Cfg::kScaleCol + stage * 32, sb = sa + 16;
      const uint64_t dsa = dsa0 + stage * (kFp4ScaleBytes / 16);
      const uint64_t dsb = dsb0 + stage * (kFp4ScaleBytes / 16);
#pragma unroll
      for (int c = 0; c < (kNv ? 4 : 2); ++c) {
        if (c * (kNv ? 1 : 2) < steps) {
          tmem_copy_scales<1>(lead, sa + 4 * c, dsa + c * (kFp4ScaleChunk / 16));
          tmem_copy_scales<1>(lead, sb + 4 * c, dsb + c * (kFp4ScaleChunk / 16));
        }
      }
      const uint64_t da = da0 + stage * (Cfg::kABytes / 16), db = db0 + stage * (Cfg::kBBytes / 16);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (j < steps) {
          if constexpr (kNv)
            umma_nvf4(lead, tmem, da + 2 * j, db + 2 * j, idesc, sa + 4 * j, sb + 4 * j, acc);
          else
            umma_mxf4(lead, tmem, da + 2 * j, db + 2 * j, idesc | umma_scale_ids(2 * (j & 1)),
                      sa + 4 * (j / 2), sb + 4 * (j / 2), acc);
          acc = 1;
        }
      }
      umma_commit_lead(lead, &empty[stage]);
      if (++stage == S) {
        stage = 0;
        phase ^= 1u;
      }
    }
    // Everything issued has completed, also after an abort.
    __syncwarp();
    umma_commit_lead(lead, done);
    drain_fp4(done, 0, globaltimer());
  } else if constexpr (kQuantize) {
    // ------------------------------------------------------------ tokens
    const int tid = static_cast<int>(threadIdx.x) - 64;
    __shared__ Borders borders;
    const TensorScale ts(p.ga);
    // rows of the tile past the last token
    for (int i = tid; i < S * Cfg::kBBytes / 16; i += 128)
      reinterpret_cast<uint4*>(sB)[i] = make_uint4(0u, 0u, 0u, 0u);
    for (int i = tid; i < S * kFp4ScaleBytes / 16; i += 128)
      reinterpret_cast<uint4*>(sSB)[i] = make_uint4(0u, 0u, 0u, 0u);
    if constexpr (kNv && sizeof(typename std::conditional<kQuantize, X, int>::type) == 2) {
      if (warp == 2) find_borders<std::is_same<X, __half>::value ? 10 : 7>(&borders, ts.g, lane);
    }
    asm volatile("bar.sync 1, 128;" ::: "memory");
    // A thread takes 16 columns of one token and K block; as many blocks at a time
    // as give every thread at most one, the next ones' values on their way.
    const int units = p.T * 16, blocks = min(S, 128 / units);
    const int mine = tid / units, t = tid % units / 16, u = tid % 16;   // block of the group, token, run
    const X* const row = static_cast<const X*>(p.x) + static_cast<int64_t>(t) * p.ld_x + 16 * u;
    Raw16<X> next;
    auto load = [&](int kb) {   // whether there is something to load
      const bool there = mine < blocks && kb < kb1 && kb * kFp4K + 16 * u < p.K;
      if (there) next.load(row + kb * kFp4K);
      return there;
    };
    bool live = load(kb0 + mine);
    int stage = 0;
    uint32_t phase = 0;
    for (int first = kb0; first < kb1; first += blocks) {
      const int n = min(blocks, kb1 - first), kb = first + mine;
      float f[16];
      uint32_t m = 0u;
      if (live) {
        next.get(f);
        m = next.amax_bits();
      }
      const bool here = live;
      live = load(kb + blocks);
      bool ok = true;
      int last = stage;
      uint32_t last_phase = phase, my_stage = 0;
      for (int i = 0; i < n; ++i) {
        ok = ok && mbar_wait(&empty[last], last_phase ^ 1u, abort_flag, ctrl, 42);
        if (i == mine) my_stage = last;
        if (++last == S) {
          last = 0;
          last_phase ^= 1u;
        }
      }
      if (!__all_sync(0xffffffffu, ok)) break;   // as mbar_wait_warp
      // columns past K are zeros (a stage holds an earlier block's)
      uint32_t q0 = 0u, q1 = 0u, code = 0u;
      if constexpr (kNv) {
        if (here) code = quantize_nv<X>(f, m, row + kb * kFp4K, ts, &borders, q0, q1);
      } else {
        m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
        if (here) code = quantize_mx(f, m, q0, q1);
      }
      if (mine < n) {
        // row t of the 128-byte swizzled tile: 16-byte chunk c lies at c ^ (t % 8)
        *reinterpret_cast<uint2*>(sB + my_stage * Cfg::kBBytes + t * 128 + (((u / 2) ^ (t & 7)) << 4) +
                                  (u & 1) * 8) = make_uint2(q0, q1);
        const int run = kNv ? u : u / 2;
        if (kNv || (u & 1) == 0)
          sSB[my_stage * kFp4ScaleBytes + run / 4 * kFp4ScaleChunk + t * 16 + run % 4] =
              static_cast<uint8_t>(code);
      }
      fence_proxy_async_smem();
      __syncwarp();
      for (int i = 0; i < n; ++i) {
        if (lane == 0) mbar_arrive(&full[stage]);
        if (++stage == S) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  float* part = reinterpret_cast<float*>(smem);   // [NT][128]
  if (warp >= 2) {
    const int q = warp & 3;   // the TMEM lanes this warp may read
    const bool failed = abort_flag[0] != 0;
    constexpr int kStep = NT < 32 ? 16 : 32;   // columns in registers at a time: twice that
    const uint32_t lanes = tmem + (static_cast<uint32_t>(q * 32) << 16);
#pragma unroll
    for (int c0 = 0; c0 < NT; c0 += 2 * kStep) {
      float v[2][kStep];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (c0 + h * kStep < NT) {
          if constexpr (kStep == 16)
            tmem_ld16(lanes + c0 + h * kStep, v[h]);
          else
            tmem_ld32(lanes + c0 + h * kStep, v[h]);
        }
      }
      tmem_ld_wait();
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (c0 + h * kStep < NT) {
#pragma unroll
          for (int j = 0; j < kStep; ++j)
            part[(c0 + h * kStep + j) * kFp4M + q * 32 + lane] = failed ? NAN : v[h][j];
        }
    }
  }
  tc_fence_before();
  if (split > 1)
    cluster_sync_all();
  else
    __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, kFp4TmemCols);
  griddep_wait();   // the output's memory may be the previous kernel's
  const OutScale alpha(p);
  const int nt = min(NT, p.T - t0);
  switch (split) {
    case 1: add_partials<1>(p, part, 0, warp, lane, nt, t0, n0, alpha); break;
    case 2: add_partials<2>(p, part, rank, warp, lane, nt, t0, n0, alpha); break;
    case 4: add_partials<4>(p, part, rank, warp, lane, nt, t0, n0, alpha); break;
    default: add_partials<8>(p, part, rank, warp, lane, nt, t0, n0, alpha); break;
  }
  if (split > 1) cluster_sync_all();   // peers may still read this CTA's sums
}

// ---------------------------------------------------------------------------
// Many tokens: a pair of CTAs (tcgen05 cta_group::2) per tile of 256 weight rows
// x 256 tokens, persistent.  Each CTA of the pair holds 128 of the weight rows
// and 128 of the tokens in its shared memory and the accumulators of its weight
// rows in its TMEM; the even CTA issues the MMAs for both.  A tile needs 38 KB
// from L2 per CTA and K block for 33.6 MFLOP, against 36 KB for 8.4 MFLOP of the
// kernel above, which L2 bounds.  Times of products of 4 to 13 tiles a pair and 4 to 28
// K blocks fit 7 us + 0.44 us a K block + 1.7 us a tile (mxfp4: 6, 0.35, 2.1).
//
// TMEM: two accumulators of 256 columns would leave no room for scales, so they
// overlap: the epilogue drains the columns that both have first and then lets the
// next tile's MMAs start.  Every stage has its scale columns: with fewer, a slot
// can only be refilled after the commit of the MMAs that read it, and waiting for
// that cost 10% (nvfp4 at T = 8192, K = 7168, N = 4096: 114 us with three slots
// and five stages).
// ---------------------------------------------------------------------------

namespace {

constexpr int kPairThreads = 384;     // warp 0: loads, warp 1: MMA, warps 4-11: epilogue
constexpr int kPairTile = 256;        // weight rows and tokens of a tile
constexpr int kPairOpBytes = 128 * 128;
template <bool kNv>
struct PairCfg {
  static constexpr int kStages = kNv ? 4 : 5;
  static constexpr int kChunks = kNv ? 4 : 2;         // 128 x 4 scale blocks of a K block
  static constexpr int kScaleRow = kChunks * kFp4ScaleChunk;
  static constexpr int kStageBytes = 2 * kPairOpBytes + 3 * kScaleRow;
  static constexpr int kSmem = 1024 + kStages * kStageBytes + 256;
  static constexpr int kSlotCols = 12 * kChunks;      // weight rows 4, tokens 8 a scale block
  static constexpr int kAcc1 = kNv ? 64 : 128;        // column of the second accumulator
  static constexpr int kScaleCol0 = kAcc1 + kPairTile;
  // columns both accumulators have: a half of the tokens and this many groups of 32
  static constexpr int kMoreGroups = (kPairTile / 2 - kAcc1) / 32;
  static_assert(kSmem <= kMaxDynSmemBytes, "ring exceeds shared memory");
  static_assert(kScaleCol0 + kStages * kSlotCols <= kFp4TmemCols, "scales exceed TMEM");
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void arrive_cluster(uint32_t addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
// Box into this CTA's shared memory, completion on a barrier of the pair.
__device__ __forceinline__ void tma_load_pair(void* dst, const CUtensorMap* map, uint32_t bar, int32_t x,
                                              int32_t y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y)
      : "memory");
}
// Arrives on the barrier at this offset in both CTAs once all tcgen05
// operations issued so far by this thread have completed.
__device__ __forceinline__ void umma_commit_pair(uint32_t lead, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred l;\n\tsetp.ne.b32 l, %2, 0;\n\t"
      "@l tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
      " [%0], %1;\n\t}" ::"r"(smem_u32(bar)),
      "h"(static_cast<uint16_t>(3)), "r"(lead)
      : "memory");
}

__device__ __forceinline__ void store_out1(__nv_bfloat16* o, float v) { *o = __float2bfloat16_rn(v); }
__device__ __forceinline__ void store_out1(__half* o, float v) { *o = __float2half_rn(v); }
__device__ __forceinline__ void store_out1(float* o, float v) { *o = v; }

}  // namespace

template <typename O, bool kNv>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
    moe_fp4_gemm_pair_kernel(const __grid_constant__ CUtensorMap tm_w,
                             const __grid_constant__ CUtensorMap tm_t,
                             const __grid_constant__ CUtensorMap tm_sw,
                             const __grid_constant__ CUtensorMap tm_st, Fp4GemmParams p) {
  using Cfg = PairCfg<kNv>;
  constexpr int S = Cfg::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* sA = smem;
  uint8_t* sB = sA + S * kPairOpBytes;
  uint8_t* sSA = sB + S * kPairOpBytes;
  uint8_t* sSB = sSA + S * Cfg::kScaleRow;
  uint64_t* full = reinterpret_cast<uint64_t*>(sSB + S * 2 * Cfg::kScaleRow);   // the even CTA's
  uint64_t* empty = full + S;
  uint64_t* tfull = empty + S;     // a tile's sums are complete
  uint64_t* tfree = tfull + 1;     // the even CTA's: the overlapping columns are drained
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tfree + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int pairs = static_cast<int>(gridDim.x) / 2, pair = static_cast<int>(blockIdx.x) / 2;
  const int n_tiles = (p.N + kPairTile - 1) / kPairTile, t_tiles = (p.T + kPairTile - 1) / kPairTile;
  const int tiles = n_tiles * t_tiles;
  const int KB = (p.K + kFp4K - 1) / kFp4K;
  CtrlBlock* ctrl = &g_fp4_ctrl;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(tfull, 1);
    mbar_init(tfree, 16);   // eight epilogue warps of each CTA
    abort_flag[0] = 0;
    abort_flag[1] = p.stall ? kStallLimitUs : static_cast<int>(kWaitLimitNs / 1000);
    fence_barrier_init();
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(tmem_slot)),
                 "r"(kFp4TmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tm_w);
    tma_prefetch_desc(&tm_t);
    tma_prefetch_desc(&tm_sw);
    tma_prefetch_desc(&tm_st);
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();   // both CTAs' barriers and TMEM exist
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  griddep_wait();   // the tokens' codes are complete; no load goes out before

  if (warp == 0) {
    // ------------------------------------------------------------ loads
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      for (int tile = pair; tile < tiles; tile += pairs) {
        const int n0 = tile % n_tiles * kPairTile + 128 * rank;
        const int tb = tile / n_tiles * kPairTile;
        const int t0 = tb + 128 * rank;
        for (int kb = 0; kb < KB; ++kb) {
          if (!mbar_wait(&empty[stage], phase ^ 1u, abort_flag, ctrl, 50)) goto loads_done;
          const uint32_t bar = map_rank(smem_u32(&full[stage]), 0);
          if (rank == 0) mbar_arrive_expect_tx(&full[stage], 2 * Cfg::kStageBytes);   // both CTAs'
          tma_load_pair(sA + stage * kPairOpBytes, &tm_w, bar, kb * 128, n0);
          tma_load_pair(sB + stage * kPairOpBytes, &tm_t, bar, kb * 128, t0);
          const int x = kb * (Cfg::kScaleRow / 8);
          tma_load_pair(sSA + stage * Cfg::kScaleRow, &tm_sw, bar, x, n0 / 128);
          tma_load_pair(sSB + stage * 2 * Cfg::kScaleRow, &tm_st, bar, x, tb / 128);
          if (++stage == S) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
    loads_done:;
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA (even CTA)
    if (rank == 0) {
      const uint32_t lead = elect_lane();
      const uint32_t idesc = umma_idesc_fp4(kPairTile, !kNv) + (1u << 27);   // M = 256
      const uint64_t da0 = umma_desc_sw128(smem_u32(sA)), db0 = umma_desc_sw128(smem_u32(sB));
      const uint64_t dsa0 = scale_desc(smem_u32(sSA)), dsb0 = scale_desc(smem_u32(sSB));
      constexpr int kChunks = Cfg::kChunks;
      int stage = 0, seq = 0;
      uint32_t phase = 0;
      // A block's wait is tried before the MMAs of the block before it are
      // issued: the answer's latency would otherwise add to every block.
      bool loaded = false;
      bool ok = !p.stall || mbar_wait(tfull, 0, abort_flag, ctrl, 54);
      for (int tile = pair; ok && tile < tiles; tile += pairs, ++seq) {
        if (seq > 0 && !mbar_wait(tfree, (seq - 1) & 1u, abort_flag, ctrl, 51)) break;
        tc_fence_after();
        const uint32_t d = tmem + ((seq & 1) ? Cfg::kAcc1 : 0);
        uint32_t acc = 0;
        for (int kb = 0; kb < KB; ++kb) {
          if (!loaded && !mbar_wait(&full[stage], phase, abort_flag, ctrl, 52)) {
            ok = false;
            break;
          }
          const int steps = min(4, (p.K - kb * kFp4K + 63) / 64);
          const uint32_t sa = tmem + Cfg::kScaleCol0 + stage * Cfg::kSlotCols;
          const uint32_t sb = sa + 4 * kChunks;
          const uint64_t dsa = dsa0 + stage * (Cfg::kScaleRow / 16);
          const uint64_t dsb = dsb0 + stage * (2 * Cfg::kScaleRow / 16);
          const uint64_t da = da0 + stage * (kPairOpBytes / 16), db = db0 + stage * (kPairOpBytes / 16);
          uint64_t* const done = &empty[stage];
          if (++stage == S) {
            stage = 0;
            phase ^= 1u;
          }
#pragma unroll
          for (int c = 0; c < kChunks; ++c) {
            if (c * (4 / kChunks) < steps) {
              tmem_copy_scales<2>(lead, sa + 4 * c, dsa + c * (kFp4ScaleChunk / 16));
              tmem_copy_scales<2>(lead, sb + 8 * c, dsb + c * (kFp4ScaleChunk / 16));
              tmem_copy_scales<2>(lead, sb + 8 * c + 4, dsb + (kChunks + c) * (kFp4ScaleChunk / 16));
            }
          }
          loaded = mbar_test_wait(&full[stage], phase);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (j < steps) {
              if constexpr (kNv)
                umma_nvf4_pair(lead, d, da + 2 * j, db + 2 * j, idesc, sa + 4 * j, sb + 8 * j, acc);
              else
                umma_mxf4_pair(lead, d, da + 2 * j, db + 2 * j, idesc | umma_scale_ids(2 * (j & 1)),
                               sa + 4 * (j / 2), sb + 8 * (j / 2), acc);
              acc = 1;
            }
          }
          umma_commit_pair(lead, done);
        }
        if (ok) umma_commit_pair(lead, tfull);
      }
      if (abort_flag[0]) {
        // Loads and MMAs in flight land before either CTA can exit: none takes
        // as long as the bound of a wait, and none is issued after an abort.
        const unsigned long long since = globaltimer();
        while (globaltimer() - since < kWaitLimitNs) __nanosleep(1000000);
      }
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------ epilogue
    // Warp quarter q reads TMEM lanes 32q.. (its weight rows), one per lane;
    // half 0 takes tokens 0-127 of the tile, half 1 the others, in groups of 32.
    const int q = warp & 3, half = (warp - 4) / 4;
    const uint32_t lanes = static_cast<uint32_t>(q * 32) << 16;
    const OutScale alpha(p);
    const uint32_t free_bar = map_rank(smem_u32(tfree), 0);
    int seq = 0;
    // After a wait that ran out all later tiles are NaN as well: the barrier's phase is
    // behind, and the parity that they wait for would be taken for complete.
    bool ok = true;
    for (int tile = pair; tile < tiles; tile += pairs, ++seq) {
      const int n = tile % n_tiles * kPairTile + 128 * rank + q * 32 + lane;
      const int tb = tile / n_tiles * kPairTile + 128 * half;
      ok = ok && mbar_wait_warp(tfull, seq & 1u, abort_flag, ctrl, 53);
      const float scale = ok ? alpha.scale : NAN;
      tc_fence_after();
      const uint32_t d = tmem + lanes + ((seq & 1) ? Cfg::kAcc1 : 0) + 128 * half;
      // The columns that the other accumulator also has, the last of the first
      // and the first of the second, are drained first: all of one half of the
      // tokens, kMoreGroups groups of the other, next to it.
      constexpr int kMore = Cfg::kMoreGroups;
      const bool whole = half != (seq & 1);
      const int more = half ? 0 : 4 - kMore, rest = half ? kMore : 0;
      float v[4][32];
      if (whole) {
#pragma unroll
        for (int g = 0; g < 4; ++g) tmem_ld32(d + 32 * g, v[g]);
      } else {
#pragma unroll
        for (int g = 0; g < kMore; ++g) tmem_ld32(d + 32 * (more + g), v[g]);
      }
      tmem_ld_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_cluster(free_bar);
      // here and not in `store`, which is there eight times: the code's size costs (T = 901,
      // K = 480: 9.7 us instead of 9.45)
      if (alpha.before != 1.f) {
#pragma unroll
        for (int g = 0; g < 4; ++g)
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (whole || g < kMore) v[g][j] *= alpha.before;
      }
      O* const col = static_cast<O*>(p.out) + n;
      auto store = [&](int group, const float (&u)[32]) {
        const int t0 = tb + 32 * group;
        if (n >= p.N) return;
        O* o = col + static_cast<int64_t>(t0) * p.ldo;
        if (t0 + 32 <= p.T) {
#pragma unroll
          for (int j = 0; j < 32; ++j, o += p.ldo) store_out1(o, u[j] * scale);
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j, o += p.ldo)
            if (t0 + j < p.T) store_out1(o, u[j] * scale);
        }
      };
      if (whole) {
#pragma unroll
        for (int g = 0; g < 4; ++g) store(g, v[g]);
      } else {
#pragma unroll
        for (int g = 0; g < kMore; ++g) store(more + g, v[g]);
#pragma unroll
        for (int g = 0; g < 4 - kMore; ++g) tmem_ld32(d + 32 * (rest + g), v[g]);
        tmem_ld_wait();
        if (alpha.before != 1.f) {
#pragma unroll
          for (int g = 0; g < 4 - kMore; ++g)
#pragma unroll
            for (int j = 0; j < 32; ++j) v[g][j] *= alpha.before;
        }
#pragma unroll
        for (int g = 0; g < 4 - kMore; ++g) store(rest + g, v[g]);
      }
      tc_fence_before();
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();   // the peer's MMAs and signals are done with this CTA
  tc_fence_after();
  if (warp == 2)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kFp4TmemCols)
                 : "memory");
}

namespace {

// Scales [row blocks, chunks * 512 bytes] as 8-byte elements, read in boxes of
// one K block x box_rows row blocks.
int fp4_scale_map(const void* base, uint64_t chunks, uint64_t row_blocks, uint32_t chunks_per_block,
                  uint32_t box_rows, CUtensorMap* out) {
  const auto fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(tensor_map_encode());
  if (!fn) return MOE_ERR_CUDA;
  cuuint64_t dims[2] = {chunks * 64, row_blocks};
  cuuint64_t strides[1] = {chunks * kFp4ScaleChunk};
  cuuint32_t box[2] = {chunks_per_block * 64, box_rows};
  cuuint32_t estr[2] = {1, 1};
  return fn(out, CU_TENSOR_MAP_DATA_TYPE_FLOAT64, 2, const_cast<void*>(base), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? MOE_OK
             : MOE_ERR_CUDA;
}

// Codes [rows, K/2] with row stride ld bytes, read in boxes of 128 bytes x box_rows.
int fp4_map(const void* base, uint64_t k_bytes, uint64_t rows, uint64_t ld, uint32_t box_rows,
            CUtensorMap* out) {
  const auto fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(tensor_map_encode());
  if (!fn) return MOE_ERR_CUDA;
  cuuint64_t dims[2] = {k_bytes, rows};
  cuuint64_t strides[1] = {ld};
  cuuint32_t box[2] = {128, box_rows};
  cuuint32_t estr[2] = {1, 1};
  return fn(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? MOE_OK
             : MOE_ERR_CUDA;
}

// Clusters of 2, 4 and 8 CTAs of the split kernel that run at once, per device: a
// graphics processing cluster holds whole ones only (of 8, fewer than 148 / 8).
int g_max_clusters[64][3];

// CTAs that share a tile: as many as run at once, each with a K block at least.
int fp4_split(const Fp4GemmParams& p, int nt) {
  const int64_t tiles = static_cast<int64_t>((p.N + kFp4M - 1) / kFp4M) * ((p.T + nt - 1) / nt);
  const int KB = (p.K + kFp4K - 1) / kFp4K;
  int dev = 0, split = 1;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 1;
  for (int i = 0; i < 3; ++i)
    if ((2 << i) <= KB && tiles <= g_max_clusters[dev][i]) split = 2 << i;
  return split;
}

template <int NT, typename X = void>
int launch_nt(Fp4GemmParams p, const void* w_codes, int64_t ld_w, const void* t_codes, int64_t ld_t,
              bool after_quantize, cudaStream_t s) {
  CUtensorMap tm_w, tm_t{};
  int st = fp4_map(w_codes, p.K / 2, p.N, ld_w, kFp4M, &tm_w);
  if (!st && t_codes) st = fp4_map(t_codes, p.K / 2, p.T, ld_t, NT, &tm_t);
  if (st) return st;
  const int n_tiles = (p.N + kFp4M - 1) / kFp4M, t_tiles = (p.T + NT - 1) / NT;
  const int split = p.split = fp4_split(p, NT);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(n_tiles * split, t_tiles);
  cfg.blockDim = dim3(kFp4Threads);
  cfg.dynamicSmemBytes = Fp4Cfg<NT>::kSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (split > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = split;
    attr[n].val.clusterDim.y = 1;
    attr[n++].val.clusterDim.z = 1;
  }
  if (after_quantize) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, p.nv ? moe_fp4_gemm_kernel<NT, true, X> : moe_fp4_gemm_kernel<NT, false, X>,
                            tm_w, tm_t, p) == cudaSuccess
             ? MOE_OK
             : MOE_ERR_CUDA;
}

template <typename O>
int launch_pair(const Fp4GemmParams& p, const void* w_codes, int64_t ld_w, const void* t_codes,
                int64_t ld_t, int sms, bool after_quantize, cudaStream_t s) {
  CUtensorMap tm_w, tm_t, tm_sw, tm_st;
  int st = fp4_map(w_codes, p.K / 2, p.N, ld_w, 128, &tm_w);
  if (!st) st = fp4_map(t_codes, p.K / 2, p.T, ld_t, 128, &tm_t);
  if (!st) st = fp4_scale_map(p.w_scales, p.chunks, (p.N + 127) / 128, p.chunks_per_block, 1, &tm_sw);
  if (!st) st = fp4_scale_map(p.t_scales, p.chunks, (p.T + 127) / 128, p.chunks_per_block, 2, &tm_st);
  if (st) return st;
  const int64_t tiles = static_cast<int64_t>((p.N + kPairTile - 1) / kPairTile) *
                        ((p.T + kPairTile - 1) / kPairTile);
  const int pairs = static_cast<int>(tiles < sms / 2 ? tiles : sms / 2);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(2 * pairs);
  cfg.blockDim = dim3(kPairThreads);
  cfg.dynamicSmemBytes = p.nv ? PairCfg<true>::kSmem : PairCfg<false>::kSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = after_quantize ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, p.nv ? moe_fp4_gemm_pair_kernel<O, true> : moe_fp4_gemm_pair_kernel<O, false>,
                            tm_w, tm_t, tm_sw, tm_st, p) == cudaSuccess
             ? MOE_OK
             : MOE_ERR_CUDA;
}

template <typename Kernel>
int set_attr(Kernel kernel, int bytes) {
  return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) == cudaSuccess
             ? MOE_OK
             : MOE_ERR_CUDA;
}
template <int NT, typename X = void>
int set_attr_nt() {
  const int st = set_attr(moe_fp4_gemm_kernel<NT, true, X>, Fp4Cfg<NT>::kSmem);
  return st ? st : set_attr(moe_fp4_gemm_kernel<NT, false, X>, Fp4Cfg<NT>::kSmem);
}
template <typename O>
int set_attr_pair() {
  const int st = set_attr(moe_fp4_gemm_pair_kernel<O, true>, PairCfg<true>::kSmem);
  return st ? st : set_attr(moe_fp4_gemm_pair_kernel<O, false>, PairCfg<false>::kSmem);
}

}  // namespace

namespace {

std::mutex g_setup_mu;
bool g_set_up[64];

// The current device's SM count; its products may use their shared memory and know how
// many clusters run at once.
int fp4_device(int* sms) {
  int st = num_sms(sms);
  if (st) return st;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return MOE_ERR_CUDA;
  std::lock_guard<std::mutex> lk(g_setup_mu);
  if (g_set_up[dev]) return MOE_OK;
  st = set_attr_nt<16>();
  if (!st) st = set_attr_nt<32>();
  if (!st) st = set_attr_nt<64>();
  if (!st) st = set_attr_nt<128>();
  if (!st) st = set_attr_nt<16, __nv_bfloat16>();
  if (!st) st = set_attr_nt<16, __half>();
  if (!st) st = set_attr_nt<16, float>();
  if (!st) st = set_attr_pair<__nv_bfloat16>();
  if (!st) st = set_attr_pair<__half>();
  if (!st) st = set_attr_pair<float>();
  for (int i = 0; i < 3 && !st; ++i) {
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2u << i;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3(2u << i);
    cfg.blockDim = dim3(kFp4Threads);
    cfg.dynamicSmemBytes = Fp4Cfg<128>::kSmem;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&g_max_clusters[dev][i], moe_fp4_gemm_kernel<128, true>, &cfg) !=
        cudaSuccess)
      st = MOE_ERR_CUDA;
  }
  g_set_up[dev] = !st;
  return st;
}

}  // namespace

// after_quantize: the kernel launched just before in this stream is the
// quantisation of the tokens, which lets this one start early.
//
// Up to 64 tokens one tile of tokens takes them all and the weights stream once.
// Above, the pair kernel and the split kernel on 128-token tiles take about as
// long for a K block (0.5 us), so the one with fewer of them after one another is
// launched; a split tile's exchange of sums counts as three.  (nvfp4, T=300:
// N=4096 K=7168 18.1 us in pairs and 19.9 split, N=512 K=7168 17.4 and 8.5.)
int launch_fp4_gemm(const Fp4GemmParams& p, const void* w_codes, int64_t ld_w, const void* t_codes,
                    int64_t ld_t, int sms, bool after_quantize, cudaStream_t s) {
  if (p.T <= 16) return launch_nt<16>(p, w_codes, ld_w, t_codes, ld_t, after_quantize, s);
  if (p.T <= 32) return launch_nt<32>(p, w_codes, ld_w, t_codes, ld_t, after_quantize, s);
  if (p.T <= 64) return launch_nt<64>(p, w_codes, ld_w, t_codes, ld_t, after_quantize, s);
  auto tiles = [&p](int m, int t) {
    return static_cast<int64_t>((p.N + m - 1) / m) * ((p.T + t - 1) / t);
  };
  const int64_t KB = (p.K + kFp4K - 1) / kFp4K, pairs = sms / 2, split = fp4_split(p, 128);
  const int64_t pair_steps = (tiles(kPairTile, kPairTile) + pairs - 1) / pairs * KB;
  const int64_t split_steps = (tiles(kFp4M, 128) * split + sms - 1) / sms * ((KB + split - 1) / split) +
                              (split > 1 ? 3 : 0);
  if (split_steps < pair_steps) return launch_nt<128>(p, w_codes, ld_w, t_codes, ld_t, after_quantize, s);
  if (p.out_dtype == MOE_BF16)
    return launch_pair<__nv_bfloat16>(p, w_codes, ld_w, t_codes, ld_t, sms, after_quantize, s);
  if (p.out_dtype == MOE_F16)
    return launch_pair<__half>(p, w_codes, ld_w, t_codes, ld_t, sms, after_quantize, s);
  return launch_pair<float>(p, w_codes, ld_w, t_codes, ld_t, sms, after_quantize, s);
}

namespace {

bool off(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) != 0; }

// Whether `rows` rows at a and as many at b (bytes of a row and of its stride) share
// memory; columns of one matrix beside each other do not.
bool rows_overlap(const void* a, int64_t row_a, int64_t ld_a, const void* b, int64_t row_b, int64_t ld_b,
                  int64_t rows) {
  const auto a0 = reinterpret_cast<uintptr_t>(a), b0 = reinterpret_cast<uintptr_t>(b);
  const uintptr_t a1 = a0 + (rows - 1) * ld_a + row_a, b1 = b0 + (rows - 1) * ld_b + row_b;
  if (a1 <= b0 || b1 <= a0) return false;
  if (ld_a != ld_b) return true;
  const uintptr_t ld = static_cast<uintptr_t>(ld_a);
  const uintptr_t d = b0 >= a0 ? (b0 - a0) % ld : (ld - (a0 - b0) % ld) % ld;   // of b's rows in a's
  return d < static_cast<uintptr_t>(row_a) || d + row_b > ld;
}

// Whether the format carries MOE_FP4_TEST_STALL, which it loses.
bool take_stall(int32_t* format) {
  const bool stall = (*format & MOE_FP4_TEST_STALL) != 0;
  *format &= ~MOE_FP4_TEST_STALL;
  return stall;
}

int gemm_params(Fp4GemmParams* p, int32_t format, int64_t T, int64_t N, int64_t K, const void* w_codes,
                int64_t ld_w, const void* w_scales, const float* w_global_scale, void* out,
                int32_t out_dtype, int64_t ldo) {
  int st = fp4_check(format, T, K);
  if (!st) st = fp4_check(format, N, K);
  if (st) return st;
  // grid.y counts tiles of 128 tokens
  if (N < 1 || T > (int64_t(1) << 22)) return MOE_ERR_SHAPE;
  if (out_dtype != MOE_BF16 && out_dtype != MOE_F16 && out_dtype != MOE_F32) return MOE_ERR_INVALID_ARG;
  if (format == MOE_MXFP4 && w_global_scale) return MOE_ERR_INVALID_ARG;
  if (ld_w < K / 2 || ld_w % 16 != 0 || ldo < N) return MOE_ERR_SHAPE;
  if (T == 0) return MOE_OK;
  if (!w_codes || !w_scales || !out) return MOE_ERR_INVALID_ARG;
  const int elem = out_dtype == MOE_F32 ? 4 : 2;
  if (off(w_codes, 16) || off(w_scales, 16) || off(w_global_scale, 4) || off(out, elem))
    return MOE_ERR_ALIGNMENT;
  p->T = static_cast<int>(T);
  p->N = static_cast<int>(N);
  p->K = static_cast<int>(K);
  p->nv = format == MOE_NVFP4;
  p->chunks = fp4_chunks(format, K);
  p->chunks_per_block = p->nv ? 4 : 2;
  p->w_scales = static_cast<const uint8_t*>(w_scales);
  p->gb = w_global_scale;
  p->out = out;
  p->out_dtype = out_dtype;
  p->ldo = ldo;
  p->vec_out = !off(out, 4 * elem) && ldo % 4 == 0;
  return MOE_OK;
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" {

int moe_fp4_matmul(const void* a_codes, int64_t ld_a, const void* a_scales,
                   const float* a_global_scale, const void* b_codes, int64_t ld_b,
                   const void* b_scales, const float* b_global_scale, int32_t format, int64_t T,
                   int64_t N, int64_t K, void* out, int32_t out_dtype, int64_t ldo, void* stream) {
  Fp4GemmParams p{};
  p.stall = take_stall(&format);
  int st = gemm_params(&p, format, T, N, K, b_codes, ld_b, b_scales, b_global_scale, out, out_dtype, ldo);
  if (st) return st;
  if (format == MOE_MXFP4 && a_global_scale) return MOE_ERR_INVALID_ARG;
  if (ld_a < K / 2 || ld_a % 16 != 0) return MOE_ERR_SHAPE;
  if (T == 0) return MOE_OK;
  if (!a_codes || !a_scales) return MOE_ERR_INVALID_ARG;
  if (off(a_codes, 16) || off(a_scales, 16) || off(a_global_scale, 4)) return MOE_ERR_ALIGNMENT;
  int sms = 0;
  if ((st = fp4_device(&sms))) return st;
  p.t_scales = static_cast<const uint8_t*>(a_scales);
  p.ga = a_global_scale;
  return launch_fp4_gemm(p, b_codes, ld_b, a_codes, ld_a, sms, false, static_cast<cudaStream_t>(stream));
}

int moe_fp4_linear_workspace_size(int32_t format, int64_t T, int64_t K, size_t* bytes) {
  if (!bytes) return MOE_ERR_INVALID_ARG;
  const int st = fp4_check(format, T, K);
  if (st) return st;
  const size_t codes = (static_cast<size_t>(T) * (K / 2) + 255) / 256 * 256;
  *bytes = T <= kFp4FusedTokens
               ? 0
               : codes + static_cast<size_t>((T + 127) / 128) * fp4_chunks(format, K) * 512;
  return MOE_OK;
}

int moe_fp4_linear(const void* x, int32_t x_dtype, int64_t ld_x, const float* x_global_scale,
                   const void* w_codes, int64_t ld_w, const void* w_scales,
                   const float* w_global_scale, int32_t format, int64_t T, int64_t N, int64_t K,
                   void* out, int32_t out_dtype, int64_t ldo, void* workspace,
                   size_t workspace_bytes, void* stream) {
  Fp4GemmParams p{};
  p.stall = take_stall(&format);
  int st = gemm_params(&p, format, T, N, K, w_codes, ld_w, w_scales, w_global_scale, out, out_dtype, ldo);
  if (!st) st = fp4_check_input(x, x_dtype, ld_x, T, K, format, x_global_scale);
  if (st) return st;
  if (T == 0) return MOE_OK;
  size_t need = 0;
  if ((st = moe_fp4_linear_workspace_size(format, T, K, &need))) return st;
  if (need && (!workspace || workspace_bytes < need)) return MOE_ERR_WORKSPACE;
  if (need && off(workspace, 256)) return MOE_ERR_ALIGNMENT;
  // a few tokens are read by every tile's blocks while others store
  const int64_t ex = x_dtype == MOE_F32 ? 4 : 2, eo = out_dtype == MOE_F32 ? 4 : 2;
  if (rows_overlap(x, K * ex, ld_x * ex, out, N * eo, ldo * eo, T)) return MOE_ERR_INVALID_ARG;
  int sms = 0;
  if ((st = fp4_device(&sms))) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  p.ga = x_global_scale;
  if (!need) {
    p.x = x;
    p.ld_x = ld_x;
    if (x_dtype == MOE_BF16) return launch_nt<16, __nv_bfloat16>(p, w_codes, ld_w, nullptr, 0, false, s);
    if (x_dtype == MOE_F16) return launch_nt<16, __half>(p, w_codes, ld_w, nullptr, 0, false, s);
    return launch_nt<16, float>(p, w_codes, ld_w, nullptr, 0, false, s);
  }
  uint8_t* codes = static_cast<uint8_t*>(workspace);
  uint8_t* scales = codes + (static_cast<size_t>(T) * (K / 2) + 255) / 256 * 256;
  if ((st = moe_fp4_quantize(x, x_dtype, ld_x, T, K, format, x_global_scale, codes, scales, stream)))
    return st;
  p.t_scales = scales;
  return launch_fp4_gemm(p, w_codes, ld_w, codes, K / 2, sms, true, s);
}

int moe_fp4_device_error(void* stream, int32_t* code, int32_t* info) {
  if (!code || !info) return MOE_ERR_INVALID_ARG;
  int sms = 0;
  const int st = num_sms(&sms);
  if (st) return st;
  CtrlBlock host;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (cudaMemcpyFromSymbolAsync(&host, g_fp4_ctrl, sizeof(host), 0, cudaMemcpyDeviceToHost, s) !=
      cudaSuccess)
    return MOE_ERR_CUDA;
  if (cudaStreamSynchronize(s) != cudaSuccess) return MOE_ERR_CUDA;
  *code = host.error;
  *info = host.error_info;
  if (host.error) {   // told once
    void* word = nullptr;
    if (cudaGetSymbolAddress(&word, g_fp4_ctrl) != cudaSuccess ||
        cudaMemsetAsync(word, 0, sizeof(host), s) != cudaSuccess ||
        cudaStreamSynchronize(s) != cudaSuccess)
      return MOE_ERR_CUDA;
  }
  return MOE_OK;
}

}  // extern "C"
