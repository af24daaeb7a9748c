// fp4_gemm.cu -- products of microscaled 4-bit rows on the sm_100 tensor cores
// (tcgen05.mma kind::mxf4 / kind::mxf4nvf4 with block scales in tensor memory, fp32 sums):
//   out[m, n] = (sum over k of x[m, k] w[n, k]) * xs[m] * ws[n] + bias[n]
// where x and w stand for code * block scale and xs, ws for the rows' scales.
//
// A K step is 256 columns: 128 bytes of codes per row (one 128-byte swizzle row, four
// products of 64 columns) and, per 128 rows, four (nvfp4) or two (mxfp4) 512-byte tiles of
// block scales.  Codes and scales come by TMA into a ring of stages; the scales go on into
// tensor memory by tcgen05.cp, into one of a few slots: the copy into a slot waits for the
// products that read it last, and the products of a step for its copies.
#include <type_traits>

#include "fp4.cuh"
#include "h3b_kernels.cuh"

namespace h3b {

constexpr int kF4Step = 128;  // bytes of codes per row and K step

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// Shared-memory matrix descriptors, of which the high word is constant and the low one the address
// in units of 16 bytes and a flag: what a step needs comes by additions to it.
__device__ __forceinline__ uint32_t sdesc_low(uint32_t smem_addr) { return ((smem_addr & 0x3FFFF) >> 4) | (1u << 16); }
// K-major in the 128-byte swizzle: 8-row atoms of 1,024 bytes (SBO)
__device__ __forceinline__ uint64_t sdesc_codes(uint32_t low) {
  constexpr uint32_t high = (1024 >> 4) | (1u << 14) | (2u << 29);
  return ((uint64_t)high << 32) | low;
}
// A tile of block scales, without swizzle: 32 rows of 16 bytes, 8-row pieces of 128 bytes (SBO)
__device__ __forceinline__ uint64_t sdesc_scales(uint32_t low) {
  constexpr uint32_t high = (128 >> 4) | (1u << 14);
  return ((uint64_t)high << 32) | low;
}
// Instruction descriptor of the block-scaled 4-bit kinds: bits 4-5 / 29-30 first byte of the
// scale word of B / A, 7-9 / 10-11 E2M1 operands (1), 17-22 N>>3, 23 E8M0 scales, 24-28 M>>4.
__host__ __device__ constexpr uint32_t idesc_fp4(int M, int N, bool e8m0, uint32_t scale_byte) {
  return (scale_byte << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | ((e8m0 ? 1u : 0u) << 23) |
         ((uint32_t)(M >> 4) << 24) | (scale_byte << 29);
}

template <int FORMAT, int CTAS>
__device__ __forceinline__ void mma_fp4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb,
                                        uint32_t accumulate) {
#define H3B_MMA_FP4(kind)                                                                          \
  asm volatile(                                                                                    \
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma." kind " [%0], %1, %2, %3, [%5], [%6], p;\n\t}" \
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(sa), "r"(sb)                      \
      : "memory")
  if constexpr (FORMAT == kMxfp4 && CTAS == 1) H3B_MMA_FP4("cta_group::1.kind::mxf4.block_scale.scale_vec::2X");
  if constexpr (FORMAT == kMxfp4 && CTAS == 2) H3B_MMA_FP4("cta_group::2.kind::mxf4.block_scale.scale_vec::2X");
  if constexpr (FORMAT == kNvfp4 && CTAS == 1) H3B_MMA_FP4("cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X");
  if constexpr (FORMAT == kNvfp4 && CTAS == 2) H3B_MMA_FP4("cta_group::2.kind::mxf4nvf4.block_scale.scale_vec::4X");
#undef H3B_MMA_FP4
}
// A 512-byte tile of block scales to four columns of tensor memory (all four lane quadrants)
template <int CTAS>
__device__ __forceinline__ void copy_scales(uint32_t taddr, uint64_t sdesc) {
  if constexpr (CTAS == 1)
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(sdesc) : "memory");
  else
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(sdesc) : "memory");
}

// A sum times its row scales.  Of two scales on the same side of 1 the first takes the sum no further
// than both do, and they follow each other; where one is below 1 and the other is not, their product
// lies between them and comes first, so that nothing leaves fp32's range on the way to a value in it.
__device__ __forceinline__ float fp4_scaled(float sum, float xs, float ws) {
  const bool apart = (fabsf(xs) < 1.0f) != (fabsf(ws) < 1.0f);
  return __fmul_rn(__fmul_rn(sum, apart ? __fmul_rn(xs, ws) : xs), apart ? 1.0f : ws);
}
// A sum to its output value; xs and ws are 1 where there are no row scales.  APART: they may lie on
// either side of 1
template <bool APART>
__device__ __forceinline__ float fp4_finish(float sum, float xs, float ws, float bias, const Fp4GemmArgs& a) {
  const float v = APART ? fp4_scaled(sum, xs, ws) : __fmul_rn(__fmul_rn(sum, xs), ws);
  return a.bias ? __fadd_rn(v, bias) : v;
}

// One thread: the scale copies of one K step.  BANDS: 128-row bands of scales of the B operand.
template <int FORMAT, int CTAS, int BANDS>
__device__ __forceinline__ void fp4_step_scales(uint32_t smem_sa, uint32_t smem_sb, uint32_t tmem_sa, uint32_t tmem_sb) {
  constexpr int kTiles = FORMAT == kMxfp4 ? 2 : 4;  // scale tiles per band and step
  const uint32_t la = sdesc_low(smem_sa), lb = sdesc_low(smem_sb);
#pragma unroll
  for (int g = 0; g < kTiles; ++g) {
    copy_scales<CTAS>(tmem_sa + (uint32_t)(4 * g), sdesc_scales(la + 32u * g));
#pragma unroll
    for (int b = 0; b < BANDS; ++b)
      copy_scales<CTAS>(tmem_sb + (uint32_t)(4 * (BANDS * g + b)), sdesc_scales(lb + 32u * (kTiles * b + g)));
  }
}
// One thread: the products of one K step into accumulator d; tmem_sb: the column of B's scales
// in which those of its first row lie.
template <int FORMAT, int CTAS, int M, int N, int BANDS>
__device__ __forceinline__ void fp4_step_products(uint32_t d, uint32_t smem_a, uint32_t smem_b, uint32_t tmem_sa,
                                                  uint32_t tmem_sb, int products, bool first) {
  const uint32_t la = sdesc_low(smem_a), lb = sdesc_low(smem_b);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (k > 0 && k >= products) break;
    const uint32_t byte = FORMAT == kMxfp4 ? 2u * (uint32_t)(k & 1) : 0u;
    const uint32_t g = FORMAT == kMxfp4 ? (uint32_t)(k >> 1) : (uint32_t)k;
    mma_fp4<FORMAT, CTAS>(d, sdesc_codes(la + 2u * k), sdesc_codes(lb + 2u * k), idesc_fp4(M, N, FORMAT == kMxfp4, byte),
                          tmem_sa + 4u * g, tmem_sb + 4u * BANDS * g, first && k == 0 ? 0u : 1u);
  }
}
// Non-blocking look at a barrier.  The warps that issue scale copies and products look at the next
// step's barriers, a lane at each, before they issue this step's: a wait costs about 100 cycles
// even where it is over, a scale copy 20 to 30, and a step of the 256 x 256 tiles has 512 in all
// (9,472 x 2,048 x 16,384 mxfp4 with plain waits 124 us, so 104 us).
__device__ __forceinline__ bool mbar_peek(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
  return ok != 0;
}
// A place in a ring of n stages: the next fill's stage and the parity of its barrier
struct RingPlace {
  uint32_t stage = 0, parity = 0;
  __device__ __forceinline__ void next(uint32_t n) {
    if (++stage == n) {
      stage = 0;
      parity ^= 1u;
    }
  }
};

// ------------------------------------------------------------------ few rows: a split over K
// A tile is 128 rows of the weight (the products' M) x TOK rows of x (their N), so that one
// token costs the reading of the weight and hardly more.  The CTAs of a cluster (1, 2, 4 or 8)
// take equal parts of K; each sends its sums to the CTAs that own their columns (equal shares of
// the tile's 128), which add them in the CTAs' order (the same sums every time) and write them.
// Without a split the sums go out as they come from tensor memory.
//   warp 0: TMA, warp 1: tensor memory and products, warp 2: scale copies, warps 3-6: sums
// Behind the quantisation of x in the stream, the first weight tiles are on their way before
// that has ended.  ROWS16: x is 16-bit, at most 16 rows, and warps 3-6 of each CTA quantise
// its part of K themselves (for nvfp4 the cluster's CTAs tell each other their rows' absmax).
template <int FORMAT, int TOK, bool ROWS16>
struct SplitCfg {
  static_assert(!ROWS16 || TOK == 16, "rows are quantised here for a tile of 16");
  static constexpr int kScaleBytes = FORMAT == kMxfp4 ? 1024 : 2048;  // of a band and step
  static constexpr int kWBytes = 128 * kF4Step;
  static constexpr int kXBytes = TOK * kF4Step;
  static constexpr int kXStep = kXBytes + kScaleBytes;
  static constexpr int kStageBytes = kWBytes + kScaleBytes + (ROWS16 ? 0 : kXStep);
  static_assert(kStageBytes % 1024 == 0 && kXStep % 1024 == 0, "swizzled tiles start at multiples of 1024");
  static constexpr int kAccCols = TOK < 32 ? 32 : TOK;
  static constexpr int kSlotCols = kScaleBytes / 64;  // both operands' scales of a step: 16 or 32 columns
  static constexpr int kSlots = 4;
  static constexpr int kTmemCols = 256;
  static_assert(kAccCols + kSlots * kSlotCols <= kTmemCols, "");
  // what a CTA needs beside its stages
  static constexpr int rest_bytes(int steps, int split) {
    return (ROWS16 ? steps * kXStep : 0) + (split > 1 ? TOK * 512 : 0) + 1024;
  }
};
constexpr int kSplitThreads = 224, kSplitMaxStages = 8;
constexpr int kSplitMost = 220 * 1024;  // dynamic shared memory of a CTA
constexpr int kRows16Steps = 16;  // K steps of a CTA that quantises x
// Pieces of 512 columns of x that one of its four warps holds.  More rows take longer here than in a
// kernel of their own in front (4,096 -> 4,096, nvfp4: 4 rows 7.2 us in one launch and 6.2 in two, 8 rows
// 8.4 and 6.1; mxfp4: 8 rows 5.8 and 5.7); a call in one launch costs the host 10 us, one in two 14.  The limits
// go by the call from the host: in a captured graph, nvfp4 rows near them would take less time in two launches.
constexpr int rows16_items(int format) { return format == kMxfp4 ? 4 : 2; }

// bounded wait for an mbarrier whose arrivals release what other CTAs of the cluster wrote here
__device__ __forceinline__ bool mbar_wait_sent(uint64_t* bar, volatile int* abort_flag) {
  const uint64_t t0 = globaltimer_ns();
  for (uint32_t n = 0;; ++n) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], 0;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(smem_u32(bar)) : "memory");
    if (ok) return true;
    if (n >= kWaitMaxTries || (n > 64 && globaltimer_ns() - t0 > kWaitLimitNs)) {
      *abort_flag = 1;
      record_status(H3B_STATUS_GEMM_TIMEOUT);
      return false;
    }
  }
}

template <int FORMAT, int TOK, bool ROWS16, bool BF16>
__global__ void __launch_bounds__(kSplitThreads)
    fp4_split_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_sw,
                     const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_sx,
                     Fp4GemmArgs a, int log_split, int num_stages) {
  using C = SplitCfg<FORMAT, TOK, ROWS16>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t full[kSplitMaxStages], empty[kSplitMaxStages], scaled[C::kSlots], done, copied, x_ready, sent;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_flag, late_flag;
  __shared__ uint32_t row_top[16];
  __shared__ float row_scale[TOK];
  __shared__ __align__(16) uint16_t pieces[ROWS16 ? 4 : 1][ROWS16 ? 512 : 8];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = 1 << log_split, rank = (int)blockIdx.x & (split - 1);
  const int n0 = ((int)blockIdx.x >> log_split) * 128, m0 = (int)blockIdx.y * TOK;
  const int num_k = (a.K + 255) / 256;
  const int kb0 = (num_k * rank) >> log_split, steps = ((num_k * (rank + 1)) >> log_split) - kb0;
  const uint32_t stages = (uint32_t)num_stages;
  const int log_share = 7 - log_split, share = 1 << log_share;  // columns of the tile that this CTA adds up
  uint8_t* x_area = smem + stages * C::kStageBytes;             // ROWS16: [steps] codes and scales
  // [split][TOK][share], at the same place in all CTAs of the cluster
  float* sums = reinterpret_cast<float*>(x_area + (ROWS16 ? ((num_k + split - 1) >> log_split) * C::kXStep : 0));

  if (warp == 0) {
    if (lane < kSplitMaxStages) {
      mbar_init(&full[lane], 1);
      mbar_init(&empty[lane], 1);
    } else if (lane < kSplitMaxStages + C::kSlots) {
      mbar_init(&scaled[lane - kSplitMaxStages], 1);
    } else if (lane == 31) {
      mbar_init(&done, 1);
      mbar_init(&copied, 1);
      mbar_init(&x_ready, 128);
      mbar_init(&sent, (uint32_t)(128 / min(32, share)));
      abort_flag = late_flag = 0;
    }
    fence_mbar_init();
    __syncwarp();
    asm volatile("bar.arrive 1, %0;" ::"n"(kSplitThreads) : "memory");
    // the first loads start before tensor memory is there
    RingPlace fill, freed;
    auto load_w = [&](int i, uint32_t stage) {
      uint8_t* at = smem + stage * C::kStageBytes;
      mbar_arrive_expect_tx(&full[stage], C::kStageBytes);
      tma_load_2d(at, &tm_w, &full[stage], (kb0 + i) * kF4Step, n0);
      tma_load_2d(at + C::kWBytes, &tm_sw, &full[stage], (kb0 + i) * (C::kScaleBytes / 8), n0 >> 7);
    };
    auto load_x = [&](int i, uint32_t stage) {
      if constexpr (!ROWS16) {
        uint8_t* at = smem + stage * C::kStageBytes + C::kWBytes + C::kScaleBytes;
        tma_load_2d(at, &tm_x, &full[stage], (kb0 + i) * kF4Step, m0);
        tma_load_2d(at + C::kXBytes, &tm_sx, &full[stage], (kb0 + i) * (C::kScaleBytes / 8), m0 >> 7);
      }
    };
    const int ahead = min(steps, num_stages);
    if (a.behind_rows) {
      if (elect_one())
        for (int i = 0; i < ahead; ++i) load_w(i, (uint32_t)i);
      __syncwarp();
      chain_wait();
      if (elect_one())
        for (int i = 0; i < ahead; ++i) load_x(i, (uint32_t)i);
    } else {
      chain_wait();
      if (elect_one())
        for (int i = 0; i < ahead; ++i) {
          load_w(i, (uint32_t)i);
          load_x(i, (uint32_t)i);
        }
    }
    __syncwarp();
    chain_next();
    if (split > 1) {
      cluster_arrive();
      cluster_wait();
      if (ROWS16 && FORMAT == kNvfp4) cluster_sync_all();
    }
    int fills = ahead;
    for (int i = 0; i < ahead; ++i) fill.next(stages);
    for (; fills < steps; ++fills) {
      if (!mbar_wait_warp(&empty[freed.stage], freed.parity, &abort_flag, H3B_STATUS_GEMM_TIMEOUT)) break;
      freed.next(stages);
      if (elect_one()) {
        load_w(fills, fill.stage);
        load_x(fills, fill.stage);
      }
      __syncwarp();
      fill.next(stages);
    }
    // every copy that was started has landed before the CTA may leave: of each slot the last fill
    for (uint32_t s = 0; s < stages; ++s)
      mbar_wait_warp(&full[s], s < fill.stage ? fill.parity : fill.parity ^ 1u, &late_flag, H3B_STATUS_GEMM_TIMEOUT);
  } else {
    if (warp == 1) {
      tmem_alloc(&tmem_slot, C::kTmemCols);
      tmem_relinquish();
    } else if (ROWS16 && threadIdx.x >= 96 && threadIdx.x < 112) {
      row_top[threadIdx.x - 96] = 0u;
    }
    tc_fence_before();
    asm volatile("bar.sync 1, %0;" ::"n"(kSplitThreads) : "memory");
    tc_fence_after();
    chain_next();
    if (split > 1) cluster_arrive();  // and wait before anything of another CTA is touched
  }
  const uint32_t tmem = tmem_slot;  // warp 0 does not use it

  if (warp == 1) {
    if (split > 1) {
      cluster_wait();
      if (ROWS16 && FORMAT == kNvfp4) cluster_sync_all();
    }
    // products: a step's operands are there, and its scales in tensor memory
    const uint32_t smem0 = smem_u32(smem), x0 = smem_u32(x_area);
    RingPlace at, scales;
    auto peek = [&]() {
      return lane == 1 ? mbar_peek(&full[at.stage], at.parity) : mbar_peek(&scaled[scales.stage], scales.parity);
    };
    bool seen = peek();
    const bool ready = !ROWS16 || mbar_wait_warp(&x_ready, 0, &abort_flag, H3B_STATUS_GEMM_TIMEOUT);
    for (int i = 0; ready && i < steps; ++i) {
      if (!__all_sync(0xffffffffu, seen) &&
          (!mbar_wait_warp(&scaled[scales.stage], scales.parity, &abort_flag, H3B_STATUS_GEMM_TIMEOUT) ||
           !mbar_wait_warp(&full[at.stage], at.parity, &abort_flag, H3B_STATUS_GEMM_TIMEOUT)))
        break;
      tc_fence_after();
      const uint32_t w = smem0 + at.stage * C::kStageBytes;
      const uint32_t x = ROWS16 ? x0 + (uint32_t)(i * C::kXStep) : w + C::kWBytes + C::kScaleBytes;
      const uint32_t ts = tmem + C::kAccCols + C::kSlotCols * scales.stage;
      uint64_t* used = &empty[at.stage];
      at.next(stages);
      scales.next(C::kSlots);
      seen = peek();
      if (elect_one()) {
        // rows m0 .. of their 128-row band: 32 to a column of the scales
        fp4_step_products<FORMAT, 1, 128, TOK, 1>(tmem, w, x, ts, ts + C::kSlotCols / 2 + ((uint32_t)(m0 >> 5) & 3u),
                                                  (a.K - (kb0 + i) * 256 + 63) / 64, i == 0);
        mma_commit(used);
      }
      __syncwarp();
    }
    if (elect_one()) mma_commit(&done);
    __syncwarp();
    mbar_wait_warp(&done, 0, &late_flag, H3B_STATUS_GEMM_TIMEOUT);
  } else if (warp == 2) {
    if (split > 1) {
      cluster_wait();
      if (ROWS16 && FORMAT == kNvfp4) cluster_sync_all();
    }
    // scale copies: into the slot that the products kSlots steps before have read
    const uint32_t smem0 = smem_u32(smem), x0 = smem_u32(x_area);
    const bool ready = !ROWS16 || mbar_wait_warp(&x_ready, 0, &abort_flag, H3B_STATUS_GEMM_TIMEOUT);
    RingPlace at, freed, scales;
    int i = 0;
    // With as many stages as slots or fewer, a stage that is full says that its slot was read; with
    // more, the slot's barrier is asked, which cannot have moved on by more than one phase.
    auto asks = [&]() { return i >= C::kSlots && num_stages > C::kSlots; };
    auto peek = [&]() {
      const bool slot = lane == 1 && asks();
      return mbar_peek(slot ? &empty[freed.stage] : &full[at.stage], slot ? freed.parity : at.parity);
    };
    bool seen = peek();
    while (ready && i < steps) {
      if (!__all_sync(0xffffffffu, seen) &&
          (!mbar_wait_warp(&full[at.stage], at.parity, &abort_flag, H3B_STATUS_GEMM_TIMEOUT) ||
           (asks() && !mbar_wait_warp(&empty[freed.stage], freed.parity, &abort_flag, H3B_STATUS_GEMM_TIMEOUT))))
        break;
      tc_fence_after();
      const uint32_t w = smem0 + at.stage * C::kStageBytes;
      const uint32_t x = ROWS16 ? x0 + (uint32_t)(i * C::kXStep) : w + C::kWBytes + C::kScaleBytes;
      const uint32_t ts = tmem + C::kAccCols + C::kSlotCols * scales.stage;
      uint64_t* there = &scaled[scales.stage];
      if (asks()) freed.next(stages);
      at.next(stages);
      scales.next(C::kSlots);
      ++i;
      seen = peek();
      if (elect_one()) {
        fp4_step_scales<FORMAT, 1, 1>(w + C::kWBytes, x + C::kXBytes, ts, ts + C::kSlotCols / 2);
        mma_commit(there);
      }
      __syncwarp();
    }
    if (elect_one()) mma_commit(&copied);
    __syncwarp();
    mbar_wait_warp(&copied, 0, &late_flag, H3B_STATUS_GEMM_TIMEOUT);
  } else if (warp > 2) {
    const int tid = (int)threadIdx.x - 96;
    chain_wait();
    const int toks = min(TOK, a.M - m0);
    if constexpr (ROWS16) {
      // A warp takes 32 chunks of 16 columns of a row at a time, and keeps them between the passes.
      const uint16_t* x = a.x16 + kb0 * 256;
      const int K = a.K - kb0 * 256, log_segs = a.x16_log_segs, items = a.M << log_segs;
      constexpr int kItems = rows16_items(FORMAT);
      uint4 raw[kItems][2];
#pragma unroll
      for (int j = 0; j < kItems; ++j) {
        const int item = warp - 3 + 4 * j;
        if (item >= items) break;
        const uint16_t* row = x + (int64_t)(item >> log_segs) * a.x16_stride;
        const int c = (item & ((1 << log_segs) - 1)) * 32 + lane;
        if (a.x16_vec) load16_raw<true>(row, c, K, pieces[warp - 3], raw[j][0], raw[j][1]);
        else load16_raw<false>(row, c, K, pieces[warp - 3], raw[j][0], raw[j][1]);
      }
      if constexpr (FORMAT == kNvfp4) {
#pragma unroll
        for (int j = 0; j < kItems; ++j) {
          const int item = warp - 3 + 4 * j;
          if (item >= items) break;
          float2 v[8];
          unpack16<BF16>(raw[j][0], raw[j][1], v);
          uint32_t top = absmax16(v);
          if (top >= kInfBits) top = 0u;
          top = __reduce_max_sync(0xffffffffu, top);
          if (lane == 0) atomicMax(&row_top[item >> log_segs], top);
        }
        if (split > 1) {
          cluster_wait();
          cluster_sync_all();
        } else {
          asm volatile("bar.sync 2, 128;" ::: "memory");
        }
      }
#pragma unroll
      for (int j = 0; j < kItems; ++j) {
        const int item = warp - 3 + 4 * j;
        if (item >= items) break;
        const int r = item >> log_segs, c = (item & ((1 << log_segs) - 1)) * 32 + lane;
        float2 v[8];
        float inv_r = 1.0f;
        unpack16<BF16>(raw[j][0], raw[j][1], v);
        if constexpr (FORMAT == kNvfp4) {
          uint32_t top = 0u;
          if (lane < split)
            asm volatile("ld.shared::cluster.u32 %0, [%1];"
                         : "=r"(top) : "r"(mapa_shared(smem_u32(&row_top[r]), (uint32_t)lane)) : "memory");
          const int e = row_exponent(__reduce_max_sync(0xffffffffu, top));
          inv_r = exp2_bits(-e);
          if (lane == 0) row_scale[r] = exp2_bits(e);
        }
        uint32_t top = absmax16(v), w[2];
        if (FORMAT == kMxfp4) top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        const uint32_t word = ScaleWord<FORMAT>::of(quantize16<FORMAT>(v, top, inv_r, w), lane);
        constexpr int kLanes = ScaleWord<FORMAT>::kLanes;
        if (c < steps * 16) {
          uint8_t* at = x_area + (c >> 4) * C::kXStep;
          // 16-byte pieces of a 128-byte row are swizzled by the row, as a TMA copy would leave them
          *reinterpret_cast<uint2*>(at + r * 128 + (((((c & 15) >> 1) ^ r) & 7) << 4) + (c & 1) * 8) = make_uint2(w[0], w[1]);
          if ((lane & (kLanes - 1)) == 0)
            *reinterpret_cast<uint32_t*>(at + C::kXBytes + (c & 15) / kLanes * 512 + r * 16) = word;
        }
      }
      if (FORMAT == kMxfp4 && tid < 16) row_scale[tid] = 1.0f;
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      mbar_arrive(&x_ready);
    } else {
      for (int i = tid; i < toks; i += 128) row_scale[i] = a.xs ? a.xs[m0 + i] : 1.0f;
    }
    // what the output needs beside the sums is fetched before they are there
    const int quad = warp & 3, row = quad * 32 + lane;
    const int n = split == 1 ? n0 + row : n0 + rank * share + ((2 * tid) & (share - 1));
    const int n1 = min(n + 1, a.N - 1);
    const float ws0 = a.ws && n < a.N ? a.ws[n] : 1.0f, bias0 = a.bias && n < a.N ? a.bias[n] : 0.0f;
    const float ws1 = a.ws && n < a.N ? a.ws[n1] : 1.0f, bias1 = a.bias && n < a.N ? a.bias[n1] : 0.0f;
    asm volatile("bar.sync 2, 128;" ::: "memory");  // row_scale
    // Whether some row's and some column's scale of this warp lie on different sides of 1: found here, while the
    // products run, since the order for it takes each sum longer (333 rows, 4,096 -> 4,096: mxfp4 12.4 us with it
    // for all sums, so 11.7, nvfp4 14.6 and 14.0).
    bool apart = a.ws && (ROWS16 ? FORMAT == kNvfp4 : a.xs != nullptr);
    if (apart) {
      const bool below0 = fabsf(ws0) < 1.0f, below1 = fabsf(ws1) < 1.0f;
      bool low = n < a.N && (below0 || below1), high = n < a.N && !(below0 && below1);
      for (int i = lane; i < toks; i += 32) {
        const bool below = fabsf(row_scale[i]) < 1.0f;
        low = low || below;
        high = high || !below;
      }
      apart = __any_sync(0xffffffffu, low) && __any_sync(0xffffffffu, high);
    }
    if (split > 1 && !(ROWS16 && FORMAT == kNvfp4)) cluster_wait();
    const bool summed = mbar_wait_warp(&done, 0, &abort_flag, H3B_STATUS_GEMM_TIMEOUT);
    tc_fence_after();
    const uint32_t taddr = tmem + ((uint32_t)(quad * 32) << 16);
    if (split == 1) {
      auto write = [&](auto order) {
#pragma unroll 1
        for (int c = 0; summed && c < toks; c += 16) {
          uint32_t r[16];
          tmem_ld16(taddr + (uint32_t)c, r);
          tmem_wait_ld();
          reg_barrier16(r);
          if (n < a.N) {
            uint16_t* dst = a.out + (int64_t)(m0 + c) * a.out_stride + n;
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              if (c + j >= toks) break;
              dst[j * a.out_stride] = f32_to_half_bits<BF16>(
                  fp4_finish<decltype(order)::value>(__uint_as_float(r[j]), row_scale[c + j], ws0, bias0, a));
            }
          }
          __syncwarp();
        }
      };
      if (__builtin_expect(!apart, 1)) write(std::false_type{});
      else write(std::true_type{});
    } else {
      const uint32_t owner = (uint32_t)(row >> log_share);
      const uint32_t to = mapa_shared(smem_u32(sums + ((rank * TOK) << log_share) + (row & (share - 1))), owner);
#pragma unroll 1
      for (int c = 0; summed && c < toks; c += 16) {
        uint32_t r[16];
        tmem_ld16(taddr + (uint32_t)c, r);
        tmem_wait_ld();
        reg_barrier16(r);
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (c + j < toks)
            asm volatile("st.shared::cluster.b32 [%0], %1;"
                         ::"r"(to + (uint32_t)(((c + j) << log_share) * 4)), "r"(r[j]) : "memory");
      }
      __syncwarp();
      if (summed && (row & (min(32, share) - 1)) == 0)
        asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];"
                     ::"r"(mapa_shared(smem_u32(&sent), owner)) : "memory");
      // also where this CTA has given up: the others' sums must find it here
      const bool got = mbar_wait_sent(&sent, &abort_flag);
      const float* mine = sums + ((2 * tid) & (share - 1));
      const int log_pairs = log_share - 1;
      auto add_up = [&](auto order) {
        for (int tok = tid >> log_pairs; got && tok < toks; tok += 128 >> log_pairs) {
          float2 p[8];
#pragma unroll
          for (int r = 0; r < 8; ++r)
            if (r < split) p[r] = *reinterpret_cast<const float2*>(mine + ((r * TOK + tok) << log_share));
          float y0 = 0.f, y1 = 0.f;
#pragma unroll
          for (int r = 0; r < 8; ++r)
            if (r < split) {
              y0 = __fadd_rn(y0, p[r].x);
              y1 = __fadd_rn(y1, p[r].y);
            }
          if (n >= a.N) continue;
          const uint16_t h0 = f32_to_half_bits<BF16>(fp4_finish<decltype(order)::value>(y0, row_scale[tok], ws0, bias0, a));
          const uint16_t h1 = f32_to_half_bits<BF16>(fp4_finish<decltype(order)::value>(y1, row_scale[tok], ws1, bias1, a));
          uint16_t* dst = a.out + (int64_t)(m0 + tok) * a.out_stride + n;
          if (n1 > n && (reinterpret_cast<uintptr_t>(dst) & 3) == 0) {
            *reinterpret_cast<uint32_t*>(dst) = (uint32_t)h0 | ((uint32_t)h1 << 16);
          } else {
            dst[0] = h0;
            if (n1 > n) dst[1] = h1;
          }
        }
      };
      if (__builtin_expect(!apart, 1)) add_up(std::false_type{});
      else add_up(std::true_type{});
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, C::kTmemCols);
  }
  __syncwarp();
  // A CTA that gave up leaves last: the others' sums may still be on their way into its shared memory.
  // Those that have all sums leave at once, and the barrier counts them.
  if (split > 1 && abort_flag) {
    cluster_arrive();
    cluster_wait();
  }
}

// ------------------------------------------------------------------ many rows: 256 x 256 tiles on two SMs
// A cluster of two CTAs computes 256 x 256 tiles (rows of x are the products' M): each CTA
// loads 128 rows of x and 128 of the weight, and the even CTA's products read both.  Its
// tensor memory holds 256 accumulator columns twice, overlapping ([0, 256) and [kSecond,
// kSecond + 256)), and behind them slots of scales.  The epilogue of a tile first takes what
// lies in the overlap into registers and lets the next tile's products begin; its output
// goes through shared memory in pieces of 32 rows x 64 columns, by TMA (16-byte stores of a
// thread per row took the same shared-memory cycles that the products read with: 8,192 x
// 12,288 x 4,096 180 us).
//   warp 0: TMA, warp 1: tensor memory and (even CTA) scale copies and products (a warp of its own
//   for the copies made it slower: they wait in the tensor pipe behind the products issued before
//   them, and what follows would wait for their barrier), warps 4-11: epilogue, two per lane quadrant
template <int FORMAT>
struct PairFp4Cfg {
  static constexpr int kScaleBytes = FORMAT == kMxfp4 ? 1024 : 2048;  // of a band and step
  static constexpr int kStageBytes = 2 * 128 * kF4Step + 3 * kScaleBytes;
  static constexpr int kStages = 5;
  static constexpr int kOutBytes = 8 * 4096;
  static constexpr int kTotal = kStages * kStageBytes + kOutBytes + 1024;
  static_assert(kStageBytes % 1024 == 0, "swizzled tiles start at multiples of 1024");
  // Scale copies run ahead of the products by kSlots - 1 steps at most.  With 2 slots the copy
  // for a step starts when the products of the step before it do and comes too late (9,472 x
  // 2,048 x 16,384 mxfp4: 124 us, with 3 104 us, with 4 the same).
  static constexpr int kSlots = 3;
  static constexpr int kSlotCols = 3 * kScaleBytes / 128;  // 24 or 48 columns
  static constexpr int kSecond = FORMAT == kMxfp4 ? 160 : 96;
  static constexpr int kScales = kSecond + 256;
  static_assert(kScales + kSlots * kSlotCols <= 512, "");
};
constexpr int kPairFp4Threads = 384;

// 32 columns of a row's sums to 16 bits, two to a word; columns: their scales and biases, four of
// each in turn, in shared memory, or null where there are none.  BOTH: there are row scales on both
// sides (nvfp4; mxfp4 rows of a caller's), and with `apart` some row's of this warp may lie on the other
// side of 1 than some column's (fp4_scaled); else the two follow each other.
template <bool BOTH, bool BF16>
__device__ __forceinline__ void fp4_pack_chunk(const uint32_t (&r)[32], uint32_t (&h)[16], float xs,
                                               const float4* columns, bool apart) {
  const float2 x2 = splat2(xs);
  if (BOTH && __builtin_expect(apart, 0)) {
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const float4 w = columns[2 * q], b = columns[2 * q + 1];
      float z[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) z[j] = fp4_scaled(__uint_as_float(r[4 * q + j]), xs, (&w.x)[j]);
      h[2 * q] = pack_halves<BF16>(__fadd_rn(z[0], b.x), __fadd_rn(z[1], b.y));
      h[2 * q + 1] = pack_halves<BF16>(__fadd_rn(z[2], b.z), __fadd_rn(z[3], b.w));
    }
  } else if (columns) {
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const float4 w = columns[2 * q], b = columns[2 * q + 1];
      const float2 y0 = mul2(make_float2(__uint_as_float(r[4 * q]), __uint_as_float(r[4 * q + 1])), x2);
      const float2 y1 = mul2(make_float2(__uint_as_float(r[4 * q + 2]), __uint_as_float(r[4 * q + 3])), x2);
      const float2 z0 = add2(mul2(y0, make_float2(w.x, w.y)), make_float2(b.x, b.y));
      const float2 z1 = add2(mul2(y1, make_float2(w.z, w.w)), make_float2(b.z, b.w));
      h[2 * q] = pack_halves<BF16>(z0.x, z0.y);
      h[2 * q + 1] = pack_halves<BF16>(z1.x, z1.y);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const float2 y = mul2(make_float2(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1])), x2);
      h[j] = pack_halves<BF16>(y.x, y.y);
    }
  }
}
// A warp's 32 x 64 piece of the output through its 4 KB of shared memory (rows of 128 bytes,
// 16-byte pieces swizzled by the row, as TMA reads them): this lane's row is m = m0 + lane, its
// columns from n0 on are lo and hi.
__device__ __forceinline__ void fp4_put_piece(const CUtensorMap* tm_out, uint8_t* buf, const uint32_t (&lo)[16],
                                              const uint32_t (&hi)[16], int m0, int n0, const Fp4GemmArgs& a) {
  const int lane = threadIdx.x & 31;
  if (a.out_tma) {  // the piece before has been read
    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
  }
  __syncwarp();
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    *reinterpret_cast<uint4*>(buf + lane * 128 + ((q ^ (lane & 7)) << 4)) =
        make_uint4(lo[4 * q], lo[4 * q + 1], lo[4 * q + 2], lo[4 * q + 3]);
    *reinterpret_cast<uint4*>(buf + lane * 128 + (((q + 4) ^ (lane & 7)) << 4)) =
        make_uint4(hi[4 * q], hi[4 * q + 1], hi[4 * q + 2], hi[4 * q + 3]);
  }
  if (a.out_tma) {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0 && m0 < a.M && n0 < a.N) {  // rows and columns beyond are not written
      asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];"
                   ::"l"(reinterpret_cast<uint64_t>(tm_out)), "r"(smem_u32(buf)), "r"(n0), "r"(m0) : "memory");
      asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    }
  } else {
    // Rows that TMA does not take: each by the whole warp, a lane for two columns.  Where a row starts
    // between words a lane stores its second column with the next lane's first, and the first and the
    // last column of the 64 go alone; without branches, which cost more than the stores (11,203 rows,
    // 896 -> 2,487 94 us with them).
    __syncwarp();
    const int n = n0 + 2 * lane, rows = min(32, a.M - m0);
    uint16_t* dst = a.out + (int64_t)m0 * a.out_stride + n;
    const bool between = (reinterpret_cast<uintptr_t>(dst) & 2) != 0, turns = (a.out_stride & 1) != 0;
    if (n0 + 64 <= a.N) {
#pragma unroll 1
      for (int r0 = 0; r0 < rows; r0 += 8) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t w =
              *reinterpret_cast<const uint32_t*>(buf + (r0 + i) * 128 + (((lane >> 2) ^ i) << 4) + (lane & 3) * 4);
          const bool off = between ^ (turns && (i & 1));
          const uint32_t next = __shfl_down_sync(0xffffffffu, w, 1);
          const bool there = r0 + i < rows;
          uint16_t* to = dst + (int64_t)(r0 + i) * a.out_stride;
          if (there && (!off || lane < 31)) *reinterpret_cast<uint32_t*>(to + off) = off ? __byte_perm(w, next, 0x5432) : w;
          if (there && off && (lane == 0 || lane == 31)) to[lane & 1] = (uint16_t)(lane ? w >> 16 : w);
        }
      }
    } else {
      for (int r = 0; r < rows; ++r, dst += a.out_stride) {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(buf + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4);
        if (n < a.N) dst[0] = (uint16_t)(w & 0xffffu);
        if (n + 1 < a.N) dst[1] = (uint16_t)(w >> 16);
      }
    }
    __syncwarp();
  }
}

// Tile t of a product: `group` tiles of columns at a time, and for them all tiles of rows
struct TilePlace {
  int m, n;
};
__device__ __forceinline__ TilePlace tile_place(int t, int num_m, int num_n, int group) {
  const int g = t / (group * num_m), in = t - g * group * num_m, width = min(group, num_n - group * g);
  return {in / width, group * g + in % width};
}

template <int FORMAT, bool BOTH, bool BF16>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairFp4Threads, 1)
    fp4_pair_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                    const __grid_constant__ CUtensorMap tm_sx, const __grid_constant__ CUtensorMap tm_sw,
                    const __grid_constant__ CUtensorMap tm_out, Fp4GemmArgs a) {
  using C = PairFp4Cfg<FORMAT>;
  constexpr uint32_t kStages = C::kStages;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t full[kStages], empty[kStages], tfull, tempty, drained;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_flag, late_flag;
  __shared__ __align__(16) float columns[128][4];  // of 256 columns: four scales, their four biases, and so on

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int num_m = (a.M + 255) / 256, num_n = (a.N + 255) / 256;
  const int tiles = num_m * num_n;
  const int num_k = (a.K + 255) / 256;

  if (threadIdx.x == 0) {
    for (uint32_t s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 2);
      mbar_init(&empty[s], 1);
    }
    mbar_init(&tfull, 1);
    mbar_init(&tempty, 16);  // the epilogue warps of both CTAs
    mbar_init(&drained, 1);
    abort_flag = late_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(&tmem_slot, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync_all();  // both CTAs' barriers are initialised; all 512 columns were taken, so both bases are 0
  tc_fence_after();
  // The kernel after this one is not let in early: where its blocks came onto SMs whose pair was done
  // first, a norm and its product took 197 us instead of 187 (8,192 rows, 4,096 -> 12,288, mxfp4).
  chain_wait();
  const uint32_t tmem = tmem_slot;
  const uint32_t full0 = mapa_shared(smem_u32(full), 0);
  const uint32_t tempty0 = mapa_shared(smem_u32(&tempty), 0);

  if (warp == 0) {
    RingPlace fill;
    bool ok = true;
    for (int t = pair; ok && t < tiles; t += pairs) {
      const auto [mb, nb] = tile_place(t, num_m, num_n, a.group);
      for (int kb = 0; kb < num_k; ++kb) {
        if (!mbar_wait_warp(&empty[fill.stage], fill.parity ^ 1, &abort_flag, H3B_STATUS_GEMM_TIMEOUT)) { ok = false; break; }
        if (elect_one()) {
          uint8_t* at = smem + fill.stage * C::kStageBytes;
          const uint32_t fb = full0 + fill.stage * 8;
          mbar_arrive_expect_tx_cluster(fb, C::kStageBytes);
          tma_load_2d_pair(at, &tm_x, fb, kb * kF4Step, mb * 256 + (int)rank * 128);
          tma_load_2d_pair(at + 128 * kF4Step, &tm_w, fb, kb * kF4Step, nb * 256 + (int)rank * 128);
          at += 2 * 128 * kF4Step;
          tma_load_2d_pair(at, &tm_sx, fb, kb * (C::kScaleBytes / 8), mb * 2 + (int)rank);
          // the scales of all 256 rows of the weight: each CTA's tensor memory holds them
          tma_load_2d_pair(at + C::kScaleBytes, &tm_sw, fb, kb * (C::kScaleBytes / 8), nb * 2);
        }
        __syncwarp();
        fill.next(kStages);
      }
    }
    // Copies have landed before the CTAs leave.  Both CTAs' are counted by the even CTA's barriers, up to its
    // own last fill, and the odd CTA's by their use, of which its barriers are told: the even one may have
    // given up before them.  Of each slot the last fill: slots before the next one in this round, the others before.
    uint64_t* landed = rank == 0 ? full : empty;
    for (uint32_t s = 0; s < kStages; ++s)
      mbar_wait_warp(&landed[s], s < fill.stage ? fill.parity : fill.parity ^ 1u, &late_flag, H3B_STATUS_GEMM_TIMEOUT);
  } else if (warp == 1) {
    if (rank == 0) {
      const uint32_t smem0 = smem_u32(smem);
      RingPlace at, freed, scales;
      uint32_t it = 0, tile = 0;  // K steps so far (up to the slots' number), tiles so far
      bool ok = true;
      // a step's operands are there, and the products kSlots steps before have read its slot of scales
      auto peek = [&]() {
        const bool slot = lane == 1 && it == C::kSlots;
        return mbar_peek(slot ? &empty[freed.stage] : &full[at.stage], slot ? freed.parity : at.parity);
      };
      bool seen = peek();
      for (int t = pair; ok && t < tiles; t += pairs, ++tile) {
        if (tile > 0 && !mbar_wait_warp(&tempty, (tile - 1) & 1, &abort_flag, H3B_STATUS_GEMM_TIMEOUT)) break;
        const uint32_t d = tmem + (tile & 1 ? (uint32_t)C::kSecond : 0u);
        int products = (a.K + 63) / 64;
        for (int kb = 0; kb < num_k; ++kb, products -= 4) {
          if (!__all_sync(0xffffffffu, seen) &&
              (!mbar_wait_warp(&full[at.stage], at.parity, &abort_flag, H3B_STATUS_GEMM_TIMEOUT) ||
               (it == C::kSlots && !mbar_wait_warp(&empty[freed.stage], freed.parity, &abort_flag, H3B_STATUS_GEMM_TIMEOUT)))) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t x = smem0 + at.stage * C::kStageBytes;
          const uint32_t sx = x + 2 * 128 * kF4Step;
          const uint32_t ts = tmem + C::kScales + C::kSlotCols * scales.stage;
          uint64_t* used = &empty[at.stage];
          if (it == C::kSlots) freed.next(kStages);
          else ++it;
          at.next(kStages);
          scales.next(C::kSlots);
          seen = peek();
          if (elect_one()) {
            fp4_step_scales<FORMAT, 2, 2>(sx, sx + C::kScaleBytes, ts, ts + C::kSlotCols / 3);
            fp4_step_products<FORMAT, 2, 256, 256, 2>(d, x, x + 128 * kF4Step, ts, ts + C::kSlotCols / 3, products, kb == 0);
            mma_commit_pair(used, 0x3);
          }
          __syncwarp();
        }
        if (ok && elect_one()) mma_commit_pair(&tfull, 0x3);
        __syncwarp();
      }
      if (elect_one()) mma_commit_pair(&drained, 0x1);
      __syncwarp();
      mbar_wait_warp(&drained, 0, &late_flag, H3B_STATUS_GEMM_TIMEOUT);
    }
  } else if (warp >= 4) {
    const int quad = warp & 3, half = (warp - 4) >> 2;
    uint8_t* buf = smem + kStages * C::kStageBytes + (warp - 4) * 4096;
    const float4* cols = a.ws || a.bias ? reinterpret_cast<const float4*>(columns) : nullptr;
    uint32_t tile = 0;
    bool live = true;
    for (int t = pair; t < tiles; t += pairs, ++tile) {
      const auto [mb, nb] = tile_place(t, num_m, num_n, a.group);
      const int m_warp = mb * 256 + (int)rank * 128 + quad * 32, m = m_warp + lane;
      const float xs = a.xs && m < a.M ? a.xs[m] : 1.0f;
      bool apart = false;
      if (a.ws || a.bias) {  // the tile's columns' scales and bias, while its products run
        const int i = (int)threadIdx.x - 128, n = nb * 256 + i;
        // where there are none, 1 and -0, which change no sum
        const float w = a.ws && n < a.N ? a.ws[n] : 1.0f, b = a.bias && n < a.N ? a.bias[n] : -0.0f;
        asm volatile("bar.sync 1, 256;" ::: "memory");  // all warps are done with the last tile's
        columns[i >> 2 << 1][i & 3] = w;
        columns[(i >> 2 << 1) + 1][i & 3] = b;
        if constexpr (BOTH) {
          // How many of the columns' scales are below 1: where none or all are, and this warp's rows' likewise, they
          // need no order.  (One code for all cases took 3,600 rows, 4,096 -> 16,384 nvfp4 126.3 us, so 123.7,
          // and 122.5 to 124.5 with no order at all.)
          uint32_t below;
          asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.popc.u32 %0, 1, 256, p;\n\t}"
                       : "=r"(below) : "r"(n < a.N && fabsf(w) < 1.0f ? 1u : 0u) : "memory");
          const bool row_below = fabsf(xs) < 1.0f;
          const bool alike = m >= a.M || (row_below ? below == (uint32_t)min(256, a.N - nb * 256) : below == 0u);
          apart = !__all_sync(0xffffffffu, alike);
        } else {
          asm volatile("bar.sync 1, 256;" ::: "memory");
        }
      }
      // a warp that has given up goes on through the tiles, since the others meet it at the barriers above
      live = live && mbar_wait_warp(&tfull, tile & 1, &abort_flag, H3B_STATUS_GEMM_TIMEOUT);
      if (!live) continue;
      tc_fence_after();
      const bool odd = tile & 1;
      const uint32_t taddr = tmem + ((uint32_t)(quad * 32) << 16) + (odd ? (uint32_t)C::kSecond : 0u);
      // This warp's two 64-column pieces.  The overlap is the end of the even tiles and the start
      // of the odd ones, 96 (mxfp4) or 160 columns: the first pieces of the two warps of a lane
      // quadrant cover 128 of them, and for nvfp4 `half` 1 takes 32 columns of its second one along.
      const int first = odd ? half : 3 - half, second = odd ? (half ? 2 : 3) : half;
      const int n0 = nb * 256;
      uint32_t r0[32], r1[32], r2[32], h0[16], h1[16];
      const int early = odd ? 2 * second : 2 * second + 1, late = odd ? 2 * second + 1 : 2 * second;  // chunks of 32
      tmem_ld32(taddr + 64u * (uint32_t)first, r0);
      tmem_ld32(taddr + 64u * (uint32_t)first + 32u, r1);
      if (FORMAT == kNvfp4) tmem_ld32(taddr + 32u * (uint32_t)early, r2);
      tmem_wait_ld_dep(r0);
      reg_barrier32(r1);
      if (FORMAT == kNvfp4) reg_barrier32(r2);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(tempty0);
      fp4_pack_chunk<BOTH, BF16>(r0, h0, xs, cols ? cols + (64 * first) / 2 : nullptr, apart);
      fp4_pack_chunk<BOTH, BF16>(r1, h1, xs, cols ? cols + (64 * first + 32) / 2 : nullptr, apart);
      fp4_put_piece(&tm_out, buf, h0, h1, m_warp, n0 + 64 * first, a);
      if (FORMAT != kNvfp4) tmem_ld32(taddr + 32u * (uint32_t)early, r2);
      tmem_ld32(taddr + 32u * (uint32_t)late, r0);
      tmem_wait_ld_dep(r0);
      reg_barrier32(r2);
      fp4_pack_chunk<BOTH, BF16>(r2, h0, xs, cols ? cols + (32 * early) / 2 : nullptr, apart);
      fp4_pack_chunk<BOTH, BF16>(r0, h1, xs, cols ? cols + (32 * late) / 2 : nullptr, apart);
      if (odd) fp4_put_piece(&tm_out, buf, h0, h1, m_warp, n0 + 64 * second, a);
      else fp4_put_piece(&tm_out, buf, h1, h0, m_warp, n0 + 64 * second, a);
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");  // written before the block leaves
    __syncwarp();
  }

  tc_fence_before();
  cluster_sync_all();  // the pair's products, copies and epilogues are done
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

// ------------------------------------------------------------------ host side

// Launch in a cluster of `ctas` (0: as the kernel declares), starting while the kernel before ends; with
// `smem` bytes of shared memory, kMost in the kernel's largest call
template <auto Kernel, int kMost, typename... A>
static cudaError_t launch_fp4(int64_t grid, int64_t grid_y, int ctas, int threads, size_t smem, cudaStream_t s,
                              const A&... args) {
  cudaError_t e = allow_shared_memory<Kernel, kMost>();
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)ctas;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)grid, (unsigned)grid_y);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = ctas ? 2 : 1;
  e = cudaLaunchKernelEx(&cfg, Kernel, args...);
  if (e == cudaSuccess) chained_launches.fetch_add(1, std::memory_order_relaxed);
  return e;
}

// Codes as [rows, pitch] bytes in boxes of box_rows x 128, swizzled; scales as [bands, groups x 512]
// bytes in boxes of box_bands x one step.  What lies outside reads as zero codes and scales.
static bool make_fp4_maps(const Fp4RowsView& v, int format, int box_rows, int box_bands, CUtensorMap* codes,
                          CUtensorMap* scales) {
  const uint64_t pitch = (uint64_t)fp4_pitch(v.K), words = (uint64_t)fp4_groups(v.K, format) * 64;
  return make_tmap_2d(codes, v.codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, pitch, (uint64_t)v.rows, pitch, kF4Step,
                      (uint32_t)box_rows, CU_TENSOR_MAP_SWIZZLE_128B) &&
         make_tmap_2d(scales, v.blocks, CU_TENSOR_MAP_DATA_TYPE_FLOAT64, 8, words, (uint64_t)(v.rows + 127) / 128,
                      words * 8, format == kMxfp4 ? 128 : 256, (uint32_t)box_bands, CU_TENSOR_MAP_SWIZZLE_NONE);
}

// How a product of few rows is divided: rows of x per tile and CTAs along K
struct SplitPlan {
  int tok, log_split;
};
static SplitPlan plan_split(int M, int N, int K) {
  const int num_k = (K + 255) / 256, sms = num_sms();
  const int64_t tiles_n = (N + 127) / 128;
  // tiles of 64 rows as long as most of them run at once (128 rows, 4,096 -> 4,096: 8.0 us, with
  // tiles of 128 10.2; 1,024 rows: 23 and 17 us)
  const int tok = M <= 16 ? 16 : 2 * tiles_n * ((M + 63) / 64) <= 3 * sms ? 64 : 128;
  const int64_t tiles = tiles_n * ((M + tok - 1) / tok);
  // K steps that the busiest SM takes, and what adding up costs in steps (48 rows, 16,384 -> 4,096:
  // one part 20.5 us, four 12.8; 128 rows, 4,096 -> 4,096: one part 8.0 us, two 10.7)
  const int joining = tok == 16 ? 2 : tok == 64 ? 12 : 24;
  SplitPlan best{tok, 0};
  int64_t least = INT64_MAX;
  for (int l = 0; l <= 3 && 1 << l <= num_k; ++l) {
    if (l && tiles << l > 2 * sms) break;  // more than run at once
    const int64_t cost = ((tiles << l) + sms - 1) / sms * ((num_k + (1 << l) - 1) >> l) + (l ? joining : 0);
    if (cost < least) {
      least = cost;
      best.log_split = l;
    }
  }
  return best;
}
template <int FORMAT, int TOK, bool ROWS16>
static int launch_split(const Fp4RowsView& x, const Fp4RowsView& w, const Fp4GemmArgs& a, int log_split, cudaStream_t s,
                        cudaError_t* err) {
  using C = SplitCfg<FORMAT, TOK, ROWS16>;
  CUtensorMap tx, tw, tsx, tsw;
  if (!make_fp4_maps(w, FORMAT, 128, 1, &tw, &tsw)) return 1;
  if (ROWS16) tx = tw, tsx = tsw;  // not used
  else if (!make_fp4_maps(x, FORMAT, TOK, 1, &tx, &tsx)) return 1;
  const int split = 1 << log_split;
  const int64_t grid = (int64_t)((a.N + 127) / 128) * split, grid_y = (a.M + TOK - 1) / TOK;
  const int steps = ((a.K + 255) / 256 + split - 1) / split, rest = C::rest_bytes(steps, split);
  // As many stages as one CTA per SM has room for, or two where there are more CTAs than SMs.  Never
  // so little shared memory that three fit: tensor memory is for two, and a third one that waited for
  // it could keep the clusters of the other two, or the kernel before, waiting.
  const int room = grid * grid_y > num_sms() ? 106 * 1024 : kSplitMost;
  static_assert(C::rest_bytes(kRows16Steps, 8) + 2 * C::kStageBytes <= kSplitMost, "two stages always fit");
  int stages = (room - rest) / C::kStageBytes;
  stages = stages < 2 ? 2 : stages > kSplitMaxStages ? kSplitMaxStages : stages;
  if (stages > steps) stages = steps;
  int smem = stages * C::kStageBytes + rest;
  if (smem < 80 * 1024) smem = 80 * 1024;
  auto launch = [&](auto bf16) {
    return launch_fp4<fp4_split_kernel<FORMAT, TOK, ROWS16, decltype(bf16)::value>, kSplitMost>(
        grid, grid_y, split, kSplitThreads, (size_t)smem, s, tw, tsw, tx, tsx, a, log_split, stages);
  };
  *err = a.bf16 ? launch(std::true_type{}) : launch(std::false_type{});
  return *err == cudaSuccess ? 0 : 2;
}
template <int FORMAT>
static int launch_pair(const Fp4RowsView& x, const Fp4RowsView& w, const Fp4GemmArgs& a, cudaStream_t s,
                       cudaError_t* err) {
  CUtensorMap tx, tw, tsx, tsw;
  if (!make_fp4_maps(x, FORMAT, 128, 1, &tx, &tsx) || !make_fp4_maps(w, FORMAT, 128, 2, &tw, &tsw)) return 1;
  // output rows that TMA takes: 16-byte aligned, and so are the steps between them
  CUtensorMap to = tx;
  Fp4GemmArgs b = a;
  b.out_tma = a.out_stride % 8 == 0 && reinterpret_cast<uintptr_t>(a.out) % 16 == 0;
  if (b.out_tma && !make_tmap_2d(&to, a.out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, (uint64_t)a.N, (uint64_t)a.M,
                                 (uint64_t)a.out_stride * 2, 64, 32, CU_TENSOR_MAP_SWIZZLE_128B))
    return 1;
  // Eight tiles of columns at a time, so that the weight is read once and x again for each eight; all of
  // them where x is the longer operand and the weight stays in L2 (4,096 x 16,384 x 16,384 nvfp4 396 us,
  // with all columns 490; 16,384 x 4,096 x 16,384 mxfp4 368 and 359).
  const int64_t num_n = (a.N + 255) / 256, tiles = (int64_t)((a.M + 255) / 256) * num_n;
  b.group = a.M >= a.N && (int64_t)a.N * fp4_pitch(a.K) <= 48 << 20 ? (int)num_n : 8;
  const int64_t pairs = tiles < num_sms() / 2 ? tiles : num_sms() / 2;
  constexpr int kTotal = PairFp4Cfg<FORMAT>::kTotal;
  auto launch = [&](auto both, auto bf16) {
    return launch_fp4<fp4_pair_kernel<FORMAT, decltype(both)::value, decltype(bf16)::value>, kTotal>(
        2 * pairs, 1, 0, kPairFp4Threads, kTotal, s, tx, tw, tsx, tsw, to, b);
  };
  auto launch_as = [&](auto both) { return a.bf16 ? launch(both, std::true_type{}) : launch(both, std::false_type{}); };
  // The order of two scales in an instance of its own (9,472 x 2,048 x 4,096 mxfp4, where there are none, with a cold
  // instruction cache: 34.6 us, with the code for both 36.9)
  *err = a.xs && a.ws ? launch_as(std::true_type{}) : launch_as(std::false_type{});
  return *err == cudaSuccess ? 0 : 2;
}
static bool uses_pair(int M, int N) {
  // from about half as many tiles as there are pairs of SMs on (1,024 rows, 4,096 -> 4,096, 64 tiles:
  // 15.8 us and 17.4 by the other kernel; 333 rows, 32 tiles: 11.1 and 10.3)
  return M > 128 && (int64_t)((M + 255) / 256) * ((N + 255) / 256) > num_sms() / 4;
}
template <int FORMAT>
static int launch_gemm_of(const Fp4RowsView& x, const Fp4RowsView& w, const Fp4GemmArgs& a, cudaStream_t s,
                          cudaError_t* err) {
  if (uses_pair(a.M, a.N)) return launch_pair<FORMAT>(x, w, a, s, err);
  const SplitPlan p = plan_split(a.M, a.N, a.K);
  return p.tok == 16   ? launch_split<FORMAT, 16, false>(x, w, a, p.log_split, s, err)
         : p.tok == 64 ? launch_split<FORMAT, 64, false>(x, w, a, p.log_split, s, err)
                       : launch_split<FORMAT, 128, false>(x, w, a, p.log_split, s, err);
}

int launch_fp4_gemm(const Fp4RowsView& x, const Fp4RowsView& w, Fp4GemmArgs a, int format, cudaStream_t s,
                    cudaError_t* err) {
  a.xs = x.row_scales;
  a.ws = w.row_scales;
  return format == kMxfp4 ? launch_gemm_of<kMxfp4>(x, w, a, s, err) : launch_gemm_of<kNvfp4>(x, w, a, s, err);
}

// K steps of a CTA, and the pieces of 512 columns that they make of a row, as a power of two
static int64_t rows16_steps(int64_t K, int log_split) { return ((K + 255) / 256 + (1 << log_split) - 1) >> log_split; }
static int rows16_log_segs(int64_t steps) { return steps <= 2 ? 0 : steps <= 4 ? 1 : steps <= 8 ? 2 : 3; }
bool fp4_takes_rows16(int64_t M, int64_t N, int64_t K, int format) {
  if (M > 16 || uses_pair((int)M, (int)N)) return false;
  const SplitPlan p = plan_split((int)M, (int)N, (int)K);
  const int64_t steps = rows16_steps(K, p.log_split);
  return p.tok == 16 && steps <= kRows16Steps && M << rows16_log_segs(steps) <= 4 * rows16_items(format);
}
int launch_fp4_gemm_rows16(const uint16_t* x, int64_t x_stride, const Fp4RowsView& w, Fp4GemmArgs a, int format,
                           cudaStream_t s, cudaError_t* err) {
  a.ws = w.row_scales;
  a.x16 = x;
  a.x16_stride = x_stride;
  a.x16_vec = a.K % 16 == 0 && rows16(x, a.M > 1 ? x_stride : 0);
  const int log_split = plan_split(a.M, a.N, a.K).log_split;
  a.x16_log_segs = rows16_log_segs(rows16_steps(a.K, log_split));
  return format == kMxfp4 ? launch_split<kMxfp4, 16, true>({}, w, a, log_split, s, err)
                          : launch_split<kNvfp4, 16, true>({}, w, a, log_split, s, err);
}

}  // namespace h3b
