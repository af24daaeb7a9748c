// fp4_gemm.cu -- products of microscaled 4-bit rows on the sm_100 tensor cores
// (tcgen05.mma kind::mxf4 / kind::mxf4nvf4 with block scales in tensor memory, fp32 sums):
//   out[m, n] = (sum over k of x[m, k] w[n, k]) * xs[m] * ws[n] + bias[n]
// where x and w stand for code * block scale and xs, ws for the rows' scales.
//
// A K step is 256 columns: 128 bytes of codes per row (one 128-byte swizzle row, four
// products of 64 columns) and, per 128 rows, four (nvfp4) or two (mxfp4) 512-byte tiles of
// block scales.  Codes and scales come by TMA into a ring of stages; the scales go on into
// tensor memory by tcgen05.cp, into one of two slots: the copy into a slot waits for the
// products of the step before last, which read it.
#include "fp4.cuh"
#include "h3b_kernels.cuh"

namespace h3b {

constexpr int kF4Step = 128;  // bytes of codes per row and K step

// Shared-memory matrix descriptor without swizzle for a tile of block scales: 32 rows of 16
// bytes, 8-row pieces of 128 bytes one after the other (SBO).
__device__ __forceinline__ uint64_t sdesc_scales(uint32_t smem_addr) {
  uint64_t d = 0;
  d |= (uint64_t)((smem_addr & 0x3FFFF) >> 4);
  d |= (uint64_t)1 << 16;
  d |= (uint64_t)(128 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  return d;
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

// A sum to its output value; xs and ws are 1 where there are no row scales
__device__ __forceinline__ float fp4_finish(float sum, float xs, float ws, float bias, const Fp4GemmArgs& a) {
  const float v = __fmul_rn(__fmul_rn(sum, xs), ws);
  return a.bias ? __fadd_rn(v, bias) : v;
}

// One thread: the scale copies and products of one K step into accumulator d.  BANDS: 128-row
// bands of scales of the B operand, whose first row's scales lie in column column_b of theirs.
template <int FORMAT, int CTAS, int M, int N, int BANDS>
__device__ __forceinline__ void fp4_step(uint32_t d, uint32_t smem_a, uint32_t smem_b, uint32_t smem_sa,
                                         uint32_t smem_sb, uint32_t tmem_sa, uint32_t tmem_sb, uint32_t column_b,
                                         int products, bool first) {
  constexpr int kTiles = FORMAT == kMxfp4 ? 2 : 4;  // scale tiles per band and step
#pragma unroll
  for (int g = 0; g < kTiles; ++g) {
    copy_scales<CTAS>(tmem_sa + (uint32_t)(4 * g), sdesc_scales(smem_sa + (uint32_t)(512 * g)));
#pragma unroll
    for (int b = 0; b < BANDS; ++b)
      copy_scales<CTAS>(tmem_sb + (uint32_t)(4 * (BANDS * g + b)),
                        sdesc_scales(smem_sb + (uint32_t)(512 * (kTiles * b + g))));
  }
  const uint64_t da = sdesc_kmajor_sw128(smem_a), db = sdesc_kmajor_sw128(smem_b);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (k >= products) break;
    const uint32_t byte = FORMAT == kMxfp4 ? 2u * (uint32_t)(k & 1) : 0u;
    const uint32_t g = FORMAT == kMxfp4 ? (uint32_t)(k >> 1) : (uint32_t)k;
    mma_fp4<FORMAT, CTAS>(d, da + (uint64_t)(2 * k), db + (uint64_t)(2 * k), idesc_fp4(M, N, FORMAT == kMxfp4, byte),
                          tmem_sa + 4u * g, tmem_sb + 4u * BANDS * g + column_b, first && k == 0 ? 0u : 1u);
  }
}

// ------------------------------------------------------------------ few rows: a split over K
// A tile is 128 rows of the weight (the products' M) x TOK rows of x (their N), so that one
// token costs the reading of the weight and hardly more.  The CTAs of a cluster take equal parts
// of K; each puts its sums into its shared memory, and every CTA adds up and writes out a part
// of the tile's tokens, from all CTAs in their order (the same sums every time).  Without a
// split the sums go out as they come from tensor memory.  Two CTAs fit an SM.
//   warp 0: TMA, warp 1: tensor memory and products, warps 2-5: sums; all: the joining
// Behind the quantisation of x in the stream, the first weight tiles are on their way before
// that has ended.  ROWS16: x is 16-bit, at most 16 rows, and warps 2-5 of each CTA quantise
// its part of K themselves (for nvfp4 the cluster's CTAs tell each other their rows' absmax).
template <int FORMAT, int TOK, bool ROWS16>
struct SplitCfg {
  static_assert(!ROWS16 || TOK == 16, "rows are quantised here for a tile of 16");
  static constexpr int kScaleBytes = FORMAT == kMxfp4 ? 1024 : 2048;  // of a band and step
  static constexpr int kWBytes = 128 * kF4Step;
  static constexpr int kXBytes = TOK * kF4Step;
  static constexpr int kXStep = kXBytes + kScaleBytes;
  static constexpr int kStageBytes = kWBytes + kScaleBytes + (ROWS16 ? 0 : kXStep);
  static constexpr int kStages = TOK == 128 ? 3 : 4;
  static constexpr int kAccCols = TOK < 32 ? 32 : TOK;
  static constexpr int kTmemCols = kAccCols + 64 <= 128 ? 128 : 256;  // and two slots of 16 + 16 columns of scales
  static_assert(kStageBytes % 1024 == 0 && kXStep % 1024 == 0, "swizzled tiles start at multiples of 1024");
  static_assert(128 * TOK * 4 <= kStages * kStageBytes, "the sums take the stages' place");
  static constexpr int smem_bytes(int steps) { return kStages * kStageBytes + (ROWS16 ? steps * kXStep : 0) + 1024; }
};
constexpr int kSplitThreads = 192;
constexpr int kRows16Steps = 8;  // K steps of a CTA that quantises x: what fits twice on an SM

template <int FORMAT, int TOK, bool ROWS16, bool BF16>
__global__ void __launch_bounds__(kSplitThreads)
    fp4_split_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_sw,
                     const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_sx,
                     Fp4GemmArgs a, int split) {
  using C = SplitCfg<FORMAT, TOK, ROWS16>;
  constexpr int kStages = C::kStages;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t full[kStages], empty[kStages], done, x_ready;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_flag, late_flag;
  __shared__ uint32_t row_top[16];
  __shared__ float row_scale[16];
  __shared__ __align__(16) uint16_t stages[ROWS16 ? 4 : 1][ROWS16 ? 512 : 8];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)cluster_ctarank();
  const int num_n = (a.N + 127) / 128;
  const int tile = blockIdx.x / split;
  const int n0 = tile % num_n * 128, m0 = tile / num_n * TOK;
  const int num_k = (a.K + 255) / 256;
  const int kb0 = (int)((int64_t)num_k * rank / split), steps = (int)((int64_t)num_k * (rank + 1) / split) - kb0;
  uint8_t* x_area = smem + kStages * C::kStageBytes;  // ROWS16: [steps] codes and scales

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(&done, 1);
    mbar_init(&x_ready, 128);
    abort_flag = late_flag = 0;
    fence_mbar_init();
  }
  if (ROWS16 && threadIdx.x < 16) row_top[threadIdx.x] = 0u;
  if (warp == 1) {
    tmem_alloc(&tmem_slot, C::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  chain_next();
  const uint32_t tmem = tmem_slot;

  if (warp == 0) {
    auto load_w = [&](int i) {
      uint8_t* at = smem + i % kStages * C::kStageBytes;
      mbar_arrive_expect_tx(&full[i % kStages], C::kStageBytes);
      tma_load_2d(at, &tm_w, &full[i % kStages], (kb0 + i) * kF4Step, n0);
      tma_load_2d(at + C::kWBytes, &tm_sw, &full[i % kStages], (kb0 + i) * (C::kScaleBytes / 8), n0 >> 7);
    };
    auto load_x = [&](int i) {
      if constexpr (!ROWS16) {
        uint8_t* at = smem + i % kStages * C::kStageBytes + C::kWBytes + C::kScaleBytes;
        tma_load_2d(at, &tm_x, &full[i % kStages], (kb0 + i) * kF4Step, m0);
        tma_load_2d(at + C::kXBytes, &tm_sx, &full[i % kStages], (kb0 + i) * (C::kScaleBytes / 8), m0 >> 7);
      }
    };
    const int ahead = steps < kStages ? steps : kStages;
    if (!a.behind_rows) chain_wait();
    if (elect_one())
      for (int i = 0; i < ahead; ++i) load_w(i);
    __syncwarp();
    if (a.behind_rows) chain_wait();
    if (!ROWS16 && elect_one())
      for (int i = 0; i < ahead; ++i) load_x(i);
    __syncwarp();
    if (ROWS16 && FORMAT == kNvfp4) cluster_sync_all();
    int fills = ahead;
    for (; fills < steps; ++fills) {
      if (!mbar_wait_warp(&empty[fills % kStages], (fills / kStages - 1) & 1, &abort_flag, H3B_STATUS_GEMM_TIMEOUT)) break;
      if (elect_one()) {
        load_w(fills);
        load_x(fills);
      }
      __syncwarp();
    }
    // every copy that was started has landed before the CTA may leave
    for (int i = fills > kStages ? fills - kStages : 0; i < fills; ++i)
      mbar_wait_warp(&full[i % kStages], (i / kStages) & 1, &late_flag, H3B_STATUS_GEMM_TIMEOUT);
  } else if (warp == 1) {
    const uint32_t smem0 = smem_u32(smem), x0 = smem_u32(x_area);
    if (ROWS16 && FORMAT == kNvfp4) cluster_sync_all();
    const bool ready = !ROWS16 || mbar_wait_warp(&x_ready, 0, &abort_flag, H3B_STATUS_GEMM_TIMEOUT);
    for (int i = 0; ready && i < steps; ++i) {
      if (!mbar_wait_warp(&full[i % kStages], (i / kStages) & 1, &abort_flag, H3B_STATUS_GEMM_TIMEOUT)) break;
      // the scale slot of this step: read by the products of the step before last
      if (i >= 2 && !mbar_wait_warp(&empty[(i - 2) % kStages], ((i - 2) / kStages) & 1, &abort_flag, H3B_STATUS_GEMM_TIMEOUT))
        break;
      tc_fence_after();
      if (elect_one()) {
        const uint32_t at = smem0 + (uint32_t)(i % kStages * C::kStageBytes);
        const uint32_t x = ROWS16 ? x0 + (uint32_t)(i * C::kXStep) : at + C::kWBytes + C::kScaleBytes;
        const uint32_t ts = tmem + C::kAccCols + 32u * (uint32_t)(i & 1);
        const int products = (a.K - (kb0 + i) * 256 + 63) / 64;
        // rows m0 .. of their 128-row band: 32 to a column of the scales in tensor memory
        fp4_step<FORMAT, 1, 128, TOK, 1>(tmem, at, x, at + C::kWBytes, x + C::kXBytes, ts, ts + 16,
                                         (uint32_t)(m0 >> 5) & 3u, products, i == 0);
        mma_commit(&empty[i % kStages]);
      }
      __syncwarp();
    }
    if (elect_one()) mma_commit(&done);
    __syncwarp();
    mbar_wait_warp(&done, 0, &late_flag, H3B_STATUS_GEMM_TIMEOUT);
    chain_wait();
  } else {
    chain_wait();
    if constexpr (ROWS16) {
      // a warp takes 32 chunks of 16 columns of a row at a time
      const uint16_t* x = a.x16 + kb0 * 256;
      const int K = a.K - kb0 * 256, segs = (steps + 1) / 2, items = a.M * segs;
      const bool vec = a.x16_vec;
      uint16_t* stage = stages[warp - 2];
      float v[16];
      auto load = [&](int item) {
        const uint16_t* row = x + (int64_t)(item / segs) * a.x16_stride;
        const int c = item % segs * 32 + lane;
        if (vec) load16<BF16, true>(row, c, K, stage, v);
        else load16<BF16, false>(row, c, K, stage, v);
      };
      if constexpr (FORMAT == kNvfp4) {
        for (int item = warp - 2; item < items; item += 4) {
          load(item);
          uint32_t top = absmax16(v);
          if (top >= kInfBits) top = 0u;
          top = __reduce_max_sync(0xffffffffu, top);
          if (lane == 0) atomicMax(&row_top[item / segs], top);
        }
        cluster_sync_all();
      }
      for (int item = warp - 2; item < items; item += 4) {
        const int r = item / segs, c = item % segs * 32 + lane;
        if (FORMAT == kMxfp4 || items > 4) load(item);  // else it is there from above
        float inv_r = 1.0f;
        if constexpr (FORMAT == kNvfp4) {
          uint32_t top = 0u;
          if (lane < split)
            asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(top) : "r"(mapa_shared(smem_u32(&row_top[r]), (uint32_t)lane)));
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
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      mbar_arrive(&x_ready);
    }
    const int quad = warp & 3, row = quad * 32 + lane, toks = min(TOK, a.M - m0);
    if (mbar_wait_warp(&done, 0, &abort_flag, H3B_STATUS_GEMM_TIMEOUT)) {
      tc_fence_after();
      float* sums = reinterpret_cast<float*>(smem);  // [TOK][128]
      const int n = n0 + row;
      const float ws = a.ws && n < a.N ? a.ws[n] : 1.0f, bias = a.bias && n < a.N ? a.bias[n] : 0.0f;
#pragma unroll 1
      for (int c = 0; c < toks; c += 16) {
        uint32_t r[16];
        tmem_ld16(tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)c, r);
        tmem_wait_ld();
        reg_barrier16(r);
        if (split > 1) {
#pragma unroll
          for (int j = 0; j < 16; ++j) sums[(c + j) * 128 + row] = __uint_as_float(r[j]);
        } else if (n < a.N) {
          uint16_t* dst = a.out + (int64_t)(m0 + c) * a.out_stride + n;
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            if (c + j >= toks) break;
            const float xs = ROWS16 ? (FORMAT == kNvfp4 ? row_scale[c + j] : 1.0f) : a.xs ? a.xs[m0 + c + j] : 1.0f;
            dst[j * a.out_stride] = f32_to_half_bits<BF16>(fp4_finish(__uint_as_float(r[j]), xs, ws, bias, a));
          }
        }
        __syncwarp();
      }
    }
    tc_fence_before();
  }
  if (split > 1) {
    cluster_sync_all();
    const int t0 = TOK * rank / split, t1 = min(TOK * (rank + 1) / split, a.M - m0);
    const uint32_t sums0 = smem_u32(smem);
    const bool wide = (a.out_stride & 3) == 0 && (reinterpret_cast<uintptr_t>(a.out) & 7) == 0;
    for (int i = (int)threadIdx.x; i < (t1 - t0) * 32; i += kSplitThreads) {
      const int tok = t0 + (i >> 5), c = (i & 31) * 4, n = n0 + c;
      if (n >= a.N) continue;
      float y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
      for (int r = 0; r < split; ++r) {
        float4 p;
        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(p.x), "=f"(p.y), "=f"(p.z), "=f"(p.w)
                     : "r"(mapa_shared(sums0 + (uint32_t)(tok * 512 + c * 4), (uint32_t)r)));
        y[0] = __fadd_rn(y[0], p.x);
        y[1] = __fadd_rn(y[1], p.y);
        y[2] = __fadd_rn(y[2], p.z);
        y[3] = __fadd_rn(y[3], p.w);
      }
      const float xs = ROWS16 ? (FORMAT == kNvfp4 ? row_scale[tok] : 1.0f) : a.xs ? a.xs[m0 + tok] : 1.0f;
      uint16_t h[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int nn = min(n + j, a.N - 1);
        h[j] = f32_to_half_bits<BF16>(fp4_finish(y[j], xs, a.ws ? a.ws[nn] : 1.0f, a.bias ? a.bias[nn] : 0.0f, a));
      }
      uint16_t* dst = a.out + (int64_t)(m0 + tok) * a.out_stride + n;
      if (wide && n + 4 <= a.N) {
        *reinterpret_cast<uint2*>(dst) =
            make_uint2((uint32_t)h[0] | ((uint32_t)h[1] << 16), (uint32_t)h[2] | ((uint32_t)h[3] << 16));
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n + j < a.N) dst[j] = h[j];
      }
    }
    cluster_sync_all();  // no CTA leaves while another reads its sums
  } else {
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, C::kTmemCols);
  }
}

// ------------------------------------------------------------------ many rows: 256 x 256 tiles on two SMs
// A cluster of two CTAs computes 256 x 256 tiles (rows of x are the products' M): each CTA
// loads 128 rows of x and 128 of the weight, and the even CTA's products read both.  Its
// tensor memory holds 256 accumulator columns twice, overlapping by 96 columns ([0, 256) and
// [160, 416)), and two slots of scales (48 columns each).  The epilogue of a tile first takes
// what lies in the overlap into registers and lets the next tile's products begin.
//   warp 0: TMA, warp 1: tensor memory and (even CTA) products, warps 4-11: epilogue, two per
//   lane quadrant
template <int FORMAT>
struct PairFp4Cfg {
  static constexpr int kScaleBytes = FORMAT == kMxfp4 ? 1024 : 2048;  // of a band and step
  static constexpr int kStageBytes = 2 * 128 * kF4Step + 3 * kScaleBytes;
  static constexpr int kStages = FORMAT == kMxfp4 ? 6 : 5;
  static constexpr int kTotal = kStages * kStageBytes + 1024;
  static_assert(kStageBytes % 1024 == 0, "swizzled tiles start at multiples of 1024");
};
constexpr int kPairFp4Threads = 384;
constexpr int kPairFp4Second = 160, kPairFp4Scales = 416;  // tensor-memory columns

template <bool BF16>
__device__ __forceinline__ void fp4_store_chunk(const uint32_t (&r)[32], int m, int n0, const Fp4GemmArgs& a, float xs,
                                                bool vec) {
  uint16_t* dst = a.out + (int64_t)m * a.out_stride + n0;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    float y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = __fmul_rn(__uint_as_float(r[8 * q + j]), xs);
    const int n = n0 + 8 * q;
    if (vec && n + 8 <= a.N) {
      if (a.ws) {
        const float4 w0 = *reinterpret_cast<const float4*>(a.ws + n), w1 = *reinterpret_cast<const float4*>(a.ws + n + 4);
        const float w[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = __fmul_rn(y[j], w[j]);
      }
      if (a.bias) {
        const float4 b0 = *reinterpret_cast<const float4*>(a.bias + n), b1 = *reinterpret_cast<const float4*>(a.bias + n + 4);
        const float b[8] = {b0.x, b0.y, b0.z, b0.w, b1.x, b1.y, b1.z, b1.w};
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = __fadd_rn(y[j], b[j]);
      }
      *reinterpret_cast<uint4*>(dst + 8 * q) = make_uint4(pack_halves<BF16>(y[0], y[1]), pack_halves<BF16>(y[2], y[3]),
                                                          pack_halves<BF16>(y[4], y[5]), pack_halves<BF16>(y[6], y[7]));
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (n + j >= a.N) continue;
        float v = y[j];
        if (a.ws) v = __fmul_rn(v, a.ws[n + j]);
        if (a.bias) v = __fadd_rn(v, a.bias[n + j]);
        dst[8 * q + j] = f32_to_half_bits<BF16>(v);
      }
    }
  }
}

template <int FORMAT, bool BF16>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairFp4Threads, 1)
    fp4_pair_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                    const __grid_constant__ CUtensorMap tm_sx, const __grid_constant__ CUtensorMap tm_sw,
                    Fp4GemmArgs a) {
  using C = PairFp4Cfg<FORMAT>;
  constexpr int kStages = C::kStages;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t full[kStages], empty[kStages], tfull, tempty, drained;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_flag, late_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int num_m = (a.M + 255) / 256, num_n = (a.N + 255) / 256;
  const int tiles = num_m * num_n;
  const int num_k = (a.K + 255) / 256;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
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
  chain_next();
  chain_wait();
  const uint32_t tmem = tmem_slot;
  const uint32_t full0 = mapa_shared(smem_u32(full), 0);
  const uint32_t tempty0 = mapa_shared(smem_u32(&tempty), 0);

  if (warp == 0) {
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int t = pair; ok && t < tiles; t += pairs) {
      const int mb = t / num_n, nb = t % num_n;
      for (int kb = 0; kb < num_k; ++kb) {
        if (!mbar_wait_warp(&empty[stage], phase ^ 1, &abort_flag, H3B_STATUS_GEMM_TIMEOUT)) { ok = false; break; }
        if (elect_one()) {
          uint8_t* at = smem + stage * C::kStageBytes;
          const uint32_t fb = full0 + (uint32_t)(stage * 8);
          mbar_arrive_expect_tx_cluster(fb, C::kStageBytes);
          tma_load_2d_pair(at, &tm_x, fb, kb * kF4Step, mb * 256 + (int)rank * 128);
          tma_load_2d_pair(at + 128 * kF4Step, &tm_w, fb, kb * kF4Step, nb * 256 + (int)rank * 128);
          at += 2 * 128 * kF4Step;
          tma_load_2d_pair(at, &tm_sx, fb, kb * (C::kScaleBytes / 8), mb * 2 + (int)rank);
          // the scales of all 256 rows of the weight: each CTA's tensor memory holds them
          tma_load_2d_pair(at + C::kScaleBytes, &tm_sw, fb, kb * (C::kScaleBytes / 8), nb * 2);
        }
        __syncwarp();
        if (++stage == kStages) { stage = 0; phase ^= 1; }
      }
    }
    // Both CTAs' copies are counted by the even CTA's barriers; the odd one waits for it at the
    // end.  Of each slot the last fill: slots before `stage` in this round, the others before.
    if (rank == 0)
      for (int s = 0; s < kStages; ++s)
        mbar_wait_warp(&full[s], s < stage ? phase : phase ^ 1u, &late_flag, H3B_STATUS_GEMM_TIMEOUT);
  } else if (warp == 1) {
    if (rank == 0) {
      const uint32_t smem0 = smem_u32(smem);
      uint32_t it = 0;  // K steps so far
      uint32_t tile = 0;
      bool ok = true;
      for (int t = pair; ok && t < tiles; t += pairs, ++tile) {
        if (tile > 0 && !mbar_wait_warp(&tempty, (tile - 1) & 1, &abort_flag, H3B_STATUS_GEMM_TIMEOUT)) break;
        tc_fence_after();
        const uint32_t d = tmem + (tile & 1 ? (uint32_t)kPairFp4Second : 0u);
        for (int kb = 0; kb < num_k; ++kb, ++it) {
          const uint32_t stage = it % kStages;
          if (!mbar_wait_warp(&full[stage], (it / kStages) & 1, &abort_flag, H3B_STATUS_GEMM_TIMEOUT) ||
              (it >= 2 && !mbar_wait_warp(&empty[(it - 2) % kStages], ((it - 2) / kStages) & 1, &abort_flag,
                                          H3B_STATUS_GEMM_TIMEOUT))) {
            ok = false;
            break;
          }
          tc_fence_after();
          if (elect_one()) {
            const uint32_t at = smem0 + stage * C::kStageBytes;
            const uint32_t ts = tmem + kPairFp4Scales + 48u * (it & 1);
            fp4_step<FORMAT, 2, 256, 256, 2>(d, at, at + 128 * kF4Step, at + 2 * 128 * kF4Step,
                                             at + 2 * 128 * kF4Step + C::kScaleBytes, ts, ts + 16, 0u,
                                             (a.K - kb * 256 + 63) / 64, kb == 0);
            mma_commit_pair(&empty[stage], 0x3);
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
    const bool vec = (a.out_stride & 7) == 0 && (reinterpret_cast<uintptr_t>(a.out) & 15) == 0 &&
                     (reinterpret_cast<uintptr_t>(a.ws) & 15) == 0 && (reinterpret_cast<uintptr_t>(a.bias) & 15) == 0;
    uint32_t tile = 0;
    for (int t = pair; t < tiles; t += pairs, ++tile) {
      const int mb = t / num_n, nb = t % num_n;
      if (!mbar_wait_warp(&tfull, tile & 1, &abort_flag, H3B_STATUS_GEMM_TIMEOUT)) break;
      tc_fence_after();
      const int m = mb * 256 + (int)rank * 128 + quad * 32 + lane;
      const float xs = a.xs && m < a.M ? a.xs[m] : 1.0f;
      const bool odd = tile & 1;
      const uint32_t taddr = tmem + ((uint32_t)(quad * 32) << 16) + (odd ? (uint32_t)kPairFp4Second : 0u);
      // this warp's four chunks of 32 columns; in the overlap lie 5, 6, 7 of the even tiles
      // and 0, 1, 2 of the odd ones, and they come first
      const int order = odd ? (half ? 0x6572 : 0x4310) : (half ? 0x3247 : 0x1065);
      uint32_t r0[32], r1[32];
      tmem_ld32(taddr + 32u * (uint32_t)(order & 15), r0);
      tmem_ld32(taddr + 32u * (uint32_t)((order >> 4) & 15), r1);
      tmem_wait_ld_dep(r0);
      reg_barrier32(r1);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(tempty0);
      const int n0 = nb * 256;
      if (m < a.M) {
        fp4_store_chunk<BF16>(r0, m, n0 + 32 * (order & 15), a, xs, vec);
        fp4_store_chunk<BF16>(r1, m, n0 + 32 * ((order >> 4) & 15), a, xs, vec);
      }
      __syncwarp();
      tmem_ld32(taddr + 32u * (uint32_t)((order >> 8) & 15), r0);
      tmem_ld32(taddr + 32u * (uint32_t)((order >> 12) & 15), r1);
      tmem_wait_ld_dep(r0);
      reg_barrier32(r1);
      if (m < a.M) {
        fp4_store_chunk<BF16>(r0, m, n0 + 32 * ((order >> 8) & 15), a, xs, vec);
        fp4_store_chunk<BF16>(r1, m, n0 + 32 * ((order >> 12) & 15), a, xs, vec);
      }
      __syncwarp();
    }
  }

  tc_fence_before();
  cluster_sync_all();  // the pair's products, copies and epilogues are done
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

// ------------------------------------------------------------------ host side

// Launch in a cluster of `ctas` (0: as the kernel declares), starting while the kernel before ends
template <typename... P, typename... A>
static cudaError_t launch_fp4(void (*kernel)(P...), int64_t grid, int ctas, int threads, size_t smem, cudaStream_t s,
                              const A&... args) {
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)ctas;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = ctas ? 2 : 1;
  e = cudaLaunchKernelEx(&cfg, kernel, args...);
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

#ifdef FORCE
#include <cstdlib>
static int env(const char* n, int d) { const char* v = getenv(n); return v ? atoi(v) : d; }
#endif
// How a product of few rows is divided: TOK and the CTAs along K
struct SplitPlan {
  int tok, split;
};
static SplitPlan plan_split(int M, int N, int K) {
#ifdef FORCE
  if (env("H3B_TOK", 0)) return {env("H3B_TOK", 0), env("H3B_SPLIT", 1)};
#endif
  const int tok = M <= 16 ? 16 : M <= 64 ? 64 : 128, num_k = (K + 255) / 256;
  const int64_t tiles = (int64_t)((N + 127) / 128) * ((M + tok - 1) / tok);
  int split = 1;
  while (split < 8 && 2 * split <= num_k && tiles * 2 * split <= 2 * num_sms()) split *= 2;
  return {tok, split};
}
template <int FORMAT, int TOK, bool ROWS16>
static int launch_split(const Fp4RowsView& x, const Fp4RowsView& w, const Fp4GemmArgs& a, int split, cudaStream_t s,
                        cudaError_t* err) {
  CUtensorMap tx, tw, tsx, tsw;
  if (!make_fp4_maps(w, FORMAT, 128, 1, &tw, &tsw)) return 1;
  if (ROWS16) tx = tw, tsx = tsw;  // not used
  else if (!make_fp4_maps(x, FORMAT, TOK, 1, &tx, &tsx)) return 1;
  const int64_t tiles = (int64_t)((a.N + 127) / 128) * ((a.M + TOK - 1) / TOK);
  const int steps = ((a.K + 255) / 256 + split - 1) / split;
  *err = launch_fp4(a.bf16 ? fp4_split_kernel<FORMAT, TOK, ROWS16, true> : fp4_split_kernel<FORMAT, TOK, ROWS16, false>,
                    tiles * split, split, kSplitThreads, SplitCfg<FORMAT, TOK, ROWS16>::smem_bytes(steps), s, tw, tsw, tx,
                    tsx, a, split);
  return *err == cudaSuccess ? 0 : 2;
}
template <int FORMAT>
static int launch_pair(const Fp4RowsView& x, const Fp4RowsView& w, const Fp4GemmArgs& a, cudaStream_t s,
                       cudaError_t* err) {
  CUtensorMap tx, tw, tsx, tsw;
  if (!make_fp4_maps(x, FORMAT, 128, 1, &tx, &tsx) || !make_fp4_maps(w, FORMAT, 128, 2, &tw, &tsw)) return 1;
  const int64_t tiles = (int64_t)((a.M + 255) / 256) * ((a.N + 255) / 256);
  const int64_t pairs = tiles < num_sms() / 2 ? tiles : num_sms() / 2;
  *err = launch_fp4(a.bf16 ? fp4_pair_kernel<FORMAT, true> : fp4_pair_kernel<FORMAT, false>, 2 * pairs, 0,
                    kPairFp4Threads, PairFp4Cfg<FORMAT>::kTotal, s, tx, tw, tsx, tsw, a);
  return *err == cudaSuccess ? 0 : 2;
}
static bool uses_pair(int M, int N) {
#ifdef FORCE
  if (env("H3B_PAIR", -1) >= 0) return env("H3B_PAIR", 0);
#endif
  return (int64_t)((M + 255) / 256) * ((N + 255) / 256) >= num_sms() / 2;
}
template <int FORMAT>
static int launch_gemm_of(const Fp4RowsView& x, const Fp4RowsView& w, const Fp4GemmArgs& a, cudaStream_t s,
                          cudaError_t* err) {
  if (uses_pair(a.M, a.N)) return launch_pair<FORMAT>(x, w, a, s, err);
  const SplitPlan p = plan_split(a.M, a.N, a.K);
  return p.tok == 16   ? launch_split<FORMAT, 16, false>(x, w, a, p.split, s, err)
         : p.tok == 64 ? launch_split<FORMAT, 64, false>(x, w, a, p.split, s, err)
                       : launch_split<FORMAT, 128, false>(x, w, a, p.split, s, err);
}

int launch_fp4_gemm(const Fp4RowsView& x, const Fp4RowsView& w, Fp4GemmArgs a, int format, cudaStream_t s,
                    cudaError_t* err) {
  a.xs = x.row_scales;
  a.ws = w.row_scales;
  return format == kMxfp4 ? launch_gemm_of<kMxfp4>(x, w, a, s, err) : launch_gemm_of<kNvfp4>(x, w, a, s, err);
}

bool fp4_takes_rows16(int64_t M, int64_t N, int64_t K) {
  if (M > 16 || uses_pair((int)M, (int)N)) return false;
  const SplitPlan p = plan_split((int)M, (int)N, (int)K);
  return p.tok == 16 && (K + 255) / 256 <= (int64_t)kRows16Steps * p.split;
}
int launch_fp4_gemm_rows16(const uint16_t* x, int64_t x_stride, const Fp4RowsView& w, Fp4GemmArgs a, int format,
                           cudaStream_t s, cudaError_t* err) {
  a.ws = w.row_scales;
  a.x16 = x;
  a.x16_stride = x_stride;
  a.x16_vec = a.K % 16 == 0 && rows16(x, a.M > 1 ? x_stride : 0);
  const int split = plan_split(a.M, a.N, a.K).split;
  return format == kMxfp4 ? launch_split<kMxfp4, 16, true>({}, w, a, split, s, err)
                          : launch_split<kNvfp4, 16, true>({}, w, a, split, s, err);
}

}  // namespace h3b
