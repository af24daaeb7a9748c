// fp4_rows.cu -- rows to microscaled 4-bit floats (mxfp4, nvfp4) and back, and the residual
// addition + RMSNorm whose output goes to INT8 or 4-bit rows in the same pass.
//
// One row is held in registers by one warp (up to 1,024 columns) or one block: each thread
// has one to four chunks of 16 columns, so the row is read once, and everything that is
// asked of the whole row (sum of squares, absmax) is a reduction over registers.  A chunk is
// an nvfp4 block, two neighbouring lanes hold an mxfp4 block, and four or eight lanes the
// four scales of a word.
//
// All scales are found exactly: mxfp4's and the nvfp4 row scale are powers of two read off
// the absmax's bits.  The remaining quotients (absmax / 6 to E4M3, x / scale to E2M1) are
// correctly rounded before they are rounded to the narrow type.  For 16-bit inputs that
// gives the nearest code of the exact quotient, ties included: quotient and border differ
// by more than the fp32 rounding or not at all, since the border times the scale has fewer
// than 24 bits.
//
// Infinities and NaN: the block's scale becomes NaN (all of it is lost, and seen to be); the
// row scale goes by the other blocks.  An INT8 row with one gets the scale NaN or infinity.
#include <cfloat>

#include "fp4.cuh"

namespace h3b {

constexpr uint32_t kInfBits = 0x7F800000u;

// two floats -> E2M1 codes, to nearest even, saturating; lo in bits 0..3
__device__ __forceinline__ uint32_t e2m1x2(float lo, float hi) {
  uint32_t r;
  asm("{\n\t.reg .b8 t;\n\tcvt.rn.satfinite.e2m1x2.f32 t, %1, %2;\n\tcvt.u32.u8 %0, t;\n\t}" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float e4m3_to_f32(uint32_t code) {
  uint32_t h2;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"((uint16_t)code));
  return __half2float(__ushort_as_half((uint16_t)(h2 & 0xffffu)));
}
__device__ __forceinline__ float e8m0_to_f32(uint32_t b) {
  return __uint_as_float(b == 0u ? 0x00400000u : b == 255u ? 0x7FC00000u : b << 23);
}

// max of non-negative floats' bits over the row's threads (a warp, or the block)
template <bool BLOCK>
__device__ __forceinline__ uint32_t row_max(uint32_t v, uint32_t* red) {
  v = __reduce_max_sync(0xffffffffu, v);
  if constexpr (BLOCK) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = blockDim.x >> 5;
    if (lane == 0) red[warp] = v;
    __syncthreads();
    v = __reduce_max_sync(0xffffffffu, lane < n ? red[lane] : 0u);
  }
  return v;
}
template <bool BLOCK>
__device__ __forceinline__ float row_sum(float v, float* red) {
  v = warp_butterfly_sum(v);
  if constexpr (BLOCK) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = blockDim.x >> 5;
    if (lane == 0) red[warp] = v;
    __syncthreads();
    v = warp_butterfly_sum(lane < n ? red[lane] : 0.0f);
  }
  return v;
}

// 16 columns from column c0 on, zeros beyond K.  VEC: all pointers and strides allow 16-byte
// accesses and K is a multiple of 16.
template <bool BF16, bool VEC>
__device__ __forceinline__ void load16(const uint16_t* row, int c0, int K, float (&v)[16]) {
  if constexpr (VEC) {
    const uint4 z = make_uint4(0u, 0u, 0u, 0u);
    const bool live = c0 < K;
    const uint4 a = live ? *reinterpret_cast<const uint4*>(row + c0) : z;
    const uint4 b = live ? *reinterpret_cast<const uint4*>(row + c0 + 8) : z;
    const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[2 * i] = half_to_f32<BF16>((uint16_t)(w[i] & 0xffffu));
      v[2 * i + 1] = half_to_f32<BF16>((uint16_t)(w[i] >> 16));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = c0 + i < K ? half_to_f32<BF16>(row[c0 + i]) : 0.0f;
  }
}
template <bool BF16, bool VEC>
__device__ __forceinline__ void store16(uint16_t* row, int c0, int K, const float (&v)[16]) {
  if constexpr (VEC) {
    if (c0 >= K) return;
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = pack_halves<BF16>(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<uint4*>(row + c0) = make_uint4(w[0], w[1], w[2], w[3]);
    *reinterpret_cast<uint4*>(row + c0 + 8) = make_uint4(w[4], w[5], w[6], w[7]);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (c0 + i < K) row[c0 + i] = f32_to_half_bits<BF16>(v[i]);
  }
}

// FORMAT 0: int8.  BLOCK: a row per block, else per warp.  CH chunks per thread.
template <int FORMAT, bool BF16, bool NORM, bool VEC, bool BLOCK, int CH>
__global__ void __launch_bounds__(512) fp4_rows_kernel(Fp4RowArgs a) {
  __shared__ uint32_t red[2][32];
  chain_wait();
  chain_next();  // behind the wait: a product that follows may read its weight before it waits
  const int t = BLOCK ? (int)threadIdx.x : (int)(threadIdx.x & 31);
  const int step = BLOCK ? (int)blockDim.x : 32;
  const int64_t row = BLOCK ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (row >= a.rows) return;  // whole warps of a warp-per-row block
  float v[CH][16];
#pragma unroll
  for (int i = 0; i < CH; ++i) load16<BF16, VEC>(a.x + row * a.x_stride, (t + i * step) * 16, a.K, v[i]);

  if constexpr (NORM) {
    if (a.res) {
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        float r[16];
        load16<BF16, VEC>(a.res + row * a.res_stride, (t + i * step) * 16, a.K, r);
#pragma unroll
        // the sum as it is stored: what a later layer reads is what is normed here
        for (int j = 0; j < 16; ++j) v[i][j] = half_to_f32<BF16>(f32_to_half_bits<BF16>(__fadd_rn(v[i][j], r[j])));
      }
#pragma unroll
      for (int i = 0; i < CH; ++i) store16<BF16, VEC>(a.sum + row * a.sum_stride, (t + i * step) * 16, a.K, v[i]);
    }
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < CH; ++i)
#pragma unroll
      for (int j = 0; j < 16; ++j) ss = fmaf(v[i][j], v[i][j], ss);
    ss = row_sum<BLOCK>(ss, reinterpret_cast<float*>(red[0]));
    const float inv = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(ss, (float)a.K), a.eps)));
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      float w[16];
      load16<BF16, VEC>(a.norm_w, (t + i * step) * 16, a.K, w);
#pragma unroll
      for (int j = 0; j < 16; ++j) v[i][j] = __fmul_rn(__fmul_rn(v[i][j], inv), w[j]);
    }
    // beyond K: zeros times inv (finite or NaN) times a weight of zero
#pragma unroll
    for (int i = 0; i < CH; ++i)
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if ((t + i * step) * 16 + j >= a.K) v[i][j] = 0.0f;
  }

  uint32_t top[CH];  // absmax bits of each block (of 16 columns for int8)
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    top[i] = 0u;
#pragma unroll
    for (int j = 0; j < 16; ++j) top[i] = max(top[i], __float_as_uint(v[i][j]) & 0x7FFFFFFFu);
    if (FORMAT == kMxfp4) top[i] = max(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
  }

  if constexpr (FORMAT == 0) {
    uint32_t m = 0u;
#pragma unroll
    for (int i = 0; i < CH; ++i) m = max(m, top[i]);
    m = row_max<BLOCK>(m, red[1]);
    const float scale = __fdiv_rn(__uint_as_float(m), 127.0f);  // NaN and infinity stay
    if (t == 0) a.row_scales[row] = scale;
    const bool some = m < kInfBits && scale >= FLT_MIN;  // a row below that is zeros
    const float rs = some ? __fdiv_rn(1.0f, scale) : 0.0f;
    uint8_t* dst = a.codes + row * (int64_t)a.K;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int c0 = (t + i * step) * 16;
      uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float q = some ? div_rn_by(v[i][j], scale, rs) : 0.0f;  // at most 127 and an fp32 rounding
        w[j >> 2] |= ((uint32_t)__float2int_rn(q) & 0xffu) << (8 * (j & 3));
      }
      if constexpr (VEC) {
        if (c0 < a.K) *reinterpret_cast<uint4*>(dst + c0) = make_uint4(w[0], w[1], w[2], w[3]);
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (c0 + j < a.K) dst[c0 + j] = (uint8_t)(w[j >> 2] >> (8 * (j & 3)));
      }
    }
    return;
  }

  const int64_t pitch = fp4_pitch(a.K);
  const int groups = (int)fp4_groups(a.K, FORMAT);
  uint8_t* dst = a.codes + row * pitch;
  uint8_t* word0 = a.blocks + (row >> 7) * groups * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4;
  float inv_r = 1.0f;
  if constexpr (FORMAT == kNvfp4) {
    uint32_t m = 0u;
#pragma unroll
    for (int i = 0; i < CH; ++i) m = max(m, top[i] < kInfBits ? top[i] : 0u);
    m = row_max<BLOCK>(m, red[1]);
    // least e with absmax <= 2688 * 2^e = 1.3125 * 2^(11 + e), at least -126
    const int e = m ? max((int)(m >> 23) - 138 + ((m & 0x7FFFFFu) > 0x280000u ? 1 : 0), -126) : 0;
    inv_r = __uint_as_float((uint32_t)(127 - e) << 23);
    if (t == 0) a.row_scales[row] = __uint_as_float((uint32_t)(127 + e) << 23);
  }
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const int c = t + i * step;
    const bool bad = top[i] >= kInfBits;
    uint32_t byte, w[2] = {0u, 0u};
    if constexpr (FORMAT == kMxfp4) {
      byte = bad ? 255u : (uint32_t)max((int)(top[i] >> 23) - 2, 0);
      const float inv = __uint_as_float((254u - byte) << 23);
#pragma unroll
      for (int j = 0; j < 16; j += 2)
        w[j >> 3] |= e2m1x2(__fmul_rn(v[i][j], inv), __fmul_rn(v[i][j + 1], inv)) << (4 * (j & 7));
    } else {
      byte = bad ? 0x7Fu : (uint32_t)f32x2_to_e4m3x2(__fdiv_rn(__fmul_rn(__uint_as_float(top[i]), inv_r), 6.0f), 0.0f) & 0xffu;
      const float s = e4m3_to_f32(byte);
      const float rs = s > 0.0f ? __fdiv_rn(1.0f, s) : 0.0f;  // under a scale of zero: zeros, with their signs
#pragma unroll
      for (int j = 0; j < 16; j += 2) {
        // the remainder of -0 is 0 and would make the quotient 0: the sign is x's
        const float q0 = copysignf(div_rn_by(__fmul_rn(v[i][j], inv_r), s, rs), v[i][j]);
        const float q1 = copysignf(div_rn_by(__fmul_rn(v[i][j + 1], inv_r), s, rs), v[i][j + 1]);
        w[j >> 3] |= e2m1x2(q0, q1) << (4 * (j & 7));
      }
    }
    if (bad) w[0] = w[1] = 0u;
    if (c * 8 < pitch) *reinterpret_cast<uint2*>(dst + c * 8) = make_uint2(w[0], w[1]);
    // four blocks' scales to a word: those of four lanes, or of four pairs
    constexpr int kLanes = FORMAT == kMxfp4 ? 8 : 4, kPer = kLanes / 4;
    uint32_t word = byte << (8 * ((t / kPer) & 3));
#pragma unroll
    for (int o = kPer; o < kLanes; o *= 2) word |= __shfl_xor_sync(0xffffffffu, word, o);
    if ((t & (kLanes - 1)) == 0 && c / kLanes < groups)
      *reinterpret_cast<uint32_t*>(word0 + (int64_t)(c / kLanes) * 512) = word;
  }
}

// Codes and scales to 16-bit values: a thread takes 16 columns.  value = code * block scale * row scale
template <int FORMAT, bool BF16, bool VEC>
__global__ void __launch_bounds__(256) fp4_dequantize_kernel(Fp4RowsView a, uint16_t* out, int64_t out_stride,
                                                             int chunks, int64_t total) {
  chain_wait();
  chain_next();
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= total) return;
  const int64_t row = at / chunks;
  const int c = (int)(at - row * chunks);
  const uint2 q = *reinterpret_cast<const uint2*>(a.codes + row * fp4_pitch(a.K) + c * 8);
  const int b = c * 16 / fp4_block(FORMAT);
  const uint32_t byte = a.blocks[((row >> 7) * fp4_groups(a.K, FORMAT) + (b >> 2)) * 512 + (row & 31) * 16 +
                                 ((row >> 5) & 3) * 4 + (b & 3)];
  const float s = FORMAT == kMxfp4 ? e8m0_to_f32(byte) : e4m3_to_f32(byte);
  const float r = a.row_scales ? a.row_scales[row] : 1.0f;
  float v[16];
#pragma unroll
  for (int j = 0; j < 16; j += 2) {
    const uint32_t pair = ((j < 8 ? q.x : q.y) >> (4 * (j & 7))) & 0xffu;
    uint32_t h2;
    asm("{\n\t.reg .b8 t;\n\tcvt.u8.u32 t, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, t;\n\t}" : "=r"(h2) : "r"(pair));
    v[j] = __fmul_rn(__fmul_rn(__half2float(__ushort_as_half((uint16_t)(h2 & 0xffffu))), s), r);
    v[j + 1] = __fmul_rn(__fmul_rn(__half2float(__ushort_as_half((uint16_t)(h2 >> 16))), s), r);
  }
  store16<BF16, VEC>(out + row * out_stride, c * 16, a.K, v);
}

// ------------------------------------------------------------------ host side

static bool rows16(const void* p, int64_t stride) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % 8 == 0; }

template <int FORMAT, bool BF16, bool NORM, bool VEC>
static cudaError_t launch_rows(const Fp4RowArgs& a, cudaStream_t s) {
  // chunks of 16 columns, up to the end of the last scale word
  const int chunks = FORMAT == 0 ? (a.K + 15) / 16 : (int)fp4_groups(a.K, FORMAT) * (fp4_block(FORMAT) / 4);
  if (chunks <= 64) {
    const int64_t grid = (a.rows + 7) / 8;
    return chunks <= 32 ? launch_chained(fp4_rows_kernel<FORMAT, BF16, NORM, VEC, false, 1>, grid, 256, 0, s, a)
                        : launch_chained(fp4_rows_kernel<FORMAT, BF16, NORM, VEC, false, 2>, grid, 256, 0, s, a);
  }
  const int ch = chunks <= 512 ? 1 : chunks <= 1024 ? 2 : 4;
  const int threads = ((chunks + ch - 1) / ch + 31) / 32 * 32;
  return ch == 1   ? launch_chained(fp4_rows_kernel<FORMAT, BF16, NORM, VEC, true, 1>, a.rows, threads, 0, s, a)
         : ch == 2 ? launch_chained(fp4_rows_kernel<FORMAT, BF16, NORM, VEC, true, 2>, a.rows, threads, 0, s, a)
                   : launch_chained(fp4_rows_kernel<FORMAT, BF16, NORM, VEC, true, 4>, a.rows, threads, 0, s, a);
}
template <int FORMAT, bool NORM>
static cudaError_t launch_rows_as(const Fp4RowArgs& a, bool bf16, cudaStream_t s) {
  bool vec = a.K % 16 == 0 && rows16(a.x, a.x_stride);
  if (NORM) vec = vec && rows16(a.norm_w, 0);
  if (NORM && a.res) vec = vec && rows16(a.res, a.res_stride) && rows16(a.sum, a.sum_stride);
  if (bf16)
    return vec ? launch_rows<FORMAT, true, NORM, true>(a, s) : launch_rows<FORMAT, true, NORM, false>(a, s);
  return vec ? launch_rows<FORMAT, false, NORM, true>(a, s) : launch_rows<FORMAT, false, NORM, false>(a, s);
}

cudaError_t launch_fp4_rows(const Fp4RowArgs& a, int format, bool bf16, cudaStream_t s) {
  if (!a.norm_w)
    return format == kMxfp4 ? launch_rows_as<kMxfp4, false>(a, bf16, s) : launch_rows_as<kNvfp4, false>(a, bf16, s);
  return format == 0         ? launch_rows_as<0, true>(a, bf16, s)
         : format == kMxfp4 ? launch_rows_as<kMxfp4, true>(a, bf16, s)
                             : launch_rows_as<kNvfp4, true>(a, bf16, s);
}

template <int FORMAT>
static cudaError_t launch_dequantize(const Fp4RowsView& a, uint16_t* out, int64_t stride, bool bf16, cudaStream_t s) {
  const int chunks = (a.K + 15) / 16;
  const int64_t total = a.rows * chunks, grid = (total + 255) / 256;
  const bool vec = a.K % 16 == 0 && rows16(out, stride);
  if (bf16)
    return vec ? launch_chained(fp4_dequantize_kernel<FORMAT, true, true>, grid, 256, 0, s, a, out, stride, chunks, total)
               : launch_chained(fp4_dequantize_kernel<FORMAT, true, false>, grid, 256, 0, s, a, out, stride, chunks, total);
  return vec ? launch_chained(fp4_dequantize_kernel<FORMAT, false, true>, grid, 256, 0, s, a, out, stride, chunks, total)
             : launch_chained(fp4_dequantize_kernel<FORMAT, false, false>, grid, 256, 0, s, a, out, stride, chunks, total);
}
cudaError_t launch_fp4_dequantize(const Fp4RowsView& a, int format, uint16_t* out, int64_t out_stride, bool bf16,
                                  cudaStream_t s) {
  return format == kMxfp4 ? launch_dequantize<kMxfp4>(a, out, out_stride, bf16, s)
                          : launch_dequantize<kNvfp4>(a, out, out_stride, bf16, s);
}

}  // namespace h3b
