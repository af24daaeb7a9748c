// fp4.cuh -- microscaled 4-bit floating-point rows: their formats and layout, argument
// structs and host launchers of the kernels over them (fp4_rows.cu, fp4_gemm.cu).
//
// An element is an E2M1 code: sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6; two columns to a
// byte, the even one in the low nibble.  Rows are padded with zero codes to a multiple of 32
// columns (16 bytes, what a TMA copy's row pitch needs).
//   mxfp4: blocks of 32 columns with an E8M0 scale 2^(byte - 127)
//   nvfp4: blocks of 16 columns with an E4M3 scale, and one fp32 scale per row
// Block scales lie as the block-scaled tensor-core products read them: tiles of 128 rows x 4
// blocks in 512 bytes, row r's four bytes at (r % 32) * 16 + (r / 32) * 4, the tiles of a
// 128-row band one after the other along the columns.  A 32 x 16-byte copy of such a tile to
// tensor memory (tcgen05.cp 32x128b) puts row r's scales into lane r % 32, column r / 32.
#pragma once

#include "h3b_common.cuh"
#include "h3b_packed.cuh"
#include "streaming.cuh"

namespace h3b {

enum Fp4Format : int { kMxfp4 = 1, kNvfp4 = 2 };

__host__ __device__ constexpr int fp4_block(int format) { return format == kMxfp4 ? 32 : 16; }
__host__ __device__ constexpr int64_t fp4_pitch(int64_t cols) { return (cols + 31) / 32 * 16; }  // bytes of a row's codes
// 512-byte tiles along a band's columns
__host__ __device__ constexpr int64_t fp4_groups(int64_t cols, int format) {
  return (cols + 4 * fp4_block(format) - 1) / (4 * fp4_block(format));
}
__host__ __device__ constexpr int64_t fp4_scale_bytes(int64_t rows, int64_t cols, int format) {
  return (rows + 127) / 128 * fp4_groups(cols, format) * 512;
}

constexpr int kFp4MaxRowCols = 32768;  // a row that the row kernels hold in registers

// Quantisation of rows, optionally behind an addition and an RMSNorm.
struct Fp4RowArgs {
  const uint16_t* x;
  int64_t x_stride;
  int64_t rows;
  int K;
  // norm (norm_w set): h = x + res (res set; stored to sum), y = h / sqrt(mean(h^2) + eps) * norm_w
  const uint16_t* res;
  int64_t res_stride;
  uint16_t* sum;
  int64_t sum_stride;
  const uint16_t* norm_w;
  float eps;
  // output
  uint8_t* codes;      // E2M1 rows of fp4_pitch(K) bytes, or int8 rows of K
  uint8_t* blocks;     // block scales
  float* row_scales;   // nvfp4's, or the int8 rows' scales
};
// format: kMxfp4, kNvfp4 or 0 for int8 (with a norm only)
cudaError_t launch_fp4_rows(const Fp4RowArgs& a, int format, bool bf16, cudaStream_t s);

struct Fp4RowsView {
  const uint8_t* codes;
  const uint8_t* blocks;
  const float* row_scales;  // null: 1
  int64_t rows;
  int K;
};
cudaError_t launch_fp4_dequantize(const Fp4RowsView& a, int format, uint16_t* out, int64_t out_stride, bool bf16,
                                  cudaStream_t s);

// out [M, N] = x [M, K] . w [N, K]^T * xs[m] * ws[n] + bias[n]
struct Fp4GemmArgs {
  int M, N, K;
  const float* xs;    // null: 1
  const float* ws;    // null: 1
  const float* bias;  // null: none
  uint16_t* out;
  int64_t out_stride;
  int bf16;
  int behind_rows;  // launched right behind the kernel that quantises x, after which w does not change
  // 16-bit rows that the product quantises itself (launch_fp4_gemm_rows16)
  const uint16_t* x16;
  int64_t x16_stride;
  int x16_vec;       // they allow 16-byte accesses
  int x16_log_segs;  // pieces of 512 columns that a CTA takes of a row, as a power of two
  // set by the launcher: the output rows go out by TMA; tiles of columns that are gone through at a time
  int out_tma, group;
};
// 0 ok, 1 tensor-map encoding failed, 2 CUDA error (*err)
int launch_fp4_gemm(const Fp4RowsView& x, const Fp4RowsView& w, Fp4GemmArgs a, int format, cudaStream_t s,
                    cudaError_t* err);

// Whether a linear of these sizes quantises its 16-bit rows inside the product, and that product
bool fp4_takes_rows16(int64_t M, int64_t N, int64_t K, int format);
int launch_fp4_gemm_rows16(const uint16_t* x, int64_t x_stride, const Fp4RowsView& w, Fp4GemmArgs a, int format,
                           cudaStream_t s, cudaError_t* err);

template <bool BF16>
__device__ __forceinline__ float half_to_f32(uint16_t b) {
  return BF16 ? bf16_bits_to_f32(b) : __half2float(__ushort_as_half(b));
}
template <bool BF16>
__device__ __forceinline__ uint16_t f32_to_half_bits(float f) {
  return BF16 ? f32_to_bf16_bits(f) : __half_as_ushort(__float2half_rn(f));
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack_halves(float lo, float hi) {
  uint32_t r;
  if constexpr (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// ------------------------------------------------------------------ a chunk of 16 columns to codes
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

// The 16 codes (w) and the block's scale byte of a chunk v, of which the block's absmax has the
// bits `top`; inv_r: 1 / row scale.
template <int FORMAT>
__device__ __forceinline__ uint32_t quantize16(const float2 (&v)[8], uint32_t top, float inv_r, uint32_t (&w)[2]) {
  const bool bad = top >= kInfBits;
  uint32_t byte;
  w[0] = w[1] = 0u;
  if constexpr (FORMAT == kMxfp4) {
    byte = bad ? 255u : (uint32_t)max((int)(top >> 23) - 2, 0);
    const float2 inv = splat2(__uint_as_float((254u - byte) << 23));
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float2 q = mul2(v[j], inv);
      w[j >> 2] |= e2m1x2(q.x, q.y) << (8 * (j & 3));
    }
  } else {
    byte = bad ? 0x7Fu : (uint32_t)f32x2_to_e4m3x2(__fdiv_rn(__fmul_rn(__uint_as_float(top), inv_r), 6.0f), 0.0f) & 0xffu;
    const float s = e4m3_to_f32(byte);
    const float2 s2 = splat2(s), r2 = splat2(inv_r);
    const float2 rs2 = splat2(s > 0.0f ? __fdiv_rn(1.0f, s) : 0.0f);  // under a scale of zero: zeros, with their signs
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      // the remainder of -0 is 0 and would make the quotient 0: the sign is x's
      const float2 q = div2_rn_by(mul2(v[j], r2), s2, rs2);
      w[j >> 2] |= e2m1x2(copysignf(q.x, v[j].x), copysignf(q.y, v[j].y)) << (8 * (j & 3));
    }
  }
  if (bad) w[0] = w[1] = 0u;
  return byte;
}
// bits of the largest magnitude; above infinity's where there is a NaN
__device__ __forceinline__ uint32_t absmax16(const float2 (&v)[8]) {
  float m = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) asm("max.NaN.abs.f32 %0, %0, %1, %2;" : "+f"(m) : "f"(v[j].x), "f"(v[j].y));
  return __float_as_uint(m) & 0x7FFFFFFFu;
}
// The exponent of an nvfp4 row's scale from its absmax's bits: least e with absmax <= 2688 * 2^e =
// 1.3125 * 2^(11 + e), at least -126; 0 for a row of zeros.
__device__ __forceinline__ int row_exponent(uint32_t top) {
  return top ? max((int)(top >> 23) - 138 + ((top & 0x7FFFFFu) > 0x280000u ? 1 : 0), -126) : 0;
}
__device__ __forceinline__ float exp2_bits(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }  // -126 <= e <= 127
// Four blocks' scale bytes to a word, in all lanes that share it: those of four lanes with a
// chunk each (nvfp4) or of four pairs of lanes (mxfp4).
template <int FORMAT>
struct ScaleWord {
  static constexpr int kLanes = FORMAT == kMxfp4 ? 8 : 4;
  __device__ __forceinline__ static uint32_t of(uint32_t byte, int lane) {
    uint32_t word = byte << (8 * ((lane / (kLanes / 4)) & 3));
#pragma unroll
    for (int o = kLanes / 4; o < kLanes; o *= 2) word |= __shfl_xor_sync(0xffffffffu, word, o);
    return word;
  }
};

}  // namespace h3b
