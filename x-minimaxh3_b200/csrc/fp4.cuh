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
};
// 0 ok, 1 tensor-map encoding failed, 2 CUDA error (*err)
int launch_fp4_gemm(const Fp4RowsView& x, const Fp4RowsView& w, Fp4GemmArgs a, int format, cudaStream_t s,
                    cudaError_t* err);

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
  return (uint32_t)f32_to_half_bits<BF16>(lo) | ((uint32_t)f32_to_half_bits<BF16>(hi) << 16);
}

}  // namespace h3b
