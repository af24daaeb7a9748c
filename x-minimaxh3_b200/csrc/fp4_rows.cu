// fp4_rows.cu -- rows to microscaled 4-bit floats (mxfp4, nvfp4) and back, and the residual
// addition + RMSNorm whose output goes to INT8 or 4-bit rows in the same pass.
//
// One row is held in registers by one warp (up to 1,024 columns) or one block: each thread
// has one to four chunks of 16 columns, so the row is read once, and everything that is
// asked of the whole row (sum of squares, absmax) is a reduction over registers.  A chunk is
// an nvfp4 block, two neighbouring lanes hold an mxfp4 block, and four or eight lanes the
// four scales of a word.
//
// mxfp4's scales and the nvfp4 row scale are powers of two read off the absmax's bits, which is
// exact.  The remaining quotients (absmax / 6 to E4M3, x / scale to E2M1) are correctly rounded
// before they are rounded to the narrow type.  For 16-bit inputs that gives the nearest code of
// the exact quotient, ties included: quotient and border differ by more than the fp32 rounding
// or not at all, since the border times the scale has fewer than 24 bits.
//
// Infinities and NaN: the block's scale becomes NaN (all of it is lost, and seen to be); the
// row scale goes by the other blocks.  An INT8 row with one gets the scale NaN or infinity.
#include <cfloat>

#include "fp4.cuh"

namespace h3b {

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

// 16 columns from chunk c (of 16 columns) on, zeros beyond K; neighbouring lanes of a warp ask for
// neighbouring chunks.  VEC: all pointers and strides allow 16-byte accesses and K is a multiple
// of 16.  Otherwise the warp moves its 512 columns together, through `stage`, in words or 16-bit
// pieces as the row's address allows (a lane's own 16 pieces would be 32 bytes apart from its
// neighbours': 3,607 rows of 1,044 columns to nvfp4 and back took 34 us that way).
template <bool VEC>
__device__ __forceinline__ void load16_raw(const uint16_t* row, int c, int K, uint16_t* stage, uint4& a, uint4& b) {
  a = b = make_uint4(0u, 0u, 0u, 0u);
  if constexpr (VEC) {
    if (c * 16 < K) {
      a = *reinterpret_cast<const uint4*>(row + c * 16);
      b = *reinterpret_cast<const uint4*>(row + c * 16 + 8);
    }
  } else {
    const int lane = threadIdx.x & 31, base = (c - lane) * 16, n = K - base;
    const uint16_t* src = row + base;
    if ((reinterpret_cast<uintptr_t>(row) & 3) == 0) {
      uint32_t w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int at = j * 64 + lane * 2;
        w[j] = at + 1 < n ? *reinterpret_cast<const uint32_t*>(src + at) : at < n ? (uint32_t)src[at] : 0u;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) reinterpret_cast<uint32_t*>(stage)[j * 32 + lane] = w[j];
    } else {
      uint16_t h[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) h[j] = j * 32 + lane < n ? src[j * 32 + lane] : (uint16_t)0;
#pragma unroll
      for (int j = 0; j < 16; ++j) stage[j * 32 + lane] = h[j];
    }
    __syncwarp();
    a = *reinterpret_cast<const uint4*>(stage + lane * 16);
    b = *reinterpret_cast<const uint4*>(stage + lane * 16 + 8);
    __syncwarp();
  }
}
template <bool BF16>
__device__ __forceinline__ float2 unpack_halves(uint32_t w) {
  if constexpr (BF16) return unpack_bf16x2(w);
  else return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <bool BF16>
__device__ __forceinline__ void unpack16(const uint4& a, const uint4& b, float2 (&v)[8]) {
  const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = unpack_halves<BF16>(w[i]);
}
template <bool BF16, bool VEC>
__device__ __forceinline__ void load16(const uint16_t* row, int c, int K, uint16_t* stage, float2 (&v)[8]) {
  uint4 a, b;
  load16_raw<VEC>(row, c, K, stage, a, b);
  unpack16<BF16>(a, b, v);
}
template <bool BF16, bool VEC>
__device__ __forceinline__ void store16(uint16_t* row, int c, int K, uint16_t* stage, const float2 (&v)[8]) {
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = pack_halves<BF16>(v[i].x, v[i].y);
  const uint4 a = make_uint4(w[0], w[1], w[2], w[3]), b = make_uint4(w[4], w[5], w[6], w[7]);
  if constexpr (VEC) {
    if (c * 16 < K) {
      *reinterpret_cast<uint4*>(row + c * 16) = a;
      *reinterpret_cast<uint4*>(row + c * 16 + 8) = b;
    }
  } else {
    const int lane = threadIdx.x & 31, base = (c - lane) * 16, n = K - base;
    *reinterpret_cast<uint4*>(stage + lane * 16) = a;
    *reinterpret_cast<uint4*>(stage + lane * 16 + 8) = b;
    __syncwarp();
    uint16_t* dst = row + base;
    if ((reinterpret_cast<uintptr_t>(row) & 3) == 0) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int at = j * 64 + lane * 2;
        if (at + 1 < n) *reinterpret_cast<uint32_t*>(dst + at) = reinterpret_cast<const uint32_t*>(stage)[j * 32 + lane];
        else if (at < n) dst[at] = stage[at];
      }
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (j * 32 + lane < n) dst[j * 32 + lane] = stage[j * 32 + lane];
    }
    __syncwarp();
  }
}
// 16 int8 codes of chunk c (w: four to a word) into a row of K bytes
template <bool VEC>
__device__ __forceinline__ void store16_bytes(uint8_t* row, int c, int K, uint8_t* stage, const uint32_t (&w)[4]) {
  if constexpr (VEC) {
    if (c * 16 < K) *reinterpret_cast<uint4*>(row + c * 16) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
    const int lane = threadIdx.x & 31, base = (c - lane) * 16, n = K - base;
    *reinterpret_cast<uint4*>(stage + lane * 16) = make_uint4(w[0], w[1], w[2], w[3]);
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (j * 32 + lane < n) row[base + j * 32 + lane] = stage[j * 32 + lane];
    __syncwarp();
  }
}

// FORMAT 0: int8.  BLOCK: a row per block, else per warp.  CH chunks per thread.
template <int FORMAT, bool BF16, bool NORM, bool VEC, bool BLOCK, int CH>
__global__ void __launch_bounds__(512, CH <= 2 ? 2 : 1) fp4_rows_kernel(Fp4RowArgs a) {
  __shared__ uint32_t red[2][32];
  __shared__ __align__(16) uint16_t stages[VEC ? 1 : 16][VEC ? 8 : 512];
  chain_wait();
  chain_next();  // behind the wait: a product that follows may read its weight before it waits
  const int lane = threadIdx.x & 31;
  const int t = BLOCK ? (int)threadIdx.x : lane;
  const int step = BLOCK ? (int)blockDim.x : 32;
  const int64_t row = BLOCK ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (row >= a.rows) return;  // whole warps of a warp-per-row block
  uint16_t* stage = stages[VEC ? 0 : threadIdx.x >> 5];
  float2 v[CH][8];
#pragma unroll
  for (int i = 0; i < CH; ++i) load16<BF16, VEC>(a.x + row * a.x_stride, t + i * step, a.K, stage, v[i]);

  if constexpr (NORM) {
    if (a.res) {
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        float2 r[8];
        load16<BF16, VEC>(a.res + row * a.res_stride, t + i * step, a.K, stage, r);
#pragma unroll
        for (int j = 0; j < 8; ++j) {  // the sum as it is stored: what a later layer reads is what is normed here
          const float2 h = add2(v[i][j], r[j]);
          v[i][j] = unpack_halves<BF16>(pack_halves<BF16>(h.x, h.y));
        }
      }
#pragma unroll
      for (int i = 0; i < CH; ++i) store16<BF16, VEC>(a.sum + row * a.sum_stride, t + i * step, a.K, stage, v[i]);
    }
    float2 ss2 = splat2(0.0f);
#pragma unroll
    for (int i = 0; i < CH; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) ss2 = fma2(v[i][j], v[i][j], ss2);
    float ss = __fadd_rn(ss2.x, ss2.y);
    ss = row_sum<BLOCK>(ss, reinterpret_cast<float*>(red[0]));
    // Within 2 ulp, and common to the row.  A correctly rounded root and quotient take every thread longer
    // (16,384 x 512 into INT8 13.5 us, so 12.1; 8,190 x 4,096 37.4 and 37.1).
    const float inv = rsqrtf(__fadd_rn(__fdiv_rn(ss, (float)a.K), a.eps));
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int c = t + i * step;
      float2 w[8];
      load16<BF16, VEC>(a.norm_w, c, a.K, stage, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[i][j] = mul2(mul2(v[i][j], splat2(inv)), w[j]);
        // beyond K inv may have made a zero NaN
        if (!(VEC ? c * 16 < a.K : c * 16 + 2 * j < a.K)) v[i][j].x = 0.0f;
        if (!(VEC ? c * 16 < a.K : c * 16 + 2 * j + 1 < a.K)) v[i][j].y = 0.0f;
      }
    }
  }

  uint32_t top[CH];  // absmax bits of each block (of 16 columns for int8)
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    top[i] = absmax16(v[i]);
    if (FORMAT == kMxfp4) top[i] = max(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
  }

  if constexpr (FORMAT == 0) {
    uint32_t m = 0u;
#pragma unroll
    for (int i = 0; i < CH; ++i) m = max(m, top[i]);
    m = row_max<BLOCK>(m, red[1]);
    float scale = __fdiv_rn(__uint_as_float(m), 127.0f);  // NaN and infinity stay
    if (t == 0) a.row_scales[row] = scale;
    if (scale > 0.0f && scale < FLT_MIN) {
      // The reciprocal of a subnormal scale may be infinite: row and scale times 2^64.  The scale's own rounding
      // may have taken it so far below absmax / 127 that values go beyond 127 of them.
      const float up = exp2_bits(64);
      scale = __fmul_rn(scale, up);
      const float most = __fmul_rn(scale, 127.0f);
#pragma unroll
      for (int i = 0; i < CH; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          v[i][j] = mul2(v[i][j], splat2(up));
          v[i][j].x = fminf(fmaxf(v[i][j].x, -most), most);
          v[i][j].y = fminf(fmaxf(v[i][j].y, -most), most);
        }
    }
    const bool some = m < kInfBits && scale > 0.0f;
    const float rs = some ? __fdiv_rn(1.0f, scale) : 0.0f;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        // at most 127 and an fp32 rounding; rounded by adding 1.5 * 2^23, whose low byte is then the code
        const float2 q = some ? div2_rn_by(v[i][j], splat2(scale), splat2(rs)) : splat2(0.0f);
        const float2 n = add2(q, splat2(12582912.0f));
        w[j >> 1] |= (__byte_perm(__float_as_uint(n.x), __float_as_uint(n.y), 0x0040) & 0xffffu) << (16 * (j & 1));
      }
      store16_bytes<VEC>(a.codes + row * (int64_t)a.K, t + i * step, a.K, reinterpret_cast<uint8_t*>(stage), w);
    }
  } else {
    const int64_t pitch = fp4_pitch(a.K);
    const int groups = (int)fp4_groups(a.K, FORMAT);
    uint8_t* dst = a.codes + row * pitch;
    uint8_t* word0 = a.blocks + (row >> 7) * groups * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4;
    float inv_r = 1.0f;
    if constexpr (FORMAT == kNvfp4) {
      uint32_t m = 0u;
#pragma unroll
      for (int i = 0; i < CH; ++i) m = max(m, top[i] < kInfBits ? top[i] : 0u);
      const int e = row_exponent(row_max<BLOCK>(m, red[1]));
      inv_r = exp2_bits(-e);
      if (t == 0) a.row_scales[row] = exp2_bits(e);
    }
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int c = t + i * step;
      uint32_t w[2];
      const uint32_t byte = quantize16<FORMAT>(v[i], top[i], inv_r, w);
      if (c * 8 < pitch) *reinterpret_cast<uint2*>(dst + c * 8) = make_uint2(w[0], w[1]);
      const uint32_t word = ScaleWord<FORMAT>::of(byte, lane);
      constexpr int kLanes = ScaleWord<FORMAT>::kLanes;
      if ((lane & (kLanes - 1)) == 0 && c / kLanes < groups)
        *reinterpret_cast<uint32_t*>(word0 + (int64_t)(c / kLanes) * 512) = word;
    }
  }
}

// A code pair to its two elements
__device__ __forceinline__ float2 elements_of(uint32_t pair) {
  uint32_t h2;
  asm("{\n\t.reg .b8 t;\n\tcvt.u8.u32 t, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, t;\n\t}" : "=r"(h2) : "r"(pair));
  return unpack_halves<false>(h2);
}
// Codes and scales to 16-bit values: value = code * block scale * row scale.  A warp takes 1,024
// columns of a row, a thread eight at a time (16 bytes of output, so that a warp's store is 512
// bytes in a row: 16,384 x 4,096 with 16 columns a thread 33 us), or, where rows do not allow
// that, 512 columns through shared memory.  ROW: there are row scales.  Of mxfp4, one below 1 goes onto
// the block's first, which is a power of two, since the largest of those times an element of 4 or 6
// leaves fp32's range.
template <int FORMAT, bool ROW, bool BF16, bool VEC>
__global__ void __launch_bounds__(256) fp4_dequantize_kernel(Fp4RowsView a, uint16_t* out, int64_t out_stride,
                                                             uint32_t parts, int64_t total) {
  __shared__ __align__(16) uint16_t stages[VEC ? 1 : 8][VEC ? 8 : 512];
  chain_wait();
  chain_next();
  const int lane = threadIdx.x & 31;
  const int64_t at = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (at >= total) return;
  const int64_t row = total <= UINT32_MAX ? (int64_t)((uint32_t)at / parts) : at / parts;
  const int part = (int)(at - row * parts);
  const uint8_t* codes = a.codes + row * fp4_pitch(a.K);
  const uint8_t* blocks = a.blocks + (row >> 7) * fp4_groups(a.K, FORMAT) * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4;
  auto scale_byte = [&](int column) -> uint32_t {
    const int b = column / fp4_block(FORMAT);
    return blocks[(int64_t)(b >> 2) * 512 + (b & 3)];
  };
  const float r = ROW ? a.row_scales[row] : 1.0f;
  const bool first = ROW && FORMAT == kMxfp4 && fabsf(r) < 1.0f;
  auto scale_of = [&](uint32_t byte) {
    const float s = FORMAT == kMxfp4 ? e8m0_to_f32(byte) : e4m3_to_f32(byte);
    return splat2(first ? __fmul_rn(s, r) : s);
  };
  auto value_of = [&](uint32_t pair, float2 s) {
    const float2 v = mul2(elements_of(pair), s);
    return ROW ? mul2(v, splat2(first ? 1.0f : r)) : v;
  };
  if constexpr (VEC) {
    uint32_t q[4], byte[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = part * 1024 + i * 256 + lane * 8;
      q[i] = c < a.K ? *reinterpret_cast<const uint32_t*>(codes + c / 2) : 0u;
      byte[i] = c < a.K ? scale_byte(c) : 0u;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = part * 1024 + i * 256 + lane * 8;
      const float2 s = scale_of(byte[i]);
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 v = value_of((q[i] >> (8 * j)) & 0xffu, s);
        w[j] = pack_halves<BF16>(v.x, v.y);
      }
      if (c < a.K) *reinterpret_cast<uint4*>(out + row * out_stride + c) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  } else {
    const int c = part * 32 + lane;
    float2 v[8] = {};
    if (c * 16 < a.K) {
      const uint2 q = *reinterpret_cast<const uint2*>(codes + c * 8);
      const float2 s = scale_of(scale_byte(c * 16));
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = value_of(((j < 4 ? q.x : q.y) >> (8 * (j & 3))) & 0xffu, s);
    }
    store16<BF16, VEC>(out + row * out_stride, c, a.K, stages[threadIdx.x >> 5], v);
  }
}

// ------------------------------------------------------------------ host side

int num_sms();

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
  // Two chunks a thread in long rows where there are some for all SMs: fewer warps meet for a row's
  // sum (4,000 x 4,096 normed into nvfp4 27.0 -> 21.6 us, from 16-bit rows 13.5 -> 10.7); one for a
  // few rows (1 x 4,096 into INT8 2.8 us, with two 3.2) and short ones (3,607 x 1,044 into nvfp4 6.2,
  // with two 7.4).
  const bool two = a.rows >= 4 * num_sms() && chunks >= (VEC ? 128 : 256);
  const int ch = chunks > 1024 ? 4 : chunks > 512 || two ? 2 : 1;
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

template <int FORMAT, bool ROW, bool BF16>
static cudaError_t launch_dequantize(const Fp4RowsView& a, uint16_t* out, int64_t stride, cudaStream_t s) {
  const bool vec = a.K % 16 == 0 && rows16(out, stride);
  const uint32_t parts = (uint32_t)(vec ? (a.K + 1023) / 1024 : (a.K + 511) / 512);
  const int64_t total = a.rows * parts, grid = (total + 7) / 8;
  return vec ? launch_chained(fp4_dequantize_kernel<FORMAT, ROW, BF16, true>, grid, 256, 0, s, a, out, stride, parts, total)
             : launch_chained(fp4_dequantize_kernel<FORMAT, ROW, BF16, false>, grid, 256, 0, s, a, out, stride, parts, total);
}
template <int FORMAT>
static cudaError_t launch_dequantize_as(const Fp4RowsView& a, uint16_t* out, int64_t stride, bool bf16, cudaStream_t s) {
  if (a.row_scales)
    return bf16 ? launch_dequantize<FORMAT, true, true>(a, out, stride, s) : launch_dequantize<FORMAT, true, false>(a, out, stride, s);
  return bf16 ? launch_dequantize<FORMAT, false, true>(a, out, stride, s) : launch_dequantize<FORMAT, false, false>(a, out, stride, s);
}
cudaError_t launch_fp4_dequantize(const Fp4RowsView& a, int format, uint16_t* out, int64_t out_stride, bool bf16,
                                  cudaStream_t s) {
  return format == kMxfp4 ? launch_dequantize_as<kMxfp4>(a, out, out_stride, bf16, s)
                          : launch_dequantize_as<kNvfp4>(a, out, out_stride, bf16, s);
}

}  // namespace h3b
