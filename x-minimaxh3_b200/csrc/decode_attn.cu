// decode_attn.cu -- attention of one new token per sequence over a paged K/V cache.
//
//   out[h] = sum_j softmax_j(scale * q[h] . k_j) v_j over the visible keys j
//
// Bound by reading K and V once: 1 flop per byte and head of a group.  The keys are cut
// into chunks of 16 (inside one page) and the chunks of all (sequence, kv head) pairs into
// one list that every warp of a persistent grid takes an equal, contiguous part of, so
// ragged lengths and few long sequences load the card alike.  A pair whose chunks span
// several warps is joined by a second kernel from fp32 partial sums with their softmax
// statistics.  Few short sequences are bound by latency and take one launch of clusters.
//
// Measured, 32 heads of 8 kv heads: 2 sequences of 150,000 bf16 tokens 182 us, 6.3 TB/s of
// K and V; 96 ragged sequences of about 3,500 E4M3 tokens 110 us, 5.4 TB/s; one of 701
// tokens 6.3 us on the device.
//
// A warp keeps its chunk in registers, without shared memory:
//   S^T = K . Q^T   m16n8k16, M = 16 keys, N = 8 heads of the group.  The products'
//                   order over the 128 channels is free, so each thread loads 16
//                   contiguous bytes of its key rows and the matching ones of Q.
//   P^T             exp2 of S^T under the running maximum, rounded to the 16-bit type of the
//                   V product (its sum is not: one more rounding of the weights, relative
//                   2^-9 in bf16 and 2^-12 in fp16, that tensor cores ask for); the accumulator
//                   layout of S^T becomes the B operand by one 8 x 8 transpose per 8 keys
//   O^T += V^T . P^T  M = 16 channels, N = 8 heads, K = 16 keys: the A operand pairs
//                   two keys of one channel, one byte permute per register
// E4M3 caches are widened to fp16 (exact), with a bf16 q in fp16 under a power of two per head
// that brings its largest channel to [1, 2).  Channels of 2^-17 and more are exact then; smaller
// ones round to multiples of 2^-24, an error of the size that an fp32 sum with the largest
// channel's product has anyway (only where that channel's keys are 0 it would not).
#include "streaming.cuh"

namespace h3b {

namespace {

constexpr int kDecodeThreads = 128;
constexpr int kChunk = 16;
// P = 2^(x - m) times 2^kHalfUp where it rounds to fp16 (16-bit fp16 caches, and E4M3 ones,
// whose V widens to fp16): its peak is then 2^15, below fp16's largest value, and a weight
// keeps fp16's 11 bits down to 2^-29 of the largest (without the factor to 2^-14, and none
// below 2^-25: 32,768 keys 23.4 octaves below a first token came out 32 % too heavy).  The
// row sum has the same factor, so it leaves in O / l, and every piece has it, so the joins
// need not know.  bf16 has fp32's exponents and needs none.
constexpr float kHalfUp = 15.f;

template <bool BF16>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  if constexpr (BF16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
// Streamed once: no place in L1.  Not a read-only (.nc) load: an append that this kernel
// follows may still be writing these pages when this kernel is launched.
__device__ __forceinline__ uint4 ld_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// two E4M3 bytes (low half of w, or high half) -> two fp16
__device__ __forceinline__ uint32_t widen_lo(uint32_t w) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ uint32_t widen_hi(uint32_t w) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}" : "=r"(r) : "r"(w));
  return r;
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  if constexpr (BF16) return bf16x2_bits(lo, hi);
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// workspace: int64 prefix[kDecodeMaxSeqs + 1] (chunks before each sequence, one kv head
// and row group), int64 share; then per (worker, slot) R rows of 128 sums and of (m, l)
constexpr int64_t kDecodeHeader = (kDecodeMaxSeqs + 2) * 8;

// The chunks of a sequence: those of the first tokens, then those of the window.
struct ChunkList {
  int first_n;  // chunks of the first tokens (0 when the window's chunks join them)
  int win;      // first chunk of the window
  int n;
};
__device__ __forceinline__ ChunkList chunk_list(const VisibleKeys& v) {
  const int end = (v.end + kChunk - 1) / kChunk, firsts = (v.sinks + kChunk - 1) / kChunk, win = v.lo / kChunk;
  if (v.lo >= v.end) return {firsts, end, firsts};  // no windowed key
  if (v.sinks == 0) return {0, win, end - win};
  if (firsts >= win) return {0, 0, end};
  return {firsts, win, firsts + end - win};
}

template <int NT>
__device__ __forceinline__ float* partial_rows(float* ws, int64_t worker, int slot) {
  return ws + kDecodeHeader / 4 + (worker * 2 + slot) * (int64_t)(NT * 8) * 128;
}
template <int NT>
__device__ __forceinline__ float* partial_stats(float* ws, int64_t workers, int64_t worker, int slot) {
  return ws + kDecodeHeader / 4 + workers * 2 * (int64_t)(NT * 8) * 128 + (worker * 2 + slot) * (int64_t)(NT * 16);
}

// A warp's chunks [c0, c1) of one sequence (b, in table row `slot`) and eight or 16 heads
// from r0 of kv head kh: unnormalised sums o, maxima m (in powers of two) and row sums l.
template <bool BF16, bool FP8, int NT>
__device__ __forceinline__ void decode_chunks(const DecodeArgs& a, int b, int slot, const VisibleKeys& see,
                                              const ChunkList& cl, int kh, int r0, int c0, int c1, float (&o)[NT][8][4],
                                              float (&m)[NT][2], float (&l)[NT][2]) {
  const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3, group = a.Hq / a.Hkv;
  // Q of head r0 + 8 t + g: the channels this thread's K loads bring
  uint32_t qf[NT][8][2];
  float sc[NT][2];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int r = r0 + t * 8 + g;
    const uint16_t* qp = a.q + b * a.q_stride + ((int64_t)kh * group + r) * 128;
    uint4 w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // 16-bit: channels 32 i + 8 c + 0..7; E4M3: 64 (i / 2) + 16 c + 8 (i % 2) + 0..7
      const int d = FP8 ? (i >> 1) * 64 + c * 16 + (i & 1) * 8 : i * 32 + c * 8;
      w[i] = r < group ? *reinterpret_cast<const uint4*>(qp + d) : make_uint4(0, 0, 0, 0);
    }
    float up = 1.f;
    if constexpr (FP8 && BF16) {
      // bf16 q -> fp16 under a power of two: the head's largest |q| comes to [1, 2)
      float mx = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t ws[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) mx = fmaxf(mx, fmaxf(fabsf(bf16_lo(ws[e])), fabsf(bf16_hi(ws[e]))));
      }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const int ex = (int)(__float_as_uint(mx) >> 23) - 127;  // of a normal, finite maximum
      float down = 1.f;
      if (mx > 0.f && ex > -126 && ex < 127) {
        up = __uint_as_float((uint32_t)(ex + 127) << 23);
        down = __uint_as_float((uint32_t)(127 - ex) << 23);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t* ws = reinterpret_cast<uint32_t*>(&w[i]);
#pragma unroll
        for (int e = 0; e < 4; ++e) ws[e] = pack16<false>(bf16_lo(ws[e]) * down, bf16_hi(ws[e]) * down);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      qf[t][2 * i][0] = w[i].x;
      qf[t][2 * i][1] = w[i].y;
      qf[t][2 * i + 1][0] = w[i].z;
      qf[t][2 * i + 1][1] = w[i].w;
    }
    const float s = a.scale_log2 * (FP8 ? a.k_scale[kh] : 1.f);
    // the score columns of this thread are heads 2c and 2c + 1 of the tile
    sc[t][0] = s * __shfl_sync(0xffffffffu, up, 8 * c);
    sc[t][1] = s * __shfl_sync(0xffffffffu, up, 8 * c + 4);
  }

#pragma unroll
  for (int t = 0; t < NT; ++t) {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[t][i][0] = o[t][i][1] = o[t][i][2] = o[t][i][3] = 0.f;
    m[t][0] = m[t][1] = -INFINITY;
    l[t][0] = l[t][1] = 0.f;
  }

  constexpr int kEB = FP8 ? 1 : 2;  // bytes per element
  constexpr int kKL = FP8 ? 2 : 4;  // 16-byte loads of a key row per thread
  constexpr int kVL = FP8 ? 1 : 2;
  constexpr int CH = FP8 ? 2 : 1;   // chunks of a step: 8 KB of K and V under way per warp either way
  uint4 kr[CH][2][kKL], vr[CH][4][kVL];
  int pgs = 0, pbase = c0 - 64;
  auto chunk_of = [&](int ord) { return ord < cl.first_n ? ord : ord - cl.first_n + cl.win; };
  // byte offset of key row 0 of chunk ordinal `ord`; page numbers come 32 chunks at a
  // time (an ordinal past the piece stands for its last)
  auto offset_of = [&](int ord) -> int64_t {
    if (ord - pbase >= 32) {
      pbase = ord;
      const int o2 = min(ord + lane, c1 - 1);
      pgs = (int)paged_page(a.paged, slot, chunk_of(o2) * kChunk / a.paged.page);
    }
    const int64_t pg = __shfl_sync(0xffffffffu, pgs, ord - pbase);
    const int j = chunk_of(min(ord, c1 - 1)) * kChunk;
    return ((pg * a.Hkv + kh) * a.paged.page + (j & (a.paged.page - 1))) * (int64_t)(128 * kEB);
  };
  auto load_k = [&](const int64_t (&off)[CH]) {
#pragma unroll
    for (int u = 0; u < CH; ++u) {
      const uint8_t* p = static_cast<const uint8_t*>(a.paged.k) + off[u] + g * (128 * kEB) + c * 16;
#pragma unroll
      for (int i = 0; i < kKL; ++i) {
        kr[u][0][i] = ld_stream(p + i * 64);
        kr[u][1][i] = ld_stream(p + i * 64 + 8 * 128 * kEB);
      }
    }
  };
  auto load_v = [&](const int64_t (&off)[CH]) {
#pragma unroll
    for (int u = 0; u < CH; ++u) {
      const uint8_t* p = static_cast<const uint8_t*>(a.paged.v) + off[u] + 2 * c * (128 * kEB) + g * 16;
#pragma unroll
      for (int i = 0; i < kVL; ++i) {
        vr[u][0][i] = ld_stream(p + i * 128);
        vr[u][1][i] = ld_stream(p + i * 128 + 128 * kEB);
        vr[u][2][i] = ld_stream(p + i * 128 + 8 * 128 * kEB);
        vr[u][3][i] = ld_stream(p + i * 128 + 9 * 128 * kEB);
      }
    }
  };
  int64_t off[CH];
#pragma unroll
  for (int u = 0; u < CH; ++u) off[u] = offset_of(c0 + u);
  load_k(off);
  load_v(off);
  for (int ord = c0; ord < c1; ord += CH) {
    float s[CH][NT][4];
#pragma unroll
    for (int u = 0; u < CH; ++u) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float(&st)[4] = s[u][t];
        st[0] = st[1] = st[2] = st[3] = 0.f;
#pragma unroll
        for (int i = 0; i < kKL; ++i) {
          const uint4 &x = kr[u][0][i], &y = kr[u][1][i];
          if constexpr (FP8) {
            const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int e = 0; e < 4; ++e)
              mma16816<false>(st, widen_lo(xs[e]), widen_lo(ys[e]), widen_hi(xs[e]), widen_hi(ys[e]),
                              qf[t][4 * i + e][0], qf[t][4 * i + e][1]);
          } else {
            mma16816<BF16>(st, x.x, y.x, x.y, y.y, qf[t][2 * i][0], qf[t][2 * i][1]);
            mma16816<BF16>(st, x.z, y.z, x.w, y.w, qf[t][2 * i + 1][0], qf[t][2 * i + 1][1]);
          }
        }
      }
    }
    const bool more = ord + CH < c1;
    if (more) {
#pragma unroll
      for (int u = 0; u < CH; ++u) off[u] = offset_of(ord + CH + u);
      load_k(off);
    }
    uint32_t hide[CH];  // bit 0: key j0 + g of the chunk is invisible, bit 1: key j0 + g + 8
#pragma unroll
    for (int u = 0; u < CH; ++u) {
      const int j0 = chunk_of(ord + u) * kChunk;
      const bool past = ord + u >= c1;
      hide[u] = 0;
      if (past || !(j0 + kChunk <= see.end && (j0 >= see.lo || j0 + kChunk <= see.sinks))) {
        auto seen = [&](int j) { return !past && j < see.end && (j >= see.lo || j < see.sinks); };
        hide[u] = (seen(j0 + g) ? 0u : 1u) | (seen(j0 + g + 8) ? 0u : 2u);
        // what lies in invisible rows (stale or never written) must not meet P = 0
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          if (!seen(j0 + 2 * c + (kk & 1) + (kk >> 1) * 8)) {
#pragma unroll
            for (int i = 0; i < kVL; ++i) vr[u][kk][i] = make_uint4(0, 0, 0, 0);
          }
        }
      }
    }
    uint32_t pb[CH][NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float x[CH][4];
      float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
      for (int u = 0; u < CH; ++u) {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[u][e] = (hide[u] >> (e >> 1)) & 1u ? -INFINITY : s[u][t][e] * sc[t][e & 1];
        mx0 = fmaxf(mx0, fmaxf(x[u][0], x[u][2]));
        mx1 = fmaxf(mx1, fmaxf(x[u][1], x[u][3]));
      }
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) {
        mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, d));
        mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, d));
      }
      const float n0 = fmaxf(m[t][0], mx0), n1 = fmaxf(m[t][1], mx1);
      if (__any_sync(0xffffffffu, n0 != m[t][0] || n1 != m[t][1])) {
        const float a0 = n0 == m[t][0] ? 1.f : exp2_fast(m[t][0] - n0);
        const float a1 = n1 == m[t][1] ? 1.f : exp2_fast(m[t][1] - n1);
        m[t][0] = n0;
        m[t][1] = n1;
        l[t][0] *= a0;
        l[t][1] *= a1;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          o[t][i][0] *= a0;
          o[t][i][1] *= a1;
          o[t][i][2] *= a0;
          o[t][i][3] *= a1;
        }
      }
      // a maximum of -inf (nothing seen yet) subtracts as 0: exp2(-inf) = 0
      constexpr float up = BF16 && !FP8 ? 0.f : kHalfUp;
      const float f0 = n0 == -INFINITY ? 0.f : n0 - up, f1 = n1 == -INFINITY ? 0.f : n1 - up;
#pragma unroll
      for (int u = 0; u < CH; ++u) {
        const float p0 = exp2_fast(x[u][0] - f0), p1 = exp2_fast(x[u][1] - f1);
        const float p2 = exp2_fast(x[u][2] - f0), p3 = exp2_fast(x[u][3] - f1);
        l[t][0] += p0 + p2;
        l[t][1] += p1 + p3;
        // P rounds to the 16-bit type of the V product; its sum stays in fp32
        pb[u][t][0] = transpose8x8(pack16<BF16 && !FP8>(p0, p1));
        pb[u][t][1] = transpose8x8(pack16<BF16 && !FP8>(p2, p3));
      }
    }
#pragma unroll
    for (int u = 0; u < CH; ++u) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        uint32_t w[4];
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          if constexpr (FP8) {
            const uint4& v = vr[u][kk][0];
            const uint32_t word = (i >> 1) == 0 ? v.x : (i >> 1) == 1 ? v.y : (i >> 1) == 2 ? v.z : v.w;
            w[kk] = (i & 1) ? widen_hi(word) : widen_lo(word);
          } else {
            const uint4& v = vr[u][kk][i >> 2];
            w[kk] = (i & 3) == 0 ? v.x : (i & 3) == 1 ? v.y : (i & 3) == 2 ? v.z : v.w;
          }
        }
        const uint32_t a0 = __byte_perm(w[0], w[1], 0x5410), a1 = __byte_perm(w[0], w[1], 0x7632);
        const uint32_t a2 = __byte_perm(w[2], w[3], 0x5410), a3 = __byte_perm(w[2], w[3], 0x7632);
#pragma unroll
        for (int t = 0; t < NT; ++t) mma16816<BF16 && !FP8>(o[t][i], a0, a1, a2, a3, pb[u][t][0], pb[u][t][1]);
      }
    }
    if (more) load_v(off);
  }

#pragma unroll
  for (int t = 0; t < NT; ++t) {
#pragma unroll
    for (int d = 4; d < 32; d <<= 1) {
      l[t][0] += __shfl_xor_sync(0xffffffffu, l[t][0], d);
      l[t][1] += __shfl_xor_sync(0xffffffffu, l[t][1], d);
    }
  }
}
// first channel of accumulator tile i of a thread: elements 0 / 1 are it, 2 / 3 the next
template <bool FP8>
__device__ __forceinline__ int tile_channel(int i) {
  const int g = (threadIdx.x & 31) >> 2;
  return FP8 ? g * 16 + 2 * i : (i >> 2) * 64 + g * 8 + (i & 3) * 2;
}

// FP8: E4M3 cache; BF16: type of q and out (and of a 16-bit cache); NT: 8-head groups
// a warp takes together.
template <bool BF16, bool FP8, int NT, int MINB>
__global__ void __launch_bounds__(kDecodeThreads, MINB) decode_kernel(DecodeArgs a) {
  extern __shared__ int64_t prefix[];  // [seqs + 1]
  __shared__ int64_t carry;
  __shared__ int64_t warp_sum[4];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
  const int group = a.Hq / a.Hkv;
  const int groups = (group + NT * 8 - 1) / (NT * 8);  // row groups of a kv head
  const int heads = a.Hkv * groups;                    // (kv head, row group) pairs

  if (threadIdx.x == 0) {
    carry = 0;
    prefix[0] = 0;
  }
  chain_next();
  chain_wait();
  __syncthreads();
  for (int base = 0; base < a.seqs; base += kDecodeThreads) {
    const int i = base + threadIdx.x;
    int64_t n = 0;
    if (i < a.seqs) {
      const int len = paged_len(a.paged, paged_slot(a.paged, i));
      n = chunk_list(visible_keys(a.rule, len - 1, len)).n;
    }
    int64_t x = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) warp_sum[warp] = x;
    __syncthreads();
    int64_t before = carry;
    for (int w = 0; w < warp; ++w) before += warp_sum[w];
    if (i < a.seqs) prefix[i + 1] = before + x;
    __syncthreads();
    if (threadIdx.x == kDecodeThreads - 1) carry = before + x;
    __syncthreads();
  }
  const int64_t total = prefix[a.seqs] * heads;
  const int64_t share = (total + a.workers - 1) / a.workers;
  if (blockIdx.x == 0) {
    int64_t* head = reinterpret_cast<int64_t*>(a.partial);
    for (int i = threadIdx.x; i <= a.seqs; i += kDecodeThreads) head[i] = prefix[i];
    if (threadIdx.x == 0) head[kDecodeMaxSeqs + 1] = share;
  }
  const int64_t worker = (int64_t)blockIdx.x * (kDecodeThreads / 32) + warp;
  int64_t at = worker * share;
  const int64_t stop = min(at + share, total);
  if (worker >= a.workers || at >= stop) return;

  int b;
  {
    int lo = 0, hi = a.seqs - 1;  // the last sequence whose chunks begin at or before `at`
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (prefix[mid] * heads <= at) lo = mid; else hi = mid - 1;
    }
    b = lo;
  }
  bool first_piece = true;
  while (at < stop) {
    while (prefix[b + 1] * heads <= at) ++b;
    const int64_t n_seq = prefix[b + 1] - prefix[b];
    const int64_t in_seq = at - prefix[b] * heads;
    const int hp = (int)(in_seq / n_seq);
    const int c0 = (int)(in_seq - hp * n_seq);
    const int c1 = (int)min(n_seq, (int64_t)c0 + (stop - at));
    const int kh = hp / groups, r0 = (hp % groups) * NT * 8;
    const int slot = paged_slot(a.paged, b);
    const int len = paged_len(a.paged, slot);
    const VisibleKeys see = visible_keys(a.rule, len - 1, len);
    const ChunkList cl = chunk_list(see);

    float o[NT][8][4];
    float m[NT][2], l[NT][2];
    decode_chunks<BF16, FP8, NT>(a, b, slot, see, cl, kh, r0, c0, c1, o, m, l);
    if (c0 == 0 && c1 == n_seq) {
      const float vs = FP8 ? a.v_scale[kh] : 1.f;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = r0 + t * 8 + 2 * c + e;
          if (r < group) {
            const float inv = (l[t][e] == 0.f ? 0.f : 1.f / l[t][e]) * vs;
            uint16_t* dst = a.out + b * a.out_stride + ((int64_t)kh * group + r) * 128;
#pragma unroll
            for (int i = 0; i < 8; i += 4) {
              uint4 w;
              w.x = pack16<BF16>(o[t][i][e] * inv, o[t][i][2 + e] * inv);
              w.y = pack16<BF16>(o[t][i + 1][e] * inv, o[t][i + 1][2 + e] * inv);
              w.z = pack16<BF16>(o[t][i + 2][e] * inv, o[t][i + 2][2 + e] * inv);
              w.w = pack16<BF16>(o[t][i + 3][e] * inv, o[t][i + 3][2 + e] * inv);
              *reinterpret_cast<uint4*>(dst + tile_channel<FP8>(i)) = w;
            }
          }
        }
      }
    } else {
      const int ps = first_piece ? 0 : 1;
      float* rows = partial_rows<NT>(a.partial, worker, ps);
      float* stats = partial_stats<NT>(a.partial, a.workers, worker, ps);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = t * 8 + 2 * c + e;
          if (r0 + r >= group) continue;
#pragma unroll
          for (int i = 0; i < 8; i += 2)
            *reinterpret_cast<float4*>(rows + r * 128 + tile_channel<FP8>(i)) =
                make_float4(o[t][i][e], o[t][i][2 + e], o[t][i + 1][e], o[t][i + 1][2 + e]);
          if (g == 0) *reinterpret_cast<float2*>(stats + r * 2) = make_float2(m[t][e], l[t][e]);
        }
      }
    }
    first_piece = false;
    at += c1 - c0;
  }
}

// Few pairs of short sequences (see launch_decode): a cluster of eight CTAs per (kv head,
// row group), its 32 warps an equal part of the chunks each, joined over distributed shared
// memory: one launch, no workspace, and no list of all chunks.
constexpr int kCluster = 8;
template <bool BF16, bool FP8, int NT>
__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kDecodeThreads, 2) decode_cluster_kernel(DecodeArgs a) {
  constexpr int kRows = NT * 8, kWarps = kDecodeThreads / 32, kParts = kCluster * kWarps;
  __shared__ float4 part[kWarps][kRows][32];
  __shared__ float2 stat[kWarps][kRows];
  __shared__ float4 acc_s[kDecodeThreads];
  __shared__ float2 stat_s[kDecodeThreads];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = lane & 3;
  const int group = a.Hq / a.Hkv, groups = (group + kRows - 1) / kRows, heads = a.Hkv * groups;
  const int pair = blockIdx.x / kCluster, b = pair / heads, hp = pair % heads;
  const int rank = (int)cluster_ctarank(), kh = hp / groups, r0 = (hp % groups) * kRows;
  chain_next();
  chain_wait();
  const int slot = paged_slot(a.paged, b), len = paged_len(a.paged, slot);
  const VisibleKeys see = visible_keys(a.rule, len - 1, len);
  const ChunkList cl = chunk_list(see);
  const int w = rank * kWarps + warp, c0 = cl.n * w / kParts, c1 = cl.n * (w + 1) / kParts;
  float o[NT][8][4], m[NT][2], l[NT][2];
  if (c0 < c1) {
    decode_chunks<BF16, FP8, NT>(a, b, slot, see, cl, kh, r0, c0, c1, o, m, l);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = t * 8 + 2 * c + e;
#pragma unroll
        for (int i = 0; i < 8; i += 2)
          part[warp][r][tile_channel<FP8>(i) / 4] = make_float4(o[t][i][e], o[t][i][2 + e], o[t][i + 1][e], o[t][i + 1][2 + e]);
        if (lane < 4) stat[warp][r] = make_float2(m[t][e], l[t][e]);
      }
    }
  } else {
    if (lane < kRows) stat[warp][lane] = make_float2(-INFINITY, 0.f);
  }
  cluster_sync_all();
  // this CTA's 16 channels of every row: four threads' pieces a row, the parts shared out
  constexpr int kPieces = kRows * 4, kSplits = kDecodeThreads / kPieces;
  const int piece = threadIdx.x % kPieces, r = piece >> 2, split = threadIdx.x / kPieces;
  float mx = -INFINITY, sum = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int i = 0; i < kParts / kSplits; ++i) {
    const int p = split * (kParts / kSplits) + i;
    const uint32_t st_at = mapa_shared(smem_u32(&stat[p % kWarps][r]), p / kWarps);
    const uint32_t at = mapa_shared(smem_u32(&part[p % kWarps][r][rank * 4 + (piece & 3)]), p / kWarps);
    float2 st;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(st.x), "=f"(st.y) : "r"(st_at));
    if (st.x == -INFINITY && st.y == 0.f) continue;  // no key: its sums were not written
    float4 x;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w) : "r"(at));
    const float m_new = st.x > mx || mx == -INFINITY ? st.x : mx;
    const float keep = mx == m_new ? 1.f : exp2f(mx - m_new), take = st.x == m_new ? 1.f : exp2f(st.x - m_new);
    mx = m_new;
    sum = sum * keep + st.y * take;
    acc = make_float4(fmaf(x.x, take, acc.x * keep), fmaf(x.y, take, acc.y * keep), fmaf(x.z, take, acc.z * keep),
                      fmaf(x.w, take, acc.w * keep));
  }
  acc_s[threadIdx.x] = acc;
  stat_s[threadIdx.x] = make_float2(mx, sum);
  cluster_sync_all();  // no CTA leaves while another reads its sums
  if (split == 0 && r0 + r < group) {
#pragma unroll
    for (int i = 1; i < kSplits; ++i) {
      const float2 st = stat_s[threadIdx.x + i * kPieces];
      const float4 x = acc_s[threadIdx.x + i * kPieces];
      if (st.x == -INFINITY && st.y == 0.f) continue;
      const float m_new = st.x > mx || mx == -INFINITY ? st.x : mx;
      const float keep = mx == m_new ? 1.f : exp2f(mx - m_new), take = st.x == m_new ? 1.f : exp2f(st.x - m_new);
      mx = m_new;
      sum = sum * keep + st.y * take;
      acc = make_float4(fmaf(x.x, take, acc.x * keep), fmaf(x.y, take, acc.y * keep), fmaf(x.z, take, acc.z * keep),
                        fmaf(x.w, take, acc.w * keep));
    }
    const float inv = (sum == 0.f ? 0.f : 1.f / sum) * (a.v_scale ? a.v_scale[kh] : 1.f);
    *reinterpret_cast<uint2*>(a.out + b * a.out_stride + ((int64_t)kh * group + r0 + r) * 128 + rank * 16 + (piece & 3) * 4) =
        make_uint2(pack16<BF16>(acc.x * inv, acc.y * inv), pack16<BF16>(acc.z * inv, acc.w * inv));
  }
}

// Joins the partial sums of a (kv head, row group): out = sum_p 2^(m_p - M) O_p /
// sum_p 2^(m_p - M) l_p.  A block per pair, its warps shared out over the rows and, where
// there are more of them, over the parts of a row; four channels per lane.  Pairs that one
// warp finished are left alone; pairs without any visible key give 0.  Blocks of 128
// threads where there are many pairs, of 512 where few pairs have many parts each.
template <bool BF16, int NT>
__global__ void __launch_bounds__(512) decode_join_kernel(DecodeArgs a) {
  __shared__ float4 acc_s[512];
  __shared__ float2 stat_s[16];
  const int group = a.Hq / a.Hkv, groups = (group + NT * 8 - 1) / (NT * 8), heads = a.Hkv * groups;
  const int b = blockIdx.x / heads, hp = blockIdx.x % heads;
  const int kh = hp / groups, first = (hp % groups) * NT * 8, rows = min(group - first, NT * 8);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int splits = max(warps / rows, 1), split = warp / rows;
  chain_next();
  chain_wait();
  const int64_t* prefix = reinterpret_cast<const int64_t*>(a.partial);
  const int64_t share = prefix[kDecodeMaxSeqs + 1], before = prefix[b], n = prefix[b + 1] - before;
  const int64_t s0 = before * heads + hp * n, s1 = s0 + n;
  const int64_t w0 = n ? s0 / share : 0, w1 = n ? (s1 - 1) / share : 0;
  if ((n && w0 == w1) || (splits == 1 && split > 0)) return;
  const int parts = (int)(w1 - w0 + 1);
  // only the first part can lie in its worker's second slot: a later worker begins in the pair
  const int head_slot = n && w0 * share < s0 ? 1 : 0;
  for (int r = warp % rows; r < rows; r += warps) {  // once, unless there are more rows than warps
    uint16_t* dst = a.out + b * a.out_stride + ((int64_t)kh * group + first + r) * 128 + lane * 4;
    float m = -INFINITY, l = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    if (split < splits && n) {
      for (int p0 = split; p0 < parts; p0 += 4 * splits) {
        float2 st[4];
        float4 x[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int p = p0 + u * splits;
          const bool in = p < parts;
          const int64_t w = w0 + (in ? p : 0);
          const int slot = p == 0 ? head_slot : 0;
          st[u] = in ? *reinterpret_cast<const float2*>(partial_stats<NT>(a.partial, a.workers, w, slot) + r * 2)
                     : make_float2(-INFINITY, 0.f);
          x[u] = in ? *reinterpret_cast<const float4*>(partial_rows<NT>(a.partial, w, slot) + r * 128 + lane * 4)
                    : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        float mx = m;
#pragma unroll
        for (int u = 0; u < 4; ++u) mx = fmaxf(mx, st[u].x);
        const float base = mx == -INFINITY ? 0.f : mx, keep = exp2f(m - base);
        m = mx;
        l *= keep;
        acc = make_float4(acc.x * keep, acc.y * keep, acc.z * keep, acc.w * keep);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const float w = exp2f(st[u].x - base);
          l = fmaf(w, st[u].y, l);
          acc = make_float4(fmaf(w, x[u].x, acc.x), fmaf(w, x[u].y, acc.y), fmaf(w, x[u].z, acc.z), fmaf(w, x[u].w, acc.w));
        }
      }
    }
    if (splits > 1) {  // then rows <= warps / 2, and every warp passes here once
      acc_s[threadIdx.x] = acc;
      if (lane == 0) stat_s[warp] = make_float2(m, l);
      __syncthreads();
      if (split > 0) return;
      const float own = m;
      for (int i = 1; i < splits; ++i) m = fmaxf(m, stat_s[r + i * rows].x);
      const float base = m == -INFINITY ? 0.f : m, keep = exp2f(own - base);
      l *= keep;
      acc = make_float4(acc.x * keep, acc.y * keep, acc.z * keep, acc.w * keep);
      for (int i = 1; i < splits; ++i) {
        const float2 st = stat_s[r + i * rows];
        const float4 x = acc_s[(r + i * rows) * 32 + lane];
        const float w = exp2f(st.x - base);
        l = fmaf(w, st.y, l);
        acc = make_float4(fmaf(w, x.x, acc.x), fmaf(w, x.y, acc.y), fmaf(w, x.z, acc.z), fmaf(w, x.w, acc.w));
      }
    }
    const float inv = (l == 0.f ? 0.f : 1.f / l) * (a.v_scale ? a.v_scale[kh] : 1.f);
    *reinterpret_cast<uint2*>(dst) =
        make_uint2(pack16<BF16>(acc.x * inv, acc.y * inv), pack16<BF16>(acc.z * inv, acc.w * inv));
  }
}

int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return 0;
  return n;
}

// One wave of clusters (two CTAs per multiprocessor) and at most eight chunks a warp.
// capacity: the tokens that a table row can name, for the host does not know the lengths.
// Decode of one 701-token sequence, 32/8 heads, on the device: 6.3 us in a table of 720
// tokens, and 10.5 us by the list of all chunks, as in a table of 32,768.
bool decode_by_clusters(int64_t seqs, int64_t Hq, int64_t Hkv, int64_t capacity) {
  const int64_t group = Hq / Hkv, rows = group > 8 ? 16 : 8;
  const int64_t pairs = seqs * Hkv * ((group + rows - 1) / rows);
  return pairs * kCluster <= 2 * (int64_t)sm_count() && capacity <= kCluster * (kDecodeThreads / 32) * 8 * kChunk;
}

template <bool BF16, bool FP8, int NT, int MINB>
cudaError_t launch_decode(DecodeArgs a, cudaStream_t s) {
  const int sms = sm_count();
  if (sms <= 0) return cudaErrorNoDevice;
  const int group = a.Hq / a.Hkv;
  const int64_t heads = (int64_t)a.Hkv * ((group + NT * 8 - 1) / (NT * 8));
  const int64_t most = (int64_t)a.seqs * heads * (((int64_t)a.paged.width * a.paged.page + kChunk - 1) / kChunk);
  if (decode_by_clusters(a.seqs, a.Hq, a.Hkv, (int64_t)a.paged.width * a.paged.page))
    return launch_chained(decode_cluster_kernel<BF16, FP8, NT>, a.seqs * heads * kCluster, kDecodeThreads, 0, s, a);
  constexpr int kWarps = kDecodeThreads / 32;
  int64_t blocks = (most + kWarps - 1) / kWarps;
  if (blocks > (int64_t)sms * MINB) blocks = (int64_t)sms * MINB;
  if (blocks < 1) blocks = 1;
  a.workers = (int)blocks * kWarps;
  const size_t smem = (size_t)(a.seqs + 1) * 8;
  const cudaError_t e = launch_chained(decode_kernel<BF16, FP8, NT, MINB>, blocks, kDecodeThreads, smem, s, a);
  if (e != cudaSuccess) return e;
  const int64_t pairs = a.seqs * heads;
  return launch_chained(decode_join_kernel<BF16, NT>, pairs, pairs >= 2 * sms ? 128 : 512, 0, s, a);
}

}  // namespace

int64_t decode_workspace_bytes(int64_t seqs, int64_t Hq, int64_t Hkv, int64_t capacity) {
  const int sms = sm_count();
  if (decode_by_clusters(seqs, Hq, Hkv, capacity)) return 0;
  // two pieces per warp; two blocks per SM with 16 rows a piece (more than three with 8)
  return kDecodeHeader + (int64_t)sms * 2 * (kDecodeThreads / 32) * 2 * 16 * (128 + 2) * 4;
}

cudaError_t launch_decode_attention(DecodeArgs a, int kind, cudaStream_t s) {
  const bool wide = a.Hq / a.Hkv > 8;
  switch (kind) {
    case 0: return wide ? launch_decode<true, false, 2, 2>(a, s) : launch_decode<true, false, 1, 3>(a, s);
    case 1: return wide ? launch_decode<false, false, 2, 2>(a, s) : launch_decode<false, false, 1, 3>(a, s);
    case 2: return wide ? launch_decode<true, true, 2, 2>(a, s) : launch_decode<true, true, 1, 3>(a, s);
    default: return wide ? launch_decode<false, true, 2, 2>(a, s) : launch_decode<false, true, 1, 3>(a, s);
  }
}

}  // namespace h3b
