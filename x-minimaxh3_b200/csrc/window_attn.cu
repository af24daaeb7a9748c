// window_attn.cu -- causal attention with a sliding window and visible first tokens
// over contiguous K/V of a ragged batch, or over a paged cache.
#include "streaming.cuh"

namespace h3b {

template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (BF16) return bf16x2_bits(lo, hi);
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// One warp per (query row, head), four channels per lane, one key at a time.
template <bool BF16>
__global__ void __launch_bounds__(256) window_row_kernel(WindowArgs a) {
  const int64_t unit = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (unit >= (int64_t)a.Tq * a.Hq) return;
  const int row = (int)(unit / a.Hq), h = (int)(unit % a.Hq), kh = h / (a.Hq / a.Hkv);
  int seq = -1;
  RowRange qr{0, 0};
  for (int i = 0; i < a.seqs; ++i) {
    qr = row_range(a.q_starts, i, a.Tq);
    if (row >= qr.a && row < qr.b) {
      seq = i;
      break;
    }
  }
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  if (seq >= 0) {
    const bool paged = a.paged.k != nullptr;
    int slot = -1, lk;
    RowRange kr{0, 0};
    if (paged) {
      slot = paged_slot(a.paged, seq);
      lk = paged_len(a.paged, slot);
    } else {
      kr = row_range(a.k_starts, seq, a.Tk);
      lk = kr.b - kr.a;
    }
    const uint2 qw = *reinterpret_cast<const uint2*>(a.q + row * a.q_stride + h * 128 + lane * 4);
    const float2 q0 = unpack2<BF16>(qw.x), q1 = unpack2<BF16>(qw.y);
    const VisibleKeys see = visible_keys(a.rule, lk - (qr.b - qr.a) + (row - qr.a), lk);
    for (int j = 0; j < see.end; ++j) {
      if (j == see.sinks && j < see.lo) j = see.lo;
      if (j >= see.end) break;
      const uint16_t *kp, *vp;
      if (paged) {
        const int64_t at = ((paged_page(a.paged, slot, j / a.paged.page) * a.Hkv + kh) * a.paged.page +
                            j % a.paged.page) * 128 + lane * 4;
        kp = static_cast<const uint16_t*>(a.paged.k) + at;
        vp = static_cast<const uint16_t*>(a.paged.v) + at;
      } else {
        kp = a.k + (kr.a + j) * a.k_stride + kh * 128 + lane * 4;
        vp = a.v + (kr.a + j) * a.v_stride + kh * 128 + lane * 4;
      }
      const uint2 kw = *reinterpret_cast<const uint2*>(kp);
      const uint2 vw = *reinterpret_cast<const uint2*>(vp);
      const float2 k0 = unpack2<BF16>(kw.x), k1 = unpack2<BF16>(kw.y);
      float s = fmaf(q0.x, k0.x, fmaf(q0.y, k0.y, fmaf(q1.x, k1.x, q1.y * k1.y)));
      s = warp_butterfly_sum(s) * a.scale_log2;
      const float mn = fmaxf(m, s);
      const float al = m == mn ? 1.f : exp2f(m - mn), p = exp2f(s - mn);
      m = mn;
      l = fmaf(l, al, p);
      const float2 v0 = unpack2<BF16>(vw.x), v1 = unpack2<BF16>(vw.y);
      acc[0] = fmaf(acc[0], al, p * v0.x);
      acc[1] = fmaf(acc[1], al, p * v0.y);
      acc[2] = fmaf(acc[2], al, p * v1.x);
      acc[3] = fmaf(acc[3], al, p * v1.y);
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  *reinterpret_cast<uint2*>(a.out + row * a.out_stride + h * 128 + lane * 4) =
      make_uint2(pack2<BF16>(acc[0] * inv, acc[1] * inv), pack2<BF16>(acc[2] * inv, acc[3] * inv));
}

int launch_window_attention(const WindowArgs& a, bool bf16, cudaStream_t s, cudaError_t* err) {
  const int64_t blocks = ((int64_t)a.Tq * a.Hq + 7) / 8;
  if (bf16)
    window_row_kernel<true><<<(unsigned)blocks, 256, 0, s>>>(a);
  else
    window_row_kernel<false><<<(unsigned)blocks, 256, 0, s>>>(a);
  *err = cudaGetLastError();
  return *err == cudaSuccess ? 0 : 2;
}

}  // namespace h3b
