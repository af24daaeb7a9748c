// window_attn.cu -- causal attention with a sliding window and visible first tokens
// over contiguous K/V of a ragged batch, or over a paged cache.
//
//   out_i = sum_j softmax_j(scale * q_i . k_j) v_j  over the keys j that query i sees
//
// One CTA per two 128-row query tiles A and B that read the same keys: two heads of one
// kv head at the same rows (even groups), else two consecutive row tiles of one head.
// It visits the 128-key tiles that any of its rows sees -- those of the first tokens,
// then those of the window -- in one pass with the running maximum and sum:
//   S = Q . K^T     tcgen05 kind::f16, fp32 in tensor memory
//   P = 2^(S c - m) the running maximum m moves only when a tile exceeds it by more than
//                   kWinTau, so P <= 2^kWinTau and O is rarely rescaled; P is rounded to
//                   the inputs' 16-bit type over S's own tensor-memory columns, its row
//                   sum is taken before the rounding, in fp32
//   O += P . V      A = P from tensor memory, B = V as it lies (rows of channels, the
//                   MN-major form), so V needs no transposition
//
// Only tiles that some row sees in part are masked, element by element; there V rows
// with an infinity or NaN are cleared first, because P = 0 does not hide them from the
// matrix product, and their rows' outputs get them added at the end (add_nonfinite).
//
// 384 threads: warp 0 loads (TMA; Q once, then K and V tiles through a ring of five
// 32 KB slots), warp 1 allocates tensor memory and clears V, warps 2 and 3 issue the
// MMAs of tile A and B, warps 4..7 and 8..11 are their softmax, one row per thread.
// An issuer runs PV(n - 1) before S(n), whose columns hold P(n - 1); the two tiles
// alternate on the tensor pipe and on the softmax units.
// Tensor memory: S_A 0..127, S_B 128..255, O_A 256..383, O_B 384..511, P over S + 64.
#include <climits>

#include "h3b_kernels.cuh"
#include "streaming.cuh"

namespace h3b {

namespace {

constexpr int kWinThreads = 384;
constexpr int kWinSlots = 5;
constexpr int kWinTile = 128 * 128 * 2;  // bytes of a 128 x 128 16-bit tile
constexpr int kWinOffRing = 2 * kWinTile;
constexpr int kWinOffBar = kWinOffRing + kWinSlots * kWinTile;
constexpr int kWinSmem = kWinOffBar + 512 + 1024;
// Register split (setmaxnreg): every thread starts with kWinRegs, the control warpgroup
// drops to kWinCtrlRegs, each softmax warpgroup rises to kWinSoftRegs; the shares may not
// exceed the launch's total, or the rise would wait forever (the host checks kWinRegs).
constexpr int kWinRegs = 168;
constexpr int kWinCtrlRegs = 72;
constexpr int kWinSoftRegs = 216;
static_assert(128 * (kWinCtrlRegs + 2 * kWinSoftRegs) <= kWinThreads * kWinRegs, "register split too large");
constexpr float kWinTau = 8.0f;

// D(tmem) (+)= A(tmem) * B(smem), 16-bit x 16-bit -> fp32
__device__ __forceinline__ void mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc,
                                           uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Rows of K (keys), 64 N elements (128 bytes, 128-byte swizzle) each: the N extent is
// contiguous (MN-major).  Leading offset: the next 64 columns; stride offset: 8 rows on.
__device__ __forceinline__ uint64_t sdesc_mnmajor_sw128(uint32_t smem_addr, uint32_t next_columns) {
  return (uint64_t)((smem_addr & 0x3FFFF) >> 4) | ((uint64_t)(next_columns >> 4) << 16) |
         ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
template <bool BF16>
__host__ __device__ constexpr uint32_t idesc_f16(int M, int N, bool b_mn_major) {
  return (1u << 4) | (BF16 ? (1u << 7) | (1u << 10) : 0u) | (b_mn_major ? 1u << 16 : 0u) | ((uint32_t)(N >> 3) << 17) |
         ((uint32_t)(M >> 4) << 24);
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (BF16) return bf16x2_bits(lo, hi);
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <bool BF16>
__device__ __forceinline__ float unpack_half(uint32_t w, int hi) {
  const uint16_t b = (uint16_t)(hi ? w >> 16 : w);
  if constexpr (BF16) return bf16_bits_to_f32(b);
  return __half2float(__ushort_as_half(b));
}
// bit 15 / 31 of the result: the low / high 16-bit value of w is an infinity or NaN
// (an exponent of ones carries into the sign's place)
template <bool BF16>
__device__ __forceinline__ uint32_t nonfinite2(uint32_t w) {
  if constexpr (BF16) return (w & 0x7f807f80u) + 0x00800080u;
  return (w & 0x7c007c00u) + 0x04000400u;
}

// The 128-key tiles that rows [p0, p1] of a tile see: [0, sn) and [w0, w1), sn <= w0.
struct TileKeys {
  int sn, w0, w1;
  int end, lo, sinks;  // what every row sees: keys below `sinks`, and [lo, end)
  __device__ bool takes(int n) const { return n < sn || (n >= w0 && n < w1); }
  __device__ bool whole(int n) const {
    return n * 128 + 128 <= end && (n * 128 >= lo || n * 128 + 128 <= sinks);
  }
};
__device__ TileKeys tile_keys(const WindowRule& r, int p0, int p1, int lk) {
  TileKeys t{0, 0, 0, 0, 0, 0};
  if (p1 < 0) return t;
  const VisibleKeys a = visible_keys(r, p0 < 0 ? 0 : p0, lk), b = visible_keys(r, p1, lk);
  t.sn = (b.sinks + 127) / 128;
  t.w0 = t.w1 = t.sn;
  if (a.lo < b.end) {
    t.w0 = max(a.lo / 128, t.sn);
    t.w1 = max((b.end + 127) / 128, t.w0);
  }
  if (p0 >= 0) {
    t.end = a.end;
    t.lo = b.lo;
    t.sinks = a.sinks;
  }
  return t;
}
struct WinPlan {
  TileKeys tile[2];
  int row[2], rows[2];  // first row (of q) and valid rows of each tile
  int sn, w0, steps;    // the union's tiles, in the order visited
  int p0[2];            // position of the tile's first row
  int lk, k_row, slot;  // keys of the sequence, its first K row or its table row
  __device__ int key_tile(int i) const { return i < sn ? i : w0 + (i - sn); }
  __device__ bool masked(int n) const {
    return (tile[0].takes(n) && !tile[0].whole(n)) || (tile[1].takes(n) && !tile[1].whole(n));
  }
};

// bits [a, b) of a word whose bit 0 stands for key `base`
__device__ __forceinline__ uint32_t key_bits(int base, int a, int b) {
  const int x = min(max(a - base, 0), 32), y = min(max(b - base, 0), 32);
  const uint32_t below_y = y >= 32 ? 0xffffffffu : (1u << y) - 1, below_x = x >= 32 ? 0xffffffffu : (1u << x) - 1;
  return below_y & ~below_x;
}

// 32 scores -> P, and their sum.  x = s c - m; one column pair in four takes the
// polynomial on the FMA pipe, the others ex2.approx.  In masked tiles all take ex2, whose
// exp2(-inf) is 0 (the polynomial ends at 2^-125, which would give a row that sees
// nothing a sum).
template <bool MASK>
__device__ __forceinline__ void win_exp32(uint32_t* s, float2 c2, float2 o2, float2& acc0, float2& acc1) {
#pragma unroll
  for (int c = 0; c < 32; c += 4) {
    const float2 x0 = __ffma2_rn(make_float2(__uint_as_float(s[c]), __uint_as_float(s[c + 1])), c2, o2);
    const float2 x1 = __ffma2_rn(make_float2(__uint_as_float(s[c + 2]), __uint_as_float(s[c + 3])), c2, o2);
    const float2 p0 = make_float2(ex2(x0.x), ex2(x0.y));
    const float2 p1 = !MASK && (c & 4) ? exp2_poly2(x1) : make_float2(ex2(x1.x), ex2(x1.y));
    acc0 = __fadd2_rn(acc0, p0);
    acc1 = __fadd2_rn(acc1, p1);
    s[c] = __float_as_uint(p0.x);
    s[c + 1] = __float_as_uint(p0.y);
    s[c + 2] = __float_as_uint(p1.x);
    s[c + 3] = __float_as_uint(p1.y);
  }
}

// One key tile for one query row.  cnt: tiles that the row's query tile has taken before
// (their PV is complete: it was issued before this S).
template <bool BF16, bool MASK>
__device__ __forceinline__ void win_softmax(uint32_t s_addr, uint32_t o_addr, float c, const VisibleKeys& see, int j0,
                                            int cnt, float& m, float& l) {
  uint32_t s[128];
  __syncwarp();
  tmem_ld32(s_addr, H3B_S32(s, 0));
  tmem_ld32(s_addr + 32, H3B_S32(s, 32));
  tmem_ld32(s_addr + 64, H3B_S32(s, 64));
  tmem_ld32(s_addr + 96, H3B_S32(s, 96));
  tmem_wait_ld_dep(H3B_S32(s, 0));
  reg_barrier32(H3B_S32(s, 32));
  reg_barrier32(H3B_S32(s, 64));
  reg_barrier32(H3B_S32(s, 96));
  if constexpr (MASK) {
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const int base = j0 + w * 32;
      const uint32_t bits = key_bits(base, see.lo, see.end) | key_bits(base, 0, see.sinks);
#pragma unroll
      for (int e = 0; e < 32; ++e)
        if (!((bits >> e) & 1u)) s[w * 32 + e] = 0xff800000u;
    }
  }
  float mx[4];
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    mx[w] = max3_nan(__uint_as_float(s[w * 32]), __uint_as_float(s[w * 32 + 1]), __uint_as_float(s[w * 32 + 2]));
#pragma unroll
    for (int e = 3; e < 31; e += 2)
      mx[w] = max3_nan(mx[w], __uint_as_float(s[w * 32 + e]), __uint_as_float(s[w * 32 + e + 1]));
    mx[w] = max3_nan(mx[w], __uint_as_float(s[w * 32 + 31]), __uint_as_float(s[w * 32 + 31]));
  }
  const float tmax = max3_nan(max3_nan(mx[0], mx[1], mx[2]), mx[3], mx[3]) * c;
  // a score of +inf or NaN: the row's result is not a number, whatever the rest does
  if (!(tmax < __int_as_float(0x7f800000))) l = __int_as_float(0x7fffffff);
  const float m_new = tmax > m + kWinTau || m == -__int_as_float(0x7f800000) ? tmax : m;
  float alpha = 1.f;
  if (__any_sync(0xffffffffu, m_new != m)) {
    alpha = m_new == m ? 1.f : ex2(m - m_new);
    m = m_new;
    if (cnt > 0) {
      __syncwarp();
#pragma unroll 1
      for (int k = 0; k < 128; k += 16) {
        uint32_t o[16];
        tmem_ld16(o_addr + k, o);
        tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
        tmem_st16(o_addr + k, o);
      }
    }
  }
  // nothing seen so far: subtract 0, so that the -inf of unseen keys gives 0
  const float off = m == -__int_as_float(0x7f800000) ? 0.f : -m;
  const float2 c2 = make_float2(c, c), o2 = make_float2(off, off);
  float2 acc0 = make_float2(0.f, 0.f), acc1 = make_float2(0.f, 0.f);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    win_exp32<MASK>(&s[h * 64], c2, o2, acc0, acc1);
    win_exp32<MASK>(&s[h * 64 + 32], c2, o2, acc0, acc1);
    uint32_t p[32];
#pragma unroll
    for (int e = 0; e < 32; ++e)
      p[e] = pack2<BF16>(__uint_as_float(s[h * 64 + 2 * e]), __uint_as_float(s[h * 64 + 2 * e + 1]));
    tmem_st32(s_addr + 64 + h * 32, p);
  }
  tmem_wait_st();
  tc_fence_before();
  const float2 t = __fadd2_rn(acc0, acc1);
  l = l * alpha + (t.x + t.y);
}

// row of V (of the tile's kv head) of key j
template <bool PAGED>
__device__ __forceinline__ const uint16_t* value_row(const WindowArgs& a, const WinPlan& pl, int kh, int j) {
  if constexpr (PAGED)
    return static_cast<const uint16_t*>(a.paged.v) +
           ((paged_page(a.paged, pl.slot, j / a.paged.page) * a.Hkv + kh) * a.paged.page + j % a.paged.page) * 128;
  else
    return a.v + (int64_t)(pl.k_row + j) * a.v_stride + kh * 128;
}

// Adds to an output row the infinities and NaN of the V rows that it sees and that were
// cleared from the masked tiles.  Only when there is such a row.
template <bool BF16, bool PAGED>
__device__ __noinline__ void add_nonfinite(const WindowArgs& a, const WinPlan& pl, int kh, const VisibleKeys& see,
                                           uint16_t* dst) {
  for (int i = 0; i < pl.steps; ++i) {
    const int n = pl.key_tile(i);
    if (!pl.masked(n)) continue;
    for (int j = n * 128; j < min(n * 128 + 128, see.end); ++j) {
      if (j < see.lo && j >= see.sinks) continue;
      const uint32_t* v = reinterpret_cast<const uint32_t*>(value_row<PAGED>(a, pl, kh, j));
      for (int e = 0; e < 64; ++e) {
        const uint32_t w = v[e], bad = nonfinite2<BF16>(w);
        if (!(bad & 0x80008000u)) continue;
        for (int hi = 0; hi < 2; ++hi) {
          if (!((bad >> (hi ? 31 : 15)) & 1u)) continue;
          uint16_t* o = dst + 2 * e + hi;
          const float sum = unpack_half<BF16>(*o, 0) + unpack_half<BF16>(w, hi);
          *o = (uint16_t)pack2<BF16>(sum, sum);
        }
      }
    }
  }
}

template <bool BF16, bool PAGED>
__global__ void __launch_bounds__(kWinThreads, 1)
    window_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                  const __grid_constant__ CUtensorMap tmV, const __grid_constant__ WindowArgs a, int rows_per_cta) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kWinOffBar);
  uint64_t* q_full = bars;              // 1
  uint64_t* full = bars + 1;            // kWinSlots
  uint64_t* empty = full + kWinSlots;   // kWinSlots
  uint64_t* v_ok = empty + kWinSlots;   // 4: V of step i (mod 4) is free of what masking cannot hide
  uint64_t* s_full = v_ok + 4;          // 2
  uint64_t* p_full = s_full + 2;        // 2
  uint64_t* o_full = p_full + 2;        // 2
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_full + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* cleared = abort_flag + 1;  // some seen V row was cleared
  int* found = const_cast<int*>(abort_flag) + 2;  // sequence, tile of it
  __shared__ WinPlan plan;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = a.Hq / a.Hkv;
  const bool by_heads = rows_per_cta == 128;  // A, B: two heads of a group; else two row tiles
  const int columns = by_heads ? a.Hq / 2 : a.Hq;
  const int head0 = (int)(blockIdx.x % columns) * (by_heads ? 2 : 1);
  const int kh = head0 / group;

  // which sequence and rows: tiles are numbered through the sequences, the last first
  // (with a causal mask they see most keys)
  if (warp == 0) {
    int t = (int)((gridDim.x - 1 - blockIdx.x) / columns), seq = -1;
    for (int base = 0; base < a.seqs; base += 32) {
      int n = 0;
      if (base + lane < a.seqs) {
        const RowRange r = row_range(a.q_starts, base + lane, a.Tq);
        n = (r.b - r.a + rows_per_cta - 1) / rows_per_cta;
      }
      int x = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, t < x);
      if (hit) {
        const int w = __ffs(hit) - 1;
        seq = base + w;
        t -= __shfl_sync(0xffffffffu, x - n, w);
        break;
      }
      t -= __shfl_sync(0xffffffffu, x, 31);
    }
    if (lane == 0) {
      found[0] = seq;
      found[1] = t;
    }
  }
  __syncthreads();
  if (found[0] < 0) return;  // the grid is an upper bound

  if (threadIdx.x == 0) {
    const int seq = found[0], t = found[1];
    const RowRange qr = row_range(a.q_starts, seq, a.Tq);
    WinPlan p;
    if constexpr (PAGED) {
      p.slot = paged_slot(a.paged, seq);
      p.lk = paged_len(a.paged, p.slot);
      p.k_row = 0;
    } else {
      const RowRange kr = row_range(a.k_starts, seq, a.Tk);
      p.slot = 0;
      p.lk = kr.b - kr.a;
      p.k_row = kr.a;
    }
    const int lq = qr.b - qr.a;
    for (int x = 0; x < 2; ++x) {
      const int first = t * rows_per_cta + (by_heads ? 0 : x * 128);
      p.row[x] = qr.a + first;
      p.rows[x] = max(0, min(128, lq - first));
      p.p0[x] = p.lk - lq + first;
      p.tile[x] = p.rows[x] > 0 ? tile_keys(a.rule, p.p0[x], p.p0[x] + p.rows[x] - 1, p.lk) : TileKeys{0, 0, 0, 0, 0, 0};
    }
    const TileKeys &ta = p.tile[0], &tb = p.tile[1];
    p.sn = max(ta.sn, tb.sn);
    int w0 = 1 << 30, w1 = 0;
    if (ta.w1 > ta.w0) {
      w0 = ta.w0;
      w1 = ta.w1;
    }
    if (tb.w1 > tb.w0) {
      w0 = min(w0, tb.w0);
      w1 = max(w1, tb.w1);
    }
    p.w0 = max(w0, p.sn);
    p.steps = p.sn + max(0, w1 - p.w0);
    plan = p;

    mbar_init(q_full, 1);
    for (int s = 0; s < kWinSlots; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 2);  // one release per tile
    }
    for (int s = 0; s < 4; ++s) mbar_init(&v_ok[s], 1);
    for (int x = 0; x < 2; ++x) {
      mbar_init(&s_full[x], 1);
      mbar_init(&p_full[x], 128);
      mbar_init(&o_full[x], 1);
    }
    *abort_flag = 0;
    *cleared = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int steps = plan.steps;

  if (warp < 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kWinCtrlRegs));
  if (warp == 0) {
    if (elect_one()) {
      mbar_arrive_expect_tx(q_full, 2 * kWinTile);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int h = by_heads ? head0 + x : head0;
        uint8_t* dst = smem + x * kWinTile;
        tma_load_3d(dst, &tmQ, q_full, 0, h, plan.row[x]);
        tma_load_3d(dst + kWinTile / 2, &tmQ, q_full, 64, h, plan.row[x]);
      }
    }
    __syncwarp();
    int slot = 0;
    uint32_t phase = 0;
    const int box = PAGED ? min(a.paged.page, 128) : 128;
    bool ok = true;
    for (int i = 0; i < 2 * steps && ok; ++i) {
      ok = mbar_wait_warp(&empty[slot], phase ^ 1, abort_flag, H3B_STATUS_ATTN_TIMEOUT);
      if (!ok) break;
      const int j0 = plan.key_tile(i >> 1) * 128;
      const CUtensorMap* tm = (i & 1) ? &tmV : &tmK;
      uint8_t* dst = smem + kWinOffRing + slot * kWinTile;
      if (lane == 0) mbar_arrive_expect_tx(&full[slot], kWinTile);
      __syncwarp();
      if constexpr (PAGED) {
        // a copy per page and half of the channels; pages that no row needs, or that the
        // table does not have, are read as zeros from outside the pool
        const int boxes = 2 * (128 / box);
        if (lane < boxes) {
          const int half = lane & 1, j = j0 + (lane >> 1) * box, col = j / a.paged.page;
          int64_t z = a.paged.pages * a.Hkv;
          if (j < plan.lk && col < a.paged.width) {
            const int pg = a.paged.table[(int64_t)plan.slot * a.paged.width + col];
            if (pg >= 0 && pg < a.paged.pages) z = (int64_t)pg * a.Hkv + kh;
          }
          tma_load_3d(dst + half * (kWinTile / 2) + (lane >> 1) * box * 128, tm, &full[slot], half * 64,
                      j & (a.paged.page - 1), (int)z);
        }
      } else if (lane < 2) {
        tma_load_3d(dst + lane * (kWinTile / 2), tm, &full[slot], lane * 64, kh, plan.k_row + j0);
      }
      __syncwarp();
      if (++slot == kWinSlots) {
        slot = 0;
        phase ^= 1;
      }
    }
  } else if (warp == 1) {
    // V tiles, in order: those that are masked somewhere lose their non-finite elements
    int item = 1;
    for (int i = 0; i < steps; ++i, item += 2) {
      const int slot = item % kWinSlots;
      if (!mbar_wait_warp(&full[slot], (item / kWinSlots) & 1, abort_flag, H3B_STATUS_ATTN_TIMEOUT)) break;
      const int n = plan.key_tile(i);
      if (plan.masked(n)) {
        uint4* v = reinterpret_cast<uint4*>(smem + kWinOffRing + slot * kWinTile);
        uint32_t any = 0;
#pragma unroll 8
        for (int x = 0; x < kWinTile / 16 / 32; ++x) {
          const uint4 w = v[x * 32 + lane];
          any |= nonfinite2<BF16>(w.x) | nonfinite2<BF16>(w.y) | nonfinite2<BF16>(w.z) | nonfinite2<BF16>(w.w);
        }
        if (__any_sync(0xffffffffu, any & 0x80008000u)) {
          for (int x = lane; x < kWinTile / 16; x += 32) {
            uint4 w = v[x];
            uint32_t* e = reinterpret_cast<uint32_t*>(&w);
            bool hit = false;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint32_t bad = nonfinite2<BF16>(e[k]);
              if (bad & 0x8000u) e[k] &= 0xffff0000u;
              if (bad & 0x80000000u) e[k] &= 0x0000ffffu;
              hit |= (bad & 0x80008000u) != 0;
            }
            if (hit) {
              v[x] = w;
              const int j = n * 128 + (x / 8) % 128;  // 8 pieces of 16 bytes per row and half
              if (j < plan.lk) *cleared = 1;
            }
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&v_ok[i & 3]);
    }
  } else if (warp < 4) {
    // MMA issuer of tile x: the whole warp walks the steps, one elected lane issues
    const int x = warp - 2;
    const TileKeys keys = plan.tile[x];
    constexpr uint32_t idesc_s = idesc_f16<BF16>(128, 128, false);
    constexpr uint32_t idesc_pv = idesc_f16<BF16>(128, 128, true);
    const uint32_t q_addr = smem_u32(smem + x * kWinTile), ring = smem_u32(smem + kWinOffRing);
    const uint32_t s_tmem = tmem + (uint32_t)(x * 128), o_tmem = tmem + 256 + (uint32_t)(x * 128);
    bool ok = mbar_wait_warp(q_full, 0, abort_flag, H3B_STATUS_ATTN_TIMEOUT);
    int pending = -1;  // step whose PV is to come
    bool first = true;
    uint32_t ppar = 0;
    auto issue_pv = [&]() -> bool {
      if (!mbar_wait_warp(&p_full[x], ppar, abort_flag, H3B_STATUS_ATTN_TIMEOUT)) return false;
      ppar ^= 1u;
      if (!mbar_wait_warp(&v_ok[pending & 3], (pending >> 2) & 1, abort_flag, H3B_STATUS_ATTN_TIMEOUT)) return false;
      tc_fence_after();
      const int slot = (2 * pending + 1) % kWinSlots;
      const uint64_t vdesc = sdesc_mnmajor_sw128(ring + slot * kWinTile, kWinTile / 2);
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          mma_f16_ts(o_tmem, s_tmem + 64 + 8 * k, vdesc + (uint64_t)(128 * k), idesc_pv, first && k == 0 ? 0u : 1u);
        mma_commit(&empty[slot]);
      }
      __syncwarp();
      first = false;
      pending = -1;
      return true;
    };
    for (int i = 0; i < steps && ok; ++i) {
      const int ks = (2 * i) % kWinSlots, vs = (2 * i + 1) % kWinSlots;
      ok = mbar_wait_warp(&full[ks], ((2 * i) / kWinSlots) & 1, abort_flag, H3B_STATUS_ATTN_TIMEOUT);
      if (!ok) break;
      if (keys.takes(plan.key_tile(i))) {
        if (pending >= 0 && !(ok = issue_pv())) break;
        tc_fence_after();
        const uint64_t qdesc = sdesc_kmajor_sw128(q_addr), kdesc = sdesc_kmajor_sw128(ring + ks * kWinTile);
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const uint64_t at = (uint64_t)((k & 3) * 2 + (k >> 2) * (kWinTile / 2 / 16));
            mma_bf16_ss(s_tmem, qdesc + at, kdesc + at, idesc_s, k == 0 ? 0u : 1u);
          }
          mma_commit(&empty[ks]);
          mma_commit(&s_full[x]);
        }
        __syncwarp();
        pending = i;
      } else {
        // a PV left to come would hold its slot until the tile's next step
        if (pending >= 0 && !(ok = issue_pv())) break;
        ok = mbar_wait_warp(&full[vs], ((2 * i + 1) / kWinSlots) & 1, abort_flag, H3B_STATUS_ATTN_TIMEOUT);
        if (!ok) break;
        if (elect_one()) {
          mbar_arrive(&empty[ks]);
          mbar_arrive(&empty[vs]);
        }
        __syncwarp();
      }
    }
    if (ok && pending >= 0) ok = issue_pv();
    if (ok && !first && elect_one()) mma_commit(&o_full[x]);
    __syncwarp();
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kWinSoftRegs));
    const int x = (warp - 4) >> 2, quad = warp & 3, r = quad * 32 + lane;
    const bool row_ok = r < plan.rows[x];
    const TileKeys keys = plan.tile[x];
    const VisibleKeys see = visible_keys(a.rule, plan.p0[x] + r, plan.lk);
    const uint32_t lane_off = (uint32_t)(quad * 32) << 16;
    const uint32_t s_addr = tmem + lane_off + (uint32_t)(x * 128);
    const uint32_t o_addr = tmem + lane_off + 256 + (uint32_t)(x * 128);
    float m = -__int_as_float(0x7f800000), l = 0.f;
    int cnt = 0;
    bool ok = true;
    for (int i = 0; i < steps; ++i) {
      const int n = plan.key_tile(i);
      if (!keys.takes(n)) continue;
      ok = mbar_wait_warp(&s_full[x], (uint32_t)(cnt & 1), abort_flag, H3B_STATUS_ATTN_TIMEOUT);
      if (!ok) break;
      tc_fence_after();
      if (keys.whole(n))
        win_softmax<BF16, false>(s_addr, o_addr, a.scale_log2, see, n * 128, cnt, m, l);
      else
        win_softmax<BF16, true>(s_addr, o_addr, a.scale_log2, see, n * 128, cnt, m, l);
      mbar_arrive(&p_full[x]);
      ++cnt;
    }
    const int h = by_heads ? head0 + x : head0;
    uint16_t* dst = a.out + (int64_t)(row_ok ? plan.row[x] + r : 0) * a.out_stride + (int64_t)h * 128;
    if (ok && cnt > 0) {
      if (mbar_wait_warp(&o_full[x], 0u, abort_flag, H3B_STATUS_ATTN_TIMEOUT)) {
        tc_fence_after();
        __syncwarp();
        const float inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll 1
        for (int c = 0; c < 128; c += 16) {
          uint32_t o[16];
          tmem_ld16(o_addr + c, o);
          tmem_wait_ld();
          uint32_t w[8];
#pragma unroll
          for (int e = 0; e < 8; ++e)
            w[e] = pack2<BF16>(__uint_as_float(o[2 * e]) * inv, __uint_as_float(o[2 * e + 1]) * inv);
          if (row_ok) {
            *reinterpret_cast<uint4*>(dst + c) = make_uint4(w[0], w[1], w[2], w[3]);
            *reinterpret_cast<uint4*>(dst + c + 8) = make_uint4(w[4], w[5], w[6], w[7]);
          }
        }
        if (*cleared && row_ok) add_nonfinite<BF16, PAGED>(a, plan, kh, see, dst);
      }
    } else if (row_ok && cnt == 0) {
      for (int c = 0; c < 128; c += 8) *reinterpret_cast<uint4*>(dst + c) = make_uint4(0, 0, 0, 0);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// [d2][d1][128] 16-bit elements, 64-channel boxes of `box1` x `box2`
bool make_rows_tmap(CUtensorMap* m, const void* base, bool bf16, uint64_t d1, uint64_t d2, uint64_t stride1,
                    uint64_t stride2, uint32_t box1, uint32_t box2) {
  const cuuint64_t dims[3] = {128, d1, d2};
  const cuuint64_t strides[2] = {stride1, stride2};
  const cuuint32_t box[3] = {64, box1, box2};
  const cuuint32_t steps[3] = {1, 1, 1};
  EncodeTiledFn encode = get_encode_tiled();
  return encode && encode(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                                const_cast<void*>(base), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <bool BF16, bool PAGED>
int launch_window(const WindowArgs& a, cudaStream_t s, cudaError_t* err) {
  CUtensorMap tq, tk, tv;
  if (!make_rows_tmap(&tq, a.q, BF16, (uint64_t)a.Hq, (uint64_t)a.Tq, 256, (uint64_t)a.q_stride * 2, 1, 128)) return 1;
  if constexpr (PAGED) {
    const uint64_t page = (uint64_t)a.paged.page, slabs = (uint64_t)a.paged.pages * a.Hkv;
    if (!make_rows_tmap(&tk, a.paged.k, BF16, page, slabs, 256, page * 256, (uint32_t)page, 1)) return 1;
    if (!make_rows_tmap(&tv, a.paged.v, BF16, page, slabs, 256, page * 256, (uint32_t)page, 1)) return 1;
  } else {
    if (!make_rows_tmap(&tk, a.k, BF16, (uint64_t)a.Hkv, (uint64_t)a.Tk, 256, (uint64_t)a.k_stride * 2, 1, 128)) return 1;
    if (!make_rows_tmap(&tv, a.v, BF16, (uint64_t)a.Hkv, (uint64_t)a.Tk, 256, (uint64_t)a.v_stride * 2, 1, 128)) return 1;
  }
  auto kern = window_kernel<BF16, PAGED>;
  cudaFuncAttributes fa;
  *err = cudaFuncGetAttributes(&fa, kern);
  if (*err != cudaSuccess) return 2;
  if (fa.numRegs != kWinRegs) return 3;  // the register split was planned for another count
  *err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kWinSmem);
  if (*err != cudaSuccess) return 2;
  const bool by_heads = (a.Hq / a.Hkv) % 2 == 0;
  const int rows = by_heads ? 128 : 256;
  const int64_t tiles = (int64_t)a.Tq / rows + a.seqs;  // sum of ceil(len / rows) is at most this
  const int64_t ctas = tiles * (by_heads ? a.Hq / 2 : a.Hq);
  if (ctas > INT_MAX) return 4;
  kern<<<(unsigned)ctas, kWinThreads, kWinSmem, s>>>(tq, tk, tv, a, rows);
  *err = cudaGetLastError();
  return *err == cudaSuccess ? 0 : 2;
}

}  // namespace

int launch_window_attention(const WindowArgs& a, bool bf16, cudaStream_t s, cudaError_t* err) {
  if (!a.paged.k && a.Tk == 0) {  // no key anywhere
    *err = cudaMemset2DAsync(a.out, (size_t)a.out_stride * 2, 0, (size_t)a.Hq * 256, (size_t)a.Tq, s);
    return *err == cudaSuccess ? 0 : 2;
  }
  if (a.paged.k) return bf16 ? launch_window<true, true>(a, s, err) : launch_window<false, true>(a, s, err);
  return bf16 ? launch_window<true, false>(a, s, err) : launch_window<false, false>(a, s, err);
}

}  // namespace h3b
