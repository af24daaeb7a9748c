// window_attn.cu -- causal attention with a sliding window and visible first tokens
// over contiguous K/V of a ragged batch, or over a paged cache.
//
//   out_i = sum_j softmax_j(scale * q_i . k_j) v_j  over the keys j that query i sees
//
// A persistent CTA per SM works through its share of the items, two 128-row query tiles
// A and B that read the same keys: two heads of one kv head at the same rows (even groups), else two
// consecutive row tiles of one head.  An item visits the 128-key tiles that any of its rows sees -- those of the first tokens,
// then those of the window -- in one pass with the running maximum and sum:
//   S = Q . K^T     tcgen05 kind::f16, fp32 in tensor memory
//   P = 2^(S c - m) the running maximum m moves only when a tile exceeds it by more than
//                   win_tau, so P <= 2^win_tau and O is rarely rescaled; P is rounded to the
//                   inputs' 16-bit type, which the matrix product asks for, over S's own
//                   tensor-memory columns; its row sum is taken before that, in fp32
//   O += P . V      A = P from tensor memory, B = V as it lies (rows of channels, the
//                   MN-major form), so V needs no transposition
//
// Only tiles that some row sees in part are masked, element by element; there V rows
// with an infinity or NaN are cleared first, because P = 0 does not hide them from the
// matrix product, and their rows' outputs get them added at the end (add_nonfinite).
//
// 512 threads: warp 0 plans the items and loads (TMA; Q once, then K and V tiles through
// a ring of five 32 KB slots), warp 1 allocates tensor memory and clears V, warps 2 and 3
// issue the MMAs of tile A and B, warps 4..7 and 8..11 are their softmax, one row per
// thread, warps 12..15 write O of finished items while the next one runs.  S of a step's
// first 64 keys is issued as soon as the step before has been read from their columns, S
// of the others after that step's PV, which reads P from theirs; PV of 64 keys starts when
// half of P is written.  The two tiles take turns.
// Tensor memory: S_A 0..127, S_B 128..255, O_A 256..383, O_B 384..511, P over S + 64.
//
// Bound by the chain of a step (S -> maximum -> P -> PV -> the next S), which two tiles hide
// in part: the tensor pipe and the exponential unit are each busy half of the time.  More
// tiles do not fit tensor memory; more code per step (unrolled columns, a second softmax
// warpgroup, wider output loops) measured slower, the instruction cache being short of it.
// Measured, bf16, 32 heads: 8,192 tokens, 8 kv heads, window 4,096: 417 to 475 us, 870 to
// 990 TFLOP/s (the lower under the power limit); a frame of 3,600 tokens over four frames
// and a prefix of 509, paged: 870 to 1,000 us, 880 to 1,010 TFLOP/s; 11 ragged prompts of
// about 500 tokens, fp16: 96 us, 422 TFLOP/s; six follow-ups of 90 tokens over 2,900 cached
// ones: 80 us.
#include <atomic>
#include <climits>

#include "h3b_kernels.cuh"
#include "streaming.cuh"

namespace h3b {

namespace {

constexpr int kWinThreads = 512;
constexpr int kWinSlots = 5;
constexpr int kWinTile = 128 * 128 * 2;  // bytes of a 128 x 128 16-bit tile
constexpr int kWinOffRing = 2 * kWinTile;
constexpr int kWinOffRest = kWinOffRing + kWinSlots * kWinTile;
constexpr int kWinSmem = kWinOffRest + 3 * 1024;  // all of a block's 227 KB
// Register split (setmaxnreg): every thread starts with kWinRegs, the control and output
// warpgroups drop to kWinCtrlRegs and kWinOutRegs, each softmax warpgroup rises to
// kWinSoftRegs; the shares may not exceed the launch's total, or the rise would wait
// forever (the host checks kWinRegs).
constexpr int kWinRegs = 128;
constexpr int kWinCtrlRegs = 104;
constexpr int kWinOutRegs = 104;
constexpr int kWinSoftRegs = 152;
static_assert(128 * (kWinCtrlRegs + kWinOutRegs + 2 * kWinSoftRegs) <= kWinThreads * kWinRegs, "register split too large");
// How far P may pass 2^0 before the maximum moves, and a factor 2^win_up of P that leaves in
// O / l (the pieces of cut items all have it).  fp16: P stays below 2^15, fp16's largest power
// of two, and a weight keeps 11 bits down to 2^-26 of the largest; without the factor down to
// 2^-14, and none below 2^-25 (800 keys 20.6 octaves below a first token: 4.2 % off).
template <bool BF16>
constexpr float win_tau = BF16 ? 8.0f : 3.0f;
template <bool BF16>
constexpr float win_up = BF16 ? 0.0f : 15.0f - win_tau<BF16>;

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
// Hand-over of tensor memory between warps: its order comes from tcgen05.wait and the
// tcgen05 fences on both sides, so neither the arrival nor the wait orders other memory
// (a releasing arrival costs about 150 cycles here, four of them a step).
__device__ __forceinline__ void tmem_arrive(uint64_t* bar) {  // one arrival of the (converged) warp
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "@p mbarrier.arrive.relaxed.cta.shared::cta.b64 _, [%0];\n\t}" ::"r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ bool tmem_try_wait(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.relaxed.cta.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool tmem_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  bool ok = tmem_try_wait(bar, parity);
  if (!__all_sync(0xffffffffu, ok)) ok = mbar_wait_warp(bar, parity, abort_flag, H3B_STATUS_ATTN_TIMEOUT);
  return ok;
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

// sum + 0 w, for both 16-bit values: stays 0 as long as they are finite
template <bool BF16>
__device__ __forceinline__ uint32_t zero_times2(uint32_t w, uint32_t sum) {
  uint32_t r;
  if constexpr (BF16)
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(w), "r"(0u), "r"(sum));
  else
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(w), "r"(0u), "r"(sum));
  return r;
}

// The 128-key tiles that rows [p0, p1] see: [0, sn) and [w0, w1), sn <= w0.
struct TileKeys {
  int sn, w0, w1;
  int end, lo, sinks;  // what every row sees: keys below `sinks`, and [lo, end)
  __device__ int steps() const { return sn + w1 - w0; }
};
__device__ __forceinline__ TileKeys tile_keys(const WindowRule& r, int p0, int p1, int lk) {
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
// One work item of a CTA.  Its steps visit the union of both tiles' key tiles in order;
// what a tile takes and what all its rows see whole are ranges of steps.
struct StepRanges {
  int head, from, to;     // a tile takes steps < head and [from, to)
  int whole_head, whole_from, whole_to;  // steps without a mask
  __device__ bool takes(int i) const { return i < head || (i >= from && i < to); }
  __device__ bool whole(int i) const { return i < whole_head || (i >= whole_from && i < whole_to); }
};
struct WinPlan {
  StepRanges tile[2];
  int row[2], rows[2];  // first row (of q) and valid rows of each tile
  int p0[2];            // position of the tile's first row
  int sn, w0, steps;    // key tiles of the steps: [0, sn), then w0 and on
  int from, to;         // the steps of this piece; from == to: no key to see; to < 0: no more work
  int part;             // -1, or where the sums of a piece of an item go
  int lk, k_row, slot;  // keys of the sequence, its first K row or its table row
  int head0, kh;        // head of tile A, kv head
  __device__ int key_tile(int i) const { return i < sn ? i : w0 + (i - sn); }
  __device__ bool masked(int i) const {
    return (tile[0].takes(i) && !tile[0].whole(i)) || (tile[1].takes(i) && !tile[1].whole(i));
  }
};
__device__ __forceinline__ StepRanges step_ranges(const TileKeys& t, int sn, int w0) {
  auto step = [&](int n) { return n < sn ? n : sn + max(n - w0, 0); };  // first step at or after key tile n
  StepRanges r;
  r.head = t.sn;
  r.from = step(t.w0);
  r.to = max(step(t.w1), r.from);
  r.whole_head = step(t.sinks / 128);
  r.whole_from = step((t.lo + 127) / 128);
  r.whole_to = step(t.end / 128);
  return r;
}

// bits [a, b) of a word whose bit 0 stands for key `base`
__device__ __forceinline__ uint32_t key_bits(int base, int a, int b) {
  const int x = min(max(a - base, 0), 32), y = min(max(b - base, 0), 32);
  const uint32_t below_y = y >= 32 ? 0xffffffffu : (1u << y) - 1, below_x = x >= 32 ? 0xffffffffu : (1u << x) - 1;
  return below_y & ~below_x;
}

// 32 scores -> P = 2^(s c - m), and their sum.  All through ex2.approx: under the power
// cap a polynomial on the FMA pipe for a share of them only adds instructions (8,192 x 32
// heads, window 4,096, in an earlier form of the kernel: none 485 us, one in eight 494, one in
// four 492, one in two 533).
__device__ __forceinline__ void win_exp32(uint32_t* s, float2 c2, float2 o2, float2& acc0, float2& acc1) {
#pragma unroll
  for (int c = 0; c < 32; c += 4) {
    const float2 x0 = __ffma2_rn(make_float2(__uint_as_float(s[c]), __uint_as_float(s[c + 1])), c2, o2);
    const float2 x1 = __ffma2_rn(make_float2(__uint_as_float(s[c + 2]), __uint_as_float(s[c + 3])), c2, o2);
    const float2 p0 = make_float2(ex2(x0.x), ex2(x0.y));
    const float2 p1 = make_float2(ex2(x1.x), ex2(x1.y));
    acc0 = __fadd2_rn(acc0, p0);
    acc1 = __fadd2_rn(acc1, p1);
    s[c] = __float_as_uint(p0.x);
    s[c + 1] = __float_as_uint(p0.y);
    s[c + 2] = __float_as_uint(p1.x);
    s[c + 3] = __float_as_uint(p1.y);
  }
}

__device__ __forceinline__ void win_load64(uint32_t s_addr, uint32_t (&s)[64]) {
  __syncwarp();
  tmem_ld32(s_addr, H3B_S32(s, 0));
  tmem_ld32(s_addr + 32, H3B_S32(s, 32));
  tmem_wait_ld_dep(H3B_S32(s, 0));
  reg_barrier32(H3B_S32(s, 32));
}

// One key tile for one query row, in two passes over the scores: the maximum, then P.
// Both are loops over halves of 64 keys, not unrolled: the softmax warps of both tiles run
// through this code every step, and with all 128 columns unrolled (and masked tiles apart)
// it did not stay in the instruction cache (11 prompts of about 500 tokens, in an earlier form
// of the kernel: 148 us with masked tiles apart, 134 us as one, 116 us as loops).
// The upper half goes first: its P lies over its own scores, and the lower half's columns
// are free for the next S as soon as they are read.
// cnt: tiles that the row's query tile has taken before (their PV is complete: it was
// issued before this S).
template <bool BF16>
__device__ __forceinline__ bool win_softmax(uint32_t s_addr, uint32_t o_addr, float c, const VisibleKeys& see,
                                            bool whole, int j0, int cnt, float& m, float& l, uint64_t* s_free,
                                            uint64_t* p_half, uint64_t* turn, uint32_t turn_parity,
                                            uint64_t* other_turn, volatile int* abort_flag) {
  uint32_t s[64];
  float tmax = -__int_as_float(0x7f800000);
#pragma unroll 1
  for (int g = 0; g < 2; ++g) {
    win_load64(s_addr + g * 64, s);
    if (!whole) {  // scores of unseen keys become -inf, for the second pass too
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const int base = j0 + g * 64 + w * 32;
        const uint32_t bits = key_bits(base, see.lo, see.end) | key_bits(base, 0, see.sinks);
#pragma unroll
        for (int e = 0; e < 32; ++e)
          if (!((bits >> e) & 1u)) s[w * 32 + e] = 0xff800000u;
        tmem_st32(s_addr + g * 64 + w * 32, H3B_S32(s, w * 32));
      }
      tmem_wait_st();
    }
    float mx[4];
#pragma unroll
    for (int w = 0; w < 4; ++w)
      mx[w] = max3_nan(__uint_as_float(s[w]), __uint_as_float(s[4 + w]), __uint_as_float(s[8 + w]));
#pragma unroll
    for (int e = 12; e < 60; e += 8)
#pragma unroll
      for (int w = 0; w < 4; ++w) mx[w] = max3_nan(mx[w], __uint_as_float(s[e + w]), __uint_as_float(s[e + 4 + w]));
#pragma unroll
    for (int w = 0; w < 4; ++w) mx[w] = max3_nan(mx[w], __uint_as_float(s[60 + w]), mx[w]);
    tmax = max3_nan(tmax, max3_nan(mx[0], mx[1], mx[2]), mx[3]);
  }
  tmax *= c;
  // a score of +inf or NaN: the row's result is not a number, whatever the rest does
  if (!(tmax < __int_as_float(0x7f800000))) l = __int_as_float(0x7fffffff);
  const float m_new = tmax > m + win_tau<BF16> || m == -__int_as_float(0x7f800000) ? tmax : m;
  if (__any_sync(0xffffffffu, m_new != m)) {
    const float alpha = m_new == m ? 1.f : ex2(m - m_new);
    m = m_new;
    l *= alpha;
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
  const float off = m == -__int_as_float(0x7f800000) ? 0.f : win_up<BF16> - m;
  const float2 c2 = make_float2(c, c), o2 = make_float2(off, off);
  if (!tmem_wait(turn, turn_parity, abort_flag)) return false;
  float2 acc0 = make_float2(0.f, 0.f), acc1 = make_float2(0.f, 0.f);
#pragma unroll 1
  for (int g = 1; g >= 0; --g) {
    win_load64(s_addr + g * 64, s);
    if (g == 0) {
      tc_fence_before();
      __syncwarp();
      tmem_arrive(s_free);
    }
    win_exp32(&s[0], c2, o2, acc0, acc1);
    win_exp32(&s[32], c2, o2, acc0, acc1);
    if (g == 0) {
      __syncwarp();
      tmem_arrive(other_turn);
    }
    uint32_t p[32];
#pragma unroll
    for (int e = 0; e < 32; ++e) p[e] = pack2<BF16>(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1]));
    tmem_st32(s_addr + 64 + g * 32, p);
    tmem_wait_st();
    tc_fence_before();
    if (g == 1) {
      __syncwarp();
      tmem_arrive(p_half);
    }
  }
  const float2 t = __fadd2_rn(acc0, acc1);
  l += t.x + t.y;
  return true;
}

// row of V (of the tile's kv head) of key j
template <bool PAGED>
__device__ __forceinline__ const uint16_t* value_row(const WindowArgs& a, const WinPlan& pl, int j) {
  if constexpr (PAGED)
    return static_cast<const uint16_t*>(a.paged.v) +
           ((paged_page(a.paged, pl.slot, j / a.paged.page) * a.Hkv + pl.kh) * a.paged.page + j % a.paged.page) * 128;
  else
    return a.v + (int64_t)(pl.k_row + j) * a.v_stride + pl.kh * 128;
}

// Adds to an output row (or a piece's sums) the infinities and NaN of the V rows that it
// sees and that were cleared from the masked tiles.  Only when there is such a row.
template <bool BF16, bool PAGED>
__device__ __noinline__ void add_nonfinite(const WindowArgs& a, const WinPlan& pl, const VisibleKeys& see,
                                           uint16_t* dst, float* sums) {
  for (int i = pl.from; i < pl.to; ++i) {
    if (!pl.masked(i)) continue;
    const int n = pl.key_tile(i);
    for (int j = n * 128; j < min(n * 128 + 128, see.end); ++j) {
      if (j < see.lo && j >= see.sinks) continue;
      const uint32_t* v = reinterpret_cast<const uint32_t*>(value_row<PAGED>(a, pl, j));
      for (int e = 0; e < 64; ++e) {
        const uint32_t w = v[e], bad = nonfinite2<BF16>(w);
        if (!(bad & 0x80008000u)) continue;
        for (int hi = 0; hi < 2; ++hi) {
          if (!((bad >> (hi ? 31 : 15)) & 1u)) continue;
          const int d = 2 * e + hi;
          const float x = unpack_half<BF16>(w, hi);
          if (sums) {
            sums[d] += x;
          } else {
            const float sum = unpack_half<BF16>(dst[d], 0) + x;
            dst[d] = (uint16_t)pack2<BF16>(sum, sum);
          }
        }
      }
    }
  }
}

// ---- the division of the work
//
// Items (a tile pair's rows and columns: head or head pair) are numbered tile by tile from
// the last (with a causal mask the late tiles see most keys), columns first; an item is
// worth its steps and kItemCost more.  Item c + r * CTAs goes to CTA c whole for the first
// rounds r, so that CTAs that read the same keys read them at the same time, as long as no
// CTA gets more than its equal share of all; what is left is dealt out along one list, to
// each CTA what it lacks.  A boundary that falls into an item there cuts it, unless the
// item is short (kCutFrom) or the piece would be (kLeastPiece): then it moves to the
// item's nearer end.  The pieces of a cut item leave their sums, and window_join_kernel
// puts them together.  Where no item is cut (window_cuts) all are dealt whole, tiles from the
// first on.
constexpr int kItemCost = 4;
constexpr int kCutFrom = 8;
constexpr int kLeastPiece = 3;
constexpr int kPieceFloats = 2 * 128 * 130;  // O [2][128][128], then (m, l) [2][128]
constexpr int kMaxTiles = kWinSlots * kWinTile / 24 - kWinThreads;  // whose sums and sequences fit the ring

struct PieceNote {  // [CTA][2]: slot 1 a piece with the item's first step, slot 0 any other
  int state;        // 0: none, 1: more pieces follow, 2: the last
  int row[2], rows[2], head0, pad[2];
};
__host__ __device__ inline int64_t window_notes_bytes(int ctas) { return (int64_t)ctas * 2 * sizeof(PieceNote); }

__device__ __forceinline__ int tiles_of(const WindowArgs& a, int seq, int rows_per_cta) {
  const RowRange r = row_range(a.q_starts, seq, a.Tq);
  return (r.b - r.a + rows_per_cta - 1) >> (rows_per_cta == 128 ? 7 : 8);  // 128 or 256
}
// A tile's sequence (-1: past the last tile) and its number in it.
struct TileAt {
  int seq, t;
};
// Where a warp looked for a tile last (in shared memory: few calls need it): the 32 sequences
// from `base`, and the tiles before them.
struct SeqsAt {
  long long before;
  int base;
};
// Tile t of all, found by the whole warp from where it looked last: a CTA's tiles follow each
// other, and a search from the first sequence for each took the square of their number (65,536
// sequences of a token 153 ms).
__device__ __forceinline__ TileAt find_tile(const WindowArgs& a, int t, int rows_per_cta, SeqsAt* last) {
  const int lane = threadIdx.x & 31;
  SeqsAt at = *last;
  TileAt found{-1, 0};
  for (;;) {
    const bool back = t < at.before && at.base > 0;
    if (back) at.base -= 32;
    else if (at.base >= a.seqs) break;
    const int n = at.base + lane < a.seqs ? tiles_of(a, at.base + lane, rows_per_cta) : 0;
    int x = n;
#pragma unroll 1
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    const int all = __shfl_sync(0xffffffffu, x, 31);
    if (back) at.before -= all;
    if (at.base == 0) at.before = 0;
    if (t < at.before) continue;
    const unsigned hit = __ballot_sync(0xffffffffu, t - at.before < x);
    if (hit) {
      const int w = __ffs(hit) - 1;
      found = {at.base + w, t - (int)at.before - __shfl_sync(0xffffffffu, x - n, w)};
      break;
    }
    at.before += all;
    at.base += 32;
  }
  if (lane == 0) *last = at;
  return found;
}
// The same out of the way of the planner's code: the paged kernel is faster with it there, the
// other one with it in place (six follow-ups of 90 tokens: 75.3 / 77.2 us, 8,192 tokens:
// 422 / 415 us; neither call comes here).
__device__ __noinline__ TileAt find_tile_apart(const WindowArgs& a, int t, int rows_per_cta, SeqsAt* last) {
  return find_tile(a, t, rows_per_cta, last);
}

// Everything about a tile's item but its column and its piece, by the whole warp: lanes 0
// and 1 find the keys of tiles A and B, lane 2 those of both, all in one run through the
// code (it runs once, from a cold instruction cache).  at.seq < 0, past the last tile:
// nothing to visit, no row to write.  Returns the number of steps.
template <bool PAGED>
__device__ __forceinline__ int plan_tile(const WindowArgs& a, TileAt at, int rows_per_cta, WinPlan* p) {
  const int lane = threadIdx.x & 31;
  RowRange qr{0, 0};
  int slot = 0, lk = 0, k_row = 0;
  if (at.seq >= 0) {
    qr = row_range(a.q_starts, at.seq, a.Tq);
    if constexpr (PAGED) {
      slot = paged_slot(a.paged, at.seq);
      lk = paged_len(a.paged, slot);
    } else {
      const RowRange kr = row_range(a.k_starts, at.seq, a.Tk);
      lk = kr.b - kr.a;
      k_row = kr.a;
    }
  }
  const int lq = qr.b - qr.a;
  // tiles A, B: two heads of a group at the same 128 rows; else two row tiles
  const int from = at.t * rows_per_cta + (lane == 1 && rows_per_cta != 128 ? 128 : 0);
  const int rows = max(0, min(lane == 2 ? rows_per_cta : 128, lq - from)), p0 = lk - lq + from;
  const TileKeys keys = rows > 0 ? tile_keys(a.rule, p0, p0 + rows - 1, lk) : TileKeys{0, 0, 0, 0, 0, 0};
  const int sn = __shfl_sync(0xffffffffu, keys.sn, 2), w0 = __shfl_sync(0xffffffffu, keys.w0, 2);
  const int steps = __shfl_sync(0xffffffffu, keys.steps(), 2);
  if (lane < 2) {
    p->row[lane] = qr.a + from;
    p->rows[lane] = rows;
    p->p0[lane] = p0;
    p->tile[lane] = step_ranges(keys, sn, w0);
  }
  if (lane == 0) {
    p->sn = sn;
    p->w0 = w0;
    p->steps = steps;
    p->lk = lk;
    p->k_row = k_row;
    p->slot = slot;
  }
  return steps;
}

// A place in the list that is dealt out: an item and a step of it.
struct WorkAt {
  int item, step;
};
// Inclusive prefix sums of x[0, n) in shared memory, by the whole block (in loops: the code
// runs once, from a cold instruction cache).
__device__ __forceinline__ void block_prefix(long long* x, int n, long long* scan) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per = (n + kWinThreads - 1) / kWinThreads, first = (int)threadIdx.x * per, last = min(first + per, n);
  long long sum = 0;
#pragma unroll 1
  for (int i = first; i < last; ++i) sum += x[i];
  long long incl = sum;
#pragma unroll 1
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  if (lane == 31) scan[warp] = incl;
  __syncthreads();
  long long run = incl - sum;
#pragma unroll
  for (int w = 0; w < kWinThreads / 32; ++w) run += w < warp ? scan[w] : 0;
#pragma unroll 1
  for (int i = first; i < last; ++i) x[i] = run += x[i];
  __syncthreads();
}
// What a CTA does: `rounds` whole items, then from bounds[0] to bounds[1].
constexpr int kListed = 48;
struct WorkShare {
  int valid, rounds;
  WorkAt bounds[2];
  TileAt tile[kListed];  // of the rounds' items, then of the dealt-out tiles in order
};

// A counter through the phases of a ring of N barriers: slot and parity of its next use.
template <int N>
struct RingAt {
  int slot = 0;
  uint32_t parity = 0;
  __device__ void next() {
    if (++slot == N) {
      slot = 0;
      parity ^= 1u;
    }
  }
};

// 32 output rows of a warp (a row per lane, N pieces of 16 bytes of it) so that N lanes
// store 16 N contiguous bytes of one row: an N x N transpose of pieces in each group of N
// lanes.  A store of own rows would touch 32 lines for 512 bytes.
template <int N>
__device__ __forceinline__ void transpose_pieces(uint4 (&u)[N]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int b = 1; b < N; b <<= 1) {
    const bool up = lane & b;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (i & b) continue;
      uint4 &lo = u[i], &hi = u[i | b];
      const uint4 give = up ? lo : hi;
      uint4 got;
      got.x = __shfl_xor_sync(0xffffffffu, give.x, b);
      got.y = __shfl_xor_sync(0xffffffffu, give.y, b);
      got.z = __shfl_xor_sync(0xffffffffu, give.z, b);
      got.w = __shfl_xor_sync(0xffffffffu, give.w, b);
      if (up)
        lo = got;
      else
        hi = got;
    }
  }
}

template <bool BF16, bool PAGED>
__global__ void __launch_bounds__(kWinThreads, 1)
    window_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                  const __grid_constant__ CUtensorMap tmV, const __grid_constant__ WindowArgs a, int rows_per_cta,
                  int tiles) {
  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) & 1023u) {  // the swizzled tiles and the room behind them count on it
    if (threadIdx.x == 0) record_status(H3B_STATUS_ATTN_TIMEOUT);
    chain_wait();
    if (a.notes && threadIdx.x < 2) reinterpret_cast<PieceNote*>(a.notes)[2 * blockIdx.x + threadIdx.x].state = 0;
    return;
  }
  struct Rest {
    uint64_t bars[48];
    uint32_t words[8];
    WinPlan plans[3];
    WorkShare work;
    long long scan[kWinThreads / 32];
    float l[2][128];  // row sums of the item that warps 12..15 write
    SeqsAt seqs_at;
  };
  static_assert(sizeof(Rest) <= kWinSmem - kWinOffRest, "shared memory");
  Rest& rest = *reinterpret_cast<Rest*>(smem + kWinOffRest);
  WinPlan(&plans)[3] = rest.plans;
  WorkShare& work = rest.work;
  long long* scan = rest.scan;
  uint64_t* bars = rest.bars;
  uint64_t* full = bars;                // kWinSlots
  uint64_t* empty = full + kWinSlots;   // kWinSlots (a release per tile)
  uint64_t* v_ok = empty + kWinSlots;   // 4: V of a step (mod 4) is free of what masking cannot hide
  uint64_t* q_full = v_ok + 4;          // 1
  uint64_t* q_empty = q_full + 1;       // 1 (per tile)
  uint64_t* s_full = q_empty + 1;       // 2: S written
  uint64_t* s_free = s_full + 2;        // 2: S read
  uint64_t* p_half = s_free + 2;        // 2: P of the last 64 keys written
  uint64_t* p_full = p_half + 2;        // 2
  uint64_t* o_full = p_full + 2;        // 2: O of an item complete
  uint64_t* o_free = o_full + 2;        // 2: O read
  uint64_t* turns = o_free + 2;         // 2 x 4: whose exponentials run, per SM sub-partition
  uint64_t* plan_full = turns + 8;      // 3
  uint64_t* plan_free = plan_full + 3;  // 3
  uint64_t* l_full = plan_free + 3;     // 2: row sums of an item written
  uint64_t* l_free = l_full + 2;        // 2: and read
  uint64_t* drained = l_free + 2;       // 2: the products of a tile's issuer are all done
  uint32_t* tmem_slot = rest.words;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* cleared = abort_flag + 1;  // [3]: some seen V row of the item was cleared
  volatile int* late_flag = cleared + 3;   // the last waits, which go on after abort_flag, gave up
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool by_heads = rows_per_cta == 128;
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    return mbar_wait_warp(bar, parity, abort_flag, H3B_STATUS_ATTN_TIMEOUT);
  };
  // A CTA that has given up still may not leave, or free its tensor memory, before its copies
  // and products in flight have landed: each warp that starts them waits at its end (at once
  // over where all went well).
  auto wait_landed = [&](uint64_t* bar, uint32_t parity) {
    mbar_wait_warp(bar, parity, late_flag, H3B_STATUS_ATTN_TIMEOUT);
  };

  if (warp == 0) {
    if (lane == 0) {
      tma_prefetch_desc(&tmQ);
      tma_prefetch_desc(&tmK);
      tma_prefetch_desc(&tmV);
    }
  } else if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  } else if (warp == 2 && lane == 0) {
    for (int s = 0; s < kWinSlots; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 2);
    }
    for (int s = 0; s < 4; ++s) mbar_init(&v_ok[s], 1);
    mbar_init(q_full, 1);
    mbar_init(q_empty, 2);
    for (int x = 0; x < 2; ++x) {
      mbar_init(&s_full[x], 1);
      mbar_init(&s_free[x], 4);  // a warp each
      mbar_init(&p_half[x], 4);
      mbar_init(&p_full[x], 4);
      mbar_init(&o_full[x], 1);
      mbar_init(&o_free[x], 4);
      mbar_init(&l_full[x], 4);
      mbar_init(&l_free[x], 4);
      mbar_init(&drained[x], 1);
    }
    for (int s = 0; s < 3; ++s) {
      mbar_init(&plan_full[s], 1);
      mbar_init(&plan_free[s], 15);  // all warps but the planning one
    }
    for (int s = 0; s < 8; ++s) mbar_init(&turns[s], 1);
    *abort_flag = *late_flag = 0;
    cleared[0] = cleared[1] = cleared[2] = 0;
    rest.seqs_at = {0, 0};
    fence_mbar_init();
  }
  chain_next();
  chain_wait();
  const int columns = by_heads ? a.Hq / 2 : a.Hq;
  {
    // Where no item is cut, all are dealt whole, in rounds.
    const bool cuts = a.notes != nullptr;
    // Else costs of all tiles, as prefix sums in the ring's memory.
    const int ctas = (int)gridDim.x, me = (int)blockIdx.x;
    if (!cuts) {
      if (threadIdx.x == 0) {
        const int items = tiles * columns;
        work.valid = tiles;
        work.rounds = me < items ? (items - me + ctas - 1) / ctas : 0;
        work.bounds[0] = work.bounds[1] = {items, 0};
      }
    } else {
      long long* lack = reinterpret_cast<long long*>(smem + kWinOffRing);  // [CTAs]: share without the rounds' items
      long long* seq_upto = lack + kWinThreads;                            // [seqs]: tiles of sequences 0..i
      long long* upto = seq_upto + a.seqs;  // [tiles] from the last tile: cost of an item of each, summed
      int2* seq_len = reinterpret_cast<int2*>(upto + tiles);  // [seqs]: rows and keys
      auto locate = [&](int tile) {
        int lo = 0, hi = a.seqs - 1;
#pragma unroll 1
        while (lo < hi) {
          const int mid = (lo + hi) >> 1;
          if (seq_upto[mid] > tile) hi = mid; else lo = mid + 1;
        }
        return TileAt{lo, tile - (lo ? (int)seq_upto[lo - 1] : 0)};
      };
      auto cost = [&](int q) { return upto[q] - (q ? upto[q - 1] : 0); };
      int valid = 0, items = 0, rounds = 0;
      long long all = 0, share = 0;
      // a loop: one copy of the prefix sums, which run from a cold instruction cache
#pragma unroll 1
      for (int stage = 0; stage < 3; ++stage) {
        long long* sums;
        int n;
        if (stage == 0) {
          sums = seq_upto;
          n = a.seqs;
          for (int i = (int)threadIdx.x; i < n; i += kWinThreads) {
            int lk;
            if constexpr (PAGED) {
              lk = paged_len(a.paged, paged_slot(a.paged, i));
            } else {
              const RowRange kr = row_range(a.k_starts, i, a.Tk);
              lk = kr.b - kr.a;
            }
            const RowRange qr = row_range(a.q_starts, i, a.Tq);
            seq_len[i] = make_int2(qr.b - qr.a, lk);
            seq_upto[i] = (qr.b - qr.a + rows_per_cta - 1) >> (by_heads ? 7 : 8);  // 128 or 256
          }
        } else if (stage == 1) {
          sums = upto;
          n = valid = (int)min(seq_upto[a.seqs - 1], (long long)tiles);  // more only where the starts overlap
#pragma unroll 1
          for (int q = (int)threadIdx.x; q < n; q += kWinThreads) {
            const TileAt at = locate(n - 1 - q);
            const int2 len = seq_len[at.seq];
            const int first = at.t * rows_per_cta, rows = min(rows_per_cta, len.x - first), p0 = len.y - len.x + first;
            upto[q] = tile_keys(a.rule, p0, p0 + rows - 1, len.y).steps() + kItemCost;
          }
        } else {
          sums = lack;
          n = ctas;
          items = valid * columns;
          all = valid ? upto[valid - 1] * columns : 0;
          share = (all + ctas - 1) / ctas;
          // whole rounds; a thread per CTA (the launch has at most kWinThreads)
          int my_q = (int)threadIdx.x / columns, my_column = (int)threadIdx.x % columns;
          const int step_q = ctas / columns, step_column = ctas % columns;
          long long load = 0;
#pragma unroll 1
          for (;; ++rounds) {
            const bool in = (rounds + 1) * ctas <= items;
            const long long next = (int)threadIdx.x < ctas && in ? load + cost(my_q) : 0;
            if (!__syncthreads_and(in && next <= share)) break;
            load = next;
            my_q += step_q;
            if ((my_column += step_column) >= columns) {
              my_column -= columns;
              ++my_q;
            }
          }
          if ((int)threadIdx.x < ctas) lack[threadIdx.x] = share - load;
        }
        __syncthreads();
        block_prefix(sums, n, scan);
      }
      if (threadIdx.x < 2) {
        // from after what the CTAs before this one lack, to after what it lacks itself
        const int i = me - 1 + (int)threadIdx.x, dealt = rounds * ctas, q0 = dealt / columns;
        const long long at = dealt >= items ? all
                                            : (q0 ? upto[q0 - 1] : 0) * columns + (dealt - q0 * columns) * cost(q0) +
                                                  (i < 0 ? 0 : lack[i]);
        WorkAt w{items, 0};
        if (at < all) {
          int lo = 0, hi = valid - 1;  // the first tile that ends beyond `at`
#pragma unroll 1
          while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (upto[mid] * columns > at) hi = mid; else lo = mid + 1;
          }
          // items of a tile are worth less than 2^31 together (the launcher sees to it)
          const unsigned worth = (unsigned)cost(lo), in = (unsigned)(at - (lo ? upto[lo - 1] : 0) * columns);
          const int steps = (int)worth - kItemCost;
          w.item = lo * columns + (int)(in / worth);
          w.step = max((int)(in % worth) - kItemCost, 0);
          const bool whole = steps < kCutFrom;  // the item may not be cut
          if (w.step > 0 && (whole ? 2 * w.step >= steps : steps - w.step < kLeastPiece)) {
            w.step = 0;
            ++w.item;
          } else if (whole || w.step < kLeastPiece) {
            w.step = 0;
          }
        }
        work.bounds[threadIdx.x] = w;
        work.valid = valid;
        work.rounds = rounds;
      }
      __syncthreads();
      const int dealt_tile = work.bounds[0].item / columns;
      for (int e = (int)threadIdx.x; e < kListed; e += kWinThreads) {
        const int q = e < rounds ? (me + e * ctas) / columns : dealt_tile + e - rounds;
        work.tile[e] = q < valid ? locate(valid - 1 - q) : TileAt{-1, 0};
      }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the ring's loads come next
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  // last step of a piece that a tile takes (-1: none)
  auto last_step = [](const WinPlan& p, int x) {
    const StepRanges& r = p.tile[x];
    int last = min(r.to, p.to) - 1;
    if (last < max(r.from, p.from)) last = min(r.head, p.to) - 1;
    return last < p.from ? -1 : last;
  };
  if (warp < 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kWinCtrlRegs));
  if (warp == 0) {
    // plans the items and loads their tiles
    RingAt<kWinSlots> at;
    const int box = PAGED ? a.paged.page : 128;
    bool ok = true;
    uint32_t q_parity = 1;
    WorkAt w = work.bounds[0];
    const WorkAt stop = work.bounds[1];
    const int rounds = work.rounds, dealt_tile = w.item / columns;
    PieceNote* notes = reinterpret_cast<PieceNote*>(a.notes) + 2 * blockIdx.x;
    if (a.notes && lane < 2) notes[lane].state = 0;
    __syncwarp();
    // An item's plan is made when the loads of the one before it are under way: they are
    // two steps ahead.
    int made = 0;
    for (RingAt<3> pr; ok; pr.next(), ++made) {
      WinPlan* pl = &plans[pr.slot];
      if (!wait(&plan_free[pr.slot], pr.parity ^ 1u)) break;
      const bool round = made < rounds;
      if (round || w.item < stop.item || (w.item == stop.item && w.step < stop.step)) {
        const int item = round ? (int)blockIdx.x + made * (int)gridDim.x : w.item, q = item / columns;
        const int entry = round ? made : rounds + q - dealt_tile;
        TileAt at_tile;
        if (__builtin_expect(a.notes && entry < kListed, 1))
          at_tile = work.tile[entry];
        else
          at_tile = (PAGED ? find_tile_apart : find_tile)(a, a.notes ? work.valid - 1 - q : q, rows_per_cta,
                                                          &rest.seqs_at);
        const int steps = plan_tile<PAGED>(a, at_tile, rows_per_cta, pl);
        const int from = round ? 0 : w.step, to = !round && item == stop.item ? stop.step : steps;
        const bool cut = from > 0 || to < steps;
        const int slot = from == 0 ? 1 : 0, head0 = (item - q * columns) * (by_heads ? 2 : 1);
        if (lane == 0) {
          pl->head0 = head0;
          pl->kh = head0 / (a.Hq / a.Hkv);
          pl->from = from;
          pl->to = to;
          pl->part = cut ? 2 * (int)blockIdx.x + slot : -1;
          cleared[pr.slot] = 0;
          if (cut) {
            notes[slot].state = to == steps ? 2 : 1;
            notes[slot].head0 = head0;
          }
        }
        if (lane < 2 && cut) {
          notes[slot].row[lane] = pl->row[lane];
          notes[slot].rows[lane] = pl->rows[lane];
        }
        if (!round) w = {w.item + 1, 0};
      } else if (lane == 0) {
        pl->to = -1;
      }
      __syncwarp();
      const int from = pl->from, to = pl->to, sn = pl->sn, w0 = pl->w0, kh = pl->kh;
      if (lane == 0) mbar_arrive(&plan_full[pr.slot]);
      if (to < 0) break;
      if (from == to) continue;
      if (!(ok = wait(q_empty, q_parity))) break;
      q_parity ^= 1u;
      if (lane == 0) mbar_arrive_expect_tx(q_full, 2 * kWinTile);
      __syncwarp();
      if (lane < 4)
        tma_load_3d(smem + lane * (kWinTile / 2), &tmQ, q_full, (lane & 1) * 64,
                    by_heads ? pl->head0 + (lane >> 1) : pl->head0, pl->row[lane >> 1]);
      __syncwarp();
      // The slab (page, kv head) of this lane's copy for a step's tiles: a copy per page and
      // half of the channels.  Pages that no row needs, or that the table does not have, are
      // read as zeros from outside the pool.  K and V of a step share it, and the next
      // step's is fetched while this one's copies are issued.
      auto slab_of = [&](int n) -> int {
        const int nowhere = (int)(a.paged.pages * a.Hkv), j = (n < sn ? n : w0 + (n - sn)) * 128 + (lane >> 1) * box;
        const int col = j / box;
        if (lane >= 256 / box || j >= pl->lk || col >= a.paged.width) return nowhere;
        const int pg = a.paged.table[(int64_t)pl->slot * a.paged.width + col];
        return pg >= 0 && pg < a.paged.pages ? pg * a.Hkv + kh : nowhere;
      };
      int slab = 0, next_slab = 0;
      if constexpr (PAGED) slab = slab_of(from);
      for (int i = 2 * from; i < 2 * to; ++i, at.next()) {
        const int n = i >> 1;
        if constexpr (PAGED) {
          if (!(i & 1) && n + 1 < to) next_slab = slab_of(n + 1);
        }
        if (!(ok = wait(&empty[at.slot], at.parity ^ 1u))) break;
        const CUtensorMap* tm = (i & 1) ? &tmV : &tmK;
        uint8_t* dst = smem + kWinOffRing + at.slot * kWinTile;
        uint64_t* bar = &full[at.slot];
        if (lane == 0) mbar_arrive_expect_tx(bar, kWinTile);
        __syncwarp();
        if constexpr (PAGED) {
          if (lane < 256 / box)
            tma_load_3d(dst + (lane & 1) * (kWinTile / 2) + (lane >> 1) * box * 128, tm, bar, (lane & 1) * 64, 0, slab);
          if (i & 1) slab = next_slab;
        } else if (lane < 2) {
          tma_load_3d(dst + lane * (kWinTile / 2), tm, bar, lane * 64, kh,
                      pl->k_row + (n < sn ? n : w0 + (n - sn)) * 128);
        }
        __syncwarp();
      }
      if (!ok) break;
    }
    // of each slot the last fill, of the slots from at.slot on that of the round before
    wait_landed(q_full, q_parity);
    for (int s = 0; s < kWinSlots; ++s) wait_landed(&full[s], s < at.slot ? at.parity : at.parity ^ 1u);
  } else if (warp == 1) {
    // V tiles, in order: those that are masked somewhere lose their non-finite elements
    RingAt<kWinSlots> at;
    RingAt<4> vo;
    bool ok = true;
    for (RingAt<3> pr; ok; pr.next()) {
      const WinPlan& pl = plans[pr.slot];
      if (!wait(&plan_full[pr.slot], pr.parity)) break;
      const int to = pl.to;
      if (to < 0) break;
      for (int i = pl.from; i < to; ++i) {
        // K first: a slot's fills alternate between K and V, and a wait that skipped K's
        // would take the fill before it for V's
        if (!(ok = wait(&full[at.slot], at.parity))) break;
        at.next();
        if (!(ok = wait(&full[at.slot], at.parity))) break;
        if (pl.masked(i)) {
          uint4* v = reinterpret_cast<uint4*>(smem + kWinOffRing + at.slot * kWinTile);
          uint32_t any[4] = {0, 0, 0, 0};  // 0, or NaN once an element was not finite
#pragma unroll 16
          for (int x = 0; x < kWinTile / 16 / 32; ++x) {
            const uint4 w = v[x * 32 + lane];
            any[0] = zero_times2<BF16>(w.x, any[0]);
            any[1] = zero_times2<BF16>(w.y, any[1]);
            any[2] = zero_times2<BF16>(w.z, any[2]);
            any[3] = zero_times2<BF16>(w.w, any[3]);
          }
          if (__any_sync(0xffffffffu, (any[0] | any[1] | any[2] | any[3]) & 0x7fff7fffu)) {
            const int j0 = pl.key_tile(i) * 128;
            for (int x = lane; x < kWinTile / 16; x += 32) {
              uint4 w = v[x];
              uint32_t* e = reinterpret_cast<uint32_t*>(&w);
              bool hit = false;
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                const uint32_t bad = nonfinite2<BF16>(e[c]);
                if (bad & 0x8000u) e[c] &= 0xffff0000u;
                if (bad & 0x80000000u) e[c] &= 0x0000ffffu;
                hit |= (bad & 0x80008000u) != 0;
              }
              if (hit) {
                v[x] = w;
                if (j0 + (x / 8) % 128 < pl.lk) cleared[pr.slot] = 1;  // 8 pieces per row and half
              }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&v_ok[vo.slot]);
        vo.next();
        at.next();
      }
      if (lane == 0) mbar_arrive(&plan_free[pr.slot]);
    }
  } else if (warp < 4) {
    // MMA issuer of tile x: the whole warp walks the steps, one elected lane issues
    const int x = warp - 2;
    constexpr uint32_t idesc_s = idesc_f16<BF16>(128, 128, false), idesc_half = idesc_f16<BF16>(128, 64, false);
    constexpr uint32_t idesc_pv = idesc_f16<BF16>(128, 128, true);
    const uint32_t ring = smem_u32(smem + kWinOffRing);
    const uint32_t s_tmem = tmem + (uint32_t)(x * 128), o_tmem = tmem + 256 + (uint32_t)(x * 128);
    const uint64_t qdesc = sdesc_kmajor_sw128(smem_u32(smem + x * kWinTile));
    // S of 64 or 128 keys from row `row` of a K tile
    auto issue_s = [&](int slot, int row, uint32_t idesc) {
      const uint64_t kdesc = sdesc_kmajor_sw128(ring + slot * kWinTile + row * 128);
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const uint64_t off = (uint64_t)((c & 3) * 2 + (c >> 2) * (kWinTile / 2 / 16));
        mma_bf16_ss(s_tmem + row, qdesc + off, kdesc + off, idesc, c == 0 ? 0u : 1u);
      }
    };
    RingAt<kWinSlots> at;
    RingAt<4> vo;
    uint32_t q_parity = 0, o_parity = 1, step_parity = 0;
    bool ok = true;
    for (RingAt<3> pr; ok; pr.next()) {
      if (!wait(&plan_full[pr.slot], pr.parity)) break;
      const int from = plans[pr.slot].from, to = plans[pr.slot].to;
      if (to < 0) break;
      const StepRanges r = plans[pr.slot].tile[x];
      const int last = last_step(plans[pr.slot], x);
      if (to > from) {
        if (!(ok = wait(q_full, q_parity))) break;
        q_parity ^= 1u;
        if (last < 0 && lane == 0) mbar_arrive(q_empty);
      }
      bool first = true, issued = false;
      for (int i = from; i < to; ++i) {
        const RingAt<kWinSlots> kt = at;
        at.next();
        const RingAt<kWinSlots> vt = at;
        at.next();
        const RingAt<4> vs = vo;
        vo.next();
        if (!r.takes(i)) {
          // V through its check, which must not fall behind the ring
          if (!(ok = wait(&full[kt.slot], kt.parity) && wait(&v_ok[vs.slot], vs.parity))) break;
          if (lane == 0) {
            mbar_arrive(&empty[kt.slot]);
            mbar_arrive(&empty[vt.slot]);
          }
          __syncwarp();
          continue;
        }
        if (!issued) {
          if (!(ok = wait(&full[kt.slot], kt.parity))) break;
          tc_fence_after();
          if (elect_one()) {
            issue_s(kt.slot, 0, idesc_s);
            mma_commit(&empty[kt.slot]);
            mma_commit(&s_full[x]);
            if (i == last) mma_commit(q_empty);
          }
          __syncwarp();
        }
        issued = i < last && r.takes(i + 1);
        if (issued) {
          // the next S of the first 64 keys, over the columns that hold neither S nor P now
          if (!(ok = wait(&full[at.slot], at.parity) && tmem_wait(&s_free[x], step_parity, abort_flag))) break;
          tc_fence_after();
          if (elect_one()) issue_s(at.slot, 0, idesc_half);
          __syncwarp();
        }
        const uint64_t vdesc = sdesc_mnmajor_sw128(ring + vt.slot * kWinTile, kWinTile / 2);
        if (first && !(ok = tmem_wait(&o_free[x], o_parity, abort_flag))) break;
        if (!(ok = wait(&v_ok[vs.slot], vs.parity) && tmem_wait(&p_half[x], step_parity, abort_flag))) break;
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int c = 4; c < 8; ++c)
            mma_f16_ts(o_tmem, s_tmem + 64 + 8 * c, vdesc + (uint64_t)(128 * c), idesc_pv, first && c == 4 ? 0u : 1u);
        }
        __syncwarp();
        first = false;
        if (!(ok = tmem_wait(&p_full[x], step_parity, abort_flag))) break;
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
            mma_f16_ts(o_tmem, s_tmem + 64 + 8 * c, vdesc + (uint64_t)(128 * c), idesc_pv, 1u);
          mma_commit(&empty[vt.slot]);
          if (issued) {
            issue_s(at.slot, 64, idesc_half);  // its columns held P
            mma_commit(&empty[at.slot]);
            mma_commit(&s_full[x]);
            if (i + 1 == last) mma_commit(q_empty);
          } else if (i == last) {
            mma_commit(&o_full[x]);
          }
        }
        __syncwarp();
        step_parity ^= 1u;
      }
      if (!ok) break;
      if (last >= 0) o_parity ^= 1u;
      if (lane == 0) mbar_arrive(&plan_free[pr.slot]);
    }
    if (elect_one()) mma_commit(&drained[x]);
    __syncwarp();
    wait_landed(&drained[x], 0);
  } else if (warp < 12) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kWinSoftRegs));
    const int x = (warp - 4) >> 2, quad = warp & 3;
    const uint32_t lane_off = (uint32_t)(quad * 32) << 16;
    const uint32_t s_addr = tmem + lane_off + (uint32_t)(x * 128);
    const uint32_t o_addr = tmem + lane_off + 256 + (uint32_t)(x * 128);
    // The two tiles' exponentials take turns in each SM sub-partition (warps q of A and B
    // share one): otherwise both softmaxes run at the same time, and then both wait for
    // the tensor pipe at the same time.
    uint64_t *turn = &turns[x * 4 + quad], *other_turn = &turns[(x ^ 1) * 4 + quad];
    uint32_t turn_parity = (uint32_t)(x ^ 1), step_parity = 0, l_parity = 1;
    bool ok = true;
    for (RingAt<3> pr; ok; pr.next()) {
      const WinPlan& pl = plans[pr.slot];
      if (!wait(&plan_full[pr.slot], pr.parity)) break;
      const int to = pl.to;
      if (to < 0) break;
      const StepRanges r = pl.tile[x];
      const VisibleKeys see = visible_keys(a.rule, pl.p0[x] + quad * 32 + lane, to > pl.from ? pl.lk : 0);
      float m = -__int_as_float(0x7f800000), l = 0.f;
      int cnt = 0;
      for (int i = pl.from; i < to; ++i, turn_parity ^= 1u) {
        if (!r.takes(i)) {
          if (!(ok = tmem_wait(turn, turn_parity, abort_flag))) break;
          tmem_arrive(other_turn);
          continue;
        }
        if (!(ok = tmem_wait(&s_full[x], step_parity, abort_flag))) break;
        tc_fence_after();
        ok = win_softmax<BF16>(s_addr, o_addr, a.scale_log2, see, r.whole(i), pl.key_tile(i) * 128, cnt, m, l, &s_free[x],
                               &p_half[x], turn, turn_parity, other_turn, abort_flag);
        if (!ok) break;
        __syncwarp();
        tmem_arrive(&p_full[x]);
        step_parity ^= 1u;
        ++cnt;
      }
      if (!ok) break;
      if (pl.part >= 0)
        *reinterpret_cast<float2*>(a.pieces + (int64_t)pl.part * kPieceFloats + 2 * 128 * 128 +
                                   (x * 128 + quad * 32 + lane) * 2) = make_float2(m, l);
      if (cnt > 0) {
        if (!(ok = wait(&l_free[x], l_parity))) break;
        l_parity ^= 1u;
        rest.l[x][quad * 32 + lane] = l;
        __syncwarp();
        if (lane == 0) mbar_arrive(&l_full[x]);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&plan_free[pr.slot]);
    }
  } else {
    // the outputs of both tiles, a row per thread in tensor memory
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kWinOutRegs));
    const int quad = warp & 3;
    uint32_t parity[2] = {0, 0};
    bool ok = true;
    for (RingAt<3> pr; ok; pr.next()) {
      const WinPlan& pl = plans[pr.slot];
      if (!wait(&plan_full[pr.slot], pr.parity)) break;
      if (pl.to < 0) break;
      const int part = pl.part;
#pragma unroll 1
      for (int x = 0; x < 2 && ok; ++x) {
        const uint32_t o_addr = tmem + ((uint32_t)(quad * 32) << 16) + 256 + (uint32_t)(x * 128);
        const int rows = pl.rows[x] - quad * 32;  // valid rows of this warp
        const int64_t row0 = pl.row[x] + quad * 32;
        uint16_t* dst = a.out + row0 * a.out_stride + (int64_t)(by_heads ? pl.head0 + x : pl.head0) * 128;
        float* sums = part < 0 ? nullptr : a.pieces + (int64_t)part * kPieceFloats + (x * 128 + quad * 32) * 128;
        if (last_step(pl, x) < 0) {
          if (part < 0) {
            for (int e = 0; e < min(rows, 32) * 16; e += 32) {
              const int row = (e + lane) >> 4;
              if (row < rows)
                *reinterpret_cast<uint4*>(dst + row * a.out_stride + ((e + lane) & 15) * 8) = make_uint4(0, 0, 0, 0);
            }
          }
          continue;
        }
        if (!(ok = wait(&l_full[x], parity[x]))) break;
        const float l = rest.l[x][quad * 32 + lane], inv = l == 0.f ? 0.f : 1.0f / l;
        __syncwarp();
        if (lane == 0) mbar_arrive(&l_free[x]);
        if (!(ok = tmem_wait(&o_full[x], parity[x], abort_flag))) break;
        parity[x] ^= 1u;
        tc_fence_after();
#pragma unroll 1
        for (int c = 0; c < 128; c += 32) {
          uint32_t o[32];
          tmem_ld32(o_addr + c, o);
          tmem_wait_ld_dep(o);
          if (c == 96) {
            tc_fence_before();
            __syncwarp();
            tmem_arrive(&o_free[x]);
          }
          if (part >= 0) {
            uint4 u[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) u[e] = make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
            transpose_pieces<8>(u);
#pragma unroll
            for (int e = 0; e < 8; ++e)
              *reinterpret_cast<uint4*>(sums + ((lane & 24) + e) * 128 + c + (lane & 7) * 4) = u[e];
          } else {
            uint4 u[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              u[e].x = pack2<BF16>(__uint_as_float(o[8 * e]) * inv, __uint_as_float(o[8 * e + 1]) * inv);
              u[e].y = pack2<BF16>(__uint_as_float(o[8 * e + 2]) * inv, __uint_as_float(o[8 * e + 3]) * inv);
              u[e].z = pack2<BF16>(__uint_as_float(o[8 * e + 4]) * inv, __uint_as_float(o[8 * e + 5]) * inv);
              u[e].w = pack2<BF16>(__uint_as_float(o[8 * e + 6]) * inv, __uint_as_float(o[8 * e + 7]) * inv);
            }
            transpose_pieces<4>(u);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int row = (lane & 28) + e;
              if (row < rows) *reinterpret_cast<uint4*>(dst + row * a.out_stride + c + (lane & 3) * 8) = u[e];
            }
          }
        }
        if (cleared[pr.slot]) {
          __syncwarp();
          if (lane < rows) {
            const VisibleKeys see = visible_keys(a.rule, pl.p0[x] + quad * 32 + lane, pl.lk);
            add_nonfinite<BF16, PAGED>(a, pl, see, dst + lane * a.out_stride, part >= 0 ? sums + lane * 128 : nullptr);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&plan_free[pr.slot]);
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

// Joins the pieces of cut items: a block per (CTA whose slot 1 begins a cut item, tile,
// 32 rows), eight threads per row.  The pieces follow in slot 0 of the next CTAs.
template <bool BF16>
__global__ void __launch_bounds__(256) window_join_kernel(const __grid_constant__ WindowArgs a, int ctas, int by_heads) {
  chain_next();
  chain_wait();
  const PieceNote* notes = reinterpret_cast<const PieceNote*>(a.notes);
  const int cta = blockIdx.x >> 3, x = (blockIdx.x >> 2) & 1, quad = blockIdx.x & 3;
  const PieceNote first = notes[2 * cta + 1];
  const int r = quad * 32 + (threadIdx.x >> 3), c = (threadIdx.x & 7) * 4;
  if (first.state != 1 || r >= first.rows[x]) return;
  float m = -__int_as_float(0x7f800000), l = 0.f;
  float4 acc[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) acc[e] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int p = cta, more = 1; more && p < ctas; ++p) {
    const int part = p == cta ? 2 * p + 1 : 2 * p;
    if (p > cta) {
      const int state = notes[part].state;
      if (state == 0) continue;  // a CTA without a share
      more = state == 1;
    }
    const float* piece = a.pieces + (int64_t)part * kPieceFloats;
    const float2 st = *reinterpret_cast<const float2*>(piece + 2 * 128 * 128 + (x * 128 + r) * 2);
    if (st.x == -__int_as_float(0x7f800000) && st.y == 0.f) continue;  // the row saw nothing there
    const float m_new = st.x > m || m == -__int_as_float(0x7f800000) ? st.x : m;
    const float keep = m == m_new ? 1.f : exp2f(m - m_new), w = st.x == m_new ? 1.f : exp2f(st.x - m_new);
    m = m_new;
    l = l * keep + st.y * w;
    const float* o = piece + (x * 128 + r) * 128 + c;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float4 v = *reinterpret_cast<const float4*>(o + e * 32);
      acc[e] = make_float4(fmaf(v.x, w, acc[e].x * keep), fmaf(v.y, w, acc[e].y * keep), fmaf(v.z, w, acc[e].z * keep),
                           fmaf(v.w, w, acc[e].w * keep));
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  uint16_t* dst = a.out + (int64_t)(first.row[x] + r) * a.out_stride + (int64_t)(first.head0 + (by_heads ? x : 0)) * 128 + c;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    *reinterpret_cast<uint2*>(dst + e * 32) =
        make_uint2(pack2<BF16>(acc[e].x * inv, acc[e].y * inv), pack2<BF16>(acc[e].z * inv, acc[e].w * inv));
}

// [d2][d1][128] 16-bit elements, 64-channel boxes of `box1` x `box2`
bool make_rows_tmap(CUtensorMap* m, const void* base, bool bf16, uint64_t d1, uint64_t d2, uint64_t stride1,
                    uint64_t stride2, uint32_t box1, uint32_t box2) {
  const cuuint64_t dims[3] = {128, d1, d2};
  const cuuint64_t strides[2] = {stride1, stride2};
  const cuuint32_t box[3] = {64, box1, box2};
  return encode_tiled(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, base, dims, strides,
                      box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// Whether items are cut.  Cutting takes a plan of all items by every CTA, a second launch
// and a pass over the pieces, together about five steps' time; dealing whole items leaves
// half an item's steps unbalanced on average.  So: where some item can have kCutFrom steps
// (a bound from what the host knows).  keys: all of them, or what a table row can name.
// Whole / cut: a 720p frame over four frames and a prefix 1,017 / 950 us; 11 prompts of about
// 500 tokens, window 1,024, 107 / 95; six follow-ups of 90 tokens 77 / 80; one causal prompt
// of 32 heads: 1,024 tokens 26 / 35, 2,048 tokens 60 / 65, 8,192 tokens, window 4,096, 420 /
// 458 in short runs and 456 / 465 under the power limit; of 8 heads: 2,048 tokens 41 / 40.
// Where whole items fill the multiprocessors evenly by themselves the rule loses by that much.
bool window_cuts(int64_t Tq, int64_t seqs, int64_t Hq, int64_t Hkv, int64_t keys, const WindowRule& r) {
  const bool by_heads = (Hq / Hkv) % 2 == 0;
  const int64_t rows = by_heads ? 128 : 256, columns = by_heads ? Hq / 2 : Hq, tiles = Tq / rows + seqs;
  const int64_t span = (int64_t)r.window + rows + (r.chunk > 1 ? 2 * (int64_t)r.chunk : 0);
  const int64_t most = (span < keys ? (span + 126) / 128 + 1 : (keys + 127) / 128) + (r.sinks + 127) / 128;
  return most >= kCutFrom && tiles <= kMaxTiles && (most + kItemCost) * columns < INT_MAX;
}

template <bool BF16, bool PAGED>
int launch_window(WindowArgs a, cudaStream_t s, cudaError_t* err) {
  CUtensorMap tq, tk, tv;
  if (!make_rows_tmap(&tq, a.q, BF16, (uint64_t)a.Hq, (uint64_t)a.Tq, 256, (uint64_t)a.q_stride * 2, 1, 128)) return 1;
  if constexpr (PAGED) {
    const uint64_t page = (uint64_t)a.paged.page, slabs = (uint64_t)a.paged.pages * a.Hkv;
    if (!make_rows_tmap(&tk, a.paged.k, BF16, page, slabs, 256, page * 256, (uint32_t)page, 1)) return 1;
    if (!make_rows_tmap(&tv, a.paged.v, BF16, page, slabs, 256, page * 256, (uint32_t)page, 1)) return 1;
  } else {
    const uint64_t rows = (uint64_t)(a.Tk ? a.Tk : a.Tq);  // no keys: the map of Q (see launch_window_attention)
    if (!make_rows_tmap(&tk, a.k, BF16, (uint64_t)a.Hkv, rows, 256, (uint64_t)a.k_stride * 2, 1, 128)) return 1;
    if (!make_rows_tmap(&tv, a.v, BF16, (uint64_t)a.Hkv, rows, 256, (uint64_t)a.v_stride * 2, 1, 128)) return 1;
  }
  auto kern = window_kernel<BF16, PAGED>;
  // the kernel's attributes are checked and set once per device
  static std::atomic<uint64_t> ready{0};
  int dev = 0;
  if ((*err = cudaGetDevice(&dev)) != cudaSuccess) return 2;
  const uint64_t bit = 1ull << (dev & 63);
  if (!(ready.load(std::memory_order_relaxed) & bit)) {
    cudaFuncAttributes fa;
    if ((*err = cudaFuncGetAttributes(&fa, kern)) != cudaSuccess) return 2;
    if (fa.numRegs != kWinRegs) return 3;  // the register split was planned for another count
    *err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kWinSmem);
    if (*err != cudaSuccess) return 2;
    ready.fetch_or(bit, std::memory_order_relaxed);
  }
  const bool by_heads = (a.Hq / a.Hkv) % 2 == 0;
  const int rows = by_heads ? 128 : 256;
  const int64_t tiles = (int64_t)a.Tq / rows + a.seqs;  // sum of ceil(len / rows) is at most this
  const int64_t items = tiles * (by_heads ? a.Hq / 2 : a.Hq);
  if (items > INT_MAX / 2) return 4;
  const bool cuts = a.pieces && window_cuts(a.Tq, a.seqs, a.Hq, a.Hkv,
                                           PAGED ? (int64_t)a.paged.width * a.paged.page : a.Tk, a.rule);
  if (!cuts) a.notes = nullptr;
  const int sms = num_sms() < kWinThreads ? num_sms() : kWinThreads;
  const int64_t ctas = !cuts && items < sms ? items : sms;
  *err = launch_chained(kern, ctas, kWinThreads, kWinSmem, s, tq, tk, tv, a, rows, (int)tiles);
  if (*err == cudaSuccess && cuts)
    *err = launch_chained(window_join_kernel<BF16>, ctas * 8, 256, 0, s, a, (int)ctas, (int)by_heads);
  return *err == cudaSuccess ? 0 : 2;
}

}  // namespace

int64_t window_workspace_bytes(int64_t Tq, int64_t seqs, int64_t Hq, int64_t Hkv, int64_t keys, const WindowRule& r) {
  if (!window_cuts(Tq, seqs, Hq, Hkv, keys, r)) return 0;
  const int sms = num_sms();
  return window_notes_bytes(sms) + (int64_t)sms * 2 * kPieceFloats * 4;
}

int launch_window_attention(WindowArgs a, bool bf16, void* workspace, cudaStream_t s, cudaError_t* err) {
  a.notes = workspace;
  a.pieces = workspace ? reinterpret_cast<float*>(static_cast<char*>(workspace) + window_notes_bytes(num_sms())) : nullptr;
  if (!a.paged.k && a.Tk == 0) {  // no key anywhere
    if (a.q_starts) {  // rows of no sequence stay: the kernel visits no key, and needs maps that can be made
      a.k = a.v = a.q;
      a.k_stride = a.v_stride = a.q_stride;
      return bf16 ? launch_window<true, false>(a, s, err) : launch_window<false, false>(a, s, err);
    }
    *err = cudaMemset2DAsync(a.out, (size_t)a.out_stride * 2, 0, (size_t)a.Hq * 256, (size_t)a.Tq, s);
    return *err == cudaSuccess ? 0 : 2;
  }
  if (a.paged.k) return bf16 ? launch_window<true, true>(a, s, err) : launch_window<false, true>(a, s, err);
  return bf16 ? launch_window<true, false>(a, s, err) : launch_window<false, false>(a, s, err);
}

}  // namespace h3b
