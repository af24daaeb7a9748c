// kv_pages.cu -- the page work of a paged K/V cache, all on the device: allocation of
// pages for new tokens with copy-on-write, writing K/V rows, forking, truncating,
// compacting and copying.
//
// The tables are small and their changes have to be seen as one step, so one block
// plans each change (validates all of it first: a call that cannot be done changes
// nothing and sets the sticky status word); the rows themselves, which are bound by
// memory bandwidth, are moved by full grids that follow in the stream.
// Pages are handed out lowest index first, so every result is a function of the calls.
#include "streaming.cuh"

namespace h3b {

namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanWarps = kPlanThreads / 32;

__device__ __forceinline__ int pages_of(int tokens, int page) { return (tokens + page - 1) / page; }

// inclusive scan over the block; *sum receives the total.  red: [kPlanWarps] shared
__device__ __forceinline__ int block_scan(int v, int* red, int* sum) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  if (lane == 31) red[warp] = v;
  __syncthreads();
  int upto = red[lane];  // of the warps 0..lane
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += y;
  }
  __syncthreads();
  *sum = __shfl_sync(0xffffffffu, upto, 31);
  const int before = __shfl_sync(0xffffffffu, upto, max(warp - 1, 0));
  return warp ? v + before : v;
}

// apply(owner, r, load(owner, r)) for r < count of every thread's `count`, spread evenly
// over the block, four at a time: owner is the thread whose count it is.  The loads of one
// round are under way together, so apply must not change what load reads.
// ends: [kPlanThreads] shared.
template <typename L, typename A>
__device__ __forceinline__ void block_expand(int count, int* red, int* ends, L load, A apply) {
  int total;
  ends[threadIdx.x] = block_scan(count, red, &total);
  __syncthreads();
  for (int e0 = threadIdx.x; e0 < total; e0 += 4 * kPlanThreads) {
    int owner[4] = {0, 0, 0, 0}, r[4], value[4];
#pragma unroll
    for (int step = kPlanThreads / 2; step; step >>= 1) {  // the first owner whose end lies beyond e
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (ends[owner[u] + step - 1] <= e0 + u * kPlanThreads) owner[u] += step;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      owner[u] = min(owner[u], kPlanThreads - 1);
      r[u] = e0 + u * kPlanThreads - (owner[u] ? ends[owner[u] - 1] : 0);
      value[u] = e0 + u * kPlanThreads < total ? load(owner[u], r[u]) : 0;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (e0 + u * kPlanThreads < total) apply(owner[u], r[u], value[u]);
  }
  __syncthreads();
}

// Every slot named by slots[0, n) lies in the table and is named once.  seen: a bit per
// row, zeroed here.  Returns false to every thread if not.  mine: the thread's slots[tid],
// loaded by the caller (n > tid).
template <int THREADS = kPlanThreads>
__device__ bool slots_valid(const int32_t* slots, int n, int rows, uint32_t* seen, int mine) {
  for (int i = threadIdx.x; i < (rows + 31) / 32; i += THREADS) seen[i] = 0;
  __syncthreads();
  bool bad = false;
  for (int i = threadIdx.x; i < n; i += THREADS) {
    const int s = i < THREADS ? mine : slots[i];
    if (s < 0 || s >= rows)
      bad = true;
    else
      bad |= (atomicOr(&seen[s >> 5], 1u << (s & 31)) >> (s & 31)) & 1u;
  }
  return !__syncthreads_or(bad);
}

// Bit x of lane g's result: page `lo` + 32 g + x is free (a ballot per 32 pages).
__device__ __forceinline__ uint32_t free_pages(const PageTables& t, int64_t lo) {
  const int lane = threadIdx.x & 31;
  uint32_t mask = 0;
  if (lo >= t.pages) return mask;
#pragma unroll 16
  for (int g = 0; g < 32; ++g) {
    const int64_t x = lo + g * 32 + lane;
    const uint32_t m = __ballot_sync(0xffffffffu, x < t.pages && t.refs[x] == 0);
    if (lane == g) mask = m;
  }
  return mask;
}

// workspace of extend: the copies' count (of 4 words), then first, asked, src, dst, part [n] each, given [pages]
struct ExtendPlan {
  int32_t *copies, *first, *asked, *src, *dst, *part, *given;
};
__host__ __device__ __forceinline__ ExtendPlan extend_plan(int32_t* ws, int n) {
  return {ws, ws + 4, ws + 4 + n, ws + 4 + 2 * (int64_t)n, ws + 4 + 3 * (int64_t)n, ws + 4 + 4 * (int64_t)n,
          ws + 4 + 5 * (int64_t)n};
}

// Bound by the latency of its dependent loads (status, slots, lengths, tables, counts): about
// half of the 10.5 us of a token's append to 200 sequences and its truncation.  One block,
// because the pages of a sequence depend on what all before it ask for.
// tokens: rows that come with the call (append), or -1: starts may not reach past them.
__global__ void __launch_bounds__(kPlanThreads) extend_plan_kernel(PageTables t, const int32_t* slots, int n,
                                                                   const int32_t* starts, int64_t tokens, int32_t* ws) {
  extern __shared__ uint32_t seen[];
  __shared__ int red[kPlanWarps], ends[kPlanThreads], col[kPlanThreads], first_of[kPlanThreads];
  __shared__ int copies, fault;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  chain_next();
  chain_wait();
  const ExtendPlan p = extend_plan(ws, n);
  // what does not depend on other loads is loaded together: each round trip counts here
  const int status = *t.status;
  const int mine = tid < n ? slots[tid] : 0;
  uint32_t free_mask = free_pages(t, warp * 1024);
  if (tid == 0) {
    copies = 0;
    fault = kPagesOk;
    *p.copies = 0;
  }
  if (status != kPagesOk) return;
  if (!slots_valid(slots, n, t.rows, seen, mine)) {
    if (tid == 0) *t.status = kPagesBadSlot;
    return;
  }
  // pages asked for by each sequence, and where its share of them begins
  int carry = 0, error = 0, my_asked = 0, my_first = 0;
  if (starts && tokens >= 0 && tid == 0 && (starts[0] < 0 || starts[n] > tokens)) error = kPagesBadCount;
  for (int base = 0; base < n; base += kPlanThreads) {
    const int i = base + tid;
    int asked = 0;
    if (i < n) {
      const int slot = slots[i], len = t.lens[slot];
      const int64_t count = starts ? (int64_t)starts[i + 1] - starts[i] : 1;
      if (count < 0 || len < 0) {
        error = kPagesBadCount;
      } else if (len + count > (int64_t)t.width * t.page) {
        error = kPagesTooLong;
      } else {
        const int have = pages_of(len, t.page);
        asked = pages_of(len + (int)count, t.page) - have;
        if (len % t.page && count > 0) {
          const int last = t.table[(int64_t)slot * t.width + have - 1];
          if (last < 0 || last >= t.pages)
            error = kPagesBadPage;
          else if (t.refs[last] > 1)
            ++asked;
        }
      }
    }
    int sum;
    const int upto = block_scan(asked, red, &sum);
    my_asked = asked;
    my_first = carry + upto - asked;
    if (i < n && n > kPlanThreads) {
      p.asked[i] = my_asked;
      p.first[i] = my_first;
    }
    // a sum that passes 31 bits is more than any pool has
    if ((int64_t)carry + sum > t.pages) error = max(error, (int)kPagesExhausted);
    carry = (int)min((int64_t)carry + sum, (int64_t)t.pages + 1);
  }
  if (error) atomicMax(&fault, error);
  __syncthreads();
  if (fault) {
    if (tid == 0) *t.status = fault;
    return;
  }
  if (carry > 0) {
    // The `carry` lowest free pages, in order: a warp looks at 1024 pages at a time, and
    // the block's 32 x 1024 pages follow each other until enough are found.
    int found = 0;
    for (int64_t block = 0; block < t.pages && found < carry; block += kPlanWarps * 1024) {
      if (block) free_mask = free_pages(t, block + warp * 1024);
      int sum;
      int rank = found + block_scan(__popc(free_mask), red, &sum) - __popc(free_mask);
      const int64_t lo = block + warp * 1024 + lane * 32;
      for (uint32_t m = free_mask; m && rank < carry; m &= m - 1, ++rank) p.given[rank] = (int)(lo + __ffs(m) - 1);
      found += sum;
    }
    if (found < carry) {
      if (tid == 0) *t.status = kPagesExhausted;
      return;
    }
    __syncthreads();
  }
  for (int base = 0; base < n; base += kPlanThreads) {
    const int i = base + tid;
    const bool kept = n <= kPlanThreads;
    const int asked = i >= n ? 0 : kept ? my_asked : p.asked[i];
    int slot = 0, grown = 0;
    if (i < n) {
      slot = slots[i];
      const int len = t.lens[slot], first = kept ? my_first : p.first[i];
      grown = len + (starts ? starts[i + 1] - starts[i] : 1);
      const int have = pages_of(len, t.page), copy = asked - (pages_of(grown, t.page) - have);
      if (copy) {
        const int old = t.table[(int64_t)slot * t.width + have - 1], at = atomicAdd(&copies, 1);
        p.src[at] = old;
        p.dst[at] = p.given[first];
        p.part[at] = len % t.page;
        atomicSub(&t.refs[old], 1);
      }
      col[tid] = have - copy;
      first_of[tid] = first;
    }
    if (carry > 0)
      block_expand(
          asked, red, ends, [&](int owner, int r) { return p.given[first_of[owner] + r]; },
          [&](int owner, int r, int page) {
            t.table[(int64_t)slots[base + owner] * t.width + col[owner] + r] = page;
            t.refs[page] = 1;
          });
    if (i < n) t.lens[slot] = grown;
  }
  __syncthreads();
  if (tid == 0) *p.copies = copies;
}

// The rows that shared last pages held, into their copies: a warp per (copy, layer, K/V, head).
__device__ __forceinline__ void copy_shared_rows(const PagePools& pool, int pages, int page, int n, const int32_t* ws,
                                                 int64_t warp, int64_t warps) {
  const ExtendPlan p = extend_plan(const_cast<int32_t*>(ws), n);
  const int64_t units = (int64_t)*p.copies * pool.layers * 2 * pool.Hkv;
  const int lane = threadIdx.x & 31, row16 = 128 * pool.elem / 16;
  for (int64_t u = warp; u < units; u += warps) {
    const int h = (int)(u % pool.Hkv), kv = (int)(u / pool.Hkv & 1);
    const int64_t rest = u / (2 * pool.Hkv), layer = rest % pool.layers;
    const int i = (int)(rest / pool.layers);
    uint4* base = reinterpret_cast<uint4*>(kv ? pool.v : pool.k);
    const int64_t slab = (int64_t)page * row16;
    const uint4* src = base + ((layer * pages + p.src[i]) * pool.Hkv + h) * slab;
    uint4* dst = base + ((layer * pages + p.dst[i]) * pool.Hkv + h) * slab;
    const int n16 = p.part[i] * row16;
    int x = lane;
    for (; x + 96 < n16; x += 128) {
      const uint4 a = src[x], b = src[x + 32], c = src[x + 64], d = src[x + 96];
      dst[x] = a;
      dst[x + 32] = b;
      dst[x + 64] = c;
      dst[x + 96] = d;
    }
    for (; x < n16; x += 32) dst[x] = src[x];
  }
}
__global__ void __launch_bounds__(256) extend_copy_kernel(PagePools pool, int pages, int page, int n, const int32_t* ws) {
  chain_next();
  chain_wait();
  copy_shared_rows(pool, pages, page, n, ws, (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5), (int64_t)gridDim.x * 8);
}

// K/V rows of the last tokens of each sequence into their pages, a warp per token.
// E4M3 pools hold x / scale, rounded to nearest even and saturated at +-448.
// The quotient is the correctly rounded one (div_rn_by) wherever rounding it to E4M3 can
// tell: above 1024 it saturates, and where the correction loses bits to underflow it is 0.
// rb = 1 / scale; 0 where that is no normal number: to_e4m3x16_div, apart from the others'
// code, whose test per element cost a tenth of the time.
__device__ __forceinline__ float over_scale(float x, float scale, float rb) {
  const float q = __fmul_rn(x, rb);
  return fabsf(q) > 1024.f ? q : div_rn_by(x, scale, rb);
}
__device__ __forceinline__ float scale_inverse(float scale) {
  return scale > 1e-30f && scale < 1e30f ? __frcp_rn(scale) : 0.f;
}
__device__ __forceinline__ uint32_t to_e4m3x4(float4 x, float scale, float rb) {
  const uint32_t lo = f32x2_to_e4m3x2(over_scale(x.x, scale, rb), over_scale(x.y, scale, rb));
  const uint32_t hi = f32x2_to_e4m3x2(over_scale(x.z, scale, rb), over_scale(x.w, scale, rb));
  return lo | (hi << 16);
}
template <bool BF16>
__device__ __forceinline__ float4 widen4(uint32_t w0, uint32_t w1) {
  if constexpr (BF16)
    return make_float4(__uint_as_float(w0 << 16), __uint_as_float(w0 & 0xffff0000u), __uint_as_float(w1 << 16),
                       __uint_as_float(w1 & 0xffff0000u));
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w0));
  const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&w1));
  return make_float4(a.x, a.y, b.x, b.y);
}
template <bool BF16>
__device__ __noinline__ uint4 to_e4m3x16_div(uint4 a, uint4 b, float scale) {
  uint32_t r[4];
  const uint32_t u[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float4 x = widen4<BF16>(u[2 * e], u[2 * e + 1]);
    const uint32_t lo = f32x2_to_e4m3x2(__fdiv_rn(x.x, scale), __fdiv_rn(x.y, scale));
    const uint32_t hi = f32x2_to_e4m3x2(__fdiv_rn(x.z, scale), __fdiv_rn(x.w, scale));
    r[e] = lo | (hi << 16);
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}
template <bool BF16>
__device__ __forceinline__ uint4 to_e4m3x16(const uint4& a, const uint4& b, float scale, float rb) {
  if (rb == 0.f) return to_e4m3x16_div<BF16>(a, b, scale);
  return make_uint4(to_e4m3x4(widen4<BF16>(a.x, a.y), scale, rb), to_e4m3x4(widen4<BF16>(a.z, a.w), scale, rb),
                    to_e4m3x4(widen4<BF16>(b.x, b.y), scale, rb), to_e4m3x4(widen4<BF16>(b.z, b.w), scale, rb));
}
// A write by itself (an append's plan has seen to it): the slots are distinct ones of the
// table, each holds as many tokens as it gets rows, the rows are there, and so are the pages.
__device__ __forceinline__ int64_t write_count(const PageWriteArgs& w, int i) {
  return w.starts ? (int64_t)w.starts[i + 1] - w.starts[i] : 1;
}
// The status for all but the pages, to every thread.
template <int THREADS>
__device__ __forceinline__ int write_fault(const PageTables& t, const PageWriteArgs& w, uint32_t* seen) {
  if (!slots_valid<THREADS>(w.slots, w.n, t.rows, seen, (int)threadIdx.x < w.n ? w.slots[threadIdx.x] : 0))
    return kPagesBadSlot;
  bool bad = w.starts && (w.starts[0] < 0 || w.starts[w.n] > w.tokens);
  for (int i = threadIdx.x; i < w.n; i += THREADS) {
    const int64_t count = write_count(w, i), len = t.lens[w.slots[i]];
    bad |= count < 0 || count > len || len > (int64_t)t.width * t.page;
  }
  return __syncthreads_or(bad) ? kPagesBadCount : kPagesOk;
}
__global__ void __launch_bounds__(kPlanThreads) write_check_kernel(PageTables t, PageWriteArgs w) {
  extern __shared__ uint32_t seen[];
  __shared__ int red[kPlanWarps], ends[kPlanThreads], col[kPlanThreads];
  const int tid = threadIdx.x;
  chain_next();
  chain_wait();
  if (*t.status != kPagesOk) return;
  int fault = write_fault<kPlanThreads>(t, w, seen);
  if (!fault) {
    bool bad = false;
    for (int base = 0; base < w.n; base += kPlanThreads) {
      const int i = base + tid;
      int pages = 0;
      if (i < w.n) {
        const int len = t.lens[w.slots[i]], count = (int)write_count(w, i);
        col[tid] = (len - count) / t.page;
        pages = count ? pages_of(len, t.page) - col[tid] : 0;
      }
      block_expand(
          pages, red, ends,
          [&](int owner, int x) { return t.table[(int64_t)w.slots[base + owner] * t.width + col[owner] + x]; },
          [&](int, int, int page) { bad |= page < 0 || page >= t.pages; });
    }
    if (__syncthreads_or(bad)) fault = kPagesBadPage;
  }
  if (fault && tid == 0) *t.status = fault;
}
// The same by each block of a small write, so that it needs no launch of its own: 200 tokens
// into one layer 9.9 us from the host, with write_check_kernel before it 13.7 us.  All blocks
// come to the same answer, whether or not one of them has already reported it.
constexpr int kOwnCheckTokens = 512, kOwnCheckRows = 8192;
__device__ __forceinline__ bool write_fits(const PageTables& t, const PageWriteArgs& w, uint32_t* seen) {
  int fault = write_fault<256>(t, w, seen);
  if (!fault) {
    bool bad = false;
    for (int i = threadIdx.x; i < w.n; i += 256) {
      const int slot = w.slots[i], len = t.lens[slot], count = (int)write_count(w, i);
      const int end = count ? pages_of(len, t.page) : 0;
      for (int col = (len - count) / t.page; col < end; ++col) {
        const int page = t.table[(int64_t)slot * t.width + col];
        bad |= page < 0 || page >= t.pages;
      }
    }
    if (__syncthreads_or(bad)) fault = kPagesBadPage;
  }
  if (fault && blockIdx.x == 0 && threadIdx.x == 0 && *t.status == kPagesOk) *t.status = fault;
  return !fault;
}

// Element offset in a layer's pool of kv head 0 of row `tok` of the new rows; -1: of no
// sequence.  (All else was checked before, by the plan, write_check_kernel or write_fits.)
__device__ __forceinline__ int64_t row_place(const PageTables& t, const PageWriteArgs& w, int Hkv, int64_t tok) {
  int i = (int)tok, back = 1;  // the token is the back-th last of sequence i
  if (w.starts) {
    int lo = 0, hi = w.n - 1;  // the last sequence that begins at or before the token
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (w.starts[mid] <= tok) lo = mid; else hi = mid - 1;
    }
    i = lo;
    if (tok < w.starts[i] || tok >= w.starts[i + 1]) return -1;  // a row of no sequence
    back = (int)(w.starts[i + 1] - tok);
  }
  const int slot = w.slots[i];
  if (slot < 0 || slot >= t.rows) return -1;
  const int pos = t.lens[slot] - back;
  if (pos < 0 || pos / t.page >= t.width) return -1;
  const int pg = t.table[(int64_t)slot * t.width + pos / t.page];
  if (pg < 0 || pg >= t.pages) return -1;
  return ((int64_t)pg * Hkv * t.page + pos % t.page) * 128;
}
// A block writes `per` (1..8) tokens: their places are looked up side by side first, then
// all their rows are under way together.  Bound by memory: 32,600 tokens of 8 kv heads into
// an E4M3 cache, with the plan before it, 51 us (3.9 TB/s; 47 where L2 holds some of the
// rows), half of the issue slots taken by the conversion.
// CHECK: the call is one that its blocks check; else it was checked before.
template <bool FP8, bool BF16, bool CHECK>
__global__ void __launch_bounds__(256) write_kernel(PageTables t, PagePools pool, int64_t layer, PageWriteArgs w,
                                                    const int32_t* ws, int copy_blocks, int per) {
  __shared__ int64_t place[8];
  chain_next();
  chain_wait();
  if constexpr (CHECK) {
    __shared__ uint32_t seen[kOwnCheckRows / 32];
    if (!write_fits(t, w, seen)) return;
  }
  if ((int)blockIdx.x < copy_blocks) {  // rows of other places of the same pages
    copy_shared_rows(pool, t.pages, t.page, w.n, ws, (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5),
                     (int64_t)copy_blocks * 8);
    return;
  }
  const int64_t tok0 = (int64_t)(blockIdx.x - copy_blocks) * per;
  const int some = (int)min((int64_t)per, w.tokens - tok0);
  if ((int)threadIdx.x < some) place[threadIdx.x] = *t.status == kPagesOk ? row_place(t, w, pool.Hkv, tok0 + threadIdx.x) : -1;
  __syncthreads();
  const int64_t base = layer * t.pages * pool.Hkv * t.page * 128, head_step = (int64_t)t.page * 128;
  // 16 channels of one head per thread and step
  const int pieces = pool.Hkv * 8;
#pragma unroll 2
  for (int u = threadIdx.x; u < some * pieces; u += 256) {
    const int j = u / pieces, x = u - j * pieces, h = x >> 3, d = (x & 7) * 16;
    const uint4* ks = reinterpret_cast<const uint4*>(w.k + (tok0 + j) * w.k_stride + h * 128 + d);
    const uint4* vs = reinterpret_cast<const uint4*>(w.v + (tok0 + j) * w.v_stride + h * 128 + d);
    const uint4 k0 = __ldcs(ks), k1 = __ldcs(ks + 1), v0 = __ldcs(vs), v1 = __ldcs(vs + 1);  // read once
    const int64_t at = place[j], o = base + at + h * head_step + d;
    if (at < 0) continue;
    if constexpr (FP8) {
      *reinterpret_cast<uint4*>(pool.k + o) = to_e4m3x16<BF16>(k0, k1, w.k_scale[h], scale_inverse(w.k_scale[h]));
      *reinterpret_cast<uint4*>(pool.v + o) = to_e4m3x16<BF16>(v0, v1, w.v_scale[h], scale_inverse(w.v_scale[h]));
    } else {
      uint4* kd = reinterpret_cast<uint4*>(pool.k + o * 2);
      uint4* vd = reinterpret_cast<uint4*>(pool.v + o * 2);
      kd[0] = k0;
      kd[1] = k1;
      vd[0] = v0;
      vd[1] = v1;
    }
  }
}

__global__ void __launch_bounds__(kPlanThreads) fork_kernel(PageTables t, const int32_t* src, const int32_t* dst, int n,
                                                            bool apply) {
  extern __shared__ uint32_t seen[];
  __shared__ int red[kPlanWarps], ends[kPlanThreads];
  __shared__ int fault;
  const int tid = threadIdx.x;
  if (tid == 0) fault = kPagesOk;
  chain_next();
  chain_wait();
  const int status = *t.status;
  const int mine = tid < n ? dst[tid] : 0;
  if (status != kPagesOk) return;
  if (!slots_valid(dst, n, t.rows, seen, mine)) {
    if (tid == 0) *t.status = kPagesBadSlot;
    return;
  }
  for (int i = tid; i < n; i += kPlanThreads) {
    const int s = src[i];
    if (s < 0 || s >= t.rows || (seen[s >> 5] >> (s & 31) & 1u))  // a slot is not both
      atomicMax(&fault, (int)kPagesBadSlot);
    else if (t.lens[dst[i]] != 0)
      atomicMax(&fault, (int)kPagesOccupied);
  }
  __syncthreads();
  if (fault) {
    if (tid == 0) *t.status = fault;
    return;
  }
  if (!apply) return;
  for (int base = 0; base < n; base += kPlanThreads) {
    const int i = base + tid;
    const int len = i < n ? t.lens[src[i]] : 0;
    block_expand(
        min(pages_of(max(len, 0), t.page), t.width), red, ends,
        [&](int owner, int x) { return t.table[(int64_t)src[base + owner] * t.width + x]; },
        [&](int owner, int x, int pg) {
          t.table[(int64_t)dst[base + owner] * t.width + x] = pg;
          if (pg >= 0 && pg < t.pages) atomicAdd(&t.refs[pg], 1);
        });
    if (i < n) t.lens[dst[i]] = len;
  }
}

// The same without the checks, a block per pair.
__global__ void __launch_bounds__(128) fork_rows_kernel(PageTables t, const int32_t* src, const int32_t* dst) {
  chain_next();
  chain_wait();
  const int status = *t.status, s = src[blockIdx.x], d = dst[blockIdx.x];
  if (status != kPagesOk) return;
  const int len = t.lens[s], end = min(pages_of(max(len, 0), t.page), t.width);
  for (int x = threadIdx.x; x < end; x += 128) {
    const int pg = t.table[(int64_t)s * t.width + x];
    t.table[(int64_t)d * t.width + x] = pg;
    if (pg >= 0 && pg < t.pages) atomicAdd(&t.refs[pg], 1);
  }
  if (threadIdx.x == 0) t.lens[d] = len;
}

// keep[i] tokens of slots[i] stay (null: none); the pages behind them lose a reference.
__global__ void __launch_bounds__(kPlanThreads) truncate_kernel(PageTables t, const int32_t* slots, const int32_t* keep,
                                                                int n, bool apply) {
  extern __shared__ uint32_t seen[];
  __shared__ int red[kPlanWarps], ends[kPlanThreads], from[kPlanThreads];
  const int tid = threadIdx.x;
  chain_next();
  chain_wait();
  const int status = *t.status;
  const int mine = tid < n ? slots[tid] : 0;
  if (status != kPagesOk) return;
  if (!slots_valid(slots, n, t.rows, seen, mine)) {
    if (tid == 0) *t.status = kPagesBadSlot;
    return;
  }
  bool bad = false;
  if (keep)
    for (int i = tid; i < n; i += kPlanThreads) bad |= keep[i] < 0 || keep[i] > t.lens[slots[i]];
  if (__syncthreads_or(bad)) {
    if (tid == 0) *t.status = kPagesBadCount;
    return;
  }
  if (!apply) return;
  for (int base = 0; base < n; base += kPlanThreads) {
    const int i = base + tid;
    int left = 0, drop = 0;
    if (i < n) {
      left = keep ? keep[i] : 0;
      from[tid] = pages_of(left, t.page);
      drop = min(pages_of(max(t.lens[slots[i]], 0), t.page), t.width) - from[tid];
    }
    block_expand(
        max(drop, 0), red, ends,
        [&](int owner, int x) { return t.table[(int64_t)slots[base + owner] * t.width + from[owner] + x]; },
        [&](int owner, int x, int pg) {
          t.table[(int64_t)slots[base + owner] * t.width + from[owner] + x] = -1;
          if (pg >= 0 && pg < t.pages) atomicSub(&t.refs[pg], 1);
        });
    if (i < n) t.lens[slots[i]] = left;
  }
}

// The same without the checks, a block per slot.
__global__ void __launch_bounds__(128) truncate_rows_kernel(PageTables t, const int32_t* slots, const int32_t* keep) {
  chain_next();
  chain_wait();
  const int status = *t.status, slot = slots[blockIdx.x], left = keep ? keep[blockIdx.x] : 0;
  if (status != kPagesOk) return;
  const int end = min(pages_of(max(t.lens[slot], 0), t.page), t.width);
  __syncthreads();
  for (int x = pages_of(left, t.page) + threadIdx.x; x < end; x += 128) {
    int32_t* entry = t.table + (int64_t)slot * t.width + x;
    const int pg = *entry;
    *entry = -1;
    if (pg >= 0 && pg < t.pages) atomicSub(&t.refs[pg], 1);
  }
  if (threadIdx.x == 0) t.lens[slot] = left;
}

// workspace of compact: moves, used, then src[pages], dst[pages], to[pages]
struct CompactPlan {
  int32_t *moves, *used, *src, *dst, *to;
};
__host__ __device__ __forceinline__ CompactPlan compact_plan(int32_t* ws, int pages) {
  return {ws, ws + 1, ws + 4, ws + 4 + (int64_t)pages, ws + 4 + 2 * (int64_t)pages};
}
__global__ void __launch_bounds__(kPlanThreads) compact_plan_kernel(PageTables t, int32_t* ws) {
  __shared__ int count_a[kPlanWarps], count_b[kPlanWarps];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const CompactPlan p = compact_plan(ws, t.pages);
  chain_next();
  chain_wait();
  if (*t.status != kPagesOk) {
    if (tid == 0) {
      *p.moves = 0;
      *p.used = t.pages;
    }
    return;
  }
  const int per = ((t.pages + kPlanWarps - 1) / kPlanWarps + 31) & ~31;
  const int lo = min(warp * per, t.pages), hi = min(lo + per, t.pages);
  int n = 0;
  for (int i = lo + lane; i < hi; i += 32) n += t.refs[i] != 0;
#pragma unroll
  for (int o = 16; o; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
  if (lane == 0) count_a[warp] = n;
  __syncthreads();
  int used = 0;
  for (int w = 0; w < kPlanWarps; ++w) used += count_a[w];
  __syncthreads();
  // the i-th used page at or after `used` moves into the i-th free page before it
  int holes = 0, movers = 0;
  for (int i = lo + lane; i < hi; i += 32) {
    const bool live = t.refs[i] != 0;
    holes += i < used && !live;
    movers += i >= used && live;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    holes += __shfl_xor_sync(0xffffffffu, holes, o);
    movers += __shfl_xor_sync(0xffffffffu, movers, o);
  }
  if (lane == 0) {
    count_a[warp] = holes;
    count_b[warp] = movers;
  }
  __syncthreads();
  int hole = 0, mover = 0, moves = 0;
  for (int w = 0; w < kPlanWarps; ++w) {
    if (w < warp) {
      hole += count_a[w];
      mover += count_b[w];
    }
    moves += count_b[w];
  }
  for (int i = lo; i < hi; i += 32) {
    const int x = i + lane;
    const bool in = x < hi, live = in && t.refs[x] != 0;
    const unsigned mh = __ballot_sync(0xffffffffu, in && x < used && !live);
    const unsigned mm = __ballot_sync(0xffffffffu, x >= used && live);
    const unsigned below = (1u << lane) - 1;
    if (mh >> lane & 1) p.dst[hole + __popc(mh & below)] = x;
    if (mm >> lane & 1) p.src[mover + __popc(mm & below)] = x;
    hole += __popc(mh);
    mover += __popc(mm);
  }
  __syncthreads();
  for (int i = tid; i < moves; i += kPlanThreads) {
    const int s = p.src[i], d = p.dst[i];
    p.to[s] = d;
    t.refs[d] = t.refs[s];
    t.refs[s] = 0;
  }
  if (tid == 0) {
    *p.moves = moves;
    *p.used = used;
  }
}
__global__ void __launch_bounds__(256) compact_table_kernel(PageTables t, const int32_t* ws) {
  const CompactPlan p = compact_plan(const_cast<int32_t*>(ws), t.pages);
  chain_next();
  chain_wait();
  const int used = *p.used;
  const int64_t n = (int64_t)t.rows * t.width;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int pg = t.table[i];
    if (pg >= used && pg < t.pages) t.table[i] = p.to[pg];
  }
}
// A copy of pages: all of them in the pool, none copied to twice, none copied from and to.
// The targets are marked in shared memory, kCheckPages pages of the pool at a time.
constexpr int kCheckPages = 1 << 18;
__global__ void __launch_bounds__(kPlanThreads) copy_check_kernel(const int32_t* src, const int32_t* dst, int n, int pages,
                                                                  int32_t* status) {
  extern __shared__ uint32_t target[];
  const int tid = threadIdx.x;
  chain_next();
  chain_wait();
  if (*status != kPagesOk) return;
  bool bad = false;
  for (int lo = 0; lo < pages; lo += kCheckPages) {
    const int some = min(pages - lo, kCheckPages);
    for (int i = tid; i < (some + 31) / 32; i += kPlanThreads) target[i] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kPlanThreads) {
      const int d = dst[i];
      if (d < 0 || d >= pages)
        bad = true;
      else if (d >= lo && d - lo < some)
        bad |= (atomicOr(&target[(d - lo) >> 5], 1u << (d & 31)) >> (d & 31)) & 1u;
    }
    __syncthreads();
    for (int i = tid; i < n; i += kPlanThreads) {
      const int s = src[i];
      if (s < 0 || s >= pages)
        bad = true;
      else if (s >= lo && s - lo < some)
        bad |= (target[(s - lo) >> 5] >> (s & 31)) & 1u;
    }
    __syncthreads();
  }
  if (__syncthreads_or(bad) && tid == 0) *status = kPagesBadPage;
}
// Whole pages, K and V of every layer: a block per (move, layer, K/V).  Bound by memory: 1.07
// GB moved in 364 us with the plan, 5.9 TB/s of reads and writes.  count: device value
// (compact), or null: n moves that copy_check_kernel let pass (status 0).
__global__ void __launch_bounds__(256) move_kernel(PagePools pool, int pages, int64_t bytes, const int32_t* src,
                                                   const int32_t* dst, const int32_t* count, int n, const int32_t* status) {
  chain_next();
  chain_wait();
  if (!count && *status != kPagesOk) return;
  const int64_t units = (int64_t)(count ? *count : n) * pool.layers * 2;
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int64_t layer = u / 2 % pool.layers;
    const int i = (int)(u / 2 / pool.layers);
    const int s = src[i], d = dst[i];
    uint8_t* base = u & 1 ? pool.v : pool.k;
    const uint4* from = reinterpret_cast<const uint4*>(base + (layer * pages + s) * bytes);
    uint4* to = reinterpret_cast<uint4*>(base + (layer * pages + d) * bytes);
    const int64_t n16 = bytes / 16;
    int64_t x = threadIdx.x;
    for (; x + 3 * 256 < n16; x += 4 * 256) {
      const uint4 a = __ldcs(from + x), b = __ldcs(from + x + 256), c = __ldcs(from + x + 512), e = __ldcs(from + x + 768);
      to[x] = a;
      to[x + 256] = b;
      to[x + 512] = c;
      to[x + 768] = e;
    }
    for (; x < n16; x += 256) to[x] = from[x];
  }
}

size_t seen_bytes(int rows) { return (size_t)((rows + 31) / 32) * 4; }

}  // namespace

int64_t pages_workspace_bytes(int64_t n, int64_t pages) {
  const int64_t extend = 4 + 5 * n + pages, compact = 4 + 3 * pages;
  return 4 * (extend > compact ? extend : compact);
}

constexpr int kFullGrid = 1184;  // eight blocks for each of 148 multiprocessors

cudaError_t launch_pages_extend(const PageTables& t, const PagePools& p, const int32_t* slots, int n,
                                const int32_t* starts, int64_t tokens, int32_t* ws, cudaStream_t s) {
  const cudaError_t e =
      launch_chained(extend_plan_kernel, 1, kPlanThreads, seen_bytes(t.rows), s, t, slots, n, starts, tokens, ws);
  if (e != cudaSuccess || tokens >= 0) return e;
  const int64_t most = ((int64_t)n * p.layers * 2 * p.Hkv + 7) / 8;
  return launch_chained(extend_copy_kernel, most < kFullGrid ? most : kFullGrid, 256, 0, s, p, t.pages, t.page, n, ws);
}

cudaError_t launch_pages_write(const PageTables& t, const PagePools& p, int64_t layer, const PageWriteArgs& w,
                               const int32_t* ws, cudaStream_t s) {
  int64_t copies = 0;
  if (ws) {
    copies = ((int64_t)w.n * p.layers * 2 * p.Hkv + 7) / 8;
    if (copies > kFullGrid / 2) copies = kFullGrid / 2;
  }
  const bool own_check = !ws && w.tokens > 0 && w.tokens <= kOwnCheckTokens && w.n <= kOwnCheckTokens && t.rows <= kOwnCheckRows;
  if (!ws && !own_check) {
    const cudaError_t e = launch_chained(write_check_kernel, 1, kPlanThreads, seen_bytes(t.rows), s, t, w);
    if (e != cudaSuccess || w.tokens == 0) return e;  // without rows the starts may name none
  }
  auto kern = p.elem == 2    ? (own_check ? write_kernel<false, true, true> : write_kernel<false, true, false>)
              : w.src_bf16 ? (own_check ? write_kernel<true, true, true> : write_kernel<true, true, false>)
                           : (own_check ? write_kernel<true, false, true> : write_kernel<true, false, false>);
  // two blocks for each multiprocessor first, then up to 8 tokens a block
  int64_t per = w.tokens / (kFullGrid / 4);
  per = per < 1 ? 1 : per > 8 ? 8 : per;
  return launch_chained(kern, copies + (w.tokens + per - 1) / per, 256, 0, s, t, p, layer, w, ws, (int)copies, (int)per);
}

// One block that checks a call also changes the tables where it can touch few entries; else
// a second launch with a block per sequence does: one multiprocessor makes about a scattered
// reference update per clock, a launch costs the host 2 to 3 us.  (fork + free, on the device
// in one launch each / in two: 16 sequences of 60 pages 10.2 / 6.8 us, 128 of 94 pages 19.5 /
// 6.9 us, 512 of 60 pages 39 / 8.0 us.)  A truncation mostly drops a few tokens (a pass that
// appends a token to 200 sequences and drops it, launched from the host: 17.1 / 19.2 us).  What
// is compared are the entries of the table's rows, which the host knows: in a table of 32,768
// tokens that pass takes the second launch.
constexpr int64_t kOneBlockEntries = 4096, kOneBlockKept = 16384;
cudaError_t launch_pages_fork(const PageTables& t, const int32_t* src, const int32_t* dst, int n, cudaStream_t s) {
  const bool one = (int64_t)n * t.width <= kOneBlockEntries;
  const cudaError_t e = launch_chained(fork_kernel, 1, kPlanThreads, seen_bytes(t.rows), s, t, src, dst, n, one);
  if (e != cudaSuccess || one) return e;
  return launch_chained(fork_rows_kernel, n, 128, 0, s, t, src, dst);
}
cudaError_t launch_pages_truncate(const PageTables& t, const int32_t* slots, const int32_t* keep, int n,
                                  cudaStream_t s) {
  const bool one = (int64_t)n * t.width <= (keep ? kOneBlockKept : kOneBlockEntries);
  const cudaError_t e = launch_chained(truncate_kernel, 1, kPlanThreads, seen_bytes(t.rows), s, t, slots, keep, n, one);
  if (e != cudaSuccess || one) return e;
  return launch_chained(truncate_rows_kernel, n, 128, 0, s, t, slots, keep);
}
cudaError_t launch_pages_compact(const PageTables& t, const PagePools& p, int32_t* ws, cudaStream_t s) {
  cudaError_t e = launch_chained(compact_plan_kernel, 1, kPlanThreads, 0, s, t, ws);
  if (e != cudaSuccess) return e;
  const CompactPlan c = compact_plan(ws, t.pages);
  const int64_t entries = ((int64_t)t.rows * t.width + 255) / 256;
  e = launch_chained(compact_table_kernel, entries < kFullGrid ? entries : kFullGrid, 256, 0, s, t, ws);
  if (e != cudaSuccess) return e;
  return launch_chained(move_kernel, kFullGrid, 256, 0, s, p, t.pages, (int64_t)p.Hkv * t.page * 128 * p.elem, c.src,
                        c.dst, c.moves, 0, nullptr);
}
cudaError_t launch_pages_copy(const PagePools& p, int pages, int page, const int32_t* src, const int32_t* dst, int n,
                              int32_t* status, cudaStream_t s) {
  const cudaError_t e = launch_chained(copy_check_kernel, 1, kPlanThreads, seen_bytes(pages < kCheckPages ? pages : kCheckPages),
                                       s, src, dst, n, pages, status);
  if (e != cudaSuccess) return e;
  const int64_t units = (int64_t)n * p.layers * 2;
  return launch_chained(move_kernel, units < kFullGrid ? units : kFullGrid, 256, 0, s, p, pages,
                        (int64_t)p.Hkv * page * 128 * p.elem, src, dst, nullptr, n, status);
}

}  // namespace h3b
