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
  int before = 0, total = 0;
  for (int w = 0; w < kPlanWarps; ++w) {
    const int x = red[w];
    if (w < warp) before += x;
    total += x;
  }
  __syncthreads();
  *sum = total;
  return v + before;
}

// Every slot named by slots[0, n) lies in the table and is named once.  seen: a bit per
// row, zeroed here.  Returns false to every thread if not.
__device__ bool slots_valid(const int32_t* slots, int n, int rows, uint32_t* seen) {
  for (int i = threadIdx.x; i < (rows + 31) / 32; i += kPlanThreads) seen[i] = 0;
  __syncthreads();
  bool bad = false;
  for (int i = threadIdx.x; i < n; i += kPlanThreads) {
    const int s = slots[i];
    if (s < 0 || s >= rows)
      bad = true;
    else
      bad |= (atomicOr(&seen[s >> 5], 1u << (s & 31)) >> (s & 31)) & 1u;
  }
  return !__syncthreads_or(bad);
}

// workspace of extend: the copies' count (of 4 words), then first, asked, src, dst, part [n] each, given [pages]
struct ExtendPlan {
  int32_t *copies, *first, *asked, *src, *dst, *part, *given;
};
__host__ __device__ __forceinline__ ExtendPlan extend_plan(int32_t* ws, int n) {
  return {ws, ws + 4, ws + 4 + n, ws + 4 + 2 * (int64_t)n, ws + 4 + 3 * (int64_t)n, ws + 4 + 4 * (int64_t)n,
          ws + 4 + 5 * (int64_t)n};
}

__global__ void __launch_bounds__(kPlanThreads) extend_plan_kernel(PageTables t, const int32_t* slots, int n,
                                                                   const int32_t* starts, int32_t* ws) {
  extern __shared__ uint32_t seen[];
  __shared__ int red[kPlanWarps];
  __shared__ int warp_free[kPlanWarps];
  __shared__ int copies, fault;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  chain_next();
  chain_wait();
  const ExtendPlan p = extend_plan(ws, n);
  if (tid == 0) {
    copies = 0;
    fault = kPagesOk;
    *p.copies = 0;
  }
  if (*t.status != kPagesOk) return;
  if (!slots_valid(slots, n, t.rows, seen)) {
    if (tid == 0) *t.status = kPagesBadSlot;
    return;
  }
  // pages asked for by each sequence, and where its share of them begins
  int carry = 0, error = 0;
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
          if (last >= 0 && last < t.pages && t.refs[last] > 1) ++asked;
        }
      }
    }
    int sum;
    const int upto = block_scan(asked, red, &sum);
    if (i < n) {
      p.asked[i] = asked;
      p.first[i] = carry + upto - asked;
    }
    // a sum that passes 31 bits is more than any pool has
    if ((int64_t)carry + sum > t.pages) error = max(error, (int)kPagesExhausted);
    carry = min(carry + sum, t.pages + 1);
  }
  if (error) atomicMax(&fault, error);
  __syncthreads();
  if (fault) {
    if (tid == 0) *t.status = fault;
    return;
  }
  if (carry > 0) {
    // the `carry` lowest free pages, in order: each warp counts the free pages of its
    // part of refs, then lists those whose rank is asked for
    const int per = ((t.pages + kPlanWarps - 1) / kPlanWarps + 31) & ~31;
    const int lo = min(warp * per, t.pages), hi = min(lo + per, t.pages);
    int count = 0;
    for (int i = lo; i < hi; i += 128) {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int x = i + u * 32 + lane;
        count += x < hi && t.refs[x] == 0;
      }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) count += __shfl_xor_sync(0xffffffffu, count, o);
    if (lane == 0) warp_free[warp] = count;
    __syncthreads();
    int rank = 0, all = 0;
    for (int w = 0; w < kPlanWarps; ++w) {
      if (w < warp) rank += warp_free[w];
      all += warp_free[w];
    }
    if (all < carry) {
      if (tid == 0) *t.status = kPagesExhausted;
      return;
    }
    for (int i = lo; i < hi && rank < carry; i += 32) {
      const int x = i + lane;
      const bool free_page = x < hi && t.refs[x] == 0;
      const unsigned mask = __ballot_sync(0xffffffffu, free_page);
      const int r = rank + __popc(mask & ((1u << lane) - 1));
      if (free_page && r < carry) {
        p.given[r] = x;
        t.refs[x] = 1;
      }
      rank += __popc(mask);
    }
    __syncthreads();
  }
  // hand them out, a warp to a sequence
  for (int i = warp; i < n; i += kPlanWarps) {
    const int slot = slots[i], len = t.lens[slot], count = starts ? starts[i + 1] - starts[i] : 1;
    const int have = pages_of(len, t.page), more = pages_of(len + count, t.page) - have;
    const int asked = p.asked[i], first = p.first[i];
    int32_t* row = t.table + (int64_t)slot * t.width;
    const int copy = asked - more;
    for (int r = lane; r < more; r += 32) row[have + r] = p.given[first + copy + r];
    if (lane == 0) {
      if (copy) {
        const int old = row[have - 1], page = p.given[first];
        const int at = atomicAdd(&copies, 1);
        p.src[at] = old;
        p.dst[at] = page;
        p.part[at] = len % t.page;
        row[have - 1] = page;
        atomicSub(&t.refs[old], 1);
      }
      t.lens[slot] = len + count;
    }
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
__device__ __forceinline__ uint32_t to_e4m3x4(const float* x, float scale) {
  const uint32_t lo = f32x2_to_e4m3x2(__fdiv_rn(x[0], scale), __fdiv_rn(x[1], scale));
  const uint32_t hi = f32x2_to_e4m3x2(__fdiv_rn(x[2], scale), __fdiv_rn(x[3], scale));
  return lo | (hi << 16);
}
template <bool FP8, bool BF16>
__global__ void __launch_bounds__(256) write_kernel(PageTables t, PagePools pool, int64_t layer, PageWriteArgs w,
                                                    const int32_t* ws, int copy_blocks) {
  const int lane = threadIdx.x & 31;
  chain_next();
  chain_wait();
  if ((int)blockIdx.x < copy_blocks) {  // rows of other places of the same pages
    copy_shared_rows(pool, t.pages, t.page, w.n, ws, (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5),
                     (int64_t)copy_blocks * 8);
    return;
  }
  const int64_t tok = (int64_t)(blockIdx.x - copy_blocks) * 8 + (threadIdx.x >> 5);
  if (tok >= w.tokens || *t.status != kPagesOk) return;
  int i = (int)tok, back = 1;  // the token is the back-th last of sequence i
  if (w.starts) {
    int lo = 0, hi = w.n - 1;  // the last sequence that begins at or before the token
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (w.starts[mid] <= tok) lo = mid; else hi = mid - 1;
    }
    i = lo;
    if (tok < w.starts[i] || tok >= w.starts[i + 1]) return;  // a row of no sequence
    back = (int)(w.starts[i + 1] - tok);
  }
  const int slot = w.slots[i];
  if (slot < 0 || slot >= t.rows) return;
  const int pos = t.lens[slot] - back;
  if (pos < 0 || pos / t.page >= t.width) return;
  const int pg = t.table[(int64_t)slot * t.width + pos / t.page];
  if (pg < 0 || pg >= t.pages) return;
  const int64_t at = ((layer * t.pages + pg) * pool.Hkv * t.page + pos % t.page) * 128;
  const int64_t head_step = (int64_t)t.page * 128;
  const uint16_t* ks = w.k + tok * w.k_stride;
  const uint16_t* vs = w.v + tok * w.v_stride;
  // 16 channels of one head per lane and step
  for (int x = lane; x < pool.Hkv * 8; x += 32) {
    const int h = x >> 3, d = (x & 7) * 16;
    uint4 a[4];
    a[0] = *reinterpret_cast<const uint4*>(ks + h * 128 + d);
    a[1] = *reinterpret_cast<const uint4*>(ks + h * 128 + d + 8);
    a[2] = *reinterpret_cast<const uint4*>(vs + h * 128 + d);
    a[3] = *reinterpret_cast<const uint4*>(vs + h * 128 + d + 8);
    const int64_t o = at + h * head_step + d;
    if constexpr (!FP8) {
      uint4* kd = reinterpret_cast<uint4*>(pool.k + o * 2);
      uint4* vd = reinterpret_cast<uint4*>(pool.v + o * 2);
      kd[0] = a[0];
      kd[1] = a[1];
      vd[0] = a[2];
      vd[1] = a[3];
    } else {
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const float scale = (kv ? w.v_scale : w.k_scale)[h];
        uint32_t r[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint4& src = a[kv * 2 + (q >> 1)];
          const uint32_t w0 = q & 1 ? src.z : src.x, w1 = q & 1 ? src.w : src.y;
          float f[4];
          if constexpr (BF16) {
            f[0] = __uint_as_float(w0 << 16);
            f[1] = __uint_as_float(w0 & 0xffff0000u);
            f[2] = __uint_as_float(w1 << 16);
            f[3] = __uint_as_float(w1 & 0xffff0000u);
          } else {
            const float2 x0 = __half22float2(*reinterpret_cast<const __half2*>(&w0));
            const float2 x1 = __half22float2(*reinterpret_cast<const __half2*>(&w1));
            f[0] = x0.x;
            f[1] = x0.y;
            f[2] = x1.x;
            f[3] = x1.y;
          }
          r[q] = to_e4m3x4(f, scale);
        }
        *reinterpret_cast<uint4*>((kv ? pool.v : pool.k) + o) = make_uint4(r[0], r[1], r[2], r[3]);
      }
    }
  }
}

__global__ void __launch_bounds__(kPlanThreads) fork_kernel(PageTables t, const int32_t* src, const int32_t* dst, int n) {
  extern __shared__ uint32_t seen[];
  __shared__ int fault;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) fault = kPagesOk;
  chain_next();
  chain_wait();
  if (*t.status != kPagesOk) return;
  if (!slots_valid(dst, n, t.rows, seen)) {
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
  for (int i = warp; i < n; i += kPlanWarps) {
    const int len = t.lens[src[i]];
    const int32_t* from = t.table + (int64_t)src[i] * t.width;
    int32_t* to = t.table + (int64_t)dst[i] * t.width;
    const int end = min(pages_of(max(len, 0), t.page), t.width);
    for (int x = lane; x < end; x += 32) {
      const int pg = from[x];
      to[x] = pg;
      if (pg >= 0 && pg < t.pages) atomicAdd(&t.refs[pg], 1);
    }
    if (lane == 0) t.lens[dst[i]] = len;
  }
}

// keep[i] tokens of slots[i] stay (null: none); the pages behind them lose a reference.
__global__ void __launch_bounds__(kPlanThreads) truncate_kernel(PageTables t, const int32_t* slots, const int32_t* keep,
                                                                int n) {
  extern __shared__ uint32_t seen[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  chain_next();
  chain_wait();
  if (*t.status != kPagesOk) return;
  if (!slots_valid(slots, n, t.rows, seen)) {
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
  for (int i = warp; i < n; i += kPlanWarps) {
    const int slot = slots[i], left = keep ? keep[i] : 0;
    int32_t* row = t.table + (int64_t)slot * t.width;
    const int end = min(pages_of(t.lens[slot], t.page), t.width);
    for (int x = pages_of(left, t.page) + lane; x < end; x += 32) {
      const int pg = row[x];
      if (pg >= 0 && pg < t.pages) atomicSub(&t.refs[pg], 1);
      row[x] = -1;
    }
    __syncwarp();
    if (lane == 0) t.lens[slot] = left;
  }
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
// Whole pages, K and V of every layer: a block per (move, layer, K/V).  count: device
// value (compact) or null (n moves, whose pages are checked here).
__global__ void __launch_bounds__(256) move_kernel(PagePools pool, int pages, int64_t bytes, const int32_t* src,
                                                   const int32_t* dst, const int32_t* count, int n, int32_t* status) {
  chain_next();
  chain_wait();
  const int64_t units = (int64_t)(count ? *count : n) * pool.layers * 2;
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int64_t layer = u / 2 % pool.layers;
    const int i = (int)(u / 2 / pool.layers);
    const int s = src[i], d = dst[i];
    if (s < 0 || s >= pages || d < 0 || d >= pages) {
      if (status && threadIdx.x == 0) *status = kPagesBadPage;
      continue;
    }
    uint8_t* base = u & 1 ? pool.v : pool.k;
    const uint4* from = reinterpret_cast<const uint4*>(base + (layer * pages + s) * bytes);
    uint4* to = reinterpret_cast<uint4*>(base + (layer * pages + d) * bytes);
    const int64_t n16 = bytes / 16;
    int64_t x = threadIdx.x;
    for (; x + 3 * 256 < n16; x += 4 * 256) {
      const uint4 a = from[x], b = from[x + 256], c = from[x + 512], e = from[x + 768];
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
                                const int32_t* starts, int32_t* ws, bool copy, cudaStream_t s) {
  const cudaError_t e = launch_chained(extend_plan_kernel, 1, kPlanThreads, seen_bytes(t.rows), s, t, slots, n, starts, ws);
  if (e != cudaSuccess || !copy) return e;
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
  auto kern = p.elem == 2 ? write_kernel<false, true> : w.src_bf16 ? write_kernel<true, true> : write_kernel<true, false>;
  return launch_chained(kern, copies + (w.tokens + 7) / 8, 256, 0, s, t, p, layer, w, ws, (int)copies);
}

cudaError_t launch_pages_fork(const PageTables& t, const int32_t* src, const int32_t* dst, int n, cudaStream_t s) {
  return launch_chained(fork_kernel, 1, kPlanThreads, seen_bytes(t.rows), s, t, src, dst, n);
}
cudaError_t launch_pages_truncate(const PageTables& t, const int32_t* slots, const int32_t* keep, int n,
                                  cudaStream_t s) {
  return launch_chained(truncate_kernel, 1, kPlanThreads, seen_bytes(t.rows), s, t, slots, keep, n);
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
  const int64_t units = (int64_t)n * p.layers * 2;
  return launch_chained(move_kernel, units < kFullGrid ? units : kFullGrid, 256, 0, s, p, pages,
                        (int64_t)p.Hkv * page * 128 * p.elem, src, dst, nullptr, n, status);
}

}  // namespace h3b
