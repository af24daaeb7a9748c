// streaming.cuh -- argument structs, host launchers and device helpers of the
// streaming-attention kernels (window_attn.cu, decode_attn.cu, kv_pages.cu).
#pragma once

#include <atomic>

#include "h3b_common.cuh"

namespace h3b {

// Kernels of one step follow each other closely: each is launched to start while the one
// before it in the stream ends (programmatic stream serialization), does what needs no
// earlier result, and waits for that kernel's completion (chain_wait) before it touches
// global memory; chain_next lets the kernel after it start that early in turn.
__device__ __forceinline__ void chain_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void chain_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
// How many have been launched (in a captured graph: once, when it was captured): an entry
// takes one, two or three, as the sizes ask for.
inline std::atomic<int64_t> chained_launches{0};
template <typename... P, typename... A>
cudaError_t launch_chained(void (*kernel)(P...), int64_t grid, int threads, size_t smem, cudaStream_t s, A... args) {
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
  if (e == cudaSuccess) chained_launches.fetch_add(1, std::memory_order_relaxed);
  return e;
}

// Which keys a query sees: key j of a sequence with lk keys is visible to the query at
// position p >= 0 when  j < lk,  j <= last(p)  and  (last(p) - j < window or j < sinks).
// last(p) = p for chunk 1; otherwise the end of p's chunk, chunks counted from the end
// of the `sinks` first tokens, which form a chunk of their own.
struct WindowRule {
  int window, sinks, chunk;
};
// The visible keys of one query: [0, sinks) and [lo, end), sinks <= lo <= end.
struct VisibleKeys {
  int sinks, lo, end;
};
__host__ __device__ __forceinline__ VisibleKeys visible_keys(const WindowRule& r, int p, int lk) {
  if (p < 0) return {0, 0, 0};
  int64_t last = p;
  if (r.chunk > 1) last = p < r.sinks ? r.sinks - 1 : r.sinks + ((int64_t)((p - r.sinks) / r.chunk) + 1) * r.chunk - 1;
  const int end = last + 1 < lk ? (int)last + 1 : lk;
  int64_t lo = last - r.window + 1;
  lo = lo < 0 ? 0 : lo > end ? end : lo;
  const int s = r.sinks < (int)lo ? r.sinks : (int)lo;
  return {s, (int)lo, end};
}

// Sequence i's rows [a, b) of a ragged batch: starts[i], starts[i + 1] (null: one
// sequence of all `total` rows), clamped so that a bad table reads and writes nothing
// outside the rows.
struct RowRange {
  int a, b;
};
__device__ __forceinline__ RowRange row_range(const int32_t* starts, int i, int total) {
  if (!starts) return {0, total};
  const int a = min(max(starts[i], 0), total);
  return {a, min(max(starts[i + 1], a), total)};
}

// One layer of a paged cache: pools [pages, kv heads, page, 128], table [rows, width].
struct PagedArgs {
  const void* k;
  const void* v;
  int64_t pages;
  int page;  // tokens per page: 16, 32, 64 or 128
  const int32_t* table;
  int width;
  int rows;
  const int32_t* lens;
  const int32_t* slots;  // [seqs] rows of the table, or null (sequence i in row i)
};
__device__ __forceinline__ int paged_slot(const PagedArgs& a, int i) {
  const int s = a.slots ? a.slots[i] : i;
  return s >= 0 && s < a.rows ? s : -1;
}
// keys held by a table row (0 for a row outside the table), never more than it can name
__device__ __forceinline__ int paged_len(const PagedArgs& a, int slot) {
  if (slot < 0) return 0;
  const int64_t cap = (int64_t)a.width * a.page;
  const int n = a.lens[slot];
  return n < 0 ? 0 : (int64_t)n > cap ? (int)cap : n;
}
// a page inside the pool whatever the table holds
__device__ __forceinline__ int64_t paged_page(const PagedArgs& a, int slot, int col) {
  const int64_t p = a.table[(int64_t)slot * a.width + col];
  return p >= 0 && p < a.pages ? p : 0;
}

struct WindowArgs {
  const uint16_t* q;
  int64_t q_stride;  // elements between tokens; heads are 128 apart
  const uint16_t* k;
  int64_t k_stride;
  const uint16_t* v;
  int64_t v_stride;
  int Tq, Tk, seqs, Hq, Hkv;
  const int32_t* q_starts;
  const int32_t* k_starts;
  WindowRule rule;
  float scale_log2;  // softmax scale * log2(e)
  uint16_t* out;
  int64_t out_stride;
  PagedArgs paged;  // paged.k set: keys come from the pages, k / v / k_starts unused
  void* notes;      // of cut items and their pieces (set by the launcher; null: none is cut)
  float* pieces;
};
// keys: all, or what a table row can name.  0 where no workspace would be used
int64_t window_workspace_bytes(int64_t Tq, int64_t seqs, int64_t Hq, int64_t Hkv, int64_t keys, const WindowRule& r);
// bf16: bfloat16, else float16.  workspace: null, or window_workspace_bytes() with which long
// items are cut.  Returns 0 ok, 1 tensor-map encoding failed, 2 CUDA error (*err), 3 the
// kernel's register count is not the planned one, 4 too many tiles
int launch_window_attention(WindowArgs a, bool bf16, void* workspace, cudaStream_t s, cudaError_t* err);

struct DecodeArgs {
  const uint16_t* q;
  int64_t q_stride;
  int seqs, Hq, Hkv;
  PagedArgs paged;
  const float* k_scale;  // [kv heads] of an 8-bit cache, else null
  const float* v_scale;
  WindowRule rule;
  float scale_log2;
  uint16_t* out;
  int64_t out_stride;
  float* partial;  // workspace
  int workers;
};
constexpr int kDecodeMaxSeqs = 4096;
// capacity: tokens that a table row can name
int64_t decode_workspace_bytes(int64_t seqs, int64_t Hq, int64_t Hkv, int64_t capacity);
// kind 0: bf16 cache, 1: fp16 cache, 2: E4M3 cache with bf16 q, 3: E4M3 cache with fp16 q
cudaError_t launch_decode_attention(DecodeArgs a, int kind, cudaStream_t s);

// The page tables that kv_pages.cu changes; status is a sticky error word: once it is
// not zero no entry changes anything until the caller clears it.
enum PageStatus : int {
  kPagesOk = 0,
  kPagesExhausted = 1,   // not enough free pages
  kPagesTooLong = 2,     // a sequence would outgrow its row of the table
  kPagesBadSlot = 3,     // a slot outside the table, or named twice in one call
  kPagesOccupied = 4,    // fork into a slot that holds tokens
  kPagesBadCount = 5,    // token counts that are negative, not ordered or beyond the length
  kPagesBadPage = 6,     // a page outside the pool; in a copy, a target named twice or also a source
};
struct PageTables {
  int32_t* table;
  int rows, width;
  int32_t* lens;
  int32_t* refs;
  int pages, page;
  int32_t* status;
};
struct PagePools {
  uint8_t* k;  // [layers, pages, kv heads, page, 128]
  uint8_t* v;
  int64_t layers;
  int Hkv, elem;  // elem: bytes per element, 1 or 2
};
constexpr int kPagesMaxRows = 1 << 18;
int64_t pages_workspace_bytes(int64_t n, int64_t pages);
// tokens: -1, or the rows that launch_pages_write will take next, which then makes the
// planned copies too
cudaError_t launch_pages_extend(const PageTables& t, const PagePools& p, const int32_t* slots, int n,
                                const int32_t* starts, int64_t tokens, int32_t* ws, cudaStream_t s);
struct PageWriteArgs {
  const uint16_t* k;
  int64_t k_stride;
  const uint16_t* v;
  int64_t v_stride;
  int64_t tokens;
  const int32_t* slots;
  int n;
  const int32_t* starts;
  const float* k_scale;  // [kv heads] of the layer, for an E4M3 pool
  const float* v_scale;
  int src_bf16;  // rows are bf16 (else fp16)
};
// ws: null, or the plan of launch_pages_extend whose copies are made by the same kernel
cudaError_t launch_pages_write(const PageTables& t, const PagePools& p, int64_t layer, const PageWriteArgs& w,
                               const int32_t* ws, cudaStream_t s);
cudaError_t launch_pages_fork(const PageTables& t, const int32_t* src, const int32_t* dst, int n, cudaStream_t s);
cudaError_t launch_pages_truncate(const PageTables& t, const int32_t* slots, const int32_t* keep, int n,
                                  cudaStream_t s);
cudaError_t launch_pages_compact(const PageTables& t, const PagePools& p, int32_t* ws, cudaStream_t s);
cudaError_t launch_pages_copy(const PagePools& p, int pages, int page, const int32_t* src, const int32_t* dst, int n,
                              int32_t* status, cudaStream_t s);

}  // namespace h3b
