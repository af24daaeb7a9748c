"""A paged K/V cache whose page work runs on the device.

    cache = PagedKVCache.create(layers=4, pages=2048, page_tokens=64, kv_heads=8, slots=32, max_tokens=16384)
    cache.extend(slots, starts)             # room for new tokens, once for all layers
    cache.write(slots, k, v, starts, layer=0)
    cache.append(slots, k, v)               # extend + write of a one-layer cache
    cache.fork(src, dst)                    # sequences that share pages until they are written to
    cache.truncate(slots, keep); cache.free(slots)
    cache.compact()                         # live pages to the front of the pool
    cache.copy_pages(src, dst)
    cache.check()                           # raises if a call could not be done

Slots, pages and token counts are int32 CUDA tensors and every call is asynchronous on
the current stream: nothing waits for the host, so whole steps can be captured in CUDA
graphs.  A call that cannot be done (no free pages, a slot named twice, ...) changes
nothing, and neither does any call after it until `check` (which reads the status word
and so waits for the stream) has reported it.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch

from ._lib import H3BError, PageCacheStruct, check, lib

HEAD_DIM = 128
PAGE_TOKENS = (16, 32, 64, 128)
DTYPE_CODES = {torch.float16: 1, torch.bfloat16: 2, torch.float8_e4m3fn: 3}
STATUS_TEXT = {
    1: "not enough free pages",
    2: "a sequence would outgrow its row of the table",
    3: "a slot lies outside the table or was named twice",
    4: "fork into a slot that holds tokens",
    5: "token counts are negative, unordered or beyond the length or the rows",
    6: "a page lies outside the pool, or was copied to twice, or both from and to",
}


_raw_stream = torch._C._cuda_getCurrentRawStream
_current_gpu = torch._C._cuda_getDevice


def _stream(gpu: int) -> int:
    """The current stream of the GPU that a call's tensors are on, as the C entries take it (a token's worth
    of calls is short enough for the stream object's construction to count).  The library launches on the
    current GPU, which has to be that one: a kernel of another would reach into memory that is not its own."""
    if _current_gpu() != gpu:
        raise RuntimeError(f"the tensors are on cuda:{gpu}, the current device is cuda:{_current_gpu()}")
    return _raw_stream(gpu)


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _index(t: torch.Tensor, what: str, gpu: int, n: int | None = None) -> torch.Tensor:
    if t.dtype is not torch.int32 or t.ndim != 1 or t.get_device() != gpu or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous int32 CUDA vector on the other tensors' GPU")
    if n is not None and t.shape[0] != n:
        raise ValueError(f"{what} must have {n} entries")
    return t


def _row_step(x: torch.Tensor) -> int:
    """Elements from one of x's rows [T, H, 128] to the next, if the kernels take them as they lie:
    contiguous heads, 16-byte aligned rows apart from each other; else 0.  Strides of dimensions of one
    entry, which may be anything, do not count."""
    row, head, channel = x.stride()
    tokens, heads, _ = x.shape
    if channel != 1 or (head != HEAD_DIM and heads != 1) or x.data_ptr() % 16:
        return 0
    if tokens <= 1:
        return heads * HEAD_DIM
    return row if row % 8 == 0 and row >= heads * HEAD_DIM else 0


def _token_rows(x: torch.Tensor, heads: int | None, what: str) -> tuple[torch.Tensor, int]:
    """[T, H, 128] fp16 / bf16 rows and the step between them; copied where they do not lie right."""
    shape = x.shape
    if len(shape) != 3 or shape[2] != HEAD_DIM or (heads is not None and shape[1] != heads):
        raise ValueError(f"{what} must be [tokens, {'heads' if heads is None else heads}, {HEAD_DIM}]")
    if x.dtype is not torch.bfloat16 and x.dtype is not torch.float16:
        raise ValueError(f"{what} must be bfloat16 or float16")
    step = _row_step(x)
    if not step:
        # not contiguous(), which returns rows at an odd address, and any single row, as they are
        x, step = x.clone(memory_format=torch.contiguous_format), shape[1] * HEAD_DIM
    return x, step


@dataclass
class PagedKVCache:
    """K/V pools of one or more layers behind one page table (h3b_page_cache).

    The tensors are changed in place and must not be replaced by others."""

    k: torch.Tensor       # [layers, pages, kv heads, page tokens, 128] fp16, bf16 or e4m3
    v: torch.Tensor
    table: torch.Tensor   # int32 [slots, pages per sequence], -1: no page
    lens: torch.Tensor    # int32 [slots]
    refs: torch.Tensor    # int32 [pages]
    status: torch.Tensor  # int32 [1]
    k_scale: torch.Tensor | None = None  # f32 [layers, kv heads] of an e4m3 cache: value = code * scale
    v_scale: torch.Tensor | None = None

    def __post_init__(self) -> None:
        k, v, t, lens, refs, status = self.k, self.v, self.table, self.lens, self.refs, self.status
        shape, dtype = k.shape, k.dtype
        if not k.is_cuda:
            raise RuntimeError("PagedKVCache runs only on CUDA tensors (the B200 library has no CPU path)")
        self._gpu = gpu = k.get_device()
        if not (v.get_device() == gpu == t.get_device() == lens.get_device() and refs.get_device() == gpu
                and status.get_device() == gpu):
            raise ValueError("cache tensors must be on one GPU")
        if len(shape) != 5 or shape[4] != HEAD_DIM or shape != v.shape or dtype is not v.dtype:
            raise ValueError("k and v must be [layers, pages, kv heads, page tokens, 128] of one type")
        if dtype not in DTYPE_CODES:
            raise ValueError("a cache holds float16, bfloat16 or float8_e4m3fn")
        layers, pages, heads, page, _ = shape
        if page not in PAGE_TOKENS:
            raise ValueError(f"page tokens must be one of {PAGE_TOKENS}")
        rows, width = t.shape
        if lens.shape != (rows,) or refs.shape != (pages,) or status.numel() != 1:
            raise ValueError("table [slots, width], lens [slots], refs [pages] and status [1] do not fit together")
        if not t.dtype is lens.dtype is refs.dtype is status.dtype is torch.int32:
            raise ValueError("table, lens, refs and status must be int32")
        if not (k.is_contiguous() and v.is_contiguous() and t.is_contiguous() and lens.is_contiguous()
                and refs.is_contiguous()):
            raise ValueError("cache tensors must be contiguous")
        k_scale = v_scale = None
        if dtype is torch.float8_e4m3fn:
            for x in (self.k_scale, self.v_scale):
                if (x is None or x.dtype is not torch.float32 or x.shape != (layers, heads) or not x.is_contiguous()
                        or x.get_device() != gpu):
                    raise ValueError("an e4m3 cache needs float32 k_scale and v_scale [layers, kv heads] on its GPU")
            k_scale, v_scale = self.k_scale.data_ptr(), self.v_scale.data_ptr()
        self.page_tokens, self.kv_heads = page, heads
        self._ref = ctypes.byref(PageCacheStruct(
            k.data_ptr(), v.data_ptr(), layers, pages, heads, page, DTYPE_CODES[dtype], k_scale, v_scale, t.data_ptr(),
            rows, width, lens.data_ptr(), refs.data_ptr(), status.data_ptr()))

    @classmethod
    def create(cls, layers: int, pages: int, page_tokens: int, kv_heads: int, slots: int, max_tokens: int,
               dtype: torch.dtype = torch.bfloat16, device="cuda", k_scale: torch.Tensor | None = None,
               v_scale: torch.Tensor | None = None) -> PagedKVCache:
        """An empty cache; a sequence grows to max_tokens at most."""
        if page_tokens not in PAGE_TOKENS:
            raise ValueError(f"page tokens must be one of {PAGE_TOKENS}")
        if min(layers, pages, kv_heads, slots, max_tokens) <= 0:
            raise ValueError("layers, pages, kv heads, slots and max tokens must be positive")
        shape = (layers, pages, kv_heads, page_tokens, HEAD_DIM)
        ints = dict(device=device, dtype=torch.int32)
        return cls(torch.empty(shape, device=device, dtype=dtype), torch.empty(shape, device=device, dtype=dtype),
                   torch.full((slots, -(-max_tokens // page_tokens)), -1, **ints), torch.zeros(slots, **ints),
                   torch.zeros(pages, **ints), torch.zeros(1, **ints), k_scale, v_scale)

    def _workspace(self, n: int) -> torch.Tensor:
        return self.status.new_empty(lib().h3b_pages_workspace_bytes(n, self.k.shape[1]), dtype=torch.uint8)

    def extend(self, slots: torch.Tensor, starts: torch.Tensor | None = None) -> None:
        """Room for starts[i + 1] - starts[i] more tokens (None: one) of each of the distinct slots,
        in every layer; a shared, partly filled last page is copied first."""
        n = _index(slots, "slots", self._gpu).numel()
        if starts is not None:
            _index(starts, "starts", self._gpu, n + 1)
        ws = self._workspace(n)
        check(lib().h3b_pages_extend(self._ref, _ptr(slots), n, _ptr(starts), _ptr(ws), ws.numel(),
                                     _stream(self._gpu)), "pages_extend")

    def write(self, slots: torch.Tensor, k: torch.Tensor, v: torch.Tensor, starts: torch.Tensor | None = None,
              layer: int = 0) -> None:
        """K/V rows [tokens, kv heads, 128] into the last tokens of each of the distinct slots, as `extend` made
        room for them."""
        self._rows_into(lib().h3b_pages_write, "pages_write", slots, k, v, starts, layer)

    def _rows_into(self, entry, what, slots, k, v, starts, layer, ws=None) -> None:
        n = _index(slots, "slots", self._gpu).shape[0]
        if starts is not None:
            _index(starts, "starts", self._gpu, n + 1)
        k, k_step = _token_rows(k, self.kv_heads, "k")
        v, v_step = _token_rows(v, self.kv_heads, "v")
        if not k.get_device() == v.get_device() == self._gpu:
            raise RuntimeError("PagedKVCache takes only CUDA tensors on its GPU (the B200 library has no CPU path)")
        if k.shape != v.shape or k.dtype is not v.dtype:
            raise ValueError("k and v must have one shape and type")
        if starts is None and k.shape[0] != n:
            raise ValueError("without starts there is one token for each slot")
        if self.k.dtype is not k.dtype and self.k.dtype is not torch.float8_e4m3fn:
            raise ValueError(f"a {self.k.dtype} cache does not take {k.dtype} rows")
        args = (self._ref, int(layer), slots.data_ptr(), n, _ptr(starts), k.data_ptr(), k_step, v.data_ptr(),
                v_step, DTYPE_CODES[k.dtype], k.shape[0])
        if ws is not None:
            args += (ws.data_ptr(), ws.shape[0])
        check(entry(*args, _stream(self._gpu)), what)

    def append(self, slots: torch.Tensor, k: torch.Tensor, v: torch.Tensor, starts: torch.Tensor | None = None,
               layer: int = 0) -> None:
        """extend, then write into `layer` (the other layers' rows are the caller's to write).  Rows outside
        every sequence are not used; starts that reach past the rows are refused."""
        self._rows_into(lib().h3b_pages_append, "pages_append", slots, k, v, starts, layer,
                        self._workspace(slots.shape[0]))

    def fork(self, src: torch.Tensor, dst: torch.Tensor) -> None:
        """Empty slots dst[i] become sequences that share the pages of src[i]."""
        n = _index(src, "src", self._gpu).numel()
        check(lib().h3b_pages_fork(self._ref, _ptr(src), _ptr(_index(dst, "dst", self._gpu, n)), n,
                                   _stream(self._gpu)), "pages_fork")

    def truncate(self, slots: torch.Tensor, keep: torch.Tensor) -> None:
        """Each of the distinct slots keeps its first keep[i] tokens."""
        n = _index(slots, "slots", self._gpu).numel()
        check(lib().h3b_pages_truncate(self._ref, _ptr(slots), _ptr(_index(keep, "keep", self._gpu, n)), n,
                                       _stream(self._gpu)), "pages_truncate")

    def free(self, slots: torch.Tensor) -> None:
        """The distinct slots become empty; pages that no other sequence shares are free again."""
        n = _index(slots, "slots", self._gpu).numel()
        check(lib().h3b_pages_truncate(self._ref, _ptr(slots), None, n, _stream(self._gpu)), "pages_truncate")

    def compact(self) -> None:
        """Pages in use move to the front of the pool."""
        ws = self._workspace(0)
        check(lib().h3b_pages_compact(self._ref, _ptr(ws), ws.numel(), _stream(self._gpu)), "pages_compact")

    def copy_pages(self, src: torch.Tensor, dst: torch.Tensor) -> None:
        """Pages src[i] over the distinct pages dst[i] in every layer (no page may be both); the tables stay."""
        n = _index(src, "src", self._gpu).numel()
        check(lib().h3b_pages_copy(self._ref, _ptr(src), _ptr(_index(dst, "dst", self._gpu, n)), n,
                                   _stream(self._gpu)), "pages_copy")

    def check(self) -> None:
        """Wait for the stream; raise, and clear the status word, if a call could not be done."""
        code = int(self.status.item())
        if code:
            self.status.zero_()
            raise H3BError(f"paged cache: {STATUS_TEXT.get(code, code)}; nothing was changed since")
