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
from .ops import _cuda, _p, _stream

HEAD_DIM = 128
PAGE_TOKENS = (16, 32, 64, 128)
DTYPE_CODES = {torch.float16: 1, torch.bfloat16: 2, torch.float8_e4m3fn: 3}
STATUS_TEXT = {
    1: "not enough free pages",
    2: "a sequence would outgrow its row of the table",
    3: "a slot lies outside the table or was named twice",
    4: "fork into a slot that holds tokens",
    5: "token counts are negative, unordered or beyond the length",
    6: "a page lies outside the pool",
}


def _index(t: torch.Tensor, what: str, n: int | None = None) -> torch.Tensor:
    if t.dtype != torch.int32 or t.ndim != 1 or not t.is_cuda or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous int32 CUDA vector")
    if n is not None and t.numel() != n:
        raise ValueError(f"{what} must have {n} entries")
    return t


def _token_rows(x: torch.Tensor, heads: int | None, what: str) -> torch.Tensor:
    """[T, H, 128] fp16 / bf16 with contiguous heads (any row stride that keeps 16-byte alignment)."""
    if x.ndim != 3 or x.shape[2] != HEAD_DIM or (heads is not None and x.shape[1] != heads):
        raise ValueError(f"{what} must be [tokens, {'heads' if heads is None else heads}, {HEAD_DIM}]")
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"{what} must be bfloat16 or float16")
    st = x.stride()
    if st[2] != 1 or st[1] != HEAD_DIM or st[0] % 8 or st[0] < x.shape[1] * HEAD_DIM or x.data_ptr() % 16:
        x = x.contiguous()
    return x


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
        k, v = self.k, self.v
        _cuda("PagedKVCache", k, v, self.table, self.lens, self.refs, self.status, self.k_scale, self.v_scale)
        if k.ndim != 5 or k.shape[4] != HEAD_DIM or k.shape != v.shape or k.dtype != v.dtype:
            raise ValueError("k and v must be [layers, pages, kv heads, page tokens, 128] of one type")
        if k.dtype not in DTYPE_CODES:
            raise ValueError("a cache holds float16, bfloat16 or float8_e4m3fn")
        if k.shape[3] not in PAGE_TOKENS:
            raise ValueError(f"page tokens must be one of {PAGE_TOKENS}")
        layers, pages, heads, page, _ = k.shape
        t = self.table
        if t.ndim != 2 or self.lens.shape != (t.shape[0],) or self.refs.shape != (pages,) or self.status.numel() != 1:
            raise ValueError("table [slots, width], lens [slots], refs [pages] and status [1] do not fit together")
        for x in (t, self.lens, self.refs, self.status):
            if x.dtype != torch.int32:
                raise ValueError("table, lens, refs and status must be int32")
        if k.dtype == torch.float8_e4m3fn:
            for x in (self.k_scale, self.v_scale):
                if x is None or x.dtype != torch.float32 or x.shape != (layers, heads) or not x.is_contiguous():
                    raise ValueError("an e4m3 cache needs float32 k_scale and v_scale [layers, kv heads]")
        for x in (k, v, t, self.lens, self.refs):
            if not x.is_contiguous():
                raise ValueError("cache tensors must be contiguous")
        scales = self.k_scale is not None and k.dtype == torch.float8_e4m3fn
        self._ref = ctypes.byref(PageCacheStruct(
            k.data_ptr(), v.data_ptr(), layers, pages, heads, page, DTYPE_CODES[k.dtype],
            self.k_scale.data_ptr() if scales else None, self.v_scale.data_ptr() if scales else None, t.data_ptr(),
            t.shape[0], t.shape[1], self.lens.data_ptr(), self.refs.data_ptr(), self.status.data_ptr()))

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

    @property
    def page_tokens(self) -> int:
        return self.k.shape[3]

    @property
    def kv_heads(self) -> int:
        return self.k.shape[2]

    def _workspace(self, n: int) -> torch.Tensor:
        return torch.empty(lib().h3b_pages_workspace_bytes(n, self.k.shape[1]), device=self.k.device, dtype=torch.uint8)

    def extend(self, slots: torch.Tensor, starts: torch.Tensor | None = None) -> None:
        """Room for starts[i + 1] - starts[i] more tokens (None: one) of each of the distinct slots,
        in every layer; a shared, partly filled last page is copied first."""
        n = _index(slots, "slots").numel()
        if starts is not None:
            _index(starts, "starts", n + 1)
        ws = self._workspace(n)
        check(lib().h3b_pages_extend(self._ref, _p(slots), n, _p(starts), _p(ws), ws.numel(), _stream(self.k)),
              "pages_extend")

    def write(self, slots: torch.Tensor, k: torch.Tensor, v: torch.Tensor, starts: torch.Tensor | None = None,
              layer: int = 0) -> None:
        """K/V rows [tokens, kv heads, 128] into the last tokens of each slot, as `extend` made room for them."""
        n = _index(slots, "slots").numel()
        if starts is not None:
            _index(starts, "starts", n + 1)
        k, v = _token_rows(k, self.kv_heads, "k"), _token_rows(v, self.kv_heads, "v")
        _cuda("PagedKVCache.write", k, v)
        if k.shape != v.shape or k.dtype != v.dtype:
            raise ValueError("k and v must have one shape and type")
        if starts is None and k.shape[0] != n:
            raise ValueError("without starts there is one token for each slot")
        if self.k.dtype not in (k.dtype, torch.float8_e4m3fn):
            raise ValueError(f"a {self.k.dtype} cache does not take {k.dtype} rows")
        check(lib().h3b_pages_write(self._ref, int(layer), _p(slots), n, _p(starts), _p(k), k.stride(0), _p(v),
                                    v.stride(0), DTYPE_CODES[k.dtype], k.shape[0], _stream(self.k)), "pages_write")

    def append(self, slots: torch.Tensor, k: torch.Tensor, v: torch.Tensor, starts: torch.Tensor | None = None,
               layer: int = 0) -> None:
        """extend, then write into `layer` (the other layers' rows are the caller's to write)."""
        self.extend(slots, starts)
        self.write(slots, k, v, starts, layer)

    def fork(self, src: torch.Tensor, dst: torch.Tensor) -> None:
        """Empty slots dst[i] become sequences that share the pages of src[i]."""
        n = _index(src, "src").numel()
        check(lib().h3b_pages_fork(self._ref, _p(src), _p(_index(dst, "dst", n)), n, _stream(self.k)), "pages_fork")

    def truncate(self, slots: torch.Tensor, keep: torch.Tensor) -> None:
        """Each of the distinct slots keeps its first keep[i] tokens."""
        n = _index(slots, "slots").numel()
        check(lib().h3b_pages_truncate(self._ref, _p(slots), _p(_index(keep, "keep", n)), n, _stream(self.k)),
              "pages_truncate")

    def free(self, slots: torch.Tensor) -> None:
        """The distinct slots become empty; pages that no other sequence shares are free again."""
        n = _index(slots, "slots").numel()
        check(lib().h3b_pages_truncate(self._ref, _p(slots), None, n, _stream(self.k)), "pages_truncate")

    def compact(self) -> None:
        """Pages in use move to the front of the pool."""
        ws = self._workspace(0)
        check(lib().h3b_pages_compact(self._ref, _p(ws), ws.numel(), _stream(self.k)), "pages_compact")

    def copy_pages(self, src: torch.Tensor, dst: torch.Tensor) -> None:
        """Pages src[i] over pages dst[i] in every layer (no page may be both); the tables stay."""
        n = _index(src, "src").numel()
        check(lib().h3b_pages_copy(self._ref, _p(src), _p(_index(dst, "dst", n)), n, _stream(self.k)), "pages_copy")

    def check(self) -> None:
        """Wait for the stream; raise, and clear the status word, if a call could not be done."""
        code = int(self.status.item())
        if code:
            self.status.zero_()
            raise H3BError(f"paged cache: {STATUS_TEXT.get(code, code)}; nothing was changed since")
