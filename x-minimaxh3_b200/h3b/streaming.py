"""Streaming attention over libh3b.so: new tokens attend to the keys before them.

Where the backends of `attention` take a whole sequence, bidirectionally and quantized,
these take the tokens that come next -- a video chunk by chunk, a prompt, one decoded
token -- in bf16 or fp16, with grouped heads and ragged batches:

* window_attention        contiguous K/V
* paged_window_attention  K/V of a 16-bit PagedKVCache
* decode_attention        one new token per sequence, 16-bit or e4m3 cache
* WindowAttentionB200     an AttentionBackend callable (q, k, v [L, H, 128]) over
                          window_attention: sinks, chunk and window follow from the
                          request's protected prefix and video layout

Of a sequence's Lk keys the Lq queries are the last Lq tokens.  The query at position
p = Lk - Lq + i sees key j when j <= last(p) and (last(p) - j < window or j < sinks).
last(p) = p, or with chunk > 1 the end of p's chunk (a latent frame sees itself whole),
chunks counted from the end of the `sinks` first tokens, which form one of their own.
A query that sees nothing gives 0.

Scores, softmax and sums are fp32.  The weights are rounded to the queries' type for the V
product (over an e4m3 cache: to fp16, as bf16 queries are, under a power of two per head); their
sum is not.
"""

from __future__ import annotations

import math

import torch

from . import context as _context
from ._lib import check, lib
from .cache import DTYPE_CODES, HEAD_DIM, PagedKVCache, _index, _ptr, _row_step, _stream, _token_rows

UNLIMITED = 1 << 30
MAX_SCALE = torch.finfo(torch.float32).max * math.log(2)  # the kernels' scores are powers of two


def _rule(window: int | None, sinks: int, chunk: int) -> tuple[int, int, int]:
    window = UNLIMITED if window is None else int(window)
    sinks, chunk = int(sinks), int(chunk)
    if window < 0 or sinks < 0 or chunk < 1:
        raise ValueError("need window >= 0, sinks >= 0 and chunk >= 1")
    return window, sinks, chunk


def _output(out: torch.Tensor | None, q: torch.Tensor) -> tuple[torch.Tensor, int]:
    if out is None:
        return torch.empty_like(q, memory_format=torch.contiguous_format), q.shape[1] * HEAD_DIM
    if out.shape != q.shape or out.dtype != q.dtype or out.get_device() != q.get_device():
        raise ValueError("out must have q's shape and type, on its GPU")
    step = _row_step(out)
    if not step:
        raise ValueError("out must have contiguous heads and 16-byte aligned rows")
    return out, step


def _scale(scale: float | None) -> float:
    if scale is None:
        return 1.0 / math.sqrt(HEAD_DIM)
    if not 0.0 < float(scale) < MAX_SCALE:
        raise ValueError("the softmax scale must be positive and finite, times log2(e) too")
    return float(scale)


def _workspace(workspace: torch.Tensor | None, need: int, q: torch.Tensor) -> torch.Tensor:
    if workspace is None:
        return q.new_empty(need, dtype=torch.uint8)
    if (workspace.numel() * workspace.element_size() < need or workspace.get_device() != q.get_device()
            or not workspace.is_contiguous()):
        raise ValueError(f"the workspace must have {need} contiguous bytes on the queries' GPU")
    return workspace


def _window_workspace(workspace, q, seqs, kv_heads, keys, rule) -> tuple[torch.Tensor | None, int]:
    need = lib().h3b_window_workspace_bytes(q.shape[0], seqs, q.shape[1], kv_heads, keys, *rule)
    return (_workspace(workspace, need, q), need) if need > 0 else (None, 0)


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, window: int | None = None, sinks: int = 0,
                     chunk: int = 1, scale: float | None = None, query_starts: torch.Tensor | None = None,
                     key_starts: torch.Tensor | None = None, out: torch.Tensor | None = None,
                     workspace: torch.Tensor | None = None) -> torch.Tensor:
    """q [Tq, Hq, 128], k / v [Tk, Hkv, 128] -> [Tq, Hq, 128]; bf16 or fp16.

    query_starts / key_starts: int32 [sequences + 1] first rows of each sequence of a
    ragged batch (from 0 to Tq / Tk); None: one sequence.  workspace: uint8, reused by
    calls on one stream."""
    if not (q.is_cuda and k.is_cuda and v.is_cuda):
        raise RuntimeError("window_attention runs only on CUDA tensors (the B200 library has no CPU path)")
    gpu = q.get_device()
    if not k.get_device() == v.get_device() == gpu:
        raise ValueError("q, k and v must be on one GPU")
    (q, q_step), (k, k_step), (v, v_step) = (_token_rows(q, None, "q"), _token_rows(k, None, "k"),
                                             _token_rows(v, None, "v"))
    if k.shape != v.shape or not q.dtype is k.dtype is v.dtype:
        raise ValueError("k and v must have one shape, and q their type")
    if k.shape[1] == 0 or q.shape[1] % k.shape[1]:
        raise ValueError("the query heads must be a multiple of the kv heads")
    window, sinks, chunk = _rule(window, sinks, chunk)
    seqs = 1
    if (query_starts is None) != (key_starts is None):
        raise ValueError("query_starts and key_starts come together")
    if query_starts is not None:
        seqs = _index(query_starts, "query_starts", gpu).numel() - 1
        _index(key_starts, "key_starts", gpu, seqs + 1)
        if seqs < 1:
            raise ValueError("query_starts needs at least two entries")
    out, out_step = _output(out, q)
    workspace, size = _window_workspace(workspace, q, seqs, k.shape[1], k.shape[0], (window, sinks, chunk))
    check(lib().h3b_window_attention(_ptr(q), q_step, _ptr(k), k_step, _ptr(v), v_step,
                                     DTYPE_CODES[q.dtype], q.shape[0], k.shape[0], _ptr(query_starts), _ptr(key_starts),
                                     seqs, q.shape[1], k.shape[1], window, sinks, chunk, _scale(scale), _ptr(out),
                                     out_step, _ptr(workspace), size, _stream(gpu)), "window_attention")
    return out


def _cached_queries(q: torch.Tensor, cache: PagedKVCache, layer: int, what: str) -> tuple[torch.Tensor, int]:
    if not q.is_cuda:
        raise RuntimeError(f"{what} runs only on CUDA tensors (the B200 library has no CPU path)")
    if q.get_device() != cache._gpu:
        raise ValueError("q must be on the cache's GPU")
    q, step = _token_rows(q, None, "q")
    heads = q.shape[1]
    if heads == 0 or heads % cache.kv_heads:
        raise ValueError("the query heads must be a multiple of the kv heads")
    if not 0 <= layer < cache.k.shape[0]:
        raise ValueError(f"the cache has no layer {layer}")
    return q, step


def paged_window_attention(q: torch.Tensor, cache: PagedKVCache, slots: torch.Tensor | None = None, *,
                           window: int | None = None, sinks: int = 0, chunk: int = 1, scale: float | None = None,
                           query_starts: torch.Tensor | None = None, layer: int = 0, out: torch.Tensor | None = None,
                           workspace: torch.Tensor | None = None) -> torch.Tensor:
    """q [Tq, Hq, 128]: the last tokens of the cache's sequences `slots` (int32; None: slot 0, 1, ...),
    already appended.  query_starts: int32 [sequences + 1]; None: one sequence."""
    q, q_step = _cached_queries(q, cache, layer, "paged_window_attention")
    if cache.k.dtype != q.dtype:
        raise ValueError(f"a {cache.k.dtype} cache does not serve {q.dtype} queries of several tokens")
    window, sinks, chunk = _rule(window, sinks, chunk)
    seqs = 1 if query_starts is None else _index(query_starts, "query_starts", cache._gpu).numel() - 1
    if seqs < 1:
        raise ValueError("query_starts needs at least two entries")
    if slots is not None:
        _index(slots, "slots", cache._gpu, seqs)
    elif seqs > cache.table.shape[0]:
        raise ValueError("more sequences than the cache has slots")
    out, out_step = _output(out, q)
    workspace, size = _window_workspace(workspace, q, seqs, cache.kv_heads, cache.table.shape[1] * cache.page_tokens,
                                        (window, sinks, chunk))
    check(lib().h3b_paged_window_attention(_ptr(q), q_step, DTYPE_CODES[q.dtype], q.shape[0], _ptr(query_starts),
                                           _ptr(slots), seqs, q.shape[1], cache._ref, layer, window, sinks, chunk,
                                           _scale(scale), _ptr(out), out_step, _ptr(workspace), size,
                                           _stream(cache._gpu)), "paged_window_attention")
    return out


def decode_attention(q: torch.Tensor, cache: PagedKVCache, slots: torch.Tensor | None = None, *,
                     window: int | None = None, sinks: int = 0, scale: float | None = None, layer: int = 0,
                     out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """q [n, Hq, 128]: the last token of each of the cache's sequences `slots` (int32 [n]; None: slots
    0..n-1), already appended -> [n, Hq, 128].  workspace: uint8, reused by calls on one stream."""
    q, q_step = _cached_queries(q, cache, layer, "decode_attention")
    if cache.k.dtype not in (q.dtype, torch.float8_e4m3fn):
        raise ValueError(f"a {cache.k.dtype} cache does not serve {q.dtype} queries")
    window, sinks, _ = _rule(window, sinks, 1)
    n = q.shape[0]
    if slots is not None:
        _index(slots, "slots", cache._gpu, n)
    elif n > cache.table.shape[0]:
        raise ValueError("more sequences than the cache has slots")
    need = lib().h3b_decode_workspace_bytes(n, q.shape[1], cache._ref)
    if need:
        workspace = _workspace(workspace, need, q)
    out, out_step = _output(out, q)
    check(lib().h3b_decode_attention(_ptr(q), q_step, DTYPE_CODES[q.dtype], _ptr(slots), n, q.shape[1], cache._ref,
                                     layer, window, sinks, _scale(scale), _ptr(out), out_step, _ptr(workspace), need,
                                     _stream(cache._gpu)), "decode_attention")
    return out


class WindowAttentionB200:
    """Streaming backend (q, k, v: bf16 [L, H, 128]; fewer queries than keys for a next chunk).

    The request's protected prefix stays visible (sinks) and its video layout sets the
    chunk: every latent frame sees itself, the prefix and the `frames` - 1 frames before
    it (all of them when `frames` is None).  Without a layout attention is causal with a
    window of `tokens` (None: unlimited).

    It is called with a chunk's rows; the long-sequence protocol of the whole-sequence
    backends (resolve_long_sequence_backend and what follows) is not its form."""

    approximate = True

    def __init__(self, frames: int | None = None, tokens: int | None = None, context=None) -> None:
        if frames is not None and frames < 1 or tokens is not None and tokens < 1:
            raise ValueError("a window holds at least one frame and one token")
        self.frames, self.tokens = frames, tokens
        self.context = context if context is not None else _context

    def rule(self) -> dict:
        """window, sinks and chunk of the current request."""
        prefix = int(_context.source_getter(self.context, "current_attention_protected_prefix", 0))
        layout = _context.source_getter(self.context, "current_attention_video_layout", None)
        if layout is None:
            return dict(window=self.tokens, sinks=prefix, chunk=1)
        chunk = int(layout[1])
        return dict(window=None if self.frames is None else self.frames * chunk, sinks=prefix, chunk=chunk)

    def __call__(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
        return window_attention(q, k, v, **self.rule())

    def cached(self, q: torch.Tensor, cache: PagedKVCache, slots: torch.Tensor, layer: int = 0,
               query_starts: torch.Tensor | None = None) -> torch.Tensor:
        """The same over a paged cache that already holds the new tokens."""
        return paged_window_attention(q, cache, slots, layer=layer, query_starts=query_starts, **self.rule())
