"""Host checks of the streaming operators and the paged cache (no GPU needed)."""

import ctypes

import pytest
import torch

import h3b
from h3b import _lib
from h3b._lib import PageCacheStruct, lib
from h3b.streaming import WindowAttentionB200, _rule


def _cache(**kw):
    f = dict(k=16, v=16, layers=1, pages=4, kv_heads=2, page_tokens=16, dtype=2, k_scale=None, v_scale=None, table=16,
             table_rows=4, table_width=8, lens=16, refs=16, status=16)
    f |= kw
    return ctypes.byref(PageCacheStruct(*[f[n] for n, _ in PageCacheStruct._fields_]))


D = ctypes.c_void_p(16)
ODD = ctypes.c_void_p(24)


def _window(q=D, qs=512, k=D, ks=256, v=D, vs=256, dtype=2, tq=8, tk=8, sq=None, sk=None, seqs=1, hq=4, hkv=2,
            window=4, sinks=0, chunk=1, out=D, os=512, ws=None, wsb=0):
    return lib().h3b_window_attention(q, qs, k, ks, v, vs, dtype, tq, tk, sq, sk, seqs, hq, hkv, window, sinks, chunk,
                                      0.1, out, os, ws, wsb, None)


@pytest.mark.parametrize("status,kw", [
    (-1, dict(q=None)), (-1, dict(out=None)), (-1, dict(k=None)), (-1, dict(hq=3)), (-1, dict(hkv=0)), (-2, dict(dtype=0)),
    (-2, dict(dtype=3)), (-1, dict(window=-1)), (-1, dict(sinks=-1)), (-1, dict(chunk=0)), (-1, dict(qs=504)),
    (-1, dict(qs=516)), (-1, dict(os=128)), (-1, dict(ks=128)), (-1, dict(vs=260)), (-2, dict(q=ODD)), (-2, dict(v=ODD)),
    (-2, dict(tq=1 << 31)), (-1, dict(tk=-1)), (-1, dict(tq=-1)), (-1, dict(seqs=2)), (-1, dict(sq=D)), (-1, dict(seqs=0)),
    (-1, dict(ws=D, wsb=100, tk=9000, window=9000)), (-2, dict(ws=ODD, wsb=1 << 40)), (0, dict(tq=0, q=None)),
])
def test_window_entry_refuses(status, kw):
    assert _window(**kw) == status


def _paged(q=D, dtype=2, tq=8, starts=None, seqs=1, hq=4, cache=None, layer=0):
    return lib().h3b_paged_window_attention(q, 512, dtype, tq, starts, None, seqs, hq, cache or _cache(), layer, 4, 0, 1,
                                            0.1, D, 512, None, 0, None)


@pytest.mark.parametrize("status,kw", [
    (-1, dict(cache=_cache(k=None))), (-1, dict(cache=_cache(table=None))), (-1, dict(cache=_cache(status=None))),
    (-1, dict(cache=_cache(pages=0))), (-1, dict(cache=_cache(layers=0))), (-2, dict(cache=_cache(page_tokens=48))),
    (-2, dict(cache=_cache(page_tokens=8))), (-2, dict(cache=_cache(page_tokens=256))), (-2, dict(cache=_cache(dtype=0))),
    (-2, dict(cache=_cache(dtype=1))), (-1, dict(cache=_cache(dtype=3))), (-2, dict(cache=_cache(k=24))),
    (-2, dict(cache=_cache(dtype=3, k_scale=16, v_scale=16))), (-2, dict(cache=_cache(pages=1 << 29))),
    (-2, dict(cache=_cache(table_rows=1 << 19))), (-2, dict(cache=_cache(table_width=1 << 27))), (-1, dict(layer=1)),
    (-1, dict(layer=-1)), (-1, dict(hq=5)), (-1, dict(seqs=2)), (-1, dict(q=None)), (0, dict(tq=0)),
])
def test_paged_entry_refuses(status, kw):
    assert _paged(**kw) == status


def _decode(q=D, dtype=2, seqs=2, hq=4, cache=None, ws=D, wsb=1 << 40, window=4):
    return lib().h3b_decode_attention(q, 512, dtype, None, seqs, hq, cache or _cache(), 0, window, 0, 0.1, D, 512, ws, wsb,
                                      None)


@pytest.mark.parametrize("status,kw", [
    (-1, dict(q=None)), (-2, dict(seqs=5000)), (-1, dict(ws=None, seqs=4000)), (-1, dict(wsb=8, seqs=4000)), (-2, dict(ws=ODD)),
    (-2, dict(dtype=1)), (-1, dict(hq=3)), (-1, dict(window=-2)), (-1, dict(cache=_cache(dtype=3, k_scale=16))),
    (0, dict(seqs=0)),
])
def test_decode_entry_refuses(status, kw):
    assert _decode(**kw) == status


def test_workspace_sizes():
    L = lib()
    assert L.h3b_window_workspace_bytes(8, 1, 4, 2, 896, 1 << 30, 0, 1) == 0          # seven tiles: items stay whole
    assert L.h3b_window_workspace_bytes(8, 1, 4, 2, 9000, 128, 0, 1) == 0             # the window keeps them short
    assert L.h3b_window_workspace_bytes(8, 1, 4, 2, 9000, 128, 4000, 1) != 0          # first tokens make them long
    for bad in ((-1, 1, 4, 2, 9, 9, 0, 1), (8, 0, 4, 2, 9, 9, 0, 1), (8, 1, 4, 3, 9, 9, 0, 1), (8, 1, 4, 2, 9, 9, 0, 0)):
        assert L.h3b_window_workspace_bytes(*bad) == -1
    assert L.h3b_decode_workspace_bytes(2, 3, _cache()) == -1
    assert L.h3b_decode_workspace_bytes(2, 4, None) == -1
    # few pairs of short sequences need none where there is a GPU; none is known here or there are 148 processors
    assert L.h3b_decode_workspace_bytes(4000, 4, _cache()) > 0


def test_page_entries_refuse():
    L, c = lib(), _cache()
    ws = L.h3b_pages_workspace_bytes(4, 4)
    assert ws >= 4 * (4 + 5 * 4 + 4) and ws % 4 == 0
    assert L.h3b_pages_extend(c, None, 1, None, D, ws, None) == -1
    assert L.h3b_pages_extend(c, D, 5, None, D, 1 << 20, None) == -1   # more slots than rows
    assert L.h3b_pages_extend(c, D, 4, None, D, ws - 4, None) == -1
    assert L.h3b_pages_extend(c, D, 0, None, None, 0, None) == 0
    assert L.h3b_pages_write(c, 0, D, 2, None, D, 256, D, 256, 1, 2, None) == -2   # fp16 rows, bf16 cache
    assert L.h3b_pages_write(c, 0, D, 2, None, D, 256, D, 256, 2, 3, None) == -1   # one token per slot
    assert L.h3b_pages_write(c, 0, D, 2, None, D, 128, D, 256, 2, 2, None) == -1
    assert L.h3b_pages_write(c, 0, D, 2, None, ODD, 256, D, 256, 2, 2, None) == -2
    assert L.h3b_pages_write(c, 1, D, 2, None, D, 256, D, 256, 2, 2, None) == -1
    assert L.h3b_pages_write(c, 0, D, 2, None, D, 256, D, 256, 2, 0, None) == 0
    assert L.h3b_pages_fork(c, D, None, 1, None) == -1
    assert L.h3b_pages_fork(c, D, D, 9, None) == -1
    assert L.h3b_pages_truncate(c, None, None, 1, None) == -1
    assert L.h3b_pages_compact(c, D, 8, None) == -1
    assert L.h3b_pages_compact(_cache(refs=None), D, 1 << 20, None) == -1
    assert L.h3b_pages_copy(c, D, D, 5, None) == -1
    assert b"pages_copy" in L.h3b_last_error()


def test_python_entries_refuse_cpu_tensors():
    x = torch.zeros(4, 2, 128, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        h3b.window_attention(x, x, x)
    with pytest.raises(RuntimeError, match="CUDA"):
        h3b.PagedKVCache.create(1, 4, 16, 2, 2, 32, device="cpu")
    with pytest.raises(ValueError, match="page tokens"):
        h3b.PagedKVCache.create(1, 4, 20, 2, 2, 32, device="cpu")
    with pytest.raises(ValueError, match="positive"):
        h3b.PagedKVCache.create(1, 0, 16, 2, 2, 32, device="cpu")


def test_rule_validation():
    assert _rule(None, 3, 1) == (1 << 30, 3, 1)
    for bad in ((-1, 0, 1), (4, -1, 1), (4, 0, 0)):
        with pytest.raises(ValueError):
            _rule(*bad)
    with pytest.raises(ValueError):
        WindowAttentionB200(frames=0)
    with pytest.raises(ValueError):
        WindowAttentionB200(tokens=0)


def test_backend_rule_reads_the_request():
    from h3b import context as C

    b = WindowAttentionB200(frames=3)
    assert b.rule() == dict(window=None, sinks=0, chunk=1)
    with C.attention_protected_prefix(50), C.attention_video_layout(7, 90):
        assert b.rule() == dict(window=270, sinks=50, chunk=90)
        assert WindowAttentionB200().rule() == dict(window=None, sinks=50, chunk=90)
    assert WindowAttentionB200(tokens=9).rule() == dict(window=9, sinks=0, chunk=1)


def test_struct_matches_the_header():
    import os
    import re

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    text = open(os.path.join(root, "include", "h3b.h")).read()
    body = re.search(r"typedef struct h3b_page_cache \{(.*?)\} h3b_page_cache;", text, re.S).group(1)
    names = []
    for decl in body.split(";"):
        decl = decl.strip()
        if decl:
            names += [re.sub(r".*[ *]", "", n.strip()) for n in decl.split(",")]
    assert names == [n for n, _ in _lib.PageCacheStruct._fields_]
