"""The launch count of calls that take a different number of kernels at different sizes (GPU)."""

import pytest
import torch

pytestmark = pytest.mark.gpu

from streaming_util import D  # noqa: E402


def _i32(x):
    return torch.tensor(list(x), dtype=torch.int32, device="cuda")


def _rows(n, heads):
    return torch.randn(n, heads, D, device="cuda").to(torch.bfloat16)


def _count(call):
    from h3b import _lib

    _lib.reset_launch_count()
    call()
    return _lib.launch_count()


def _cache(slots, tokens):
    from h3b import PagedKVCache

    return PagedKVCache.create(1, 4096, 16, 2, slots, tokens)


def test_attention_launches():
    from h3b import decode_attention, window_attention

    q, k = _rows(64, 4), _rows(64, 2)
    assert _count(lambda: window_attention(q, k, k)) == 1            # no item is cut
    assert _count(lambda: window_attention(_rows(2000, 4), _rows(2000, 2), _rows(2000, 2))) == 2
    assert _count(lambda: window_attention(q[:0], k, k)) == 0
    assert _count(lambda: window_attention(q, k[:0], k[:0])) == 0    # cleared, not computed
    short, long = _cache(4, 256), _cache(4, 8192)
    for cache, launches in ((short, 1), (long, 2)):                  # a cluster per pair, or a list and a join
        cache.append(_i32(range(4)), k[:4], k[:4])
        assert _count(lambda: decode_attention(q[:4], cache)) == launches


def test_page_launches():
    cache = _cache(100, 1600)
    k = _rows(1000, 2)
    first = _i32(range(10))
    assert _count(lambda: cache.append(first, k[:100], k[:100], _i32(range(0, 101, 10)))) == 2
    assert _count(lambda: cache.extend(_i32([20, 21]), _i32([0, 600, 1000]))) == 2
    assert _count(lambda: cache.write(_i32([20, 21]), k[:10], k[:10], _i32([0, 6, 10]))) == 1
    assert _count(lambda: cache.write(_i32([20, 21]), k, k, _i32([0, 600, 1000]))) == 2
    assert _count(lambda: cache.fork(_i32([0]), _i32([30]))) == 1
    assert _count(lambda: cache.fork(_i32([0] * 60), _i32(range(31, 91)))) == 2      # 6,000 entries of the table
    assert _count(lambda: cache.free(_i32([30]))) == 1
    assert _count(lambda: cache.free(_i32(range(31, 91)))) == 2
    assert _count(lambda: cache.truncate(first, _i32([5] * 10))) == 1
    assert _count(cache.compact) == 3
    assert _count(lambda: cache.copy_pages(_i32([0]), _i32([4000]))) == 2
    cache.check()
