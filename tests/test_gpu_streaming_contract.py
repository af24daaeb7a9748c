"""What a cache's refused calls leave as it was, and what they are refused for (GPU)."""

import pytest
import torch

pytestmark = pytest.mark.gpu

from streaming_util import D, HostCache  # noqa: E402


def _i32(x):
    return torch.tensor(list(x), dtype=torch.int32, device="cuda")


def _rows(n, heads=2, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(n, heads, D, device="cuda", generator=g).to(torch.bfloat16)


def _filled(pages=8, layers=1):
    """Slots 0 and 1 with 20 and 30 tokens; every page holds values of its own."""
    from h3b import PagedKVCache

    cache = PagedKVCache.create(layers, pages, 16, 2, 6, 64)
    g = torch.Generator(device="cuda").manual_seed(3)
    for pool in (cache.k, cache.v):
        pool.copy_(torch.randn(pool.shape, device="cuda", generator=g))
    cache.append(_i32([0, 1]), _rows(50), _rows(50, seed=2), _i32([0, 20, 50]))
    cache.check()
    return cache, HostCache(cache)


# ------------------------------------------------------------------------------ copy_pages

@pytest.mark.parametrize("src,dst", [([0, 99], [7, 6]), ([0], [8]), ([-1, 0], [6, 7]), ([0, 1], [7, -3]),
                                     ([0, 1, 2], [7, 6, 7]), ([0, 6], [6, 7]), ([5], [5]), ([0, 1 << 30], [6, 7])], ids=str)
def test_refused_page_copies_change_nothing(src, dst):
    """Pages outside the pool, targets named twice, pages both copied from and to: no pair is copied."""
    from h3b import H3BError

    cache, host = _filled(layers=2)
    cache.copy_pages(_i32(src), _i32(dst))
    host.assert_equal(cache)
    with pytest.raises(H3BError, match="outside the pool"):
        cache.check()
    cache.copy_pages(_i32([0, 0]), _i32([7, 6]))
    cache.check()
    assert torch.equal(cache.k[:, 7], cache.k[:, 0]) and torch.equal(cache.v[:, 6], cache.v[:, 0])


def test_page_copies_after_a_refusal_do_nothing():
    from h3b import H3BError

    for pair in ((0, 7), (0, 99)):
        cache, host = _filled()
        cache.extend(_i32([6]))
        cache.copy_pages(_i32([pair[0]]), _i32([pair[1]]))
        host.assert_equal(cache)
        with pytest.raises(H3BError, match="a slot lies outside"):  # the first reason stays
            cache.check()


def test_page_copies_of_a_pool_of_many_pages():
    """Pages on both sides of what one pass of the check marks."""
    from h3b import H3BError, PagedKVCache

    pages = (1 << 18) + 5000
    cache = PagedKVCache.create(1, pages, 16, 1, 1, 16, torch.float8_e4m3fn, k_scale=torch.ones(1, 1, device="cuda"),
                                v_scale=torch.ones(1, 1, device="cuda"))
    for pool in (cache.k, cache.v):
        pool.view(torch.uint8).zero_()
        pool.view(torch.uint8)[0, :, 0, 0, 0] = (torch.arange(pages, device="cuda") % 101).to(torch.uint8)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(4)).to(torch.int32).cuda()
    src, dst = order[: pages // 3].contiguous(), order[pages // 3: 2 * (pages // 3)].contiguous()
    want = cache.k.view(torch.uint8).clone()
    for spoil in ((0, pages - 1), (pages // 3 - 1, 5)):  # a target twice, beyond and within the first pass
        i, page = spoil
        bad = dst.clone()
        bad[i] = page
        bad[i + 1 if i == 0 else i - 1] = page
        cache.copy_pages(src, bad)
        with pytest.raises(H3BError):
            cache.check()
        assert torch.equal(cache.k.view(torch.uint8), want)
    cache.copy_pages(src, dst)
    cache.check()
    want[0, dst.long()] = want[0, src.long()]
    assert torch.equal(cache.k.view(torch.uint8), want) and torch.equal(cache.v.view(torch.uint8), want)


# ------------------------------------------------------------------------------ append

@pytest.mark.parametrize("slots,starts", [([2], [0, 9]), ([2, 3], [0, 2, 5]), ([2, 3], [0, 5, 5]), ([2], [-1, 2]),
                                          ([4, 2, 3], [-4, 0, 2, 4])], ids=str)
def test_appends_of_more_tokens_than_rows_are_refused(slots, starts):
    """Four rows come with the call; lengths would grow over rows that are never written."""
    from h3b import H3BError

    cache, host = _filled()
    cache.append(_i32(slots), _rows(4), _rows(4), _i32(starts))
    host.assert_equal(cache)
    with pytest.raises(H3BError, match="beyond the length or the rows"):
        cache.check()


def test_appends_may_leave_rows_unused():
    """A buffer of more rows than the starts name, as a captured graph has, and rows before the first."""
    for starts in ([0, 1, 3], [2, 3, 4], [1, 1, 1]):
        cache, host = _filled()
        k, v = _rows(4, seed=5), _rows(4, seed=6)
        cache.append(_i32([2, 0]), k, v, _i32(starts))
        counts = [starts[1] - starts[0], starts[2] - starts[1]]
        host.extend([2, 0], counts)
        host.write([2, 0], counts, k[starts[0]:], v[starts[0]:])
        cache.check()
        host.assert_equal(cache, str(starts))


def test_an_append_behind_a_page_that_is_gone_is_refused():
    """A table whose partly filled last page is no page of the pool: the rows would have no place."""
    from h3b import H3BError

    for page in (-1, 8, 1 << 28):
        for call in (lambda c: c.append(_i32([2, 0]), _rows(2), _rows(2)), lambda c: c.extend(_i32([2, 0]))):
            cache, host = _filled()
            cache.table[0, 1] = page
            host.table[0, 1] = page
            call(cache)
            host.assert_equal(cache)
            with pytest.raises(H3BError, match="outside the pool"):
                cache.check()
