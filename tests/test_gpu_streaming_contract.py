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


# ------------------------------------------------------------------------------ write

@pytest.mark.parametrize("slots,starts,why", [
    ([6], [0, 2], "a slot lies outside"), ([-1], [0, 2], "a slot lies outside"), ([0, 7], [0, 2, 4], "a slot lies outside"),
    ([0, 0], [0, 1, 2], "named twice"), ([2], [0, 1], "beyond the length"), ([0], [0, 21], "beyond the length"),
    ([1, 0], [0, 30, 51], "beyond the length"), ([0, 1], [0, 20, 51], "beyond the length"), ([0, 1], [0, 2, 1], "unordered"),
    ([0], [-1, 2], "negative"), ([0], None, None), ([2], None, "beyond the length"), ([0, 1], [0, 20, 50], None),
    ([0, 2, 1], [3, 9, 9, 12], None),
], ids=str)
def test_writes_are_done_whole_or_not_at_all(slots, starts, why):
    from h3b import H3BError

    cache, host = _filled()
    rows = len(slots) if starts is None else 50
    k, v = _rows(rows, seed=7), _rows(rows, seed=8)
    cache.write(_i32(slots), k, v, None if starts is None else _i32(starts))
    if why is None:
        first = 0 if starts is None else starts[0]
        host.write(slots, [1] if starts is None else [b - a for a, b in zip(starts, starts[1:])], k[first:], v[first:])
        cache.check()
    else:
        with pytest.raises(H3BError, match=why):
            cache.check()
    host.assert_equal(cache)


def test_writes_into_pages_that_are_gone_are_refused():
    """Also where the page lies among the many that a long write fills."""
    from h3b import H3BError, PagedKVCache

    cache = PagedKVCache.create(1, 3200, 16, 1, 1100, 16 * 2100)
    slots = list(range(1099, -1, -1))
    counts = [16 * 2000 - 3] + [1] * 1023 + [2] * 76
    at = [0]
    for n in counts:
        at.append(at[-1] + n)
    k = _rows(at[-1], heads=1)
    cache.extend(_i32(slots[:1024]), _i32(at[:1025]))
    cache.extend(_i32(slots[1024:]), _i32(at[1024:]))
    cache.check()
    want = cache.k.clone()
    for slot, col in ((1099, 1234), (3, 0)):
        page = int(cache.table[slot, col])
        for gone in (-1, 3200):
            cache.table[slot, col] = gone
            cache.write(_i32(slots), k, k, _i32(at))
            with pytest.raises(H3BError, match="outside the pool"):
                cache.check()
            assert torch.equal(cache.k.view(torch.int16), want.view(torch.int16))
        cache.table[slot, col] = page
    cache.write(_i32(slots), k, k, _i32(at))
    cache.check()
    got = cache.k[0, cache.table[1099, :2000].long()].reshape(-1, 1, D)[: at[1]]
    assert torch.equal(got, k[: at[1]])
    assert torch.equal(cache.k[0, cache.table[3, 0].long(), 0, :2], k[at[1096]:at[1097], 0])


@pytest.mark.parametrize("slots,tokens", [(8192, 512), (8192, 513), (8193, 500), (600, 100)], ids=str)
def test_writes_around_what_each_block_checks_itself(slots, tokens):
    """Ragged writes on both sides of the sizes at which a launch of its own checks the call."""
    from h3b import H3BError, PagedKVCache

    cache = PagedKVCache.create(1, 1400, 16, 1, slots, 1024)
    n = 600 if slots == 600 else 17
    order = torch.randperm(slots, generator=torch.Generator().manual_seed(slots))[:n].tolist()
    counts = [0] * n
    for i in range(n):
        counts[i] = tokens // n + (i < tokens % n)
    counts[0], counts[5] = counts[0] + counts[5], 0
    at = [0]
    for c in counts:
        at.append(at[-1] + c)
    assert at[-1] == tokens
    cache.extend(_i32(order), _i32(at))
    cache.check()
    host = HostCache(cache)
    k, v = _rows(tokens, heads=1, seed=3), _rows(tokens, heads=1, seed=4)
    for bad_slots, bad_at, why in ((order[:-1] + order[:1], at, "named twice"), (order[:-1] + [slots], at, "outside the table"),
                                   (order[5:6] + order[1:5] + order[:1] + order[6:], at, "beyond the length")):
        cache.write(_i32(bad_slots), k, v, _i32(bad_at))
        with pytest.raises(H3BError, match=why):
            cache.check()
    page = int(cache.table[order[0], 0])
    cache.table[order[0], 0] = 1400
    cache.write(_i32(order), k, v, _i32(at))
    with pytest.raises(H3BError, match="outside the pool"):
        cache.check()
    cache.table[order[0], 0] = page
    host.assert_equal(cache)
    cache.write(_i32(order), k, v, _i32(at))
    host.write(order, counts, k, v)
    cache.check()
    host.assert_equal(cache)


def test_writes_and_appends_without_rows():
    """No row comes with the call: starts that name none are done, others are refused."""
    from h3b import H3BError

    none = _rows(0)
    for call in (lambda c, *a: c.write(*a), lambda c, *a: c.append(*a)):
        cache, host = _filled()
        call(cache, _i32([1, 0]), none, none, _i32([0, 0, 0]))
        cache.check()
        host.assert_equal(cache)
        for starts in ([0, 0, 3], [0, 2, 2], [-1, 0, 0]):
            call(cache, _i32([1, 0]), none, none, _i32(starts))
            with pytest.raises(H3BError, match="beyond the length or the rows"):
                cache.check()
            host.assert_equal(cache)
