"""Copy-on-write inside an append, against the host's page work step by step (GPU)."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from streaming_util import D, HostCache  # noqa: E402


def _i32(x):
    return torch.tensor([int(i) for i in x], dtype=torch.int32, device="cuda")


def _cache(layers, hkv, page, pages, slots, tokens, store):
    """Pools of bytes that differ everywhere; scales for E4M3."""
    from h3b import PagedKVCache

    g = torch.Generator(device="cuda").manual_seed(pages)
    scale = {} if store is not torch.float8_e4m3fn else {
        x: torch.rand(layers, hkv, device="cuda", generator=g) * 0.02 + 0.01 for x in ("k_scale", "v_scale")}
    cache = PagedKVCache.create(layers, pages, page, hkv, slots, tokens, store, **scale)
    for pool in (cache.k, cache.v):
        raw = pool.view(torch.uint8)
        raw.copy_(torch.randint(0, 120, raw.shape, device="cuda", dtype=torch.uint8, generator=g))
    return cache, HostCache(cache)


def _rows(g, n, heads, store):
    return torch.randn(n, heads, D, device="cuda", generator=g).to(torch.float16 if store is torch.float16 else torch.bfloat16)


@pytest.mark.parametrize("store", [torch.bfloat16, torch.float16, torch.float8_e4m3fn], ids=str)
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("layers,hkv,kids", [(1, 1, 3), (3, 8, 40), (4, 16, 40)])
def test_many_children_append_to_one_shared_page(store, page, layers, hkv, kids):
    """The copies of the shared page in every layer beside the new rows of one, with as many blocks for the
    copies as a call may have (640 would be asked for at the last size, 592 are taken)."""
    past = 2 * page + page // 2 + 3
    cache, host = _cache(layers, hkv, page, 3 + kids * 2, kids + 1, 8 * page, store)
    g = torch.Generator(device="cuda").manual_seed(page)
    k, v = (_rows(g, past, hkv, store) for _ in range(2))
    at = layers - 1
    cache.append(_i32([0]), k, v, _i32([0, past]), layer=at)
    host.extend([0], [past])
    host.write([0], [past], k, v, at)
    children = list(range(kids, 0, -1))
    cache.fork(_i32([0] * kids), _i32(children))
    host.fork([0] * kids, children)
    k, v = (_rows(g, kids, hkv, store) for _ in range(2))
    cache.append(_i32(children), k, v, layer=0)
    host.extend(children, [1] * kids)
    host.write(children, [1] * kids, k, v, 0)
    cache.check()
    host.assert_equal(cache)


@pytest.mark.parametrize("store", [torch.bfloat16, torch.float8_e4m3fn], ids=str)
@pytest.mark.parametrize("layers,hkv", [(1, 5), (3, 2)])
def test_cache_life_by_appends(store, layers, hkv):
    """Appends, forks, truncations and compactions at random; every append copies what it has to."""
    rng = np.random.RandomState(layers)
    g = torch.Generator(device="cuda").manual_seed(layers)
    page, slots, pages = 16, 12, 70
    cache, host = _cache(layers, hkv, page, pages, slots, page * 9, store)
    copied = 0
    for step in range(120):
        live = [s for s in range(slots) if host.lens[s]]
        empty = [s for s in range(slots) if not host.lens[s]]
        what = rng.choice(["append", "append", "append", "fork", "truncate", "compact"])
        if what == "append":
            some = rng.permutation(slots)[:rng.randint(1, 6)]
            counts = [int(rng.choice([0, 1, 1, 2, rng.randint(1, 2 * page)])) for _ in some]
            need = sum(host.pages_of(host.lens[s] + n) - host.pages_of(host.lens[s]) + 1 for s, n in zip(some, counts))
            if need > (host.refs == 0).sum() or any(host.lens[s] + n > page * 9 for s, n in zip(some, counts)):
                continue
            copied += sum(bool(n and host.lens[s] % page and host.refs[host.table[s, host.lens[s] // page]] > 1)
                          for s, n in zip(some, counts))
            layer = int(rng.randint(layers))
            k, v = (_rows(g, sum(counts), hkv, store) for _ in range(2))
            cache.append(_i32(some), k, v, _i32(np.concatenate([[0], np.cumsum(counts)])), layer=layer)
            host.extend(some, counts)
            host.write(some, counts, k, v, layer)
        elif what == "fork" and live and empty:
            n = rng.randint(1, min(4, len(empty)) + 1)
            src, dst = [int(rng.choice(live)) for _ in range(n)], empty[:n]
            cache.fork(_i32(src), _i32(dst))
            host.fork(src, dst)
        elif what == "truncate" and live:
            some = live[:rng.randint(1, len(live) + 1)]
            keep = [int(rng.choice([0, rng.randint(0, host.lens[s] + 1)])) for s in some]
            cache.truncate(_i32(some), _i32(keep))
            host.truncate(some, keep)
        elif what == "compact":
            cache.compact()
            host.compact()
        else:
            continue
        cache.check()
        host.assert_equal(cache, f"step {step} {what}")
    assert copied > 5, copied


def test_pages_beyond_the_first_pass_of_the_search():
    """Free pages on both sides of the 32,768 that the planning block looks at together, lowest first."""
    from h3b import H3BError

    pages = 70000
    cache, host = _cache(1, 1, 16, pages, 3, 16 * 300, torch.float8_e4m3fn)
    cache.refs.fill_(1)
    free = [5, 32767, 32768, 32800, 65535, 65536] + list(range(69700, pages))
    cache.refs[torch.tensor(free, device="cuda")] = 0
    host.refs[:] = 1
    host.refs[free] = 0
    for counts in ([16 * 4, 16 * 3, 16 * 100], [0, 16 * 199 - 5, 0]):
        at = _i32(np.concatenate([[0], np.cumsum(counts)]))
        cache.extend(_i32([2, 0, 1]), at)
        host.extend([2, 0, 1], counts)
        cache.check()
        host.assert_equal(cache)
    assert (host.refs == 1).all()
    cache.extend(_i32([1]))
    with pytest.raises(H3BError, match="free pages"):
        cache.check()
    host.assert_equal(cache)


def test_many_entries_are_changed_by_a_grid():
    """Forks and frees of more than 4,096 table entries, truncations of more than 16,384."""
    slots, tokens = 300, 16 * 100
    cache, host = _cache(1, 1, 16, 4000, slots, tokens, torch.float8_e4m3fn)
    rng = np.random.RandomState(3)
    some = rng.permutation(slots)[:60]
    counts = rng.randint(0, 900, 60)
    counts[:3] = 0, 1, 16
    cache.extend(_i32(some), _i32(np.concatenate([[0], np.cumsum(counts)])))
    host.extend(some, counts)
    empty = np.setdiff1d(np.arange(slots), some)
    dst = rng.permutation(empty)[:200]
    src = rng.choice(some, 200)
    cache.fork(_i32(src), _i32(dst))
    host.fork(src, dst)
    cache.check()
    host.assert_equal(cache, "fork")
    every = rng.permutation(slots)
    keep = [rng.randint(0, host.lens[s] + 1) if rng.rand() < 0.7 else host.lens[s] for s in every]
    cache.truncate(_i32(every), _i32(keep))
    host.truncate(every, keep)
    cache.check()
    host.assert_equal(cache, "truncate")
    cache.free(_i32(every[:250]))
    host.truncate(every[:250], [0] * 250)
    cache.check()
    host.assert_equal(cache, "free")
