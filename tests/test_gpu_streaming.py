"""Streaming attention and the paged cache against plain 64-bit forms (GPU)."""

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from streaming_util import D, HostCache, assert_close, attend, visible  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    yield
    import h3b
    assert h3b.device_status(0) == 0


def _i32(x):
    return torch.tensor(list(x), dtype=torch.int32, device="cuda")


def _starts(lens):
    return _i32(np.concatenate([[0], np.cumsum(lens)]).astype(int).tolist())


def _rand(g, *shape, dtype, scale=1.0):
    return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ------------------------------------------------------------------------------ contiguous

WINDOW_CASES = [
    # lens of the queries, keys before them, Hq, Hkv, window, sinks, chunk
    ([1], 0, 1, 1, None, 0, 1),
    ([1], 700, 8, 2, None, 0, 1),
    ([127], 0, 2, 1, None, 0, 1),
    ([128], 0, 2, 2, 64, 0, 1),
    ([129], 0, 3, 1, 100, 4, 1),
    ([300], 0, 5, 5, 1, 0, 1),
    ([300], 0, 4, 2, 0, 7, 1),
    ([513], 0, 2, 1, 130, 300, 1),
    ([257], 400, 4, 1, 333, 65, 1),
    ([64, 1, 200, 5], 0, 4, 2, 48, 3, 1),
    ([64, 1, 200, 5], 130, 6, 2, 150, 17, 1),
    ([3, 260, 2, 2, 129, 1, 1], 9, 2, 2, None, 0, 1),
    ([600], 0, 2, 1, 200, 10, 50),
    ([384], 384, 2, 2, 256, 0, 128),
    ([700], 41, 2, 1, 260, 130, 130),
    ([90], 1000, 1, 1, 90, 20, 90),
    ([1100], 0, 16, 1, 700, 0, 1),
    ([2100], 0, 2, 2, 1024, 128, 1),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", WINDOW_CASES, ids=lambda c: "-".join(str(x) for x in c).replace(" ", ""))
def test_window_attention(case, dtype):
    from h3b import window_attention

    lens, past, hq, hkv, window, sinks, chunk = case
    g = _gen(len(lens) * 7 + lens[0])
    tq, keys = sum(lens), [n + past for n in lens]
    q = _rand(g, tq, hq, D, dtype=dtype, scale=1.5)
    k = _rand(g, sum(keys), hkv, D, dtype=dtype)
    v = _rand(g, sum(keys), hkv, D, dtype=dtype)
    out = window_attention(q, k, v, window=window, sinks=sinks, chunk=chunk, query_starts=_starts(lens),
                           key_starts=_starts(keys))
    a = b = 0
    for lq, lk in zip(lens, keys):
        see = visible(lq, lk, window, sinks, chunk, "cuda")
        ref, spread = attend(q[a:a + lq], k[b:b + lk], v[b:b + lk], see)
        assert_close(out[a:a + lq], ref, spread, lk, 6.0, f"sequence at {a}")
        a, b = a + lq, b + lk
    if len(lens) == 1:
        one = window_attention(q, k, v, window=window, sinks=sinks, chunk=chunk)
        assert torch.equal(one, out)


@pytest.mark.parametrize("heads", [(8, 4), (6, 2), (12, 12)], ids=str)
@pytest.mark.parametrize("rule", [(None, 0, 1), (100, 3, 1), (1, 0, 700), (129, 260, 1)], ids=str)
def test_window_more_work_than_multiprocessors(heads, rule):
    """Many items per persistent block: ragged sequences, empty ones and gaps between first tokens and window."""
    from h3b import window_attention

    hq, hkv = heads
    window, sinks, chunk = rule
    rng = np.random.RandomState(hq)
    lens = [int(x) for x in rng.choice([0, 1, 5, 127, 128, 129, 300, 700, 1100], 40)]
    keys = [n + int(rng.choice([0, 0, 3, 400])) if i % 7 else n // 2 for i, n in enumerate(lens)]
    g = _gen(hq)
    q = _rand(g, sum(lens), hq, D, dtype=torch.bfloat16, scale=1.5)
    k, v = (_rand(g, sum(keys), hkv, D, dtype=torch.bfloat16) for _ in range(2))
    out = window_attention(q, k, v, window=window, sinks=sinks, chunk=chunk, query_starts=_starts(lens),
                           key_starts=_starts(keys))
    a = b = 0
    for lq, lk in zip(lens, keys):
        if lq:
            ref, spread = attend(q[a:a + lq], k[b:b + lk], v[b:b + lk], visible(lq, lk, window, sinks, chunk, "cuda"))
            assert_close(out[a:a + lq], ref, spread, lk, 6.0, f"sequence at {a}")
        a, b = a + lq, b + lk


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", [([200], 9000, 4, 2, None, 0, 1), ([5], 20000, 3, 1, None, 0, 1), ([1], 30011, 2, 2, 29000, 70, 1),
                                  ([300, 1, 40], 7000, 6, 2, 5000, 300, 1), ([260], 6000, 5, 5, None, 100, 260),
                                  ([1500], 0, 1, 1, None, 0, 1), ([2500], 0, 3, 3, 2000, 128, 1)],
                         ids=lambda c: "-".join(str(x) for x in c).replace(" ", ""))
def test_window_few_rows_over_many_keys(case, dtype):
    """Items cut along their keys and joined; twice the same bits."""
    from h3b import window_attention

    lens, past, hq, hkv, window, sinks, chunk = case
    g = _gen(lens[0])
    keys = [n + past for n in lens]
    q = _rand(g, sum(lens), hq, D, dtype=dtype, scale=2.0)
    k, v = (_rand(g, sum(keys), hkv, D, dtype=dtype) for _ in range(2))
    kw = dict(window=window, sinks=sinks, chunk=chunk, query_starts=_starts(lens), key_starts=_starts(keys))
    out = window_attention(q, k, v, **kw)
    a = b = 0
    for lq, lk in zip(lens, keys):
        ref, spread = attend(q[a:a + lq], k[b:b + lk], v[b:b + lk], visible(lq, lk, window, sinks, chunk, "cuda"))
        assert_close(out[a:a + lq], ref, spread, lk, 6.0, f"sequence at {a}")
        a, b = a + lq, b + lk
    assert torch.equal(window_attention(q, k, v, **kw), out)


@pytest.mark.parametrize("n", [6000, 6150, 6400])
def test_window_thousands_of_sequences(n):
    """Sequences of a few tokens, on both sides of the number whose plan fits shared memory."""
    from h3b import window_attention

    rng = np.random.RandomState(n)
    lens = rng.choice([0, 1, 2, 3], n)
    keys = lens + 1
    g = _gen(n)
    q = _rand(g, int(lens.sum()), 2, D, dtype=torch.bfloat16, scale=1.5)
    k, v = (_rand(g, int(keys.sum()), 1, D, dtype=torch.bfloat16) for _ in range(2))
    out = window_attention(q, k, v, query_starts=_starts(lens.tolist()), key_starts=_starts(keys.tolist()))
    a = b = 0
    for i in range(0, n, 100):
        see = torch.block_diag(*[visible(int(lq), int(lk), None, 0, 1).float()
                                 for lq, lk in zip(lens[i:i + 100], keys[i:i + 100])]).bool().cuda()
        rows, cols = see.shape
        ref, spread = attend(q[a:a + rows], k[b:b + cols], v[b:b + cols], see)
        assert_close(out[a:a + rows], ref, spread, 4, 6.0, f"sequences from {i}")
        a, b = a + rows, b + cols


def test_window_cut_items_keep_unseen_rows_apart():
    """Non-finite V and K rows inside and outside what the rows of cut items see."""
    from h3b import window_attention

    g = _gen(12)
    n, past = 130, 8000
    q = _rand(g, n, 2, D, dtype=torch.bfloat16)
    k, v = (_rand(g, n + past, 1, D, dtype=torch.bfloat16) for _ in range(2))
    kw = dict(window=7000, sinks=5)
    see = visible(n, n + past, 7000, 5, 1, "cuda")
    clean = window_attention(q, k, v, **kw)
    for j in (6, 500, past + n - 7000 - 20, past + n - 7000 + 3, past + 10, past + 129):
        dirty_k, dirty_v = k.clone(), v.clone()
        dirty_v[j, 0, 3] = math.inf
        got = window_attention(q, dirty_k, dirty_v, **kw)
        hit = see[:, j]
        assert torch.equal(got[~hit], clean[~hit]) and not torch.isfinite(got[hit][..., 3].float()).any()
        keep = [c for c in range(D) if c != 3]
        assert torch.equal(got[..., keep], clean[..., keep])
        dirty_k[j] = math.nan
        got = window_attention(q, dirty_k, v, **kw)
        assert torch.equal(got[~hit], clean[~hit]) and torch.isnan(got[hit].float()).all()


def test_window_overlapping_starts_stay_in_bounds():
    """Starts that run backwards: rows may be anything, memory is not left."""
    from h3b import window_attention

    g = _gen(13)
    q = _rand(g, 400, 2, D, dtype=torch.bfloat16)
    k, v = (_rand(g, 400, 2, D, dtype=torch.bfloat16) for _ in range(2))
    window_attention(q, k, v, query_starts=_i32([0, 400, 0, 400, -7, 900, 3]), key_starts=_i32([0, 400, 0, 400, -9, 4000, 1]))
    torch.cuda.synchronize()


def test_window_rows_that_see_nothing_give_zero():
    """More queries than keys, a window of nothing, and sequences without keys."""
    from h3b import window_attention

    g = _gen(3)
    q = _rand(g, 300, 2, D, dtype=torch.bfloat16)
    k, v = (_rand(g, 100, 1, D, dtype=torch.bfloat16) for _ in range(2))
    out = window_attention(q, k, v)
    assert torch.equal(out[:200], torch.zeros_like(out[:200]))
    ref, spread = attend(q[200:], k, v, visible(100, 100, None, 0, 1, "cuda"))
    assert_close(out[200:], ref, spread, 100, 6.0)
    assert not window_attention(q, k, v, window=0).any()
    assert not window_attention(q, k[:0], v[:0]).any()
    out = window_attention(q, k, v, query_starts=_i32([0, 50, 200, 300]), key_starts=_i32([0, 50, 50, 100]))
    assert not out[50:200].any() and not out[200:250].any() and out[:50].any() and out[250:].any()
    assert window_attention(q[:0], k, v).shape == (0, 2, D)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("where", ["k", "v", "kv"])
def test_window_unseen_rows_may_hold_anything(bad, where):
    """Non-finite rows behind the window, in the future or in another sequence reach no query that does
    not see them; those that see a non-finite V row are not finite there."""
    from h3b import window_attention

    g = _gen(11)
    lens, hkv = [420, 33, 260], 2
    keys = lens
    q = _rand(g, sum(lens), 4, D, dtype=torch.bfloat16)
    k, v = (_rand(g, sum(keys), hkv, D, dtype=torch.bfloat16) for _ in range(2))
    dirty_k, dirty_v = k.clone(), v.clone()
    spoiled = [0, 5, 130, 300, 419, 420 + 32, 420 + 33, 420 + 33 + 255]
    for j in spoiled:
        if "k" in where:
            dirty_k[j, 1] = bad
        if "v" in where:
            dirty_v[j, 1, 7:9] = bad
    kw = dict(window=70, sinks=3, query_starts=_starts(lens), key_starts=_starts(keys))
    clean, dirty = window_attention(q, k, v, **kw), window_attention(q, dirty_k, dirty_v, **kw)
    a = 0
    for n in lens:
        see = visible(n, n, 70, 3, 1, "cuda")
        hit = torch.zeros(n, dtype=torch.bool, device="cuda")
        for j in spoiled:
            if a <= j < a + n:
                hit |= see[:, j - a]
        rows = slice(a, a + n)
        assert torch.equal(dirty[rows, :2], clean[rows, :2])          # the clean kv head
        assert torch.equal(dirty[rows, 2:][~hit], clean[rows, 2:][~hit])
        if "v" in where:
            assert not torch.isfinite(dirty[rows, 2:, 7:9][hit].float()).any()
            if where == "v":
                keep = [c for c in range(D) if c not in (7, 8)]
                assert torch.equal(dirty[rows, 2:][hit][..., keep], clean[rows, 2:][hit][..., keep])
        elif math.isnan(bad):
            assert torch.isnan(dirty[rows, 2:][hit].float()).all()
        a += n


def test_window_strides_and_views():
    """Q, K and V as slices of the rows of one projection, into a slice of a wider output."""
    from h3b import window_attention

    g = _gen(4)
    rows = _rand(g, 333, 8 + 2 + 2, D, dtype=torch.bfloat16)
    q, k, v = rows[:, :8], rows[:, 8:10], rows[:, 10:]
    wide = torch.full((333, 10, D), 7.0, dtype=torch.bfloat16, device="cuda")
    got = window_attention(q, k, v, window=100, sinks=2, out=wide[:, 1:9])
    want = window_attention(q.contiguous(), k.contiguous(), v.contiguous(), window=100, sinks=2)
    assert torch.equal(got, want) and torch.equal(wide[:, 1:9], want)
    assert (wide[:, 0] == 7).all() and (wide[:, 9] == 7).all()
    odd = rows.transpose(0, 1).contiguous().transpose(0, 1)  # heads outermost: copied first
    assert torch.equal(window_attention(odd[:, :8], odd[:, 8:10], odd[:, 10:], window=100, sinks=2), want)


def test_window_large_scores_and_scale():
    """Scores of +-600 after scaling: the running maximum has to move and rescale."""
    from h3b import window_attention

    g = _gen(5)
    q, k = _rand(g, 400, 2, D, dtype=torch.bfloat16, scale=8.0), _rand(g, 400, 1, D, dtype=torch.bfloat16, scale=8.0)
    k *= torch.linspace(0.1, 1.0, 400, device="cuda")[:, None, None].to(k.dtype)
    v = _rand(g, 400, 1, D, dtype=torch.bfloat16)
    out = window_attention(q, k, v, scale=0.5)
    ref, spread = attend(q, k, v, visible(400, 400, None, 0, 1, "cuda"), 0.5)
    # fp32 scores up to 2000: 2^-23 of that, times ln 2 per octave of the exponential
    err = (out.double() - ref).abs()
    assert (err <= 2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2e-3) * spread * 1.01).all()


def test_window_on_another_stream():
    from h3b import window_attention

    g = _gen(6)
    q, k, v = (_rand(g, 700, h, D, dtype=torch.bfloat16) for h in (4, 2, 2))
    want = window_attention(q, k, v, window=256)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = [window_attention(q, k, v, window=256) for _ in range(3)]
    side.synchronize()
    assert all(torch.equal(x, want) for x in got)


# ------------------------------------------------------------------------------ paged

def _cache(g, lens, page, hkv, dtype, layers=1, spare=3, slots=None, extra=0):
    """A cache whose unused rows, tails of pages and free pages hold NaN."""
    from h3b import PagedKVCache

    need = [-(-n // page) for n in lens]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(pages))
    store = torch.float8_e4m3fn if dtype == "e4m3" else dtype
    slots = slots or len(lens)
    scale = dict(k_scale=torch.rand(layers, hkv, device="cuda", generator=g) * 0.02 + 0.01,
                 v_scale=torch.rand(layers, hkv, device="cuda", generator=g) * 0.02 + 0.005) if dtype == "e4m3" else {}
    cache = PagedKVCache.create(layers, pages, page, hkv, slots, max(max(need) * page + extra, page), store, **scale)
    for pool, s in ((cache.k, scale.get("k_scale")), (cache.v, scale.get("v_scale"))):
        pool.view(torch.uint8).fill_(0x7f if dtype == "e4m3" else 0xff)
        at = 0
        for i, n in enumerate(lens):
            x = torch.randn(layers, hkv, need[i] * page, D, device="cuda", generator=g)
            if s is not None:
                x = (x / s[:, :, None, None]).clamp(-448, 448)
            x = x.to(store)
            for p in range(need[i]):
                m = min(page, n - p * page)
                pool[:, int(order[at + p]), :, :m] = x[:, :, p * page:p * page + m]
            at += need[i]
    at = 0
    for i, n in enumerate(lens):
        cache.table[i, :need[i]] = order[at:at + need[i]].to(torch.int32)
        cache.lens[i] = n
        at += need[i]
    cache.refs[order[:at].cuda()] = 1
    return cache


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rule", [(None, 0, 1), (200, 5, 1), (150, 140, 1), (256, 33, 128)], ids=str)
def test_paged_window_attention(page, dtype, rule):
    from h3b import paged_window_attention

    window, sinks, chunk = rule
    g = _gen(page)
    lens, new = [700, 129, 1, 300, 64], [200, 129, 1, 7, 64]
    slots = [3, 0, 4, 2, 1]
    cache = _cache(g, lens, page, 2, dtype, layers=2)
    q = _rand(g, sum(new[s] for s in slots), 6, D, dtype=dtype, scale=1.5)
    out = paged_window_attention(q, cache, _i32(slots), window=window, sinks=sinks, chunk=chunk, layer=1,
                                 query_starts=_starts([new[s] for s in slots]))
    host = HostCache(cache)
    a = 0
    for s in slots:
        k, v = host.rows(s, 1)
        see = visible(new[s], lens[s], window, sinks, chunk, "cuda")
        ref, spread = attend(q[a:a + new[s]], k, v, see)
        assert_close(out[a:a + new[s]], ref, spread, lens[s], 6.0, f"slot {s}")
        a += new[s]


def test_paged_window_unseen_pages_are_not_needed():
    """Pages that the window has left behind may be anything, even gone from the table."""
    from h3b import paged_window_attention

    g = _gen(8)
    cache = _cache(g, [1000], 16, 1, torch.bfloat16)
    q = _rand(g, 40, 2, D, dtype=torch.bfloat16)
    want = paged_window_attention(q, cache, window=100, sinks=10)
    gone = cache.table[0, 1:(960 - 99) // 16].clone()
    cache.k[0, gone.long()] = math.nan
    cache.v[0, gone.long()] = math.nan
    cache.table[0, 1:(960 - 99) // 16] = -1
    assert torch.equal(paged_window_attention(q, cache, window=100, sinks=10), want)


# ------------------------------------------------------------------------------ decode

@pytest.mark.parametrize("page", [16, 64, 128])
@pytest.mark.parametrize("dtype,store", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16),
                                         (torch.bfloat16, "e4m3"), (torch.float16, "e4m3")], ids=str)
@pytest.mark.parametrize("heads", [(1, 1), (8, 2), (5, 5), (24, 2), (32, 2), (20, 1), (16, 2), (3, 1), (14, 2)], ids=str)
@pytest.mark.parametrize("room", [0, 20000])
def test_decode_attention(page, dtype, store, heads, room):
    """room: tokens that the table could name beyond the lengths; with much of it, and with many pairs, the
    chunks of all sequences are dealt out over the grid, else a cluster serves each pair."""
    from h3b import decode_attention

    hq, hkv = heads
    g = _gen(page + hq)
    lens = [1, 15, 16, 17, 0, 130, 1000, 333, 64, 2500]
    cache = _cache(g, lens, page, hkv, store, layers=2, extra=room)
    slots = [9, 0, 3, 4, 2, 8, 1, 7, 5, 6]
    q = _rand(g, len(slots), hq, D, dtype=dtype, scale=1.5)
    host = HostCache(cache)
    for window, sinks in ((None, 0), (100, 5), (1, 0), (0, 3), (0, 0), (40, 200)):
        out = decode_attention(q, cache, _i32(slots), window=window, sinks=sinks, layer=1)
        for i, s in enumerate(slots):
            k, v = host.rows(s, 1)
            see = visible(1, lens[s], window, sinks, 1, "cuda") if lens[s] else torch.zeros(1, 0, dtype=torch.bool, device="cuda")
            ref, spread = attend(q[i:i + 1], k, v, see)
            assert_close(out[i:i + 1], ref, spread, lens[s], 14.0, f"slot {s} window {window} sinks {sinks}")


@pytest.mark.parametrize("store", [torch.bfloat16, "e4m3"], ids=str)
def test_decode_one_long_sequence(store):
    """A single sequence is split over the whole grid and joined; twice the same bits."""
    from h3b import decode_attention

    g = _gen(21)
    cache = _cache(g, [70001], 32, 1, store)
    q = _rand(g, 1, 4, D, dtype=torch.bfloat16, scale=2.0)
    out = decode_attention(q, cache)
    k, v = HostCache(cache).rows(0)
    ref, spread = attend(q, k, v, visible(1, 70001, None, 0, 1, "cuda"))
    assert_close(out, ref, spread, 70001, 14.0)
    work = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
    assert torch.equal(decode_attention(q, cache, workspace=work), out)
    assert torch.equal(decode_attention(q, cache, workspace=work), out)


@pytest.mark.parametrize("store", [torch.bfloat16, "e4m3"], ids=str)
@pytest.mark.parametrize("heads", [(3, 1), (14, 2), (24, 8), (16, 1)], ids=str)
def test_decode_many_short_sequences(store, heads):
    """More pairs than warps have parts: most are one warp's, some are joined, some are empty."""
    from h3b import decode_attention

    hq, hkv = heads
    g = _gen(hq)
    rng = np.random.RandomState(hq)
    lens = [int(x) for x in rng.choice([0, 1, 7, 16, 40, 130, 400, 1500], 310)]
    cache = _cache(g, lens, 16, hkv, store)
    q = _rand(g, len(lens), hq, D, dtype=torch.bfloat16, scale=1.5)
    out = decode_attention(q, cache, window=700, sinks=9)
    host = HostCache(cache)
    for i, n in enumerate(lens):
        k, v = host.rows(i)
        see = visible(1, n, 700, 9, 1, "cuda") if n else torch.zeros(1, 0, dtype=torch.bool, device="cuda")
        ref, spread = attend(q[i:i + 1], k, v, see)
        assert_close(out[i:i + 1], ref, spread, n, 14.0, f"sequence {i} of {n}")


def test_decode_extreme_queries_of_an_8_bit_cache():
    """bf16 queries outside fp16's range, all-zero heads, and scores that need the power of two per head."""
    from h3b import decode_attention

    g = _gen(22)
    cache = _cache(g, [300, 300, 300, 300], 16, 1, "e4m3")
    q = _rand(g, 4, 3, D, dtype=torch.bfloat16)
    q[0] *= 1e30
    q[1] *= 1e-30
    q[2, 1] = 0
    scales = torch.tensor([1e-30, 1e30, 1.0, 1.0])
    host = HostCache(cache)
    for i in range(4):
        s = float(scales[i]) * 0.09
        out = decode_attention(q[i:i + 1], cache, _i32([i]), scale=s)
        k, v = host.rows(i)
        ref, spread = attend(q[i:i + 1], k, v, visible(1, 300, None, 0, 1, "cuda"), s)
        assert_close(out, ref, spread, 300, 14.0, f"query {i}")


def test_decode_slots_and_pages_outside_the_cache_read_nothing():
    """Slots outside the table give 0; pages outside the pool stay inside the pool's memory."""
    from h3b import decode_attention, paged_window_attention

    g = _gen(23)
    cache = _cache(g, [100, 200], 16, 1, torch.bfloat16)
    q = _rand(g, 4, 2, D, dtype=torch.bfloat16)
    out = decode_attention(q, cache, _i32([-1, 0, 2, 1]))
    assert not out[0].any() and not out[2].any() and out[1].any() and out[3].any()
    out = paged_window_attention(q, cache, _i32([5]), query_starts=_i32([0, 4]))
    assert not out.any()
    cache.table[0, 2] = 1 << 28
    cache.table[1, 1] = -7
    decode_attention(q[:2], cache)
    paged_window_attention(q, cache, _i32([1]), query_starts=_i32([0, 4]))
    torch.cuda.synchronize()


# ------------------------------------------------------------------------------ pages

def _nan_cache(page, hkv, layers, pages, slots, max_tokens, store=torch.bfloat16):
    from h3b import PagedKVCache

    scale = {}
    if store == torch.float8_e4m3fn:
        scale = dict(k_scale=torch.linspace(0.01, 0.05, layers * hkv, device="cuda").view(layers, hkv),
                     v_scale=torch.linspace(0.02, 0.004, layers * hkv, device="cuda").view(layers, hkv))
    cache = PagedKVCache.create(layers, pages, page, hkv, slots, max_tokens, store, **scale)
    cache.k.view(torch.uint8).fill_(1)
    cache.v.view(torch.uint8).fill_(2)
    return cache


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("store", [torch.bfloat16, torch.float16, torch.float8_e4m3fn], ids=str)
@pytest.mark.parametrize("layers,hkv", [(1, 8), (3, 1), (2, 5)])
def test_cache_life(page, store, layers, hkv):
    """A random life of appends, forks, truncations, frees and compactions, equal to the host's step by step."""
    rng = np.random.RandomState(page + layers)
    g = _gen(page)
    slots, pages = 12, 61 if page < 64 else 40
    cache = _nan_cache(page, hkv, layers, pages, slots, page * 9, store)
    host = HostCache(cache)
    row_type = torch.float16 if store == torch.float16 else torch.bfloat16
    done = {}
    for step in range(70):
        what = rng.choice(["append", "append", "append", "fork", "truncate", "free", "compact"])
        live = [s for s in range(slots) if host.lens[s]]
        empty = [s for s in range(slots) if not host.lens[s]]
        if what == "append":
            some = rng.permutation(slots)[:rng.randint(1, 6)]
            counts = [int(rng.choice([0, 1, 1, 2, page, rng.randint(1, 2 * page)])) for _ in some]
            ones = rng.rand() < 0.3
            if ones:
                counts = [1] * len(some)
            need = sum(host.pages_of(host.lens[s] + n) - host.pages_of(host.lens[s]) + 1 for s, n in zip(some, counts))
            if need > (host.refs == 0).sum() or any(host.lens[s] + n > page * 9 for s, n in zip(some, counts)):
                continue
            k, v = (_rand(g, sum(counts), hkv, D, dtype=row_type, scale=3.0) for _ in range(2))
            starts = None if ones else _starts(counts)
            cache.extend(_i32(some), starts)
            host.extend(some, counts)
            for layer in range(layers):
                cache.write(_i32(some), k, v, starts, layer)
                host.write(some, counts, k, v, layer)
        elif what == "fork" and live and empty:
            n = rng.randint(1, min(4, len(empty)) + 1)
            src, dst = [int(rng.choice(live)) for _ in range(n)], empty[:n]
            cache.fork(_i32(src), _i32(dst))
            host.fork(src, dst)
        elif what == "truncate" and live:
            some = live[:rng.randint(1, len(live) + 1)]
            keep = [rng.randint(0, host.lens[s] + 1) for s in some]
            cache.truncate(_i32(some), _i32(keep))
            host.truncate(some, keep)
        elif what == "free" and live:
            some = live[::2]
            cache.free(_i32(some))
            host.truncate(some, [0] * len(some))
        elif what == "compact":
            cache.compact()
            host.compact()
        else:
            continue
        done[what] = done.get(what, 0) + 1
        cache.check()
        host.assert_equal(cache, f"step {step} {what}")
    assert len(done) == 5, done


def test_cache_large_pools_and_many_slots():
    """More slots and pages than one pass of the planning block."""
    slots, page = 2500, 16
    cache = _nan_cache(page, 1, 1, 9001, slots, 96)
    host = HostCache(cache)
    g = _gen(2)
    order = np.random.RandomState(1).permutation(slots)
    counts = np.random.RandomState(2).randint(0, 50, slots).tolist()
    k, v = (_rand(g, sum(counts), 1, D, dtype=torch.bfloat16) for _ in range(2))
    cache.append(_i32(order), k, v, _starts(counts))
    host.extend(order, counts)
    cache.free(_i32(order[::3]))
    host.truncate(order[::3], [0] * len(order[::3]))
    cache.compact()
    for name in ("lens",):
        assert np.array_equal(cache.lens.cpu().numpy(), host.lens)
    before = host.refs.copy()
    host.write([s for s in order], [0] * slots, k, v)
    host.compact()
    assert np.array_equal(cache.table.cpu().numpy(), host.table) and np.array_equal(cache.refs.cpu().numpy(), host.refs)
    assert before.sum() == host.refs.sum()
    cache.check()
    # the rows survived the moves
    at = np.concatenate([[0], np.cumsum(counts)])
    for i in (1, 2, 1000, 2499):
        s = int(order[i])
        if counts[i] and host.lens[s]:
            rows = torch.cat([cache.k[0, p, 0] for p in host.table[s, :host.pages_of(counts[i])].tolist()])[:counts[i]]
            assert torch.equal(rows, k[at[i]:at[i + 1], 0])


def test_cache_refusals_change_nothing_and_stick():
    from h3b import H3BError

    g = _gen(9)
    page = 16
    k1, v1 = (_rand(g, 64, 2, D, dtype=torch.bfloat16) for _ in range(2))

    def fresh():
        cache = _nan_cache(page, 2, 1, 8, 6, 64)
        cache.append(_i32([0, 1]), k1[:30], v1[:30], _i32([0, 20, 30]))
        cache.check()
        return cache, HostCache(cache)

    refused = [
        ("not enough free pages", lambda c: c.extend(_i32([2, 3, 0]), _i32([0, 50, 64, 77]))),
        ("outgrow", lambda c: c.extend(_i32([0]), _i32([0, 45]))),
        ("named twice", lambda c: c.extend(_i32([2, 2]))),
        ("outside the table", lambda c: c.extend(_i32([6]))),
        ("outside the table", lambda c: c.extend(_i32([-1]))),
        ("unordered", lambda c: c.extend(_i32([2, 3]), _i32([0, 9, 4]))),
        ("holds tokens", lambda c: c.fork(_i32([0]), _i32([1]))),
        ("outside the table", lambda c: c.fork(_i32([9]), _i32([2]))),
        ("named twice", lambda c: c.fork(_i32([0, 1]), _i32([2, 2]))),
        ("named twice", lambda c: c.fork(_i32([0, 2]), _i32([2, 3]))),
        ("beyond the length", lambda c: c.truncate(_i32([0]), _i32([21]))),
        ("negative", lambda c: c.truncate(_i32([0]), _i32([-1]))),
        ("named twice", lambda c: c.free(_i32([1, 1]))),
    ]
    cache, host = fresh()  # five pages for five: the last free ones are taken
    cache.extend(_i32([2, 3, 0]), _i32([0, 50, 64, 65]))
    host.extend([2, 3, 0], [50, 14, 1])
    host.assert_equal(cache)
    cache.check()
    assert (host.refs == 1).all()
    for text, call in refused:
        cache, host = fresh()
        call(cache)
        # sticky: later calls, the row write that would have followed among them, do nothing either
        cache.write(_i32([0]), k1[:1], v1[:1])
        cache.append(_i32([4]), k1[:1], v1[:1])
        cache.free(_i32([1]))
        cache.fork(_i32([0]), _i32([5]))
        cache.compact()
        host.assert_equal(cache, text)
        with pytest.raises(H3BError, match=text):
            cache.check()
        cache.append(_i32([4]), k1[:1], v1[:1])
        cache.check()
        assert int(cache.lens[4]) == 1
    cache, host = fresh()
    cache.copy_pages(_i32([0, 99]), _i32([7, 6]))
    with pytest.raises(H3BError, match="outside the pool"):
        cache.check()


def test_cache_copy_pages():
    cache = _nan_cache(32, 3, 2, 10, 2, 64)
    cache.k.copy_(torch.randn(cache.k.shape, device="cuda"))
    cache.v.copy_(torch.randn(cache.v.shape, device="cuda"))
    k, v = cache.k.clone(), cache.v.clone()
    cache.copy_pages(_i32([3, 0, 3]), _i32([9, 2, 4]))
    k[:, [9, 2, 4]] = k[:, [3, 0, 3]]
    v[:, [9, 2, 4]] = v[:, [3, 0, 3]]
    assert torch.equal(cache.k, k) and torch.equal(cache.v, v)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_e4m3_write_rounds_and_saturates(dtype):
    cache = _nan_cache(16, 1, 1, 4, 1, 64, torch.float8_e4m3fn)
    x = torch.zeros(8, 1, D, dtype=dtype, device="cuda")
    x[0] = torch.linspace(-30, 30, D, device="cuda").to(dtype)
    x[1, 0, :6] = torch.tensor([math.inf, -math.inf, math.nan, 6e4, -6e4, 0.0]).to(dtype)
    x[2] = torch.linspace(0, 2e-4, D, device="cuda").to(dtype)
    cache.append(_i32([0]), x, x.flip(0), _i32([0, 8]))
    cache.check()
    for pool, rows, scale in ((cache.k, x, cache.k_scale), (cache.v, x.flip(0), cache.v_scale)):
        want = (rows[:, 0].float() / scale[0, 0]).clamp(-448, 448).to(torch.float8_e4m3fn)
        page = int(cache.table[0, 0])
        got = pool[0, page, 0, :8]
        nan = torch.isnan(want.float())
        assert torch.equal(torch.isnan(got.float()), nan)
        assert torch.equal(got.float()[~nan], want.float()[~nan])


@pytest.mark.parametrize("scale", [3e-39, 7e-31, 1.1e-30, 0.013, 0.25, 9e29, 3e30, 5e37])
def test_e4m3_write_divides_exactly_at_any_scale(scale):
    """Scales whose reciprocal is usable and scales whose is not: the codes are those of the fp32 quotient."""
    cache = _nan_cache(16, 2, 1, 40, 1, 640, torch.float8_e4m3fn)
    cache.k_scale.fill_(scale)
    cache.v_scale.fill_(scale * 0.5)
    g = _gen(31)
    rows = (torch.randn(601, 2, D, device="cuda", generator=g).double() * scale * 20).float().to(torch.bfloat16)
    cache.append(_i32([0]), rows, rows, starts=_i32([0, 601]))
    cache.check()
    pages = cache.table[0, :-(-601 // 16)].long()
    for pool, by in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        got = pool[0, pages].permute(0, 2, 1, 3).reshape(-1, 2, D)[:601]
        # the quotient in 64 bits, rounded to 32 and then to 8: the fp32 quotient is correctly rounded
        want = (rows.double() / by[0, 0].double()).float().clamp(-448, 448).to(torch.float8_e4m3fn)
        assert torch.equal(got.view(torch.uint8), want.view(torch.uint8))


def test_cache_step_in_a_cuda_graph():
    """Append and decode captured once and replayed: the tables grow on the device."""
    from h3b import decode_attention

    g = _gen(31)
    cache = _cache(g, [100, 37], 16, 2, torch.bfloat16, spare=20, extra=64)
    slots = _i32([1, 0])
    q, k, v = (_rand(g, 2, h, D, dtype=torch.bfloat16) for h in (4, 2, 2))
    work = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
    out = torch.empty_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        cache.append(slots, k, v)
        decode_attention(q, cache, slots, out=out, workspace=work)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        cache.append(slots, k, v)
        decode_attention(q, cache, slots, out=out, workspace=work)
    for _ in range(19):
        graph.replay()
    cache.check()
    assert cache.lens.tolist() == [120, 57]
    host = HostCache(cache)
    for i, s in enumerate((1, 0)):
        rk, rv = host.rows(s)
        ref, spread = attend(q[i:i + 1], rk, rv, visible(1, rk.shape[0], None, 0, 1, "cuda"))
        assert_close(out[i:i + 1], ref, spread, rk.shape[0], 6.0)


# ------------------------------------------------------------------------------ backend

def test_window_backend_follows_the_request():
    from h3b import context as C
    from h3b.streaming import WindowAttentionB200, window_attention

    g = _gen(40)
    prefix, frames, tokens = 37, 4, 60
    L = prefix + frames * tokens
    q, k, v = (_rand(g, L, 2, D, dtype=torch.bfloat16) for _ in range(3))
    backend = WindowAttentionB200(frames=2)
    with C.attention_protected_prefix(prefix), C.attention_video_layout(frames, tokens):
        out = backend(q, k, v)
    see = visible(L, L, 2 * tokens, prefix, tokens, "cuda")
    # the frames' own description of it: prefix whole, frame f sees the prefix and frames f - 1, f
    f = (torch.arange(L, device="cuda") - prefix).div(tokens, rounding_mode="floor")
    f[:prefix] = -1
    want = (f[None] == -1) | ((f[:, None] >= 0) & (f[None] >= 0) & (f[:, None] - f[None] >= 0) & (f[:, None] - f[None] < 2))
    assert torch.equal(see, want)
    ref, spread = attend(q, k, v, see)
    assert_close(out, ref, spread, L, 6.0)
    assert torch.equal(WindowAttentionB200(tokens=50)(q, k, v), window_attention(q, k, v, window=50))


@pytest.mark.parametrize("e4m3", [False, True])
def test_streaming_example(e4m3):
    """Frame by frame over the cache is the whole sequence at once; forked continuations end where they should."""
    import importlib.util
    import os

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    spec = importlib.util.spec_from_file_location("streaming_example", os.path.join(root, "examples", "streaming.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    r = example.stream(frames=4, tokens=200, e4m3=e4m3)
    # the same sums in another division: two roundings to bf16 apart at most, P's and the output's
    assert ((r["frames"].float() - r["whole"].float()).abs() <= 2.0 ** -6 * (r["whole"].float().abs() + 1)).all()
    assert torch.isfinite(r["decoded"].float()).all() and r["decoded"].abs().amax() > 0
    cache = r["cache"]
    assert cache.lens.tolist() == [0] + [r["total"] + 10] * 3
    used = cache.refs > 0
    n = int(used.sum())
    assert used[:n].all() and not used[n:].any()
    # shared pages carry three references, the last pages of each continuation are its own
    full = r["total"] // 64
    assert cache.refs[cache.table[1, :full].long()].tolist() == [3] * full
