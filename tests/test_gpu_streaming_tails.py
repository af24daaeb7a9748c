"""Long tails of small softmax weights under one dominant key (GPU).

The dominant key has V = 0, so the output is what the tail leaves: weights that get lost in
the rounding of P, but not in its sum, show in full."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from streaming_util import D, UNIT  # noqa: E402


def _tail(n, octaves, v):
    """Key 0 with a score of 0 and V 0, n - 1 keys `octaves` powers of two below with V = v."""
    w = 2.0 ** -octaves * (n - 1)
    return v * w / (1 + w)


def _close(out, ref, dtype, p_unit):
    """The output's rounding, that of the weights (all equal, so it does not average out) and 2e-4 for
    the exponential and the fp32 scores and sums, all relative to the output."""
    rel = ((out.double() - ref).abs() / ref).amax()
    assert rel <= (UNIT[dtype] + p_unit + 2e-4) * 1.01, f"relative error {float(rel):.2e}"


def _cache(store, heads, page, pages, slots, n, v):
    """Every slot reads the same pages: key 0 with 8 in channel 0 and V 0, the others 0 with V = v."""
    from h3b import PagedKVCache

    dtype = torch.float8_e4m3fn if store == "e4m3" else store
    ones = lambda: torch.ones(1, heads, device="cuda")  # noqa: E731
    scale = dict(k_scale=ones(), v_scale=ones()) if store == "e4m3" else {}
    cache = PagedKVCache.create(1, pages, page, heads, slots, pages * page, dtype, **scale)
    k = torch.zeros(cache.k.shape, device="cuda")
    k[0, 0, :, 0, 0] = 8
    cache.k.copy_(k.to(dtype))
    k.fill_(v)[0, 0, :, 0] = 0
    cache.v.copy_(k.to(dtype))
    cache.table.copy_(torch.arange(pages, device="cuda", dtype=torch.int32).expand(slots, -1))
    cache.lens.fill_(n)
    cache.refs.fill_(slots)
    return cache


def _query(rows, heads, dtype):
    q = torch.zeros(rows, heads, D, device="cuda", dtype=dtype)
    q[..., 0] = 8
    return q


@pytest.mark.parametrize("store,dtype", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16),
                                         ("e4m3", torch.bfloat16), ("e4m3", torch.float16)], ids=str)
@pytest.mark.parametrize("octaves", [20.6, 23.4, 25.2, 26.0])
@pytest.mark.parametrize("group", [1, 12])
def test_decode_keeps_a_long_tail(store, dtype, octaves, group):
    """As many pairs as warps, so that one warp has the dominant key and thousands of the others."""
    from h3b import decode_attention

    n, kv, slots = 32768, 8, 250
    cache = _cache(store, kv, 128, n // 128, slots, n, 1.0)
    out = decode_attention(_query(slots, kv * group, dtype), cache, scale=octaves * math.log(2) / 64)
    p_unit = UNIT[torch.bfloat16 if store is torch.bfloat16 else torch.float16]
    _close(out, _tail(n, octaves, 1.0), dtype, p_unit)


@pytest.mark.parametrize("store,dtype", [(torch.float16, torch.float16), ("e4m3", torch.bfloat16)], ids=str)
def test_decode_of_one_short_sequence_keeps_a_tail(store, dtype):
    """One chunk of 16 keys in a table that the cluster launch takes."""
    from h3b import decode_attention

    cache = _cache(store, 1, 16, 1, 1, 16, 384.0)
    out = decode_attention(_query(1, 1, dtype), cache, scale=20.6 * math.log(2) / 64)
    _close(out, _tail(16, 20.6, 384.0), dtype, UNIT[torch.float16])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("octaves", [20.6, 23.4, 25.2, 26.0])
@pytest.mark.parametrize("n", [100, 800])
def test_window_keeps_a_tail(dtype, octaves, n):
    """Few keys, with a V that keeps the output in fp16's range."""
    from h3b import window_attention

    k = torch.zeros(n, 1, D, device="cuda", dtype=dtype)
    k[0, 0, 0] = 8
    v = torch.full((n, 1, D), 30000.0, device="cuda", dtype=dtype)
    ref = _tail(n, octaves, float(v[0, 0, 0]))
    v[0] = 0
    out = window_attention(_query(1, 1, dtype), k, v, scale=octaves * math.log(2) / 64)
    _close(out, ref, dtype, UNIT[dtype])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("octaves", [23.4, 26.0])
@pytest.mark.parametrize("slots", [1, 64])
def test_paged_window_keeps_a_long_tail(dtype, octaves, slots):
    """One sequence, whose keys are divided over the multiprocessors, and more than there are of those."""
    from h3b import paged_window_attention

    n, kv = 32768, 4
    cache = _cache(dtype, kv, 128, n // 128, slots, n, 1.0)
    starts = torch.arange(slots + 1, device="cuda", dtype=torch.int32)
    out = paged_window_attention(_query(slots, kv, dtype), cache, query_starts=starts, scale=octaves * math.log(2) / 64)
    _close(out, _tail(n, octaves, 1.0), dtype, UNIT[dtype])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_window_maximum_that_creeps_up(dtype):
    """Tiles whose maxima rise by less, about and more than the running maximum tolerates: the weights
    before and after each move keep their proportions."""
    from h3b import window_attention

    n = 1280  # ten tiles
    for octaves in (0.7, 2.9, 3.1, 7.9, 8.1, 20.0):
        k = torch.zeros(n, 1, D, device="cuda", dtype=dtype)
        rise = (torch.arange(n, device="cuda") // 128).double()
        k[:, 0, 0] = rise.to(dtype)  # whole numbers up to 9
        v = torch.randn(n, 1, D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(5)).to(dtype)
        out = window_attention(_query(1, 1, dtype), k, v, scale=octaves * math.log(2) / 8)
        w = torch.exp2((rise - rise.max()) * octaves)
        w /= w.sum()
        ref, spread = (w @ v[:, 0].double()), (w @ v[:, 0].double().abs())
        u = UNIT[dtype]
        assert ((out[0, 0].double() - ref).abs() <= u * ref.abs() + (u + 2e-4) * spread * 1.01).all(), octaves


def test_decode_of_queries_with_channels_far_apart():
    """bf16 queries over an E4M3 cache whose channels span 2^42: a channel errs by at most 2^-25 of the
    head's power of two (fp16's subnormal step), a score by 128 of those times the largest key."""
    from h3b import decode_attention
    from streaming_util import HostCache, attend, visible

    g = torch.Generator(device="cuda").manual_seed(11)
    heads, n = 6, 1000
    cache = _cache("e4m3", 1, 16, 63, 1, n, 1.0)
    for pool in (cache.k, cache.v):
        pool.copy_(torch.randn(pool.shape, device="cuda", generator=g).to(pool.dtype))
    size = 2.0 ** -(torch.arange(D, device="cuda") / 3)
    sign = torch.randint(0, 2, (1, heads, D), device="cuda", generator=g) * 2 - 1
    factor = 2.0 ** torch.tensor([-30, -10, 0, 3, 20, 60], device="cuda").view(1, heads, 1)
    order = torch.stack([torch.randperm(D, device="cuda", generator=g) for _ in range(heads)])
    q = (size[order][None] * sign * factor).to(torch.bfloat16)
    k, v = HostCache(cache).rows(0)
    for h in range(heads):
        scale = float(0.7 / factor[0, h, 0])
        out = decode_attention(q, cache, scale=scale)[:, h]
        ref, spread = attend(q[:, h:h + 1], k, v, visible(1, n, None, 0, 1, "cuda"), scale)
        score = scale * 128 * 2.0 ** -25 * float(factor[0, h, 0]) * float(k.abs().max())
        u = UNIT[torch.bfloat16]
        err = (out.double() - ref[:, 0]).abs()
        assert (err <= u * ref[:, 0].abs() + (u + 2e-4 + 2 * score) * spread[:, 0] * 1.01).all(), h
