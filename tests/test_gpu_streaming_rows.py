"""Single tokens and odd addresses in every layout that torch gives them (GPU)."""

import pytest
import torch

pytestmark = pytest.mark.gpu

from streaming_util import D  # noqa: E402


def _i32(x):
    return torch.tensor(list(x), dtype=torch.int32, device="cuda")


def _values(tokens, heads, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(tokens, heads, D, device="cuda", generator=g).to(torch.bfloat16)


def _heads_first(x):
    return x.transpose(0, 1).contiguous().transpose(0, 1)


def _odd_address(x):
    y = torch.zeros(x.numel() + 4, dtype=x.dtype, device="cuda")[4:].view(x.shape)
    return y.copy_(x)


def _slice(x):
    y = torch.zeros(x.shape[0], x.shape[1] + 3, D, dtype=x.dtype, device="cuda")[:, 1:-2]
    return y.copy_(x)


@pytest.mark.parametrize("tokens", [1, 2])
@pytest.mark.parametrize("heads", [(4, 2), (4, 1), (1, 1)], ids=str)
@pytest.mark.parametrize("layout", [_heads_first, _odd_address, _slice])
def test_layouts_of_few_tokens(tokens, heads, layout):
    from h3b import PagedKVCache, decode_attention, paged_window_attention, window_attention

    hq, hkv = heads
    q, k, v = _values(tokens, hq, 1), _values(tokens, hkv, 2), _values(tokens, hkv, 3)
    lq, lk, lv = layout(q), layout(k), layout(v)
    want = window_attention(q, k, v)
    assert torch.equal(window_attention(lq, lk, lv), want)

    def cache(k, v):
        c = PagedKVCache.create(1, 4, 16, hkv, 2, 32)
        c.append(_i32([0]), k, v, starts=_i32([0, tokens]))
        c.check()
        return c

    plain, other = cache(k, v), cache(lk, lv)
    page = int(plain.table[0, 0])
    assert torch.equal(plain.k[0, page, :, :tokens], other.k[0, page, :, :tokens])
    assert torch.equal(plain.v[0, page, :, :tokens], other.v[0, page, :, :tokens])
    assert torch.equal(paged_window_attention(lq, other), want)
    slots = _i32([0] * tokens)
    assert torch.equal(decode_attention(lq, other, slots), decode_attention(q, plain, slots))


@pytest.mark.parametrize("tokens", [1, 3])
def test_layouts_of_the_output(tokens):
    from h3b import PagedKVCache, decode_attention, window_attention

    q, k, v = _values(tokens, 4, 1), _values(tokens, 2, 2), _values(tokens, 2, 3)
    want = window_attention(q, k, v)
    out = _slice(torch.zeros_like(q))
    assert window_attention(q, k, v, out=out) is out and torch.equal(out, want)
    out = _heads_first(torch.zeros_like(q))
    if tokens == 1:
        assert window_attention(q, k, v, out=out) is out and torch.equal(out, want)
        cache = PagedKVCache.create(1, 4, 16, 2, 2, 32)
        cache.append(_i32([0]), k, v)
        assert decode_attention(q, cache, out=out.zero_()) is out
        assert torch.equal(out, decode_attention(q, cache))
    else:
        with pytest.raises(ValueError, match="out"):
            window_attention(q, k, v, out=out)
    with pytest.raises(ValueError, match="out"):
        window_attention(q, k, v, out=_odd_address(torch.zeros_like(q)))
