"""Query rows that belong to no sequence stay as they are (GPU)."""

import pytest
import torch

pytestmark = pytest.mark.gpu

from streaming_util import D, assert_close, attend, visible  # noqa: E402


@pytest.mark.parametrize("heads", [(4, 2), (3, 3)], ids=str)
@pytest.mark.parametrize("keys", [0, 1, 400])
@pytest.mark.parametrize("starts", [[2, 5, 9], [130, 131, 300], [0, 0, 0], [7, 400, 400]], ids=str)
def test_rows_of_no_sequence_are_not_written(heads, keys, starts):
    from h3b import window_attention

    hq, hkv = heads
    g = torch.Generator(device="cuda").manual_seed(keys + starts[1])
    q = torch.randn(450, hq, D, device="cuda", generator=g).to(torch.bfloat16)
    k, v = (torch.randn(2 * keys, hkv, D, device="cuda", generator=g).to(torch.bfloat16) for _ in range(2))
    out = torch.full_like(q, 7.0)
    ints = dict(dtype=torch.int32, device="cuda")
    window_attention(q, k, v, query_starts=torch.tensor(starts, **ints),
                     key_starts=torch.tensor([0, keys, 2 * keys], **ints), out=out)
    assert (out[: starts[0]] == 7).all() and (out[starts[-1]:] == 7).all()
    for i, (a, b) in enumerate(zip(starts, starts[1:])):
        if a < b and keys == 0:
            assert not out[a:b].any()
        elif a < b:
            n = b - a
            ref, spread = attend(q[a:b], k[i * keys:(i + 1) * keys], v[i * keys:(i + 1) * keys],
                                 visible(n, keys, None, 0, 1, "cuda"))
            assert_close(out[a:b], ref, spread, keys, 6.0)
