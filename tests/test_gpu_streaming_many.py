"""Window attention over more sequences than its plan lists: results and how the time grows (GPU)."""

import pytest
import torch

pytestmark = pytest.mark.gpu

from streaming_util import D, assert_close, attend, visible  # noqa: E402


def _starts(lens):
    return torch.cat([torch.zeros(1, dtype=torch.int64), torch.cumsum(torch.as_tensor(lens), 0)]).to(torch.int32).cuda()


def _milliseconds(call):
    best = float("inf")
    for _ in range(3):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        call()
        b.record()
        torch.cuda.synchronize()
        best = min(best, a.elapsed_time(b))
    return best


def test_window_time_grows_with_the_sequences_not_with_their_square():
    """One token per sequence: the output is V.  Four times the sequences may take eight times as long."""
    from h3b import window_attention

    times = []
    for n in (16384, 65536):
        q, k, v = (torch.randn(n, 1, D, device="cuda").to(torch.bfloat16) for _ in range(3))
        starts = _starts([1] * n)
        assert torch.equal(window_attention(q, k, v, query_starts=starts, key_starts=starts), v)
        times.append(_milliseconds(lambda: window_attention(q, k, v, query_starts=starts, key_starts=starts)))
    assert times[1] < 8 * times[0], times


def test_window_over_many_items_of_a_listed_plan():
    """Sequences whose plan fits, but so many heads that a block has more items than its list of tiles."""
    from h3b import window_attention

    times = []
    for n in (1500, 6000):
        q, v = (torch.randn(n, h, D, device="cuda").to(torch.bfloat16) for h in (32, 16))
        starts = _starts([1] * n)
        assert torch.equal(window_attention(q, v, v, query_starts=starts, key_starts=starts), v.repeat_interleave(2, 1))
        times.append(_milliseconds(lambda: window_attention(q, v, v, query_starts=starts, key_starts=starts)))
    assert times[1] < 8 * times[0], times


@pytest.mark.parametrize("heads", [(2, 1), (3, 3)], ids=str)
@pytest.mark.parametrize("window", [1, 60, None])
def test_window_over_many_ragged_sequences(heads, window):
    """Runs of empty sequences, long ones among them, and more tiles than the plan lists."""
    from h3b import window_attention

    hq, hkv = heads
    g = torch.Generator().manual_seed(7)
    n = 20000
    lens = torch.randint(0, 4, (n,), generator=g)
    lens[3000:9000] = 0
    lens[torch.randperm(n, generator=g)[:40]] = 300
    lens[-1], lens[0], lens[12000:12100] = 0, 513, 140
    rows = int(lens.sum())
    q = torch.randn(rows, hq, D, generator=g).to(torch.bfloat16).cuda()
    k, v = (torch.randn(rows, hkv, D, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    starts = _starts(lens)
    out = window_attention(q, k, v, window=window, query_starts=starts, key_starts=starts)
    at = starts.tolist()
    step = 250
    for i in range(0, n, step):
        a, b = at[i], at[min(i + step, n)]
        if a == b:
            continue
        see = torch.block_diag(*[visible(m, m, window, 0, 1).float() for m in lens[i:i + step].tolist() if m]).bool().cuda()
        ref, spread = attend(q[a:b], k[a:b], v[a:b], see)
        assert_close(out[a:b], ref, spread, 513, 6.0, f"sequences from {i}")


def test_window_over_many_sequences_with_starts_that_run_backwards():
    """Rows may be anything where sequences overlap; the search ends and stays in bounds."""
    from h3b import device_status, window_attention

    g = torch.Generator().manual_seed(8)
    n, rows = 9000, 4000
    starts = torch.randint(-5, rows + 100, (n + 1,), generator=g).to(torch.int32)
    starts[:4000] = torch.sort(starts[:4000]).values
    q, k, v = (torch.randn(rows, 2, D, generator=g).to(torch.bfloat16).cuda() for _ in range(3))
    window_attention(q, k, v, window=100, query_starts=starts.cuda(), key_starts=starts.cuda())
    torch.cuda.synchronize()
    assert device_status(0) == 0
