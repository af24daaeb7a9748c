"""Fp4Rows' own layout work, on host tensors (no GPU needed)."""

import pytest
import torch

import h3b
import test_fp4_host as H
from h3b import cache, fp4

from_blocks = h3b.Fp4Rows.from_blocks.__func__


@pytest.mark.parametrize("format,block", [("mxfp4", 32), ("nvfp4", 16)])
@pytest.mark.parametrize("rows,cols", [(0, 64), (0, 4096), (1, 32), (130, 96), (3, 0), (0, 0)])
def test_rows_from_elsewhere_of_any_number(format, block, rows, cols):
    """What the constructor is given.  Rows without columns reach it too, which refuses them."""
    codes = torch.arange(rows * (cols // 2)).to(torch.uint8).view(rows, cols // 2)
    blocks = -(-cols // block)
    scales = torch.arange(rows * blocks).to(torch.uint8).view(rows, blocks)
    got, tiles, n, *_ = from_blocks(lambda *a: a, codes, scales, format)
    assert n == cols and got.shape == (rows, -(-cols // 32) * 16) and torch.equal(got[:, : cols // 2], codes)
    assert tiles.shape == (-(-rows // 128), -(-blocks // 4), 512)
    for r in range(0, rows, 7):
        for b in range(blocks):
            assert tiles[r // 128, b // 4, (r % 32) * 16 + (r % 128 // 32) * 4 + b % 4] == scales[r, b]


@pytest.mark.parametrize("format", ("mxfp4", "nvfp4"))
def test_parts_asked_for_by_two_threads(format):
    """The parts become tensors where they are first asked for.  While one thread makes them, another asks for them
    between any two steps of the first."""
    rows = h3b.Fp4Rows._room(5, 64, format, torch.empty(0, dtype=torch.bfloat16))
    buffer, other = rows._buffer, []

    class Watched:
        """The buffer; each part that is cut from it lets the other thread ask for all of them first."""
        def __getitem__(self, part):
            if len(other) < 3:
                other.append(None)
                rows._buffer, found = buffer, rows._codes is not None
                other[-1] = (rows.codes, rows.scales, rows.row_scales)
                if not found:  # nothing was there: what the other thread made is taken away again
                    rows._codes = rows._scales = rows._row_scales = None
                rows._buffer = self
            return buffer[part]
    rows._buffer = Watched()
    assert rows.codes.shape == (5, 32)
    assert other
    for codes, scales, row_scales in other:
        assert codes.shape == (5, 32) and scales is not None and scales.shape[-1] == 512
        assert (row_scales is None) == (format == "mxfp4")


def test_more_rows_than_a_call_takes_reach_the_refusal(monkeypatch):
    """2^30 + 1 rows of one column: no workspace is made for them, and the library's own words are the answer."""
    monkeypatch.setattr(cache, "_current_gpu", lambda: 0)
    monkeypatch.setattr(cache, "_raw_stream", lambda gpu: 0)
    weight = h3b.Fp4Rows(H._on(0, (4, 16), torch.uint8), H._on(0, (1, 1, 512), torch.uint8), 1, "mxfp4")
    x = H._on(0, (2, 1))
    x.shape, x.new_empty = torch.Size(((1 << 30) + 1, 1)), lambda shape, **k: H._on(0, (2, 4)) if isinstance(shape, tuple) else torch.empty(shape)
    with pytest.raises(h3b.H3BError, match="bad sizes"):
        fp4.fp4_linear(x, weight)
