"""Which outputs of the 4-bit operators are refused for what they share with inputs (no GPU needed)."""

import itertools

import pytest

import h3b
import test_fp4_host as H
from h3b import cache, fp4


def _bytes(piece):
    at, rows, row, step = piece
    return {at + r * step + i for r in range(rows) for i in range(row)}


def test_pieces_that_share_a_byte_are_found():
    """Against the sets of their bytes.  Pieces of unequal steps may be taken to meet where they only reach into each
    other, pieces that share a byte never to be apart."""
    pieces = [(at, rows, row, step) for at in (0, 1, 4, 7, 9, 16) for rows in (0, 1, 2, 4) for row in (1, 3, 4, 8) for step in (4, 8, 10)
              if row <= step or rows < 2]
    for a, b in itertools.product(pieces, pieces):
        b = (b[0] + 6, *b[1:])
        share = bool(_bytes(a) & _bytes(b))
        assert fp4._meet(a, b) == fp4._meet(b, a)
        if a[3] == b[3] or a[1] < 2 or b[1] < 2:
            assert fp4._meet(a, b) == share, (a, b)
        else:
            assert fp4._meet(a, b) or not share


def _reached():
    raise H._Reached


@pytest.mark.parametrize("left,right,met", [(0, 64, False), (64, 0, False), (0, 63, True), (63, 0, True), (8, 80, False), (0, 0, True)])
def test_columns_of_one_buffer_beside_each_other(monkeypatch, left, right, met):
    """x and out as 64 columns each of rows of 144; `same` place and step is the norm's sum in place."""
    monkeypatch.setattr(cache, "_current_gpu", lambda: 0)
    monkeypatch.setattr(fp4, "lib", _reached)
    x, out, far = H._at(4096 + 2 * left, (4, 64), 144), H._at(4096 + 2 * right, (4, 64), 144), H._at(1 << 20, (4, 64))
    square = h3b.Fp4Rows(H._on(0, (64, 32), H.torch.uint8), H._on(0, (1, 1, 512), H.torch.uint8), 64, "nvfp4")
    with pytest.raises(ValueError if met else H._Reached, match="overlap" if met else None):
        h3b.fp4_linear(x, square, out=out)
    if left != right:
        for a, b in ((x, far), (far, x)):
            with pytest.raises(ValueError if met else H._Reached, match="overlap" if met else None):
                h3b.add_rms_norm_quantize(a, b, H._at(1 << 21, (64,)), out=out)
