"""Which outputs of the 4-bit operators are refused for what they share with inputs (no GPU needed)."""

import itertools
from types import SimpleNamespace

import pytest
import torch

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
    square = h3b.Fp4Rows(H._on(0, (64, 32), torch.uint8), H._on(0, (1, 1, 512), torch.uint8), 64, "nvfp4")
    with pytest.raises(ValueError if met else H._Reached, match="overlap" if met else None):
        h3b.fp4_linear(x, square, out=out)
    if left != right:
        for a, b in ((x, far), (far, x)):
            with pytest.raises(ValueError if met else H._Reached, match="overlap" if met else None):
                h3b.add_rms_norm_quantize(a, b, H._at(1 << 21, (64,)), out=out)


def _at(address, shape, dtype=torch.bfloat16):
    t = H._on(0, shape, dtype)
    t.data_ptr = lambda: address
    return t


def _rows(address, rows):
    """Rows of 64 columns; the scales 64 KB behind the codes, the row scales 128 KB."""
    return h3b.Fp4Rows(_at(address, (rows, 32), torch.uint8), _at(address + (1 << 16), (1, 1, 512), torch.uint8), 64, "nvfp4",
                       _at(address + (2 << 16), (rows,), torch.float32))


class _Library:
    def __getattr__(self, name):
        return (lambda *a: 4096) if name.endswith("workspace_bytes") else lambda *a: _reached()


BIAS = 1 << 23


@pytest.mark.parametrize("at,met", [
    (0, False), ((2 << 20) - 512, False), ((2 << 20) - 510, True), (2 << 20, True), ((2 << 20) + 127, True), ((2 << 20) + 128, False),
    ((2 << 20) + (1 << 16) + 511, True), ((2 << 20) + (1 << 16) + 512, False), ((2 << 20) + (2 << 16) + 14, True),
    ((2 << 20) + (2 << 16) + 16, False), ((2 << 20) + (3 << 15), False)])
def test_outputs_on_4_bit_rows_are_refused(monkeypatch, at, met):
    """4-bit rows of 4 x 64 at 2 MB as either operand; the outputs and the workspace are 512 bytes from `at` on or longer."""
    monkeypatch.setattr(cache, "_current_gpu", lambda: 0)
    monkeypatch.setattr(cache, "_raw_stream", lambda gpu: 0)
    monkeypatch.setattr(fp4, "lib", lambda: _Library())
    q, far = _rows(2 << 20, 4), _rows(8 << 20, 64)
    x, y = _at(3 << 20, (40, 64)), _at(6 << 20, (40, 4))
    calls = [lambda: h3b.dequantize_fp4(q, out=_at(at, (4, 64))),
             lambda: h3b.fp4_linear_prequantized(q, far, out=_at(at, (4, 64))),
             lambda: h3b.fp4_linear_prequantized(_rows(5 << 20, 64), q, out=_at(at, (64, 4)))]
    if at % 2 == 0:
        calls.append(lambda: h3b.fp4_linear(_at(3 << 20, (64, 64)), q, out=_at(at, (64, 4))))
    if at % 16 == 0 and at + 4096 <= 2 << 20 or met and at % 16 == 0:
        calls.append(lambda: h3b.fp4_linear(x, q, out=y, workspace=_at(at, (4096,), torch.uint8)))
    for call in calls:
        with pytest.raises(ValueError if met else H._Reached, match="overlap" if met else None):
            call()


def test_outputs_and_workspaces_on_anything_else_are_refused(monkeypatch):
    monkeypatch.setattr(cache, "_current_gpu", lambda: 0)
    monkeypatch.setattr(cache, "_raw_stream", lambda gpu: 0)
    monkeypatch.setattr(fp4, "lib", lambda: _Library())
    q, x, y = _rows(2 << 20, 4), _at(3 << 20, (40, 64)), _at(6 << 20, (40, 4))
    bias = _at(BIAS, (4,), torch.float32)
    room = lambda at: _at(at, (4096,), torch.uint8)
    for call in (lambda: h3b.fp4_linear(x, q, bias, out=_at(BIAS - 306, (40, 4))),
                 lambda: h3b.fp4_linear_prequantized(q, q, bias, out=_at(BIAS + 14, (4, 4))),
                 lambda: h3b.fp4_linear(x, q, bias, out=y, workspace=room(BIAS - 4080)),
                 lambda: h3b.fp4_linear(x, q, bias, out=y, workspace=room((3 << 20) + 5104)),
                 lambda: h3b.fp4_linear(x, q, out=y, workspace=room((6 << 20) - 4080)),
                 lambda: h3b.fp4_linear(x, q, out=y, workspace=room((6 << 20) + 304))):
        with pytest.raises(ValueError, match="overlap"):
            call()
    for call in (lambda: h3b.fp4_linear(x, q, bias, out=_at(BIAS - 320, (40, 4))),
                 lambda: h3b.fp4_linear(x, q, bias, out=y, workspace=room(BIAS - 4096)),
                 lambda: h3b.fp4_linear(x, q, out=y, workspace=room((6 << 20) + 320))):
        with pytest.raises(H._Reached):
            call()


def test_rows_without_any_memory():
    empty = h3b.Fp4Rows(_at(0, (0, 32), torch.uint8), _at(0, (0, 1, 512), torch.uint8), 64, "nvfp4")
    assert empty._pieces() == [] and not fp4._meet((0, 4, 8, 8), (0, 0, 8, 8)) and not fp4._meet((0, 4, 0, 8), (0, 1, 8, 8))


def test_sums_into_part_of_a_batchs_rows_are_refused(monkeypatch):
    """[batch, 3 of 5 rows, columns]: these rows have no one step.  All of the batch's rows, in part of their columns, do."""
    monkeypatch.setattr(cache, "_current_gpu", lambda: 0)
    monkeypatch.setattr(fp4, "lib", _reached)
    x, residual, weight = _at(4096, (2, 3, 64)), _at(1 << 20, (2, 3, 64)), _at(1 << 21, (64,))
    for buffer, met in ((torch.zeros(2, 5, 64, dtype=torch.bfloat16)[:, :3], True), (torch.zeros(2, 3, 80, dtype=torch.bfloat16)[..., :64], False)):
        def rows(t, at=1 << 22):
            return SimpleNamespace(get_device=lambda: 0, shape=t.shape, ndim=t.ndim, dtype=t.dtype, stride=t.stride,
                                   data_ptr=lambda: at, is_contiguous=t.is_contiguous, view=lambda *s: rows(t.view(*s)))
        with pytest.raises(ValueError if met else H._Reached, match="one step" if met else None):
            h3b.add_rms_norm_quantize(x, residual, weight, out=rows(buffer))
