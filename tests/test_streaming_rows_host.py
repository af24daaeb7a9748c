"""Which token rows the streaming operators take as they lie (no GPU needed)."""

import pytest
import torch

from h3b.cache import HEAD_DIM, _row_step, _token_rows


def _heads_first(tokens, heads):
    return torch.zeros(heads, tokens, HEAD_DIM, dtype=torch.bfloat16).transpose(0, 1)


def _odd_address(tokens, heads):
    return torch.zeros(tokens * heads * HEAD_DIM + 4, dtype=torch.bfloat16)[4:].view(tokens, heads, HEAD_DIM)


def _slice(tokens, heads):
    return torch.zeros(tokens, heads + 3, HEAD_DIM, dtype=torch.bfloat16)[:, 1:heads + 1]


def _expanded(tokens, heads):
    return torch.zeros(1, heads, HEAD_DIM, dtype=torch.bfloat16).expand(tokens, -1, -1)


@pytest.mark.parametrize("tokens", [0, 1, 2, 7])
@pytest.mark.parametrize("heads", [1, 4])
@pytest.mark.parametrize("layout", [_heads_first, _odd_address, _slice, _expanded])
def test_rows_of_any_layout_become_rows_that_fit(tokens, heads, layout):
    x = layout(tokens, heads)
    y, step = _token_rows(x, heads, "x")
    assert step == _row_step(y) >= heads * HEAD_DIM and step % 8 == 0
    assert y.shape == x.shape and y.data_ptr() % 16 == 0 and (y is x) == bool(_row_step(x))


@pytest.mark.parametrize("layout,tokens,heads,fits", [
    (_slice, 5, 2, True), (_slice, 1, 2, True), (_heads_first, 1, 4, True), (_heads_first, 5, 4, False),
    (_heads_first, 5, 1, True), (_expanded, 1, 4, True), (_expanded, 3, 4, False), (_odd_address, 1, 4, False),
    (_odd_address, 5, 4, False),
])
def test_rows_that_fit_are_not_copied(layout, tokens, heads, fits):
    assert bool(_row_step(layout(tokens, heads))) == fits
