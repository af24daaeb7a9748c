"""Softmax scales that the attention entries take (no GPU needed)."""

import ctypes
import math

import pytest

from h3b._lib import PageCacheStruct, lib
from h3b.streaming import _scale

D = ctypes.c_void_p(16)
CACHE = ctypes.byref(PageCacheStruct(16, 16, 1, 4, 2, 16, 2, None, None, 16, 4, 8, 16, 16, 16))
BAD = [0.0, -1.0, math.nan, math.inf, 2.4e38, 3e38]  # the last two are not finite in powers of two


@pytest.mark.parametrize("scale", BAD)
def test_entries_refuse_scales_that_are_not_finite_in_powers_of_two(scale):
    L = lib()
    assert L.h3b_window_attention(D, 512, D, 256, D, 256, 2, 8, 8, None, None, 1, 4, 2, 4, 0, 1, scale, D, 512, None, 0,
                                  None) == -1
    assert b"scale" in L.h3b_last_error()
    assert L.h3b_paged_window_attention(D, 512, 2, 8, None, None, 1, 4, CACHE, 0, 4, 0, 1, scale, D, 512, None, 0, None) == -1
    assert L.h3b_decode_attention(D, 512, 2, None, 2, 4, CACHE, 0, 4, 0, scale, D, 512, D, 1 << 40, None) == -1


@pytest.mark.parametrize("scale", BAD + [1e300])
def test_python_refuses_them_too(scale):
    with pytest.raises(ValueError, match="scale"):
        _scale(scale)


def test_scales_that_are_taken():
    assert _scale(None) == pytest.approx(1 / math.sqrt(128)) and _scale(2.3e38) == 2.3e38 and _scale(1) == 1.0
