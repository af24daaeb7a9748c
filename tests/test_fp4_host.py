"""Host side of the 4-bit operators: what is refused before a launch (no GPU needed)."""

import ctypes
import os
import re
from types import SimpleNamespace

import pytest
import torch

import fp4_util as U
import h3b
from h3b._lib import Fp4RowsStruct, lib

A = 4096  # an address that no call below reads: each is refused before a launch


def _rows(codes=A, scales=A, row_scales=None, rows=4, cols=64, fmt=1):
    return ctypes.byref(Fp4RowsStruct(codes, scales, row_scales, rows, cols, fmt))


def _refused(status, code, text):
    assert status == code, lib().h3b_last_error()
    assert text in lib().h3b_last_error().decode()


def test_quantize_refuses_before_a_launch():
    f = lib().h3b_fp4_quantize
    _refused(f(A, 2, 64, None, None), -1, "null")
    _refused(f(None, 2, 64, _rows(), None), -1, "null")
    _refused(f(A, 2, 64, _rows(codes=None), None), -1, "null")
    _refused(f(A, 2, 64, _rows(codes=A + 4), None), -2, "aligned")
    _refused(f(A, 2, 64, _rows(scales=A + 8), None), -2, "aligned")
    _refused(f(A + 1, 2, 64, _rows(), None), -2, "aligned")
    _refused(f(A, 0, 64, _rows(), None), -2, "dtype")
    _refused(f(A, 2, 63, _rows(), None), -1, "stride")
    _refused(f(A, 2, 64, _rows(fmt=3), None), -1, "format")
    _refused(f(A, 2, 64, _rows(fmt=2), None), -1, "row scales")
    _refused(f(A, 2, 64, _rows(cols=0), None), -1, "sizes")
    _refused(f(A, 2, 64, _rows(rows=-1), None), -1, "sizes")
    _refused(f(A, 2, 40000, _rows(cols=32769), None), -2, "32768")
    assert f(None, 2, 64, _rows(codes=None, scales=None, rows=0), None) == 0


def test_dequantize_and_gemm_refuse_before_a_launch():
    f = lib().h3b_fp4_dequantize
    _refused(f(_rows(), None, 2, 64, None), -1, "null")
    _refused(f(_rows(), A, 0, 64, None), -2, "dtype")
    _refused(f(_rows(), A, 2, 10, None), -1, "stride")
    assert f(_rows(rows=0), None, 2, 64, None) == 0
    f = lib().h3b_fp4_gemm
    _refused(f(_rows(), _rows(fmt=2), None, A, 2, 64, None), -1, "one format")
    _refused(f(_rows(), _rows(cols=32), None, A, 2, 64, None), -1, "columns")
    _refused(f(_rows(), _rows(rows=65), None, A, 2, 64, None), -1, "stride")
    _refused(f(_rows(), _rows(), None, None, 2, 64, None), -1, "null")
    _refused(f(_rows(), _rows(), None, A, 0, 64, None), -2, "dtype")
    _refused(f(_rows(rows=1 << 30), _rows(rows=1 << 30), None, A, 2, 1 << 30, None), -2, "tiles")
    assert f(_rows(rows=0), _rows(), None, None, 2, 64, None) == 0
    assert f(_rows(), _rows(rows=0), None, None, 2, 64, None) == 0


def test_linear_refuses_before_a_launch():
    f, size = lib().h3b_fp4_linear, lib().h3b_fp4_linear_workspace_bytes
    need = size(40, _rows())
    assert need == 40 * 32 + 512
    assert size(200, _rows(cols=100, fmt=2, row_scales=A)) == 200 * 64 + 2 * 2 * 512 + 800
    assert size(4, _rows(fmt=3)) == -1 and size(4, _rows(cols=32769)) == -1 and size(-1, _rows()) == -1
    assert size(4, None) == -1 and size(0, _rows()) == 0 and size(4, _rows(rows=0)) == 0
    assert size(4, _rows()) == 0  # few rows are quantised by the product itself
    _refused(f(A, 2, 40, 64, _rows(), None, A, 4, A, need - 1, None), -1, "workspace")
    _refused(f(A, 2, 40, 64, _rows(), None, A, 4, None, 0, None), -1, "workspace")
    _refused(f(A, 2, 40, 64, _rows(), None, A, 4, A + 8, need, None), -2, "aligned")
    _refused(f(A, 2, 4, 64, None, None, A, 4, A, need, None), -1, "null")
    _refused(f(A, 2, 4, 60, _rows(), None, A, 4, A, need, None), -1, "stride")
    _refused(f(A, 2, 4, 64, _rows(), None, A, 3, A, need, None), -1, "stride")
    _refused(f(A, 2, -4, 64, _rows(), None, A, 4, A, need, None), -1, "sizes")
    _refused(f(A, 2, 4, 40000, _rows(cols=32769), None, A, 4, A, 1 << 30, None), -2, "32768")
    assert f(None, 2, 0, 64, _rows(), None, None, 4, None, 0, None) == 0


def test_norm_refuses_before_a_launch():
    f = lib().h3b_add_rms_norm_int8
    ok = dict(x=A, xs=64, r=A, rs=64, s=A, ss=64, w=A, dt=2, m=4, k=64, eps=1e-5, q=A, sc=A)

    def call(**changed):
        a = ok | changed
        return f(*(a[n] for n in ("x", "xs", "r", "rs", "s", "ss", "w", "dt", "m", "k", "eps", "q", "sc")), None)
    for name in ("x", "s", "w", "q", "sc"):
        _refused(call(**{name: None}), -1, "null")
    for name in ("xs", "rs", "ss"):
        _refused(call(**{name: 63}), -1, "stride")
    _refused(call(dt=0), -2, "dtype")
    _refused(call(eps=-1.0), -1, "eps")
    _refused(call(eps=float("nan")), -1, "eps")
    _refused(call(eps=float("inf")), -1, "eps")
    _refused(call(k=0), -1, "sizes")
    _refused(call(k=32769, xs=40000, rs=40000, ss=40000), -2, "32768")
    _refused(call(q=A + 4), -2, "aligned")
    assert call(m=0) == 0
    f4 = lib().h3b_add_rms_norm_fp4
    _refused(f4(A, 64, A, 64, A, 64, A, 2, 1e-5, None, None), -1, "null")
    _refused(f4(A, 64, A, 64, None, 64, A, 2, 1e-5, _rows(), None), -1, "null")
    _refused(f4(A, 64, A, 64, A, 64, A, 2, 1e-5, _rows(fmt=2), None), -1, "row scales")
    assert f4(A, 64, A, 64, A, 64, A, 2, 1e-5, _rows(rows=0), None) == 0


def test_host_tensors_are_refused():
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    for call in (lambda: h3b.quantize_fp4(x), lambda: h3b.add_rms_norm_quantize(x, x, x[0]),
                 lambda: h3b.Fp4Linear.from_weight(x),
                 lambda: h3b.Fp4Rows(torch.zeros(2, 32, dtype=torch.uint8), torch.zeros(1, 1, 512, dtype=torch.uint8), 64,
                                     "mxfp4")):
        with pytest.raises(RuntimeError, match="only (on )?CUDA tensors"):
            call()


def _on(gpu, shape, dtype=torch.bfloat16):
    x = torch.zeros(shape, dtype=dtype)
    return SimpleNamespace(get_device=lambda: gpu, is_cuda=gpu >= 0, shape=x.shape, ndim=x.ndim, dtype=dtype,
                           stride=x.stride, data_ptr=lambda: 4096, is_contiguous=lambda: True, numel=x.numel,
                           element_size=x.element_size, new_empty=x.new_empty)


def _rows_on(gpu, other=None):
    u8 = torch.uint8
    return h3b.Fp4Rows(_on(gpu, (4, 32), u8), _on(gpu if other is None else other, (1, 1, 512), u8), 64, "nvfp4",
                       _on(gpu, (4,), torch.float32))


@pytest.mark.parametrize("gpu", [1, -1])  # -1: not a GPU's
def test_tensors_of_another_gpu_are_refused(gpu):
    x, w, norm = _on(0, (2, 64)), _rows_on(0), _on(0, (64,))
    other = _on(gpu, (2, 64))
    for call in (lambda: _rows_on(0, gpu), lambda: h3b.fp4_linear(other, w), lambda: h3b.fp4_linear(x, w, _on(gpu, (4,))),
                 lambda: h3b.fp4_linear(x, w, out=_on(gpu, (2, 4))),
                 lambda: h3b.fp4_linear_prequantized(w, w, _on(gpu, (4,))),
                 lambda: h3b.fp4_linear_prequantized(w, w, out=_on(gpu, (4, 4))),
                 lambda: h3b.dequantize_fp4(w, out=_on(gpu, (4, 64))),
                 lambda: h3b.add_rms_norm_quantize(x, other, norm), lambda: h3b.add_rms_norm_quantize(other, x, norm),
                 lambda: h3b.add_rms_norm_quantize(x, x, _on(gpu, (64,))),
                 lambda: h3b.add_rms_norm_quantize(x, x, norm, out=other)):
        with pytest.raises((ValueError, RuntimeError), match="GPU|CUDA"):
            call()
    if gpu == 1:
        with pytest.raises(ValueError, match="one GPU"):
            h3b.fp4_linear_prequantized(w, _rows_on(1))


def test_calls_on_another_gpu_than_the_current_one_are_refused(monkeypatch):
    from h3b import cache
    monkeypatch.setattr(cache, "_current_gpu", lambda: 1)
    w = _rows_on(0)
    for call in (lambda: h3b.fp4_linear_prequantized(w, w, out=_on(0, (4, 4))),
                 lambda: h3b.dequantize_fp4(w, out=_on(0, (4, 64)))):
        with pytest.raises(RuntimeError, match="the current device is cuda:1"):
            call()


def _at(address, shape, step=None):
    t = _on(0, shape)
    t.data_ptr = lambda: address
    if step is not None and step != shape[-1]:
        t.stride, t.is_contiguous = (lambda d: (step, 1)[d]), lambda: False
    return t


class _Reached(Exception):
    pass


@pytest.mark.parametrize("at,step,met", [
    (4096, 64, True), (4096 + 3 * 128, 64, True), (4096 + 4 * 128, 64, False), (4096 - 4 * 128, 64, False),
    (4096 - 4 * 128 + 2, 64, True), (4096, 72, True), (4096 - 3 * 144 - 128, 72, False), (4096 - 3 * 144 - 126, 72, True)])
def test_outputs_that_overlap_an_input_are_refused(monkeypatch, at, step, met):
    """Rows of 64 columns, four of x at 4,096; what is not refused reaches the library."""
    from h3b import cache, fp4

    def reached():
        raise _Reached
    square = h3b.Fp4Rows(_on(0, (64, 32), torch.uint8), _on(0, (1, 1, 512), torch.uint8), 64, "nvfp4")
    monkeypatch.setattr(cache, "_current_gpu", lambda: 0)
    monkeypatch.setattr(fp4, "lib", reached)
    x, out, far = _at(4096, (4, 64)), _at(at, (4, 64), step), _at(1 << 20, (4, 64))
    with pytest.raises(ValueError if met else _Reached, match="overlap" if met else None):
        h3b.fp4_linear(x, square, out=out)
    norm = _at(1 << 21, (64,))
    same = at == 4096 and step == 64
    for a, b in ((x, far), (far, x)):
        with pytest.raises(ValueError if met and not same else _Reached, match="overlap" if met and not same else None):
            h3b.add_rms_norm_quantize(a, b, norm, out=out)
    if same:
        with pytest.raises(ValueError, match="overlap"):
            h3b.add_rms_norm_quantize(far, far, _at(4096 + 64, (64,)), out=out)


def test_the_64_bit_form_on_known_values():
    """Elements, ties and scales worked out by hand."""
    x = torch.zeros(1, 32, dtype=torch.float64)
    x[0, :10] = torch.tensor([4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.3, 7.9])
    code, byte, _ = U.quantize(x, "mxfp4")
    assert byte.item() == 127  # 2^(floor(log2 7.9) - 2) = 1
    assert code[0, 0, :10].tolist() == [6, 0, 2, 2, 4, 4, 6, 6, 9, 7]
    x = torch.zeros(1, 16, dtype=torch.float64)
    x[0, :3] = torch.tensor([6.0, 3.0, -1.0])
    code, byte, e = U.quantize(x, "nvfp4")
    assert e.item() == -8  # 6 <= 2688 * 2^-8 = 10.5, and not 2688 * 2^-9
    assert U.scale_values(byte, "nvfp4").item() == 256.0
    assert code[0, 0, :3].tolist() == [7, 5, 10]


def test_no_read_only_loads_in_chained_kernels():
    """These kernels start while the one before them runs, and wait for it: what it writes may not come through
    the read-only path."""
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "x-minimaxh3_b200", "csrc")
    for name in ("fp4_rows.cu", "fp4_gemm.cu", "fp4.cuh"):
        code = re.sub(r"//[^\n]*", "", open(os.path.join(csrc, name)).read())
        assert not re.search(r"ld\.global(\.\w+)*\.nc|__ldg\b|__restrict__", code), name
        assert code.count("chain_wait();") >= code.count("__global__")
    rows = re.sub(r"//[^\n]*", "", open(os.path.join(csrc, "fp4_rows.cu")).read())
    # a product may read its weight before it waits, so the rows' kernels let it start only behind their own wait
    assert len(re.findall(r"chain_wait\(\);\s*chain_next\(\);", rows)) == rows.count("__global__")
