"""Calls from host threads: a thread's first one (B200)."""

import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def h3b():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    import h3b
    h3b.lib()
    yield h3b
    torch.cuda.synchronize()
    assert h3b.device_status(0) == 0


def _first_calls(h3b):
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(200, 512, device="cuda", generator=g).bfloat16()
    w = torch.randn(640, 512, device="cuda", generator=g).bfloat16()
    q8, s8 = h3b.ops.quantize_int8_rowwise(x)
    w8, ws = h3b.ops.quantize_int8_rowwise(w)
    w4 = h3b.quantize_fp4(w, "nvfp4")
    rows, heads = h3b.quantize_fp4(x, "nvfp4"), x.view(200, 4, 128)
    return {
        "fp4_linear": lambda: h3b.fp4_linear(x[:3], w4),
        "fp4_linear_prequantized": lambda: h3b.fp4_linear_prequantized(rows, w4),
        "int8_linear_prequantized": lambda: h3b.ops.int8_linear_prequantized(q8, s8, w8, ws),
        "window_attention": lambda: h3b.window_attention(heads, heads, heads, window=64),
    }


@pytest.mark.parametrize("name", ["fp4_linear", "fp4_linear_prequantized", "int8_linear_prequantized", "window_attention"])
def test_first_call_of_a_thread(h3b, name):
    """The thread has made no other call to the GPU, so that no context is its own yet."""
    call = _first_calls(h3b)[name]
    want, got = call(), []
    torch.cuda.synchronize()

    def work():
        try:
            got.append(call())
        except Exception as e:  # noqa: BLE001 - told to the thread that asserts
            got.append(e)
    t = threading.Thread(target=work)
    t.start()
    t.join()
    torch.cuda.synchronize()
    assert isinstance(got[0], torch.Tensor), got[0]
    assert torch.equal(got[0], want)
