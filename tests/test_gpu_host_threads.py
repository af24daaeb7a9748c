"""Calls from host threads: a thread's first one, and one operator from two threads, each on a stream of its own (B200)."""

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


def _at_once(calls, times):
    """Each call `times` times in a thread of its own; their last results."""
    errors, last = [], [None] * len(calls)
    start = threading.Barrier(len(calls))

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                torch.zeros(1, device="cuda")
                start.wait()
                for _ in range(times):
                    last[i] = calls[i]()
                    if errors:
                        return
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001 - told to the thread that asserts
            errors.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(calls))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors[0]
    return last


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


def _check(calls, times):
    want = [c() for c in calls]
    torch.cuda.synchronize()
    for got, w in zip(_at_once(calls, times), want):
        pairs = zip(got, w) if isinstance(w, tuple) else [(got, w)]
        assert all(torch.equal(a, b) for a, b in pairs)


@pytest.mark.parametrize("fmt", ("mxfp4", "nvfp4"))
@pytest.mark.parametrize("m,wide,narrow", [(1, (12288, 4096), (512, 4096)), (24, (4096, 4096), (20000, 256)),
                                           (100, (2048, 8192), (256, 512))])
def test_4_bit_linears_of_unequal_size(h3b, fmt, m, wide, narrow):
    """Calls whose kernels take unequal amounts of shared memory."""
    calls = []
    for n, k in (wide, narrow):
        g = torch.Generator(device="cuda").manual_seed(n)
        x = torch.randn(m, k, device="cuda", generator=g).bfloat16()
        w = h3b.quantize_fp4(torch.randn(n, k, device="cuda", generator=g).bfloat16(), fmt)
        out = torch.empty(m, n, device="cuda", dtype=torch.bfloat16)
        need = h3b.lib().h3b_fp4_linear_workspace_bytes(m, w._ref)
        ws = torch.empty(max(need, 16), device="cuda", dtype=torch.uint8)
        calls.append(lambda x=x, w=w, out=out, ws=ws: h3b.fp4_linear(x, w, out=out, workspace=ws))
    _check(calls, 3000)


def _entry(h3b, name, *args):
    """A C entry as its own call: hardly any of a thread's time is spent outside it."""
    from h3b._lib import check
    entry, stream = getattr(h3b.lib(), name), lambda: torch.cuda.current_stream().cuda_stream
    return lambda: check(entry(*args, stream()), name)


def test_row_quantisers_of_unequal_width(h3b):
    calls, results = [], []
    for k in (16384, 12288):
        x = torch.randn(2, k, device="cuda").bfloat16()
        q, s = torch.empty(2, k, device="cuda", dtype=torch.int8), torch.empty(2, 1, device="cuda")
        call = _entry(h3b, "h3b_quantize_int8_rowwise", x.data_ptr(), 2, k, k, q.data_ptr(), s.data_ptr())
        calls.append(lambda call=call, keep=x, out=(q, s): (call(), out)[1])
    _check(calls, 20000)


def test_block_masks_of_unequal_length(h3b):
    from h3b import attention as A
    calls = []
    for blocks in (2000, 10):
        g = torch.Generator(device="cuda").manual_seed(blocks)
        pooled = lambda n: torch.randn(1, n, 128, device="cuda", generator=g).bfloat16()
        same = lambda n: torch.ones(1, n, device="cuda", dtype=torch.uint8)
        q = A.PreparedBlocks(pooled(2), same(2), None, None, 256, 128, 256)
        k = A.PreparedBlocks(pooled(blocks), same(blocks), None, None, 64 * blocks, 64, 64 * blocks)
        calls.append(lambda q=q, k=k: A.block_mask(q, k, A.MaskConfig("topk", 0.3)))
    _check(calls, 10000)
