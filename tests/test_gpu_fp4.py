"""4-bit floating-point rows, their product and the linear over them, against 64-bit forms (B200)."""

import pytest
import torch

import fp4_util as U

pytestmark = pytest.mark.gpu

FORMATS = ("mxfp4", "nvfp4")
HALVES = (torch.bfloat16, torch.float16)


@pytest.fixture(scope="module")
def h3b():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    import h3b
    h3b.lib()
    yield h3b
    torch.cuda.synchronize()
    assert h3b.device_status(0) == 0


def _rows(m, k, dtype, seed=0, spread=1.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(m, k, device="cuda", generator=g) * torch.exp(spread * torch.randn(m, k, device="cuda", generator=g))
    return x.to(dtype)


def _check_quantised(q, x):
    """q's codes and scales are those of the 64-bit form, and its padding is zero."""
    code, byte, r = U.quantize(x.double(), q.format)
    m, k = x.shape
    assert (q.rows, q.cols) == (m, k)
    got = U.codes_of(q)
    assert torch.equal(got[:, :k], code.flatten(1)[:, :k])
    assert not got[:, k:].any()
    assert torch.equal(q.blocks().to(torch.int64), byte)
    groups = q.scales.shape[1] * 4
    tail = q.scales.view(-1, q.scales.shape[1], 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(-1, groups)[:m, byte.shape[1]:]
    assert not tail.any()
    if q.format == "nvfp4":
        assert torch.equal(q.row_scales.double(), torch.exp2(r.double()))
    else:
        assert q.row_scales is None


# ------------------------------------------------------------------------------------ quantisation


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("m,k", [(1, 1), (1, 15), (2, 16), (3, 17), (5, 31), (33, 32), (127, 33), (129, 64), (7, 130),
                                 (260, 512), (9, 1024), (6, 1040), (4, 4096), (3, 4111), (2, 8192), (3, 8208), (2, 16383),
                                 (2, 16384), (1, 20008), (2, 32768)])
def test_quantised_rows_are_those_of_the_formula(h3b, fmt, dtype, m, k):
    x = _rows(m, k, dtype, seed=m * 7 + k)
    _check_quantised(h3b.quantize_fp4(x, fmt), x)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", HALVES)
def test_every_16_bit_value_under_every_kind_of_scale(h3b, fmt, dtype):
    """All finite values as elements of blocks whose largest value lies one to four binades above: all borders
    between codes, with their ties, under many scales."""
    bits = torch.arange(0, 1 << 16, device="cuda", dtype=torch.int32).to(torch.int16)
    v = bits.view(dtype)
    v = v[torch.isfinite(v)].double()
    tops = torch.tensor([1.0, 1.2, 1.5, 1.75, 2.0, 3.0, 5.5, 7.0, 12.0], device="cuda", dtype=torch.float64)
    x = torch.zeros(v.numel(), tops.numel(), 32, device="cuda", dtype=torch.float64)
    x[..., 3], x[..., 20] = v[:, None], -v[:, None]
    x[..., 9], x[..., 30] = v[:, None] * tops, v[:, None] * tops
    x = x.flatten(1).to(dtype)
    x[~torch.isfinite(x)] = 0
    x = x.view(-1, 64 * 9 // 2)
    for at in range(0, x.shape[0], 1 << 16):
        part = x[at: at + (1 << 16)].contiguous()
        _check_quantised(h3b.quantize_fp4(part, fmt), part)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", HALVES)
def test_blocks_far_apart_and_empty(h3b, fmt, dtype):
    x = torch.zeros(8, 192, device="cuda", dtype=torch.float64)
    x[1, 5] = 1.0
    x[2] = torch.exp2(torch.arange(192, device="cuda") // 16 * 2.0 - 20)          # blocks from 2^-20 to 2^2
    x[3] = torch.exp2(torch.arange(192, device="cuda").double() / 12 - 24)        # down to fp16's subnormals
    x[4] = torch.finfo(dtype).max
    x[5] = torch.finfo(dtype).smallest_normal
    x[6, ::2] = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps       # the least subnormal
    x[7, :16], x[7, 16:] = torch.finfo(dtype).max, 1e-3
    x = x.to(dtype)
    _check_quantised(h3b.quantize_fp4(x, fmt), x)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("k", [96, 100, 4096])
def test_infinities_and_nan_take_their_block_with_them(h3b, fmt, dtype, k):
    x = _rows(6, k, dtype, seed=3)
    x[0, 5], x[1, 40], x[2, k - 1] = float("inf"), float("-inf"), float("nan")
    x[3] = float("nan")
    x[4, ::2] = float("inf")
    q = h3b.quantize_fp4(x, fmt)
    _check_quantised(q, x)
    back = h3b.dequantize_fp4(q, dtype)
    b = U.BLOCK[fmt]
    lost = torch.nn.functional.pad(~torch.isfinite(x), (0, -k % b)).view(6, -1, b).any(-1).repeat_interleave(b, 1)[:, :k]
    assert torch.equal(torch.isnan(back), lost)


@pytest.mark.parametrize("fmt", FORMATS)
def test_rows_with_any_step_and_address(h3b, fmt):
    base = _rows(20, 200, torch.bfloat16, seed=5)
    for x in (base[:, 1:129], base[::3, 8:72], base[:, ::2], base.T, base[:, 3:4], base[2:3, 7:50], base[:1].expand(5, 200)):
        _check_quantised(h3b.quantize_fp4(x, fmt), x)
    q = h3b.quantize_fp4(base.view(4, 5, 200), fmt)
    assert torch.equal(q.codes, h3b.quantize_fp4(base, fmt).codes)
    q = h3b.quantize_fp4(base[:0], fmt)
    assert q.rows == 0 and h3b.dequantize_fp4(q).shape == (0, 200)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("m,k", [(1, 1), (3, 17), (130, 48), (65, 1000)])
def test_dequantised_rows(h3b, fmt, dtype, m, k):
    """Codes under scales and row scales that 16-bit values hold exactly come back as they are."""
    q = U.random_rows(h3b, m, k, fmt, 11, row_scales=True)
    want = U.values(q)
    assert torch.equal(h3b.dequantize_fp4(q, dtype).double(), want)
    room = torch.full((m + 2, k + 9), 7.0, device="cuda", dtype=dtype)
    got = h3b.dequantize_fp4(q, dtype, out=room[1:-1, 4: 4 + k])
    assert torch.equal(got.double(), want) and got.data_ptr() == room[1:-1, 4: 4 + k].data_ptr()
    room[1:-1, 4: 4 + k] = 7.0
    assert (room == 7.0).all()


def test_quantised_rows_beyond_32_bit_offsets(h3b):
    m, k = 67000, 32768
    x = torch.zeros(m, k, device="cuda", dtype=torch.bfloat16)
    some = torch.tensor([0, 1, 32767, 65535, 65536, 66000, m - 1], device="cuda")
    x[some] = _rows(some.numel(), k, torch.bfloat16, seed=9)
    for fmt in FORMATS:
        q = h3b.quantize_fp4(x, fmt)
        want = h3b.quantize_fp4(x[some], fmt)
        assert torch.equal(q.codes[some], want.codes)
        assert torch.equal(q.codes.sum(dtype=torch.int64), want.codes.sum(dtype=torch.int64))
        back = h3b.dequantize_fp4(q)
        assert torch.equal(back[some], h3b.dequantize_fp4(want))
        assert torch.equal(back.count_nonzero(), h3b.dequantize_fp4(want).count_nonzero())
        del q, back


# ------------------------------------------------------------------------------------ layouts


@pytest.mark.parametrize("fmt", FORMATS)
def test_blocks_from_elsewhere(h3b, fmt):
    """from_blocks is the inverse of blocks(), and takes the scale types themselves."""
    for m, k in ((1, 32), (130, 96), (257, 1056)):
        q = h3b.quantize_fp4(_rows(m, k, torch.bfloat16, seed=k), fmt)
        again = h3b.Fp4Rows.from_blocks(q.codes[:, : k // 2], q.blocks(), fmt, q.row_scales)
        assert torch.equal(again.codes, q.codes)
        assert torch.equal(again.blocks(), q.blocks())
        typed = q.blocks().view(torch.float8_e8m0fnu if fmt == "mxfp4" else torch.float8_e4m3fn)
        assert torch.equal(h3b.Fp4Rows.from_blocks(q.codes[:, : k // 2], typed, fmt).blocks(), q.blocks())
        layer = h3b.Fp4Linear(q)
        assert torch.equal(layer.dense_weight().double(), U.values(q))


# ------------------------------------------------------------------------------------ products

SMALL = [(1, 1, 1), (1, 128, 64), (2, 7, 31), (3, 129, 32), (15, 64, 65), (16, 130, 256), (17, 127, 257), (33, 1003, 96),
         (64, 256, 1056), (65, 128, 100), (128, 384, 512), (129, 100, 4096), (257, 65, 2080), (300, 1003, 1041),
         (1, 4096, 4096), (8, 512, 16384), (5, 12288, 320), (16, 40000, 64), (5, 30000, 4160), (100, 30000, 1100),
         (60, 30000, 1100), (300, 4500, 1100), (1, 24000, 260), (40, 300, 5000)]
LARGE = [(2300, 2050, 32), (10000, 8, 96), (10001, 1, 300), (9900, 72, 64), (2304, 2304, 257),
         (2301, 2051, 1056), (256, 18950, 100), (19000, 250, 640), (1300, 4096, 4096)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("m,n,k", SMALL + LARGE)
def test_products_whose_sums_are_exact(h3b, fmt, dtype, m, n, k):
    """Elements are multiples of 1/2 up to 6 under scales 1/2, 1 and 2: products are multiples of 1/16 up to 144, so
    fp32 sums of up to 2^24 / (144 * 16) = 7,281 of them are exact in any order (random signs keep longer ones far
    below that), and the output is the exact value rounded once."""
    x, w = U.random_rows(h3b, m, k, fmt, 1), U.random_rows(h3b, n, k, fmt, 2)
    want = (U.values(x) @ U.values(w).T).to(torch.float32)
    got = h3b.fp4_linear_prequantized(x, w, out_dtype=dtype)
    assert torch.equal(got, want.to(dtype))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("m,n,k", [(1, 4096, 4096), (1, 12288, 4096), (7, 1003, 1044), (16, 333, 4100), (2, 70, 24),
                                   (11, 8192, 16384), (3, 40000, 8192), (48, 520, 16384), (333, 384, 2048), (1111, 1003, 1056),
                                   (2300, 2050, 700)])
def test_linear_against_the_definition(h3b, fmt, dtype, m, n, k):
    x, w = _rows(m, k, dtype, seed=m, spread=0.7), _rows(n, k, torch.bfloat16, seed=n, spread=0.3) / 64
    bias = torch.randn(n, device="cuda", generator=torch.Generator(device="cuda").manual_seed(4))
    weight = h3b.quantize_fp4(w, fmt)
    xq = h3b.quantize_fp4(x, fmt)
    for b in (None, bias):
        want, bound = U.product(xq, weight, b)
        got = h3b.fp4_linear(x, weight, b)
        assert got.dtype is dtype
        U.assert_product(got, want, bound)
        assert torch.equal(got, h3b.fp4_linear_prequantized(xq, weight, b, out_dtype=dtype))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m,n", [(5, 200), (200, 300), (2300, 2050)])
def test_row_scales_on_either_side(h3b, fmt, m, n):
    k = 224
    for rx, rw in ((False, True), (True, False), (True, True)):
        x, w = U.random_rows(h3b, m, k, fmt, 5, row_scales=rx), U.random_rows(h3b, n, k, fmt, 6, row_scales=rw)
        if rw:
            w.row_scales.mul_(1.1)
        want, bound = U.product(x, w)
        U.assert_product(h3b.fp4_linear_prequantized(x, w), want, bound)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m,n", [(5, 200), (130, 301), (2300, 2050)])
def test_output_rows_with_any_step_and_nothing_beside_them(h3b, fmt, m, n):
    k = 96
    x, w = U.random_rows(h3b, m, k, fmt, 7), U.random_rows(h3b, n, k, fmt, 8)
    want = (U.values(x) @ U.values(w).T).to(torch.bfloat16)
    for left, right in ((0, 0), (8, 16), (4, 4), (2, 5), (1, 0)):
        room = torch.full((m + 2, left + n + right), 3.25, device="cuda", dtype=torch.bfloat16)
        out = room[1: m + 1, left: left + n]
        assert h3b.fp4_linear_prequantized(x, w, out=out).data_ptr() == out.data_ptr()
        assert torch.equal(out, want)
        out.fill_(3.25)
        assert (room == 3.25).all()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m,n", [(3, 70), (100, 130), (2300, 2050)])
def test_what_lies_behind_the_rows_does_not_matter(h3b, fmt, m, n):
    """Scales behind the last row are anything, NaN too; the rows' own NaN stays in its row or column."""
    k = 160
    x, w = U.random_rows(h3b, m, k, fmt, 9), U.random_rows(h3b, n, k, fmt, 10)
    want = (U.values(x) @ U.values(w).T).to(torch.bfloat16)
    for q in (x, w):
        tiles = q.scales.view(-1, q.scales.shape[1], 32, 4, 4).permute(0, 3, 2, 1, 4)  # bands, row / 32, row % 32, ...
        last = tiles[-1]
        r = torch.arange(128, device="cuda").view(4, 32)
        last[r >= (q.rows - 1) % 128 + 1] = 255 if fmt == "mxfp4" else 127
    assert torch.equal(h3b.fp4_linear_prequantized(x, w), want)
    nan = 255 if fmt == "mxfp4" else 127

    def set_scale(q, row, byte):
        q.scales.view(-1, q.scales.shape[1], 32, 4, 4)[row // 128, 0, row % 32, row // 32 % 4, 1] = byte
    set_scale(x, m - 1, nan)
    set_scale(w, n // 2, nan)
    got = h3b.fp4_linear_prequantized(x, w)
    lost = torch.zeros_like(got, dtype=torch.bool)
    lost[m - 1], lost[:, n // 2] = True, True
    assert torch.equal(torch.isnan(got), lost) and torch.equal(got[~lost], want[~lost])


@pytest.mark.parametrize("fmt", FORMATS)
def test_scales_at_the_ends_of_their_range(h3b, fmt):
    """Products of the largest and least scales; what fp32 cannot hold is infinite or zero, and nothing is NaN."""
    k = 64
    ends = (127 - 60, 127 + 60) if fmt == "mxfp4" else (121, 135)
    x, w = U.random_rows(h3b, 40, k, fmt, 12, scales=ends), U.random_rows(h3b, 70, k, fmt, 13, scales=ends)
    want, bound = U.product(x, w)
    U.assert_product(h3b.fp4_linear_prequantized(x, w), want, bound)
    if fmt == "mxfp4":
        a = h3b.Fp4Rows.from_blocks(torch.full((2, 16), 0x77, device="cuda", dtype=torch.uint8),
                                    torch.tensor([[254], [0]], device="cuda", dtype=torch.uint8), fmt)
        got = h3b.fp4_linear_prequantized(a, a)
        assert torch.equal(got, torch.tensor([[float("inf"), 1152.0], [1152.0, 0.0]], device="cuda").bfloat16())


def test_outputs_beyond_32_bit_offsets(h3b):
    m, n, k = 66000, 33000, 32
    x, w = U.random_rows(h3b, m, k, "mxfp4", 14), U.random_rows(h3b, n, k, "mxfp4", 15)
    got = h3b.fp4_linear_prequantized(x, w)
    some = torch.tensor([0, 255, 256, 32767, 65071, 65072, 65300, m - 1], device="cuda")
    want = (U.values(x)[some] @ U.values(w).T).to(torch.bfloat16)
    assert torch.equal(got[some], want)


def test_long_rows_of_prequantised_operands(h3b):
    """Products take rows longer than those that are quantised here."""
    k = 40000 * 2
    x, w = U.random_rows(h3b, 3, k, "nvfp4", 16), U.random_rows(h3b, 200, k, "nvfp4", 17)
    want, bound = U.product(x, w)
    U.assert_product(h3b.fp4_linear_prequantized(x, w), want, bound)


# ------------------------------------------------------------------------------------ calls


@pytest.mark.parametrize("fmt", FORMATS)
def test_linear_takes_leading_dimensions_and_no_rows(h3b, fmt):
    layer = h3b.Fp4Linear.from_weight(_rows(96, 80, torch.bfloat16, seed=1), torch.randn(96, device="cuda").bfloat16(), fmt)
    x = _rows(12, 80, torch.bfloat16, seed=2)
    want = layer(x)
    assert (layer.in_features, layer.out_features) == (80, 96)
    assert torch.equal(layer(x.view(3, 4, 80)), want.view(3, 4, 96))
    assert torch.equal(layer(x[5]), want[5])
    assert torch.equal(layer(x.view(3, 4, 80).transpose(0, 1)), want.view(3, 4, 96).transpose(0, 1))
    assert layer(x[:0]).shape == (0, 96) and layer(x.view(3, 4, 80)[:, :0]).shape == (3, 0, 96)
    assert torch.equal(layer.forward_prequantized(layer.quantize(x)), want)
    empty = h3b.Fp4Linear(h3b.quantize_fp4(_rows(96, 80, torch.bfloat16)[:0], fmt))
    assert empty(x).shape == (12, 0)
    x = x.repeat(10, 1)
    need = h3b.lib().h3b_fp4_linear_workspace_bytes(120, layer.weight._ref)
    ws = torch.full((need + 64,), 0x5A, device="cuda", dtype=torch.uint8)
    out = torch.empty(120, 96, device="cuda", dtype=torch.bfloat16)
    assert h3b.fp4_linear(x, layer.weight, layer.bias, out=out, workspace=ws) is out
    assert torch.equal(out, want.repeat(10, 1)) and (ws[need:] == 0x5A).all()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m", [1, 2, 3, 4, 8, 9, 16, 17])
@pytest.mark.parametrize("n,k", [(96, 200), (4096, 1024), (300, 4096), (12288, 4096)])
def test_few_rows_of_any_step_and_address(h3b, fmt, m, n, k):
    """The product that quantises its rows itself, and the one behind a kernel that does, give what the two
    calls give; infinities and NaN in x stay in their rows."""
    base = _rows(m + 1, k + 24, torch.bfloat16, seed=m, spread=1.0)
    w = h3b.quantize_fp4(_rows(n, k, torch.bfloat16, seed=n, spread=0.3), fmt)
    bias = torch.randn(n, device="cuda")
    for x in (base[1:, 8: k + 8], base[1:, 1: k + 1], base[:m, : k].contiguous(), base[1:, 2: k + 2]):
        want = h3b.fp4_linear_prequantized(h3b.quantize_fp4(x, fmt), w, bias)
        assert torch.equal(h3b.fp4_linear(x, w, bias), want)
    x = base[1:, :k].clone()
    x[m // 2, k // 3], x[0, k - 1] = float("nan"), float("inf")
    got, want = h3b.fp4_linear(x, w), h3b.fp4_linear_prequantized(h3b.quantize_fp4(x, fmt), w)
    lost = torch.zeros(m, device="cuda", dtype=torch.bool)
    lost[m // 2] = lost[0] = True
    assert torch.equal(torch.isnan(got).all(1), lost) and torch.equal(got[~lost], want[~lost])
    assert torch.equal(torch.isnan(got), torch.isnan(want))


@pytest.mark.parametrize("m", [40, 700])
def test_graphs_that_share_a_workspace(h3b, m):
    """Two captured calls with one workspace, replayed one after the other on a stream, in either order."""
    k, n = 1024, 768
    w = [h3b.quantize_fp4(_rows(n, k, torch.bfloat16, seed=s, spread=0.3), "nvfp4") for s in (1, 2)]
    x = [_rows(m, k, torch.bfloat16, seed=s) for s in (3, 4)]
    ws = torch.empty(h3b.lib().h3b_fp4_linear_workspace_bytes(m, w[0]._ref), device="cuda", dtype=torch.uint8)
    graphs, outs = [], []
    for i in range(2):
        h3b.fp4_linear(x[i], w[i], workspace=ws)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(h3b.fp4_linear(x[i], w[i], workspace=ws))
        graphs.append(g)
    for order in ((0, 1), (1, 0), (1, 1, 0)):
        for i in range(2):
            x[i].copy_(torch.randn(m, k, device="cuda"))
        want = [h3b.fp4_linear(x[i], w[i]) for i in range(2)]
        for i in order:
            graphs[i].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(outs[i], want[i]) for i in set(order))


@pytest.mark.parametrize("m", [1, 40, 2300])
def test_same_sums_every_time(h3b, m):
    x = _rows(m, 2048, torch.bfloat16, seed=8)
    w = h3b.quantize_fp4(_rows(2050, 2048, torch.bfloat16, seed=9), "nvfp4")
    first = h3b.fp4_linear(x, w)
    for _ in range(10):
        assert torch.equal(h3b.fp4_linear(x, w), first)


@pytest.mark.parametrize("m", [3, 300, 2300])
def test_a_weight_quantised_right_before_its_use(h3b, m):
    """The product reads the weight that the kernel in front of it in the stream wrote, on a stream of its own."""
    side = torch.cuda.Stream()
    raw = [_rows(2050, 512, torch.bfloat16, seed=s) for s in range(4)]
    x = _rows(m, 512, torch.bfloat16, seed=20)
    want = [h3b.fp4_linear(x, h3b.quantize_fp4(w, "mxfp4")) for w in raw]
    torch.cuda.synchronize()
    weight = h3b.quantize_fp4(raw[0], "mxfp4")
    side.wait_stream(torch.cuda.current_stream())
    got = []
    with torch.cuda.stream(side):
        for w in raw:
            new = h3b.quantize_fp4(w, "mxfp4")
            weight.codes.copy_(new.codes)
            weight.scales.copy_(new.scales)
            got.append(h3b.fp4_linear(x, weight))
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_two_streams_at_once(h3b):
    w = [h3b.quantize_fp4(_rows(4096, 4096, torch.bfloat16, seed=s), "nvfp4") for s in (1, 2)]
    x = [_rows(24, 4096, torch.bfloat16, seed=s) for s in (3, 4)]
    want = [h3b.fp4_linear(a, b) for a, b in zip(x, w)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(h3b.fp4_linear(x[i], w[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


def test_refusals_on_the_gpu(h3b):
    x = torch.zeros(4, 64, device="cuda", dtype=torch.bfloat16)
    q = h3b.quantize_fp4(x, "mxfp4")
    other = h3b.quantize_fp4(x, "nvfp4")
    refused = [
        lambda: h3b.quantize_fp4(x.float()),
        lambda: h3b.quantize_fp4(x, "fp4"),
        lambda: h3b.quantize_fp4(x[:, :0]),
        lambda: h3b.quantize_fp4(torch.zeros(1, 32769, device="cuda", dtype=torch.bfloat16)),
        lambda: h3b.dequantize_fp4(q, torch.float32),
        lambda: h3b.dequantize_fp4(q, out=torch.empty(4, 65, device="cuda", dtype=torch.bfloat16)),
        lambda: h3b.dequantize_fp4(q, out=torch.empty(64, 4, device="cuda", dtype=torch.bfloat16).T),
        lambda: h3b.fp4_linear_prequantized(q, other),
        lambda: h3b.fp4_linear_prequantized(q, h3b.quantize_fp4(x[:, :32], "mxfp4")),
        lambda: h3b.fp4_linear_prequantized(q, q, torch.zeros(3, device="cuda")),
        lambda: h3b.fp4_linear_prequantized(q, q, out_dtype=torch.float32),
        lambda: h3b.fp4_linear_prequantized(q, q, out=torch.empty(1, 4, device="cuda", dtype=torch.bfloat16).expand(4, 4)),
        lambda: h3b.fp4_linear(x[:, :32], q),
        lambda: h3b.fp4_linear(x.float(), q),
        lambda: h3b.fp4_linear(x.repeat(10, 1), q, workspace=torch.empty(16, device="cuda", dtype=torch.uint8)),
        lambda: h3b.fp4_linear(x.repeat(10, 1), q, workspace=torch.empty(1 << 16, device="cuda", dtype=torch.uint8)[1:]),
        lambda: h3b.fp4_linear(x, q, torch.zeros(4)),
        lambda: h3b.fp4_linear(x, q, out=x[:, :4]),
        lambda: h3b.Fp4Rows(q.codes, q.scales, 65, "mxfp4"),
        lambda: h3b.Fp4Rows(q.codes, q.scales, 64, "nvfp4x"),
        lambda: h3b.Fp4Rows(q.codes, q.scales[:, :, :256], 64, "mxfp4"),
        lambda: h3b.Fp4Rows(q.codes, q.scales.int(), 64, "mxfp4"),
        lambda: h3b.Fp4Rows(q.codes, q.scales, 64, "mxfp4", torch.zeros(5, device="cuda")),
        lambda: h3b.Fp4Rows.from_blocks(q.codes, q.blocks()[:, :1], "mxfp4"),
        lambda: h3b.Fp4Linear.from_weight(x[0]),
    ]
    for i, call in enumerate(refused):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")
    assert torch.equal(h3b.fp4_linear(x, q), torch.zeros(4, 4, device="cuda").bfloat16())
