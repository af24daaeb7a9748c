"""4-bit floating-point operators at the ends of their scales' range, and long sums that are exact (B200)."""

import math

import pytest
import torch

import fp4_util as U

pytestmark = pytest.mark.gpu

HALVES = (torch.bfloat16, torch.float16)
SIZES = [(1, 300), (5, 4096), (40, 200), (300, 333), (2300, 2050)]  # a split over K or none, and pairs of SMs
FAR = (-126, -100, -60, -20, -1, 0, 1, 30, 75, 116)  # of nvfp4 row scales


@pytest.fixture(scope="module")
def h3b():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    import h3b
    h3b.lib()
    yield h3b
    torch.cuda.synchronize()
    assert h3b.device_status(0) == 0


def _assert_in_range(got, want, bound):
    """`want` within the bound where the output type holds it, infinite where it does not: from half a step above
    the largest finite value on.  So near to that that the bound reaches over it either may come."""
    most = torch.finfo(got.dtype).max
    top = most + 2.0 ** (math.frexp(most)[1] - 1) * U.UNIT[got.dtype]
    inside, outside = want.abs() + bound < top, want.abs() - bound > top
    assert torch.equal(got[outside].double(), torch.copysign(torch.full_like(want, float("inf")), want)[outside])
    U.assert_product(got[inside], want[inside], bound[inside])
    return inside


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("m,n", SIZES)
@pytest.mark.parametrize("fmt,scales,exponents", [
    ("nvfp4", (126, 127, 128), FAR), ("nvfp4", (134, 135), FAR), ("nvfp4", (121, 122), FAR),
    ("mxfp4", (127 + 40, 127 + 41), (-120, -50, 0, 20)), ("mxfp4", (127 - 40, 127 - 41), (120, 50, 0, -20)),
    ("mxfp4", (127 + 50, 127 + 51), (-120, -50, 0, 30)), ("mxfp4", (127 - 55, 127 - 56), (120, 50, 0, -50))])
def test_row_scales_far_apart(h3b, fmt, scales, exponents, m, n, dtype):
    """A large scale on one side and a small one on the other, whole powers of two and others, with a bias and
    without: what lies in the output's range is finite and right."""
    k = 224
    x, w = (U.random_rows(h3b, rows, k, fmt, 21 + rows, scales=scales, row_scales=True) for rows in (m, n))
    e = torch.tensor(exponents, device="cuda").float()
    for factor in (1.0, 1.1):
        x.row_scales.copy_(torch.exp2(e[torch.arange(m, device="cuda") % len(e)]) * factor)
        # the other side's go through all of them for each of these
        w.row_scales.copy_(torch.exp2(e[(torch.arange(n, device="cuda") * 7 + 3) % len(e)]) * factor)
        for bias in (None, torch.randn(n, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))):
            want, bound = U.product(x, w, bias)
            inside = _assert_in_range(h3b.fp4_linear_prequantized(x, w, bias, out_dtype=dtype), want, bound)
            assert inside.any() or m == 1  # a single row may have nothing but large sums


@pytest.mark.parametrize("m,n", SIZES)
def test_linear_of_far_rows(h3b, m, n):
    """Rows near the end of bf16's range times a small weight, and the other way round."""
    k = 160
    g = torch.Generator(device="cuda").manual_seed(m)
    x, w = (torch.randn(rows, k, device="cuda", generator=g) for rows in (m, n))
    for a, b in ((x * 2.0 ** 108, w * 2.0 ** -100), (x * 2.0 ** -122, w * 2.0 ** 124)):
        a, b = a.bfloat16(), b.bfloat16()
        weight = h3b.quantize_fp4(b, "nvfp4")
        want, bound = U.product(h3b.quantize_fp4(a, "nvfp4"), weight)
        got = h3b.fp4_linear(a, weight)
        assert torch.isfinite(got).all()
        U.assert_product(got, want, bound)
    one = torch.zeros(m, 16, device="cuda", dtype=torch.bfloat16)
    one[:, 0] = 1.5 * 2.0 ** 127
    small = torch.zeros(n, 16, device="cuda", dtype=torch.bfloat16)
    small[:, 0] = 2.0 ** -100
    got = h3b.fp4_linear(one, h3b.quantize_fp4(small, "nvfp4"))
    want, bound = U.product(h3b.quantize_fp4(one, "nvfp4"), h3b.quantize_fp4(small, "nvfp4"))
    U.assert_product(got, want, bound)


@pytest.mark.parametrize("dtype", HALVES)
def test_few_scales_apart_among_others(h3b, dtype):
    """One row, or one column of a tile, whose scale lies on the other side: it changes nothing beside it."""
    m, n, k = 2300, 2050, 96
    x, w = (U.random_rows(h3b, rows, k, "nvfp4", 31, row_scales=True) for rows in (m, n))
    x.row_scales.fill_(2.0 ** -3)
    w.row_scales.fill_(2.0 ** -4)
    x.row_scales[70], x.row_scales[m - 1], w.row_scales[300], w.row_scales[n - 1] = 2.0 ** 100, 2.0 ** 2, 2.0 ** 90, 2.0 ** -99
    want, bound = U.product(x, w)
    inside = _assert_in_range(h3b.fp4_linear_prequantized(x, w, out_dtype=dtype), want, bound)
    assert inside[:70, :300].all()


def test_dequantised_rows_under_far_scales(h3b):
    """A block scale that a row scale brings back into the range."""
    for bytes_, e in (((254, 253, 200), -60), ((254, 253, 200), -127), ((0, 1, 60), 60), ((0, 1, 60), 100), ((120, 127, 130), 0)):
        codes = torch.arange(256, device="cuda").to(torch.uint8).repeat(3).view(3, 256)
        scales = torch.tensor(bytes_, device="cuda", dtype=torch.uint8)[:, None].expand(3, 16)
        for factor in (1.0, -1.0):
            q = h3b.Fp4Rows.from_blocks(codes, scales, "mxfp4", torch.full((3,), factor * 2.0 ** e, device="cuda"))
            want = U.values(q)
            got = h3b.dequantize_fp4(q)
            inside = want.abs() <= torch.finfo(torch.bfloat16).max
            assert torch.equal(got[inside].double(), want[inside].bfloat16().double()) and not got[~inside].isfinite().any()
            assert not got.isnan().any()


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("m,n,k", [(1, 4096, 4096), (2, 700, 16384), (11, 520, 16384), (48, 520, 16384), (100, 4100, 4096),
                                   (333, 700, 16384), (2300, 2050, 4096), (1300, 2050, 16384)])
def test_long_sums_of_scales_with_mantissas(h3b, dtype, m, n, k):
    """E4M3 scales 1 to 1.875: products are multiples of 1/4 * 1/64, and while the sum of magnitudes is below 2^24 of
    those fp32 sums are exact in any order.  In rows of 16,384 a block in four of x is not zero, in each row others."""
    g = torch.Generator(device="cuda").manual_seed(k + m)
    rows = []
    for r in (m, n):
        codes = torch.randint(0, 256, (r, k // 2), device="cuda", dtype=torch.uint8, generator=g)
        scales = torch.randint(56, 64, (r, k // 16), device="cuda", generator=g)
        if r == m and not rows and k > 4096:
            empty = (torch.arange(k // 16, device="cuda") + torch.arange(r, device="cuda")[:, None]) % 4 > 0
            codes.masked_fill_(empty.repeat_interleave(8, 1), 0)
        rows.append(h3b.Fp4Rows.from_blocks(codes, scales.to(torch.uint8), "nvfp4"))
    a, b = (U.values(r) for r in rows)
    assert (a.abs() @ b.abs().T).max().item() * 256 < 2 ** 24
    want = (a @ b.T).to(torch.float32).to(dtype)
    assert torch.equal(h3b.fp4_linear_prequantized(*rows, out_dtype=dtype), want)


# ------------------------------------------------------------------------------------ the norm's INT8 rows


@pytest.mark.parametrize("k", [40, 1024, 4096])
def test_int8_rows_whose_scale_is_subnormal(h3b, k):
    """Rows whose absmax / 127 is below fp32's normal numbers have codes like any others.  y is off by half of
    2^-149 in each of two roundings besides what the norm's tests count, and so is the scale."""
    g = torch.Generator(device="cuda").manual_seed(k)
    x = torch.randn(12, k, device="cuda", generator=g).bfloat16()
    sign = torch.sign(torch.randn(k, device="cuda", generator=g))
    for e in (-125, -128, -131, -133):
        w = (sign * 2.0 ** e).bfloat16()
        h, (q, s) = h3b.add_rms_norm_quantize(x, None, w)
        y = x.double() / torch.sqrt((x.double() ** 2).mean(1, keepdim=True) + 1e-5) * w.double()
        off, step = 44 * 2.0 ** -24, 2.0 ** -149
        top = y.abs().amax(1, keepdim=True)
        assert (s > 0).all() and (s < 2.0 ** -126).any()
        assert ((s.double() * 127 - top).abs() <= (off + 2.0 ** -23) * top + 64 * step).all()
        ratio = y / s.double()
        want = ratio.clamp(-127, 127)
        assert ((q.double() - want).abs() <= 0.5 + 127 * (off + 2.0 ** -23) + 2 * step / s.double()).all()
    # rows on either side of the border in one call, and one of zeros
    x[3] = 0
    x[5:, k // 2:] = 0
    w = torch.full((k,), 1.0, device="cuda").bfloat16()
    w[: k // 2] = 2.0 ** -130
    x[0, : k // 2] = 0
    x[1, k // 2:] = 0
    h, (q, s) = h3b.add_rms_norm_quantize(x, None, w)
    assert s[0] > 1e-3 and q[0].any() and 0 < s[1] < 2.0 ** -126 and q[1].abs().max() >= 126 and s[3] == 0 and not q[3].any()


# ------------------------------------------------------------------------------------ outputs beside inputs


@pytest.mark.parametrize("m", [1, 5, 40, 700])
def test_inputs_and_outputs_in_the_columns_of_one_buffer(h3b, m):
    k = n = 384
    for gap in (0, 8, 3):
        buffer = torch.randn(m, 2 * k + gap, device="cuda", generator=torch.Generator(device="cuda").manual_seed(m)).bfloat16()
        x, out = buffer[:, :k], buffer[:, k + gap:]
        first, kept = x.clone(), buffer[:, k: k + gap].clone()
        weight = h3b.quantize_fp4(torch.randn(n, k, device="cuda").bfloat16(), "nvfp4")
        want = h3b.fp4_linear(first, weight)
        h3b.fp4_linear(x, weight, out=out)
        assert torch.equal(out, want) and torch.equal(x, first) and torch.equal(buffer[:, k: k + gap], kept)
        residual, norm = torch.randn(m, k, device="cuda").bfloat16(), torch.randn(k, device="cuda").bfloat16()
        total, (q, s) = h3b.add_rms_norm_quantize(first, residual, norm)
        h, (q2, s2) = h3b.add_rms_norm_quantize(x, residual, norm, out=out)
        assert h is out and torch.equal(out, total) and torch.equal(q, q2) and torch.equal(s, s2) and torch.equal(x, first)
        assert torch.equal(buffer[:, k: k + gap], kept)
