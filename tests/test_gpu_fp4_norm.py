"""Residual addition + RMSNorm into INT8 and 4-bit rows, and the 4-bit operators run together (B200)."""

import pytest
import torch

import fp4_util as U

pytestmark = pytest.mark.gpu

HALVES = (torch.bfloat16, torch.float16)
SHAPES = [(1, 1), (2, 15), (3, 16), (9, 33), (130, 64), (5, 1000), (9, 1024), (17, 1056), (3, 4096), (2, 4100), (2, 8200),
          (3, 16384), (2, 16385), (2, 32768), (1, 32767)]


@pytest.fixture(scope="module")
def h3b():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    import h3b
    h3b.lib()
    yield h3b
    torch.cuda.synchronize()
    assert h3b.device_status(0) == 0


def _inputs(m, k, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed * 1000 + m * 7 + k)
    x = torch.randn(m, k, device="cuda", generator=g) * torch.exp(torch.randn(m, 1, device="cuda", generator=g))
    r = 3 * torch.randn(m, k, device="cuda", generator=g)
    w = 1 + 0.3 * torch.randn(k, device="cuda", generator=g)
    return x.to(dtype), r.to(dtype), w.to(dtype)


def _normed(h, w, eps):
    """RMSNorm(h) * w in fp64, and a bound on the relative error of a kernel's fp32 value, in units of 2^-24: a
    thread's squares are added one after the other, at most 64 of them, then in a tree of 10 levels (half of a sum's
    error is left after the root); quotient, sum and products are off by one unit at most, and a root and reciprocal of
    two units of 2^-23 take up what threads of fewer squares leave (the longest chain is 33)."""
    h = h.double()
    y = h / torch.sqrt((h * h).mean(1, keepdim=True) + eps) * w.double()
    return y, ((64 + 10 + 2) / 2 + 6) * 2.0 ** -24


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("m,k", SHAPES)
def test_sum_norm_and_int8_rows(h3b, dtype, m, k):
    x, r, w = _inputs(m, k, dtype)
    h, (q, s) = h3b.add_rms_norm_quantize(x, r, w, eps=1e-5)
    assert torch.equal(h, (x.float() + r.float()).to(dtype)) and h.shape == x.shape
    y, off = _normed(h, w, 1e-5)
    assert q.shape == (m, k) and s.shape == (m, 1)
    top = y.abs().amax(1, keepdim=True)
    assert ((s.double() * 127 - top).abs() <= (off + 2.0 ** -23) * top).all()
    # a code is the nearest to y / s: off by at most a half and what 127 steps off by `off` come to
    assert ((q.double() - y / s.double()).abs() <= 0.5 + 127 * (off + 2.0 ** -23)).all()


def _near_border(ratio, borders, off):
    near = torch.zeros(ratio.shape, dtype=torch.bool, device=ratio.device)
    for b in borders:
        near |= (ratio - b).abs() <= 2 * off * b
    return near


@pytest.mark.parametrize("fmt", ("mxfp4", "nvfp4"))
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("m,k", SHAPES)
def test_sum_norm_and_4_bit_rows(h3b, fmt, dtype, m, k):
    """Scales and codes are those of the exact norm, but where a value lies so near a border between two codes that
    fp32 cannot tell; with this few values hardly any does."""
    x, r, w = _inputs(m, k, dtype, seed=1)
    h, q = h3b.add_rms_norm_quantize(x, r, w, eps=1e-6, to=fmt)
    assert torch.equal(h, (x.float() + r.float()).to(dtype))
    y, off = _normed(h, w, 1e-6)
    code, byte, e = U.quantize(y, fmt)
    b = U.BLOCK[fmt]
    blocks = torch.nn.functional.pad(y.abs(), (0, -k % b)).view(m, -1, b)
    top = blocks.amax(-1)
    if fmt == "nvfp4":
        row = top.amax(-1)
        sure = (torch.frexp(row / 2688).mantissa - 0.5).abs() > 2 * off
        sure &= (torch.frexp(row / 2688).mantissa - 1.0).abs() > 2 * off
        assert torch.equal(q.row_scales[sure].double(), torch.exp2(e.double())[sure])
        t = top / q.row_scales.double()[:, None] / 6
        step = torch.exp2(torch.floor(torch.log2(t.clamp_min(2.0 ** -6))) - 3)
        sure = sure[:, None] & ((t / step - torch.floor(t / step) - 0.5).abs() * step > 4 * off * t)
    else:
        sure = ((torch.frexp(top).mantissa - 0.5).abs() > 2 * off) & ((torch.frexp(top).mantissa - 1.0).abs() > 2 * off)
    assert torch.equal(q.blocks()[sure].to(torch.int64), byte[sure])
    assert (~sure).sum() <= 2 + sure.numel() // 1000
    scale = U.scale_values(q.blocks(), fmt)
    if fmt == "nvfp4":
        scale = scale * q.row_scales.double()[:, None]
    ratio = blocks / torch.where(scale > 0, scale, 1.0)[..., None]
    near = _near_border(ratio, (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0), off)
    settled = sure[..., None] & ~near
    got = torch.nn.functional.pad(U.codes_of(q)[:, :k], (0, -k % b)).view(m, -1, b)
    sign = code >= 8
    assert torch.equal((got & 7)[settled], (code & 7)[settled])
    assert torch.equal((got >= 8)[settled & (code & 7 > 0)], sign[settled & (code & 7 > 0)])
    assert not U.codes_of(q)[:, k:].any()


@pytest.mark.parametrize("to", ("int8", "mxfp4", "nvfp4"))
def test_without_a_residual_and_with_the_sum_in_place(h3b, to):
    def parts(q):
        return list(q) if to == "int8" else [q.codes, q.blocks()] + ([q.row_scales] if to == "nvfp4" else [])

    for k in (96, 4096, 4100):
        x, r, w = _inputs(40, k, torch.bfloat16, seed=2)
        total, want = h3b.add_rms_norm_quantize(x, r, w, to=to)
        h, got = h3b.add_rms_norm_quantize(total, None, w, to=to)
        assert h is total and all(torch.equal(a, b) for a, b in zip(parts(got), parts(want)))
        for i in range(2):  # into the residual, into x
            a, b = x.clone(), r.clone()
            out = (b, a)[i]
            h, got = h3b.add_rms_norm_quantize(a, b, w, to=to, out=out)
            assert h is out and torch.equal(out, total)
            assert all(torch.equal(p, s) for p, s in zip(parts(got), parts(want)))
            assert torch.equal((a, b)[i], (x, r)[i])
        room = torch.full((42, k + 16), 5.0, device="cuda", dtype=torch.bfloat16)
        h, got = h3b.add_rms_norm_quantize(x.view(8, 5, k), r.view(8, 5, k), w, to=to)
        assert torch.equal(h, total.view(8, 5, k)) and all(torch.equal(p, s) for p, s in zip(parts(got), parts(want)))
        h, got = h3b.add_rms_norm_quantize(x, r, w, to=to, out=room[1:-1, 3: 3 + k])
        assert torch.equal(h, total) and all(torch.equal(p, s) for p, s in zip(parts(got), parts(want)))
        room[1:-1, 3: 3 + k] = 5.0
        assert (room == 5.0).all()


def test_rows_of_zeros_and_of_no_number(h3b):
    x, r, w = _inputs(6, 128, torch.float16, seed=3)
    x[0], r[0] = 0, 0
    x[1, 7] = float("nan")
    x[2, 9] = float("inf")
    x[3, 5], r[3, 5] = 60000, 60000  # the fp16 sum is infinite
    h, (q, s) = h3b.add_rms_norm_quantize(x, r, w)
    assert s[0] == 0 and not q[0].any()
    assert not torch.isfinite(s[1:4]).any() and torch.isfinite(s[4:]).all()
    for fmt in ("mxfp4", "nvfp4"):
        _, z = h3b.add_rms_norm_quantize(x, r, w, to=fmt)
        v = h3b.dequantize_fp4(z)
        assert not v[0].any() and torch.isnan(v[1]).all() and torch.isfinite(v[4:]).all()
        assert torch.isnan(v[2]).any() and torch.isnan(v[3]).any()
    empty = h3b.add_rms_norm_quantize(x[:0], r[:0], w)
    assert empty[0].shape == (0, 128) and empty[1][0].shape == (0, 128)


def test_refusals(h3b):
    x, r, w = _inputs(4, 64, torch.bfloat16)
    both = torch.zeros(5, 64, device="cuda", dtype=torch.bfloat16)
    for call in (lambda: h3b.add_rms_norm_quantize(x, r, w, to="int4"),
                 lambda: h3b.add_rms_norm_quantize(x, r[:3], w),
                 lambda: h3b.add_rms_norm_quantize(x, r.half(), w),
                 lambda: h3b.add_rms_norm_quantize(x, r, w.float()),
                 lambda: h3b.add_rms_norm_quantize(x, r, w[:32]),
                 lambda: h3b.add_rms_norm_quantize(x.float(), r.float(), w.float()),
                 lambda: h3b.add_rms_norm_quantize(x, r, w, eps=-1e-6),
                 lambda: h3b.add_rms_norm_quantize(x, r, w, eps=float("nan")),
                 lambda: h3b.add_rms_norm_quantize(x, None, w, out=r),
                 lambda: h3b.add_rms_norm_quantize(x, r, w, out=r[:, :32]),
                 lambda: h3b.add_rms_norm_quantize(both[:4], r, w, out=both[1:]),
                 lambda: h3b.add_rms_norm_quantize(x, both[:4], w, out=both[1:]),
                 lambda: h3b.add_rms_norm_quantize(x, r, w, out=torch.empty(64, 4, device="cuda", dtype=torch.bfloat16).T)):
        with pytest.raises(ValueError):
            call()


# ------------------------------------------------------------------------------------ together


def _layer(h3b, x, residual, norms, up, down, weight8, scale8):
    """A pre-norm step in 4 bits, then a projection in INT8."""
    h, q = h3b.add_rms_norm_quantize(x, residual, norms[0], to="nvfp4")
    y = up.forward_prequantized(q)
    h, q = h3b.add_rms_norm_quantize(down(torch.nn.functional.silu(y)), h, norms[1], to="int8")
    return h, h3b.ops.int8_linear_prequantized(*q, weight8, scale8)


@pytest.mark.parametrize("m", [1, 19, 700])
def test_operators_run_together_eagerly_and_from_a_graph(h3b, m):
    k, n = 512, 1024
    g = torch.Generator(device="cuda").manual_seed(m)
    draw = lambda *s: torch.randn(*s, device="cuda", generator=g)
    norms = [(1 + 0.1 * draw(k)).bfloat16() for _ in range(2)]
    up = h3b.Fp4Linear.from_weight((draw(n, k) / k ** 0.5).bfloat16(), draw(n), "nvfp4")
    down = h3b.Fp4Linear.from_weight((draw(k, n) / n ** 0.5).bfloat16(), None, "mxfp4")
    weight8 = torch.randint(-127, 128, (256, k), device="cuda", generator=g, dtype=torch.int16).to(torch.int8)
    scale8 = torch.rand(256, device="cuda", generator=g) * 1e-2
    x, r = draw(m, k).bfloat16(), draw(m, k).bfloat16()
    args = (norms, up, down, weight8, scale8)

    # step by step in fp64 from what each operator was given
    h, q = h3b.add_rms_norm_quantize(x, r, norms[0], to="nvfp4")
    y = up.forward_prequantized(q)
    U.assert_product(y, *U.product(q, up.weight, up.bias))
    t = torch.nn.functional.silu(y)
    z = down(t)
    U.assert_product(z, *U.product(down.quantize(t), down.weight))
    h2, (q8, s8) = h3b.add_rms_norm_quantize(z, h, norms[1], to="int8")
    want = (q8.double() @ weight8.double().T) * s8.double() * scale8.double()
    eager = _layer(h3b, x, r, *args)
    assert torch.equal(eager[0], h2)
    # int8 sums are exact; two products and the output's rounding
    assert ((eager[1].double() - want).abs() <= (2.0 ** -8 + 2.0 ** -22) * want.abs() + 1e-30).all()

    graph = torch.cuda.CUDAGraph()
    xs, rs = x.clone(), r.clone()
    with torch.cuda.graph(graph):
        captured = _layer(h3b, xs, rs, *args)
    for seed in range(3):
        g2 = torch.Generator(device="cuda").manual_seed(100 + seed)
        xs.copy_(torch.randn(m, k, device="cuda", generator=g2))
        rs.copy_(torch.randn(m, k, device="cuda", generator=g2))
        want = _layer(h3b, xs, rs, *args)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, want))


def test_launches_are_counted(h3b):
    from h3b._lib import launch_count, reset_launch_count
    x, r, w = _inputs(3, 256, torch.bfloat16)
    layer = h3b.Fp4Linear.from_weight(x.repeat(40, 1))
    reset_launch_count()
    layer(x)
    assert launch_count() == 1  # few rows are quantised by the product
    h3b.add_rms_norm_quantize(x, r, w)
    assert launch_count() == 2
    layer.forward_prequantized(layer.quantize(x))
    assert launch_count() == 4
    layer(x.repeat(40, 1))
    assert launch_count() == 6
