"""64-bit forms of the 4-bit floating-point operators, for their tests."""

import torch

BLOCK = {"mxfp4": 32, "nvfp4": 16}
ELEMENTS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # largest relative rounding error
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}  # and the largest among subnormal numbers


def scale_values(byte, fmt):
    """What scale bytes stand for, in fp64."""
    b = byte.to(torch.int64)
    if fmt == "mxfp4":
        v = torch.exp2(b.double() - 127)
        return torch.where(b == 255, float("nan"), v)
    e, m = b >> 3, (b & 7).double()
    v = torch.where(e == 0, m / 8 * 2.0 ** -6, (1 + m / 8) * torch.exp2(e.double() - 7))
    return torch.where(b == 127, float("nan"), v)


def nearest_element(x, scale):
    """Codes (without sign) of the elements nearest to |x| / scale, ties to the even code: |x| is compared with
    the borders between neighbours times the scale, which is exact in fp64."""
    a = x.abs()
    code = torch.zeros(a.shape, dtype=torch.int64, device=x.device)
    for i in range(7):
        border = (ELEMENTS[i] + ELEMENTS[i + 1]).item() / 2 * scale
        code += (a >= border) if i % 2 else (a > border)
    return torch.where(scale > 0, code, 0)


def nearest_e4m3(t):
    """Bytes of the E4M3 values nearest to t >= 0 (at most 448), ties to the even code."""
    t = t.clamp_max(448.0)
    step = torch.exp2(torch.floor(torch.log2(t.clamp_min(2.0 ** -6))) - 3)
    v = torch.round(t / step) * step
    e = torch.floor(torch.log2(v.clamp_min(2.0 ** -6)))
    return torch.where(v < 2.0 ** -6, v * 2.0 ** 9, (e + 7) * 8 + (v / torch.exp2(e) - 1) * 8).to(torch.int64)


def row_exponent(top):
    """Least e >= -126 with top <= 2688 * 2^e, 0 for top = 0."""
    e = torch.full(top.shape, -126, dtype=torch.int64, device=top.device)
    for bit in (128, 64, 32, 16, 8, 4, 2, 1):
        fits = top <= 2688.0 * torch.exp2((e + bit - 1).double())
        e = torch.where(fits, e, e + bit)
    return torch.where(top > 0, e, 0)


def quantize(x, fmt):
    """(codes with the sign in bit 3 [rows, blocks, block], scale bytes [rows, blocks], row exponents [rows]) of
    fp64 rows."""
    m, k = x.shape
    b = BLOCK[fmt]
    x = torch.nn.functional.pad(x, (0, -k % b)).view(m, -1, b)
    lost = ~torch.isfinite(x).all(-1)
    x = torch.where(lost[..., None], 0.0, x)
    top = x.abs().amax(-1)
    if fmt == "mxfp4":
        e = torch.frexp(top).exponent.to(torch.int64) - 3
        byte = torch.where(top > 0, e, -127).clamp_min(-127) + 127
        r = torch.zeros(m, dtype=torch.int64, device=x.device)
    else:
        r = row_exponent(top.amax(-1))
        byte = nearest_e4m3(top * torch.exp2(-r[:, None].double()) / 6)
        x = x * torch.exp2(-r[:, None, None].double())
    code = nearest_element(x, scale_values(byte, fmt)[..., None])
    code = torch.where(torch.signbit(x), code + 8, code)
    byte = torch.where(lost, 255 if fmt == "mxfp4" else 127, byte)
    return torch.where(lost[..., None], 0, code), byte, r


def codes_of(rows):
    """The codes of Fp4Rows as [rows, all columns with the padding]."""
    c = rows.codes.to(torch.int64)
    return torch.stack((c & 15, c >> 4), -1).flatten(1)


def values(rows):
    """What Fp4Rows stand for, in fp64, [rows, cols]."""
    c = codes_of(rows)[:, : rows.cols]
    v = ELEMENTS.to(c.device)[c & 7]
    v = torch.where(c >= 8, -v, v)
    v = v * scale_values(rows.blocks(), rows.format).repeat_interleave(BLOCK[rows.format], 1)[:, : rows.cols]
    return v if rows.row_scales is None else v * rows.row_scales.double()[:, None]


def product(x, w, bias=None):
    """(out, bound) of Fp4Rows in fp64.  The bound on a kernel's error before its output is rounded: products of
    4-bit elements and their scales are exact or, with fp32 partial sums, off by 2^-23 of the sum of magnitudes per
    addition (a tensor core may cut instead of rounding); there are at most K additions, two row scales and a bias."""
    a, b = values(x), values(w)
    out, size = a @ b.T, a.abs() @ b.abs().T
    bound = (x.cols + 4) * 2.0 ** -23 * size
    if bias is not None:
        out = out + bias.double()
        bound = bound + 2.0 ** -23 * (size + bias.double().abs())
    return out, bound


def assert_product(got, want, bound):
    limit = bound + UNIT[got.dtype] * (want.abs() + bound) + TINY[got.dtype]
    off = (got.double() - want).abs()
    worst = (off - limit).max().item() if off.numel() else 0.0
    assert not off.isnan().any() and worst <= 0, worst


def random_rows(h3b, rows, cols, fmt, seed, scales=(126, 127, 128), row_scales=False):
    """Fp4Rows of arbitrary codes and a few block scales (bytes of E8M0; for nvfp4 the same powers of two), so that
    sums of products are exact in fp32."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.randint(0, 256, (rows, (cols + 1) // 2), device="cuda", dtype=torch.uint8, generator=g)
    if cols % 2:
        codes[:, -1] &= 15
    blocks = -(-cols // BLOCK[fmt])
    s = torch.tensor(scales, device="cuda")[torch.randint(0, len(scales), (rows, blocks), device="cuda", generator=g)]
    if fmt == "nvfp4":
        s = (s - 127 + 7) * 8  # 2^e in E4M3
    r = None
    if row_scales:
        r = torch.exp2(torch.randint(-3, 4, (rows,), device="cuda", generator=g).float())
    out = h3b.Fp4Rows.from_blocks(codes, s.to(torch.uint8), fmt, r)
    return out if cols % 2 == 0 else h3b.Fp4Rows(out.codes, out.scales, cols, fmt, out.row_scales)
