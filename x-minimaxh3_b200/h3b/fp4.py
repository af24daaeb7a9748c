"""Microscaled 4-bit floating-point linears over libh3b.so.

Beside the INT8 and W4A8 linears of `ops` and `quantization`, whose 4-bit weights are decoded
to INT8, these keep weight and activations in 4-bit floats for the tensor cores' block-scaled
products (fp16 / bf16 in and out, fp32 sums):

* quantize_fp4, dequantize_fp4   rows to 4-bit floats and back
* fp4_linear                     16-bit rows times a 4-bit weight, one or many rows
* fp4_linear_prequantized        the same for rows that are quantised already
* add_rms_norm_quantize          residual addition, RMSNorm, and an INT8 or 4-bit output: what
                                 stands in front of a linear in a pre-norm layer
* Fp4Linear                      the layer

Elements are E2M1: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign.  Two formats:

    "mxfp4"  blocks of 32 columns; scale 2^(floor(log2(absmax)) - 2), within 2^-127 .. 2^127
    "nvfp4"  blocks of 16 columns; scale e4m3(absmax / 6 / r), with r = 2^e one power of two per
             row, the least (e >= -126) with the row's absmax <= 2688 r

An element is the nearest to x / scale, ties to the even code, and 6 at most.  A block with an
infinity or a NaN becomes NaN.  Every step is exact or rounded once, so the same rows give the
same codes everywhere.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch

from ._lib import Fp4RowsStruct, check, lib
from .cache import _ptr, _stream

FORMATS = {"mxfp4": 1, "nvfp4": 2}
BLOCK = {"mxfp4": 32, "nvfp4": 16}
MAX_ROW = 32768  # columns of a row that is quantised here
_DTYPES = {torch.float16: 1, torch.bfloat16: 2}
_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _format(name: str) -> int:
    try:
        return FORMATS[name]
    except KeyError:
        raise ValueError(f"unknown 4-bit format {name!r} (expected one of {sorted(FORMATS)})") from None


@dataclass
class Fp4Rows:
    """Rows of 4-bit floats (h3b_fp4_rows).  The tensors must not be replaced by others.

    codes: two columns to a byte, the even one in the low nibble; rows end at a multiple of 32 columns.
    scales: block scales in tiles of 128 rows x 4 blocks, the order in which the products read them
    (`from_blocks` and `blocks` convert from and to [rows, blocks])."""

    codes: torch.Tensor              # uint8 [rows, ceil(cols / 32) * 16]
    scales: torch.Tensor             # uint8 [ceil(rows / 128), ceil(cols / (4 * block)), 512]
    cols: int
    format: str
    row_scales: torch.Tensor | None = None  # f32 [rows]; None: 1

    def __post_init__(self) -> None:
        codes, scales, row_scales = self.codes, self.scales, self.row_scales
        code = _format(self.format)
        if not codes.is_cuda:
            raise RuntimeError("Fp4Rows takes only CUDA tensors (the B200 library has no CPU path)")
        self._gpu = gpu = codes.get_device()
        if codes.ndim != 2 or self.cols < 1:
            raise ValueError("codes must be [rows, bytes] of at least one column")
        rows = codes.shape[0]
        group = 4 * BLOCK[self.format]
        if codes.shape[1] != (self.cols + 31) // 32 * 16:
            raise ValueError(f"{self.cols} columns take {(self.cols + 31) // 32 * 16} bytes of codes per row")
        if scales.shape != ((rows + 127) // 128, (self.cols + group - 1) // group, 512):
            raise ValueError("scales must be [ceil(rows / 128), ceil(cols / (4 * block)), 512]")
        if not codes.dtype is scales.dtype is torch.uint8 or not (codes.is_contiguous() and scales.is_contiguous()):
            raise ValueError("codes and scales must be contiguous uint8")
        if row_scales is not None and (row_scales.dtype is not torch.float32 or row_scales.shape != (rows,)
                                       or not row_scales.is_contiguous() or row_scales.get_device() != gpu):
            raise ValueError("row_scales must be a contiguous float32 vector with an entry for each row, on the codes' GPU")
        if scales.get_device() != gpu:
            raise ValueError("codes and scales must be on one GPU")
        self._ref = ctypes.byref(Fp4RowsStruct(codes.data_ptr(), scales.data_ptr(), _ptr(row_scales), rows, self.cols,
                                               code))

    @property
    def rows(self) -> int:
        return self.codes.shape[0]

    @property
    def device(self) -> torch.device:
        return self.codes.device

    @classmethod
    def empty(cls, rows: int, cols: int, format: str, device="cuda", row_scales: bool | None = None) -> Fp4Rows:
        """Room for rows; with row scales by default where the format has them."""
        _format(format)
        group = 4 * BLOCK[format]
        codes = torch.empty((rows, (cols + 31) // 32 * 16), device=device, dtype=torch.uint8)
        scales = torch.empty(((rows + 127) // 128, (cols + group - 1) // group, 512), device=device, dtype=torch.uint8)
        with_rows = format == "nvfp4" if row_scales is None else row_scales
        return cls(codes, scales, cols, format, torch.empty(rows, device=device, dtype=torch.float32) if with_rows else None)

    @classmethod
    def from_blocks(cls, codes: torch.Tensor, block_scales: torch.Tensor, format: str,
                    row_scales: torch.Tensor | None = None) -> Fp4Rows:
        """Rows quantised elsewhere: packed codes [rows, cols / 2] (even column in the low nibble) and one scale
        byte per block, [rows, ceil(cols / block)] (uint8, or the E8M0 / E4M3 type itself)."""
        _format(format)
        if codes.ndim != 2 or codes.dtype is not torch.uint8:
            raise ValueError("codes must be uint8 [rows, cols / 2]")
        rows, cols = codes.shape[0], 2 * codes.shape[1]
        blocks = -(-cols // BLOCK[format])
        if block_scales.shape != (rows, blocks) or block_scales.element_size() != 1:
            raise ValueError(f"block scales must be one byte each, [{rows}, {blocks}]")
        if block_scales.device != codes.device:
            raise ValueError("codes and scales must be on one GPU")
        pad = torch.nn.functional.pad
        b = pad(block_scales.contiguous().view(torch.uint8), (0, -blocks % 4, 0, -rows % 128))
        b = b.view(b.shape[0] // 128, 4, 32, -1, 4).permute(0, 3, 2, 1, 4)  # band, group, row % 32, row / 32, block
        return cls(pad(codes, (0, -codes.shape[1] % 16)).contiguous(), b.reshape(b.shape[0], b.shape[1], 512), cols, format,
                   None if row_scales is None else row_scales.to(torch.float32).reshape(-1).contiguous())

    def blocks(self) -> torch.Tensor:
        """The scale bytes as uint8 [rows, ceil(cols / block)]."""
        bands, groups, _ = self.scales.shape
        b = self.scales.view(bands, groups, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(bands * 128, groups * 4)
        return b[: self.rows, : -(-self.cols // BLOCK[self.format])].contiguous()


def _half_rows(x: torch.Tensor, what: str) -> torch.Tensor:
    """[..., K] as fp16 / bf16 rows [M, K] of unit column stride; copied where they do not lie so."""
    if x.dtype not in _DTYPES:
        raise ValueError(f"{what} must be bfloat16 or float16")
    if x.ndim == 0 or x.shape[-1] == 0:
        raise ValueError(f"{what} must have at least one column")
    if x.ndim != 2:
        x = x.reshape(x.numel() // x.shape[-1], x.shape[-1])
    if x.shape[1] > 1 and x.stride(1) != 1 or x.shape[0] > 1 and x.stride(0) < x.shape[1]:
        x = x.contiguous()
    return x


def _row_step(x: torch.Tensor) -> int:
    """Elements between x's rows (of a single row, whose stride may be anything, its length)."""
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def _cuda(name: str, *tensors: torch.Tensor | None) -> int:
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise RuntimeError(f"{name} runs only on CUDA tensors (the B200 library has no CPU path)")
    gpu = tensors[0].get_device()
    for t in tensors[1:]:
        if t is not None and t.get_device() != gpu:
            raise ValueError("all tensors must be on one GPU")
    return gpu


def _row_length(cols: int) -> None:
    if cols > MAX_ROW:
        raise ValueError(f"rows of more than {MAX_ROW} columns are not quantised")


def quantize_fp4(x: torch.Tensor, format: str = "nvfp4") -> Fp4Rows:
    """Rows x [..., K] (bf16 or fp16) to 4-bit floats [M, K]."""
    gpu = _cuda("quantize_fp4", x)
    _format(format)
    x = _half_rows(x, "x")
    _row_length(x.shape[1])
    out = Fp4Rows.empty(x.shape[0], x.shape[1], format, x.device)
    check(lib().h3b_fp4_quantize(_ptr(x), _DTYPES[x.dtype], _row_step(x), out._ref, _stream(gpu)), "fp4_quantize")
    return out


def _rows_out(out: torch.Tensor | None, like: torch.Tensor, rows: int, cols: int, dtype: torch.dtype) -> torch.Tensor:
    if out is None:
        return torch.empty((rows, cols), device=like.device, dtype=dtype)
    if out.shape != (rows, cols) or out.dtype is not dtype or out.get_device() != like.get_device():
        raise ValueError(f"out must be {dtype} [{rows}, {cols}] on the operands' GPU")
    if cols > 1 and out.stride(1) != 1 or rows > 1 and out.stride(0) < cols:
        raise ValueError("out must have unit column stride and rows apart from each other")
    return out


def dequantize_fp4(rows: Fp4Rows, dtype: torch.dtype = torch.bfloat16, out: torch.Tensor | None = None) -> torch.Tensor:
    """The values that 4-bit rows stand for, [M, K]."""
    if dtype not in _DTYPES:
        raise ValueError("dequantize_fp4 writes bfloat16 or float16")
    out = _rows_out(out, rows.codes, rows.rows, rows.cols, dtype)
    check(lib().h3b_fp4_dequantize(rows._ref, _ptr(out), _DTYPES[dtype], _row_step(out), _stream(rows._gpu)),
          "fp4_dequantize")
    return out


def _bias(bias: torch.Tensor | None, n: int, gpu: int) -> torch.Tensor | None:
    if bias is None:
        return None
    if bias.numel() != n:
        raise ValueError("bias does not match the weight's output rows")
    if bias.get_device() != gpu:
        raise ValueError("all tensors must be on one GPU")
    return bias.to(torch.float32).reshape(-1).contiguous()


def fp4_linear_prequantized(xq: Fp4Rows, weight: Fp4Rows, bias: torch.Tensor | None = None,
                            out_dtype: torch.dtype = torch.bfloat16, out: torch.Tensor | None = None) -> torch.Tensor:
    """xq [M, K] . weight [N, K]^T + bias -> bf16 or fp16 [M, N], for rows of one format; bias is added in fp32."""
    gpu = xq._gpu
    if weight._gpu != gpu:
        raise ValueError("all tensors must be on one GPU")
    if xq.format != weight.format:
        raise ValueError(f"{xq.format} rows do not go with a {weight.format} weight")
    if xq.cols != weight.cols:
        raise ValueError(f"Input and weight inner dimensions must match, got {xq.cols} and {weight.cols}")
    if out_dtype not in _DTYPES:
        raise ValueError("fp4_linear writes bfloat16 or float16")
    bias = _bias(bias, weight.rows, gpu)
    out = _rows_out(out, xq.codes, xq.rows, weight.rows, out_dtype)
    check(lib().h3b_fp4_gemm(xq._ref, weight._ref, _ptr(bias), _ptr(out), _DTYPES[out_dtype], _row_step(out),
                             _stream(gpu)), "fp4_gemm")
    return out


def fp4_linear(x: torch.Tensor, weight: Fp4Rows, bias: torch.Tensor | None = None, out: torch.Tensor | None = None,
               workspace: torch.Tensor | None = None) -> torch.Tensor:
    """x [..., K] (bf16 or fp16), quantised to the weight's format, times weight [N, K]^T, + bias -> x's type [..., N].

    out: rows [M, N] that receive the result.  workspace: uint8, reused by calls on one stream."""
    gpu = _cuda("fp4_linear", x)
    if weight._gpu != gpu:
        raise ValueError("all tensors must be on one GPU")
    if x.ndim == 0 or x.shape[-1] != weight.cols:
        raise ValueError(f"Input and weight inner dimensions must match, got {x.shape[-1] if x.ndim else 0} and "
                         f"{weight.cols}")
    lead = x.shape[:-1]
    x = _half_rows(x, "x")
    _row_length(weight.cols)
    m = x.shape[0]
    bias = _bias(bias, weight.rows, gpu)
    given = out is not None
    out = _rows_out(out, x, m, weight.rows, x.dtype)
    need = lib().h3b_fp4_linear_workspace_bytes(m, weight.cols, FORMATS[weight.format])
    if workspace is None:
        workspace = torch.empty(need, device=x.device, dtype=torch.uint8)
    elif (workspace.numel() * workspace.element_size() < need or workspace.get_device() != gpu
          or not workspace.is_contiguous() or workspace.data_ptr() % 16):
        raise ValueError(f"the workspace must have {need} contiguous, 16-byte aligned bytes on the operands' GPU")
    check(lib().h3b_fp4_linear(_ptr(x), _DTYPES[x.dtype], m, _row_step(x), weight._ref, _ptr(bias), _ptr(out),
                               _row_step(out), _ptr(workspace), need, _stream(gpu)), "fp4_linear")
    return out if given or len(lead) == 1 else out.view(*lead, weight.rows)


def add_rms_norm_quantize(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor, *, eps: float = 1e-5,
                          to: str = "int8", out: torch.Tensor | None = None):
    """(h, quantised RMSNorm(h) * weight) of h = x + residual; x, residual [..., K], weight [K], one 16-bit type.

    h is rounded to that type, and normed as it is stored, in fp32; `out` receives it (x or residual
    themselves may, and no other tensor that overlaps them).  Without a residual h is x, and nothing is
    written to it.  to "int8": (codes int8 [M, K], scales f32 [M, 1] = absmax / 127), as
    ops.int8_linear_prequantized takes them; "mxfp4" or "nvfp4": Fp4Rows, as fp4_linear_prequantized does."""
    gpu = _cuda("add_rms_norm_quantize", x, residual, weight, out)
    if to != "int8":
        _format(to)
    shape = x.shape
    if weight.dtype is not x.dtype or weight.ndim != 1 or x.ndim == 0 or weight.shape[0] != shape[-1]:
        raise ValueError("weight must be a vector of x's type with an entry for each column")
    if not 0.0 <= eps <= torch.finfo(torch.float32).max:
        raise ValueError("eps must be finite and not negative")
    if residual is None and out is not None:
        raise ValueError("without a residual there is no sum to write")
    rows = _half_rows(x, "x")
    m, k = rows.shape
    _row_length(k)
    weight = weight.contiguous()
    res = None
    h = x
    if residual is not None:
        if residual.shape != shape or residual.dtype is not x.dtype:
            raise ValueError("residual must have x's shape and type")
        res = _half_rows(residual, "residual")
        if out is None:
            out = torch.empty(shape, device=x.device, dtype=x.dtype)
        elif out.shape != shape or out.dtype is not x.dtype:
            raise ValueError("out must have x's shape and type")
        h, out = out, out.view(m, k)  # refused by view() where the rows do not lie in one step
        if k > 1 and out.stride(1) != 1 or m > 1 and out.stride(0) < k:
            raise ValueError("out must have unit column stride and rows apart from each other")
    args = (_ptr(rows), _row_step(rows), _ptr(res), 0 if res is None else _row_step(res), _ptr(out),
            0 if out is None else _row_step(out), _ptr(weight), _DTYPES[x.dtype])
    if to == "int8":
        q = torch.empty((m, k), device=x.device, dtype=torch.int8)
        scales = torch.empty((m, 1), device=x.device, dtype=torch.float32)
        check(lib().h3b_add_rms_norm_int8(*args, m, k, float(eps), _ptr(q), _ptr(scales), _stream(gpu)),
              "add_rms_norm_int8")
        return h, (q, scales)
    quantised = Fp4Rows.empty(m, k, to, x.device)
    check(lib().h3b_add_rms_norm_fp4(*args, float(eps), quantised._ref, _stream(gpu)), "add_rms_norm_fp4")
    return h, quantised


class Fp4Linear:
    """A linear layer with a 4-bit weight and activations; bias [N] optional."""

    def __init__(self, weight: Fp4Rows, bias: torch.Tensor | None = None) -> None:
        self.weight = weight
        self.bias = _bias(bias, weight.rows, weight._gpu)

    @classmethod
    def from_weight(cls, weight: torch.Tensor, bias: torch.Tensor | None = None, format: str = "nvfp4") -> Fp4Linear:
        """From a 16-bit weight [N, K], quantised here."""
        if weight.ndim != 2:
            raise ValueError("weight must be [out_features, in_features]")
        return cls(quantize_fp4(weight, format), bias)

    @property
    def in_features(self) -> int:
        return self.weight.cols

    @property
    def out_features(self) -> int:
        return self.weight.rows

    def quantize(self, x: torch.Tensor) -> Fp4Rows:
        """x's rows in this layer's format."""
        return quantize_fp4(x, self.weight.format)

    def forward_prequantized(self, xq: Fp4Rows, out_dtype: torch.dtype = torch.bfloat16,
                             out: torch.Tensor | None = None) -> torch.Tensor:
        return fp4_linear_prequantized(xq, self.weight, self.bias, out_dtype, out)

    def dense_weight(self) -> torch.Tensor:
        """fp32 [N, K] weight the layer applies."""
        w = self.weight
        codes = torch.stack((w.codes & 15, w.codes >> 4), -1).flatten(1)[:, : w.cols].long()
        values = torch.tensor(_VALUES + tuple(-v for v in _VALUES), device=w.device)[codes]
        scale_type = torch.float8_e8m0fnu if w.format == "mxfp4" else torch.float8_e4m3fn
        scales = w.blocks().view(scale_type).float().repeat_interleave(BLOCK[w.format], 1)[:, : w.cols]
        return values * scales * (1.0 if w.row_scales is None else w.row_scales[:, None])

    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        return fp4_linear(x, self.weight, self.bias)
