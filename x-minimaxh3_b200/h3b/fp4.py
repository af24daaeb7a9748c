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
infinity or a NaN becomes NaN.  Every step of quantize_fp4 is exact or rounded once, so the same
rows give the same codes everywhere.  The norm in front of add_rms_norm_quantize's codes is fp32: the
order in which its squares are added goes by the row's length and address and by the number of rows,
and where their sum is beyond fp32's range, the normed row is 0.
"""

from __future__ import annotations

import ctypes
import math

import torch

from ._lib import Fp4RowsStruct, check, lib
from .cache import _ptr, _stream

FORMATS = {"mxfp4": 1, "nvfp4": 2}
BLOCK = {"mxfp4": 32, "nvfp4": 16}
MAX_ROW = 32768  # columns of a row that is quantised here
_DTYPES = {torch.float16: 1, torch.bfloat16: 2}
_FLOAT_MAX = torch.finfo(torch.float32).max
_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _format(name: str) -> int:
    try:
        return FORMATS[name]
    except KeyError:
        raise ValueError(f"unknown 4-bit format {name!r} (expected one of {sorted(FORMATS)})") from None


def _scale_tiles(rows: int, cols: int, format: str) -> tuple[int, int]:
    group = 4 * BLOCK[format]
    return (rows + 127) // 128, (cols + group - 1) // group


class Fp4Rows:
    """Rows of 4-bit floats (h3b_fp4_rows).

    codes: uint8 [rows, ceil(cols / 32) * 16], two columns to a byte, the even one in the low nibble; zero codes
    behind the last column, and zero scales behind the last block.
    scales: uint8 [ceil(rows / 128), ceil(cols / (4 * block)), 512], block scales in tiles of 128 rows x 4
    blocks, the order in which the products read them (`from_blocks` and `blocks` convert from and to
    [rows, blocks]).  row_scales: f32 [rows], or None for 1; quantize_fp4 makes some for nvfp4."""

    __slots__ = ("rows", "cols", "format", "_gpu", "_ref", "_buffer", "_codes", "_scales", "_row_scales", "_from", "_to")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, cols: int, format: str,
                 row_scales: torch.Tensor | None = None) -> None:
        code = _format(format)
        if not codes.is_cuda:
            raise RuntimeError("Fp4Rows takes only CUDA tensors (the B200 library has no CPU path)")
        gpu = codes.get_device()
        if codes.ndim != 2 or cols < 1:
            raise ValueError("codes must be [rows, bytes] of at least one column")
        rows = codes.shape[0]
        if codes.shape[1] != (cols + 31) // 32 * 16:
            raise ValueError(f"{cols} columns take {(cols + 31) // 32 * 16} bytes of codes per row")
        if scales.shape != (*_scale_tiles(rows, cols, format), 512):
            raise ValueError("scales must be [ceil(rows / 128), ceil(cols / (4 * block)), 512]")
        if not codes.dtype is scales.dtype is torch.uint8 or not (codes.is_contiguous() and scales.is_contiguous()):
            raise ValueError("codes and scales must be contiguous uint8")
        if codes.data_ptr() % 16 or scales.data_ptr() % 16:
            raise ValueError("codes and scales must be 16-byte aligned")
        if row_scales is not None and (row_scales.dtype is not torch.float32 or row_scales.shape != (rows,)
                                       or not row_scales.is_contiguous() or row_scales.get_device() != gpu):
            raise ValueError("row_scales must be a contiguous float32 vector with an entry for each row, on the codes' GPU")
        if scales.get_device() != gpu:
            raise ValueError("codes and scales must be on one GPU")
        self.rows, self.cols, self.format, self._gpu = rows, cols, format, gpu
        self._buffer, self._codes, self._scales, self._row_scales = None, codes, scales, row_scales
        self._ref = ctypes.byref(Fp4RowsStruct(codes.data_ptr(), scales.data_ptr(), _ptr(row_scales), rows, cols, code))
        pieces = self._pieces()
        self._from, self._to = min((p[0] for p in pieces), default=0), max((p[0] + p[2] for p in pieces), default=0)

    @classmethod
    def _room(cls, rows: int, cols: int, format: str, like: torch.Tensor) -> Fp4Rows:
        """Room for rows that a kernel writes, in one buffer on `like`'s GPU: a decoded token's calls are short
        enough for each tensor's making to count, so the parts become tensors where they are asked for."""
        self = object.__new__(cls)
        code = FORMATS[format]
        bands, groups = _scale_tiles(rows, cols, format)
        size = rows * ((cols + 31) // 32 * 16)
        end = size + bands * groups * 512
        whole = end + (4 * rows if code == 2 else 0)
        self._buffer = buffer = like.new_empty(whole, dtype=torch.uint8)
        self._from = at = buffer.data_ptr()
        self._to = at + whole
        self.rows, self.cols, self.format, self._gpu = rows, cols, format, like.get_device()
        self._codes = self._scales = self._row_scales = None
        self._ref = ctypes.byref(Fp4RowsStruct(at, at + size, at + end if code == 2 else None, rows, cols, code))
        return self

    def _pieces(self) -> list[tuple[int, int, int, int]]:
        """The memory it lies in (see _meet), between _from and _to."""
        r = self._ref._obj
        bands, groups = _scale_tiles(self.rows, self.cols, self.format)
        sizes = ((r.codes, self.rows * ((self.cols + 31) // 32 * 16)), (r.scales, bands * groups * 512),
                 (r.row_scales, 4 * self.rows))
        return [(at, 1, size, size) for at, size in sizes if at and size]

    def _parts(self) -> None:
        bands, groups = _scale_tiles(self.rows, self.cols, self.format)
        pitch = (self.cols + 31) // 32 * 16
        size = self.rows * pitch
        end = size + bands * groups * 512
        if self.format == "nvfp4":
            self._row_scales = self._buffer[end:].view(torch.float32)
        self._scales = self._buffer[size:end].view(bands, groups, 512)
        self._codes = self._buffer[:size].view(self.rows, pitch)  # last: another thread takes it as a sign that all are there

    @property
    def codes(self) -> torch.Tensor:
        if self._codes is None:
            self._parts()
        return self._codes

    @property
    def scales(self) -> torch.Tensor:
        if self._codes is None:
            self._parts()
        return self._scales

    @property
    def row_scales(self) -> torch.Tensor | None:
        if self._codes is None:
            self._parts()
        return self._row_scales

    @property
    def device(self) -> torch.device:
        return (self._codes if self._buffer is None else self._buffer).device

    def _new(self, shape: tuple[int, ...], dtype: torch.dtype) -> torch.Tensor:
        return (self._codes if self._buffer is None else self._buffer).new_empty(shape, dtype=dtype)

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
        b = b.view(b.shape[0] // 128, 4, 32, b.shape[1] // 4, 4).permute(0, 3, 2, 1, 4)  # band, group, row % 32, row / 32, block
        return cls(pad(codes, (0, -codes.shape[1] % 16)).contiguous(), b.reshape(b.shape[0], b.shape[1], 512), cols, format,
                   None if row_scales is None else row_scales.to(torch.float32).reshape(-1).contiguous())

    def blocks(self) -> torch.Tensor:
        """The scale bytes as uint8 [rows, ceil(cols / block)]."""
        bands, groups, _ = self.scales.shape
        b = self.scales.view(bands, groups, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(bands * 128, groups * 4)
        return b[: self.rows, : -(-self.cols // BLOCK[self.format])].contiguous()


def _half_rows(x: torch.Tensor, what: str) -> tuple[torch.Tensor, int, int, int]:
    """[..., K] as fp16 / bf16 rows of unit column stride (copied where they do not lie so): the tensor, the number
    of rows, K and the elements between rows (of a single row, whose stride may be anything, its length)."""
    if x.dtype not in _DTYPES:
        raise ValueError(f"{what} must be bfloat16 or float16")
    shape = x.shape
    if not shape or shape[-1] == 0:
        raise ValueError(f"{what} must have at least one column")
    k = shape[-1]
    if x.is_contiguous():
        return x, (shape[0] if len(shape) == 2 else math.prod(shape[:-1])), k, k
    if len(shape) != 2:
        x = x.reshape(math.prod(shape[:-1]), k)
    if k > 1 and x.stride(1) != 1 or x.shape[0] > 1 and x.stride(0) < k:
        x = x.contiguous()
    return x, x.shape[0], k, x.stride(0) if x.shape[0] > 1 else k


def _meet(a: tuple[int, int, int, int], b: tuple[int, int, int, int]) -> bool:
    """Whether two pieces of memory (address, rows, bytes of a row, bytes between rows) share any.  Of pieces that reach
    into each other only those of one step are looked at more closely: their rows may lie beside each other, as
    column ranges of one buffer do."""
    (a_at, a_rows, a_row, a_step), (b_at, b_rows, b_row, b_step) = a, b
    if not (a_rows and a_row and b_rows and b_row):
        return False
    if a_at + (a_rows - 1) * a_step + a_row <= b_at or b_at + (b_rows - 1) * b_step + b_row <= a_at:
        return False
    if a_rows == 1:
        a_step = b_step
    elif b_rows == 1:
        b_step = a_step
    if a_rows == b_rows == 1 or a_step != b_step:
        return True
    beside = (b_at - a_at) % a_step
    return beside < a_row or beside + b_row > a_step


def _refuse_overlap(what: str, piece: tuple[int, int, int, int], quantised, others=()) -> None:
    """Refuses a piece of memory that a call writes and that shares any with what it reads."""
    at, rows, row, step = piece
    end = at + (rows - 1) * step + row
    for q in quantised:
        if at < q._to and q._from < end and any(_meet(piece, p) for p in q._pieces()):
            raise ValueError(f"{what} must not overlap the call's 4-bit rows")
    for p in others:
        if _meet(piece, p):
            raise ValueError(f"{what} must not overlap what the call reads or writes besides")


def _vector(t: torch.Tensor | None) -> tuple[tuple[int, int, int, int], ...]:
    """A contiguous float32 vector as a piece of memory, if there is one."""
    return () if t is None else ((t.data_ptr(), 1, 4 * t.numel(), 0),)


def _gpu_of(x: torch.Tensor, name: str) -> int:
    if not x.is_cuda:
        raise RuntimeError(f"{name} runs only on CUDA tensors (the B200 library has no CPU path)")
    return x.get_device()


def _on(gpu: int, *tensors: torch.Tensor | None) -> None:
    for t in tensors:
        if t is not None and t.get_device() != gpu:
            raise ValueError("all tensors must be on one GPU")


def _row_length(cols: int) -> None:
    if cols > MAX_ROW:
        raise ValueError(f"rows of more than {MAX_ROW} columns are not quantised")


def quantize_fp4(x: torch.Tensor, format: str = "nvfp4") -> Fp4Rows:
    """Rows x [..., K] (bf16 or fp16) to 4-bit floats [M, K]."""
    gpu = _gpu_of(x, "quantize_fp4")
    _format(format)
    x, m, k, step = _half_rows(x, "x")
    _row_length(k)
    out = Fp4Rows._room(m, k, format, x)
    check(lib().h3b_fp4_quantize(x.data_ptr(), _DTYPES[x.dtype], step, out._ref, _stream(gpu)), "fp4_quantize")
    return out


def _check_out(out: torch.Tensor, rows: int, cols: int, dtype: torch.dtype, gpu: int) -> int:
    """The step between the rows of a caller's output."""
    if out.shape != (rows, cols) or out.dtype is not dtype or out.get_device() != gpu:
        raise ValueError(f"out must be {dtype} [{rows}, {cols}] on the operands' GPU")
    if out.is_contiguous():
        return cols
    if cols > 1 and out.stride(1) != 1 or rows > 1 and out.stride(0) < cols:
        raise ValueError("out must have unit column stride and rows apart from each other")
    return out.stride(0) if rows > 1 else cols


def dequantize_fp4(rows: Fp4Rows, dtype: torch.dtype = torch.bfloat16, out: torch.Tensor | None = None) -> torch.Tensor:
    """The values that 4-bit rows stand for, [M, K]."""
    if dtype not in _DTYPES:
        raise ValueError("dequantize_fp4 writes bfloat16 or float16")
    step = rows.cols
    given = out is not None
    if not given:
        out = rows._new((rows.rows, rows.cols), dtype)
    else:
        step = _check_out(out, rows.rows, rows.cols, dtype, rows._gpu)
    stream = _stream(rows._gpu)
    if given:
        _refuse_overlap("out", (out.data_ptr(), rows.rows, 2 * rows.cols, 2 * step), (rows,))
    check(lib().h3b_fp4_dequantize(rows._ref, out.data_ptr(), _DTYPES[dtype], step, stream), "fp4_dequantize")
    return out


def _bias(bias: torch.Tensor | None, n: int, gpu: int) -> torch.Tensor | None:
    if bias is None:
        return None
    if bias.numel() != n:
        raise ValueError("bias does not match the weight's output rows")
    _on(gpu, bias)
    if bias.dtype is torch.float32 and bias.is_contiguous():
        return bias
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
    step = n = weight.rows
    bias = _bias(bias, n, gpu)
    given = out is not None
    if not given:
        out = xq._new((xq.rows, n), out_dtype)
    else:
        step = _check_out(out, xq.rows, n, out_dtype, gpu)
    stream = _stream(gpu)
    if given:
        _refuse_overlap("out", (out.data_ptr(), xq.rows, 2 * n, 2 * step), (xq, weight), _vector(bias))
    check(lib().h3b_fp4_gemm(xq._ref, weight._ref, _ptr(bias), out.data_ptr(), _DTYPES[out_dtype], step, stream), "fp4_gemm")
    return out


def fp4_linear(x: torch.Tensor, weight: Fp4Rows, bias: torch.Tensor | None = None, out: torch.Tensor | None = None,
               workspace: torch.Tensor | None = None) -> torch.Tensor:
    """x [..., K] (bf16 or fp16), quantised to the weight's format, times weight [N, K]^T, + bias -> x's type [..., N].

    out: rows [M, N] that receive the result.  workspace: uint8, reused by calls on one stream.  Neither may share
    memory with the call's other tensors."""
    gpu = _gpu_of(x, "fp4_linear")
    if weight._gpu != gpu:
        raise ValueError("all tensors must be on one GPU")
    shape, k, n = x.shape, weight.cols, weight.rows
    if not shape or shape[-1] != k:
        raise ValueError(f"Input and weight inner dimensions must match, got {shape[-1] if shape else 0} and {k}")
    x, m, k, x_step = _half_rows(x, "x")
    _row_length(k)
    step = n
    bias = _bias(bias, n, gpu)
    given = out is not None
    if given:
        step = _check_out(out, m, n, x.dtype, gpu)
        at, x_at = out.data_ptr(), x.data_ptr()
        if (m and n and at < x_at + 2 * ((m - 1) * x_step + k) and x_at < at + 2 * ((m - 1) * step + n)
                and _meet((at, m, 2 * n, 2 * step), (x_at, m, 2 * k, 2 * x_step))):
            raise ValueError("out must not overlap x")
    else:
        out = x.new_empty((m, n))
    library = lib()
    if given:
        _refuse_overlap("out", (at, m, 2 * n, 2 * step), (weight,), _vector(bias))
    need = library.h3b_fp4_linear_workspace_bytes(m, weight._ref)
    ws_at = None
    if need > 0:  # below 0: sizes that the call refuses
        shared = workspace is not None
        if not shared:
            workspace = x.new_empty(need, dtype=torch.uint8)
        elif (workspace.numel() * workspace.element_size() < need or workspace.get_device() != gpu
              or not workspace.is_contiguous() or workspace.data_ptr() % 16):
            raise ValueError(f"the workspace must have {need} contiguous, 16-byte aligned bytes on the operands' GPU")
        ws_at = workspace.data_ptr()
        if shared:
            _refuse_overlap("the workspace", (ws_at, 1, need, 0), (weight,),
                            ((x.data_ptr(), m, 2 * k, 2 * x_step), (out.data_ptr(), m, 2 * n, 2 * step), *_vector(bias)))
    check(library.h3b_fp4_linear(x.data_ptr(), _DTYPES[x.dtype], m, x_step, weight._ref, _ptr(bias),
                                 out.data_ptr(), step, ws_at, need, _stream(gpu)), "fp4_linear")
    return out if given or len(shape) == 2 else out.view(*shape[:-1], n)


def add_rms_norm_quantize(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor, *, eps: float = 1e-5,
                          to: str = "int8", out: torch.Tensor | None = None):
    """(h, quantised RMSNorm(h) * weight) of h = x + residual; x, residual [..., K], weight [K], one 16-bit type.

    h is rounded to that type, and normed as it is stored, in fp32; `out`, whose rows lie at one step from
    each other, receives it (x or residual themselves may, and no other tensor that overlaps them).  Without
    a residual h is x, and nothing is written to it.  to "int8": (codes int8 [M, K], scales f32 [M, 1] =
    absmax / 127), as ops.int8_linear_prequantized takes them; "mxfp4" or "nvfp4": Fp4Rows, as
    fp4_linear_prequantized does."""
    gpu = _gpu_of(x, "add_rms_norm_quantize")
    int8 = to == "int8"
    if not int8:
        _format(to)
    rows, m, k, step = _half_rows(x, "x")
    _row_length(k)
    dtype = x.dtype
    if weight.dtype is not dtype or weight.ndim != 1 or weight.shape[0] != k:
        raise ValueError("weight must be a vector of x's type with an entry for each column")
    if not 0.0 <= eps <= _FLOAT_MAX:
        raise ValueError("eps must be finite and not negative")
    if weight.get_device() != gpu:
        raise ValueError("all tensors must be on one GPU")
    if not weight.is_contiguous():
        weight = weight.contiguous()
    at, w_at = rows.data_ptr(), weight.data_ptr()
    h, res_at, res_step, sum_at, sum_step = x, None, 0, None, 0
    if residual is not None:
        shape = x.shape
        if residual.shape != shape or residual.dtype is not dtype or residual.get_device() != gpu:
            raise ValueError("residual must have x's shape and type, on its GPU")
        if residual.is_contiguous():
            res, res_step = residual, k
        else:
            res, _, _, res_step = _half_rows(residual, "residual")
        res_at, sum_step = res.data_ptr(), k
        if out is None:
            h = x.new_empty(shape)
            sum_at = h.data_ptr()
        else:
            if out.shape != shape or out.dtype is not dtype or out.get_device() != gpu:
                raise ValueError("out must have x's shape and type, on its GPU")
            h, sum_at = out, out.data_ptr()
            if not out.is_contiguous():
                try:
                    flat = out if len(shape) == 2 else out.view(m, k)
                except RuntimeError:  # a part of a batch's rows, say
                    raise ValueError("out's rows must lie at one step from each other") from None
                sum_step = _check_out(flat, m, k, dtype, gpu)
            end = sum_at + 2 * ((m - 1) * sum_step + k)
            for i, i_rows, i_step in ((at, m, step), (res_at, m, res_step), (w_at, 1, 0)):
                if (i < end and sum_at < i + 2 * ((m - 1) * i_step + k) and (i != sum_at or i_step != sum_step) and m
                        and _meet((sum_at, m, 2 * k, 2 * sum_step), (i, i_rows, 2 * k, 2 * i_step))):
                    raise ValueError("out may be x or residual, and must not overlap them or the weight otherwise")
    elif out is not None:
        raise ValueError("without a residual there is no sum to write")
    args = (at, step, res_at, res_step, sum_at, sum_step, w_at, _DTYPES[dtype])
    if int8:
        q, scales = x.new_empty((m, k), dtype=torch.int8), x.new_empty((m, 1), dtype=torch.float32)
        check(lib().h3b_add_rms_norm_int8(*args, m, k, eps, q.data_ptr(), scales.data_ptr(), _stream(gpu)),
              "add_rms_norm_int8")
        return h, (q, scales)
    quantised = Fp4Rows._room(m, k, to, x)
    check(lib().h3b_add_rms_norm_fp4(*args, eps, quantised._ref, _stream(gpu)), "add_rms_norm_fp4")
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
