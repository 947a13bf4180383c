"""The 8-bit linear path: rows of int8 codes with a scale each (tokens of an activation, output channels of a weight),
the RMSNorm that writes them together with the residual stream, and the matrix product of two of them.

``MambaLM.quantize_linears`` runs a model's in_proj and out_proj through these; each can be called by itself.  Tensors are
on CUDA, in float32, bfloat16 or float16, rows may be strided (``xz[:, :es]``); leading dimensions that do not lie on one
stride are copied.  Calls run on the current stream of their tensors' device, allocate through torch only and keep nothing,
so they can be captured in a CUDA graph.  No gradient: call them under ``torch.no_grad()``.  The reference has no 8-bit
linear layer; the nearest is the quantiser of its int8 collective (``mamba_lite/tp_utils.py:103-131``)."""
from __future__ import annotations

from typing import NamedTuple

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from . import _lib as L
from .logprobs import _call, _refuse_tangent

__all__ = ["MAX_COLS", "Int8Rows", "quantize_rows", "dequantize_rows", "rms_norm_int8", "add_rms_norm_int8", "int8_linear"]

MAX_COLS = 131071  # of a row: sums of int8 products stay within int32
MAX_ROWS = (1 << 31) - 1


class Int8Rows(NamedTuple):
    """Rows that stand for ``codes * scale[..., None]``: codes [..., C] int8, scale [...] float32."""
    codes: torch.Tensor
    scale: torch.Tensor


# ------------------------------------------------------------------ arguments
# A call's time on the host is most of a decode step's small calls, so the common arguments (two dimensions, dense rows) are
# taken after one row of tests, and everything else, refusals among it, by the functions that name what is wrong.
def _refuse_grad(what: str, *tensors) -> None:
    grad = torch.is_grad_enabled()
    dual = forward_ad._current_level >= 0
    if not (grad or dual):
        return
    for t in tensors:
        if t is None:
            continue
        if grad and t.requires_grad:
            raise RuntimeError(f"{what} has no gradient; call it under torch.no_grad()")
        if dual:
            _refuse_tangent(t, what)


def _check_shape(x: torch.Tensor, what: str, name: str) -> None:
    L.require_cuda(x, what)
    shape = x.shape
    if not shape or not 1 <= shape[-1] <= MAX_COLS:
        raise ValueError(f"{what}: {name} needs a last dimension of 1 to {MAX_COLS}, got shape {tuple(shape)}")
    if x.numel() > MAX_ROWS * shape[-1]:
        raise ValueError(f"{what}: {name} has more than {MAX_ROWS} rows")


def _same_device(t: torch.Tensor, x: torch.Tensor, what: str, name: str) -> None:
    if t.device != x.device:
        raise ValueError(f"{what}: {name} is on {t.device}, expected {x.device}")


def _as_rows(x: torch.Tensor, what: str, name: str):
    """(x as [rows, C] with dense rows, rows, C, the stride between rows); copied where the leading dimensions have no common
    stride."""
    if x.dim() == 2 and x.is_cuda:
        (rows, c), (ld, step) = x.shape, x.stride()
        if step == 1 and 1 <= c <= MAX_COLS and 1 < rows <= MAX_ROWS and ld >= c:
            return x, rows, c, ld
        if rows == 1 and step == 1 and 1 <= c <= MAX_COLS:
            return x, 1, c, c
    _check_shape(x, what, name)
    c = x.shape[-1]
    if x.dim() != 2:
        x = x.reshape(-1, c)
    rows, (ld, step) = x.shape[0], x.stride()
    if (step != 1 and c > 1) or (rows > 1 and ld < c):
        x, ld = x.contiguous(), c
    return x, rows, c, (ld if rows > 1 else c)


def _as_codes(r: Int8Rows, what: str, name: str):
    """``_as_rows`` of the codes, with their scales in one dimension."""
    codes, scale = r
    if codes.dtype != torch.int8 or scale.dtype != torch.float32:
        raise TypeError(f"{what}: {name} needs int8 codes and float32 scales, got {codes.dtype} and {scale.dtype}")
    rows2 = _as_rows(codes, what, name)
    if scale.shape != codes.shape[:-1]:
        raise ValueError(f"{what}: {name} has scales of shape {tuple(scale.shape)} for codes of shape {tuple(codes.shape)}")
    if scale.device != codes.device:
        raise ValueError(f"{what}: {name} has its scales on {scale.device}, its codes on {codes.device}")
    if scale.dim() != 1:
        scale = scale.reshape(-1)
    return *rows2, (scale if scale.is_contiguous() else scale.contiguous())


def _extent(x: torch.Tensor):
    """(first byte of x, the byte after its last)."""
    at, n = x.data_ptr(), x.numel()
    if not x.is_contiguous() and n:
        n = 1 + sum((size - 1) * st for size, st in zip(x.shape, x.stride()))
    return at, at + n * x.element_size()


def _overlap(x: torch.Tensor, y: torch.Tensor) -> bool:
    """Whether two tensors may share memory; of rows (two dimensions) on the same stride it is told exactly."""
    (x0, x1), (y0, y1) = _extent(x), _extent(y)
    if x1 <= y0 or y1 <= x0:
        return False
    if x.dim() == 2 and y.dim() == 2:  # columns beside each other in the same wider rows
        step = x.stride(0) * x.element_size()
        if step == y.stride(0) * y.element_size():
            at, x_row, y_row = (y0 - x0) % max(step, 1), x.shape[1] * x.element_size(), y.shape[1] * y.element_size()
            return at < x_row or at + y_row > step
    return True


def _new_rows(x: torch.Tensor, rows: int, c: int):
    """Uninitialised (codes, scale, stride) for rows like those of x; each row of codes starts on a 16-byte boundary, as the
    tensor-core product wants it."""
    wide = (c + 15) // 16 * 16
    if x.dim() == 2:
        codes, scale = x.new_empty(rows, wide, dtype=torch.int8), x.new_empty(rows, dtype=torch.float32)
    else:
        lead = x.shape[:-1]
        codes, scale = x.new_empty(*lead, wide, dtype=torch.int8), x.new_empty(lead, dtype=torch.float32)
    return (codes if wide == c else codes[..., :c]), scale, wide


def _new_like(x: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """Uninitialised, dense, of x's shape."""
    return torch.empty_like(x, dtype=dtype) if x.is_contiguous() else x.new_empty(x.shape, dtype=dtype)


# ------------------------------------------------------------------ operators
def quantize_rows(x: torch.Tensor) -> Int8Rows:
    """int8 rows of x [..., C]: scale = max(max |x|, 1e-8) / 127 in float32, a code is the nearest multiple of it (ties to
    even), -127 to 127.  A row with a NaN or an infinity has scale NaN and codes 0."""
    what = "quantize_rows"
    x2, rows, c, ld = _as_rows(x, what, "x")
    code = L.dtype_code(x.dtype)
    _refuse_grad(what, x)
    codes, scale, ld_codes = _new_rows(x, rows, c)
    _call(x2, "mtp_quantize_rows", x2.data_ptr(), code, ld, rows, c, codes.data_ptr(), ld_codes, scale.data_ptr())
    return Int8Rows(codes, scale)


def dequantize_rows(rows: Int8Rows, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """What the rows stand for: codes * scale, the float32 product rounded to ``dtype``."""
    what = "dequantize_rows"
    codes, n, c, ld, scale = _as_codes(rows, what, "rows")
    code = L.dtype_code(dtype)
    _refuse_grad(what, rows.scale)
    out = _new_like(rows.codes, dtype)
    _call(codes, "mtp_dequantize_rows", codes.data_ptr(), ld, scale.data_ptr(), n, c, out.data_ptr(), code, c)
    return out


def _norm(x, residual, weight, eps, inplace, what):
    x2, rows, c, ld = _as_rows(x, what, "x")
    x_code, w_code = L.dtype_code(x.dtype), L.dtype_code(weight.dtype)
    if weight.shape != (c,):
        raise ValueError(f"{what}: weight has shape {tuple(weight.shape)}, expected {(c,)}")
    _same_device(weight, x, what, "weight")
    eps = float(eps)
    if not eps >= 0.0:
        raise ValueError(f"{what}: eps must not be negative, got {eps}")
    _refuse_grad(what, x, residual, weight)
    if not weight.is_contiguous():
        weight = weight.contiguous()
    h, res_args = None, (None, 0, 0, None, 0)
    if residual is not None:
        if residual.shape != x.shape:
            raise ValueError(f"{what}: residual has shape {tuple(residual.shape)}, expected {tuple(x.shape)}")
        _same_device(residual, x, what, "residual")
        r_code = L.dtype_code(residual.dtype)
        res, _, _, ld_res = _as_rows(residual, what, "residual")
        if inplace:
            if res.data_ptr() != residual.data_ptr():
                raise ValueError(f"{what}: a residual that is updated in place needs rows on one stride")
            if _overlap(x2, res) or _overlap(weight, residual):
                raise ValueError(f"{what}: a residual that is updated in place must not share memory with x or weight")
            increment_version(residual)  # a backward pass that has kept it shall see that it changed
            h, ld_h = residual, ld_res
        else:
            h, ld_h = _new_like(residual, residual.dtype), c
        res_args = (res.data_ptr(), r_code, ld_res, h.data_ptr(), ld_h)
    codes, scale, ld_codes = _new_rows(x, rows, c)
    _call(x2, "mtp_rmsnorm_int8", x2.data_ptr(), x_code, ld, *res_args, rows, c, weight.data_ptr(), w_code, eps, codes.data_ptr(),
          ld_codes, scale.data_ptr())
    return Int8Rows(codes, scale), h


def rms_norm_int8(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5) -> Int8Rows:
    """``quantize_rows`` of weight * x / sqrt(mean(x^2) + eps) over the last dimension, without the norm in memory; the
    statistics are held in 64 bits and the norm is not rounded in between."""
    return _norm(x, None, weight, eps, False, "rms_norm_int8")[0]


def add_rms_norm_int8(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5, *,
                      inplace: bool = False):
    """A layer's boundary in one call: (int8 rows of the norm of h, h) with h = x + residual, added in float32 and rounded
    to the residual's dtype.  ``inplace`` writes h over the residual (its rows on one stride, no two the same memory)."""
    return _norm(x, residual, weight, eps, inplace, "add_rms_norm_int8")


def int8_linear(x: Int8Rows, weight: Int8Rows, bias: torch.Tensor | None = None, *,
                dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """x [..., K] times weight [N, K]^T: (the exact int32 sum of the codes' products) * x's scale * weight's scale (+ bias),
    in float32 in this order, rounded to ``dtype``; [..., N].  A row's results depend on no other row."""
    what = "int8_linear"
    a, m, k, ld_a, a_scale = _as_codes(x, what, "x")
    wc, n, wk, ld_w, w_scale = _as_codes(weight, what, "weight")
    if wk != k or weight.codes.dim() != 2:
        raise ValueError(f"{what}: x {tuple(x.codes.shape)} and weight {tuple(weight.codes.shape)} do not fit")
    _same_device(wc, a, what, "weight")
    code, b_code = L.dtype_code(dtype), 0
    if bias is not None:
        if bias.shape != (n,):
            raise ValueError(f"{what}: bias has shape {tuple(bias.shape)}, expected {(n,)}")
        _same_device(bias, a, what, "bias")
        b_code = L.dtype_code(bias.dtype)
        bias = bias.contiguous()
    _refuse_grad(what, x.scale, weight.scale, bias)
    out = wc.new_empty(m, n, dtype=dtype) if x.codes.dim() == 2 else wc.new_empty(*x.codes.shape[:-1], n, dtype=dtype)
    _call(a, "mtp_int8_linear", a.data_ptr(), ld_a, a_scale.data_ptr(), m, k, wc.data_ptr(), ld_w, w_scale.data_ptr(), n,
          L.ptr(bias), b_code, out.data_ptr(), code, n)
    return out
