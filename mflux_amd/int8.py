"""A linear layer in 8-bit integers, and the norm in front of it: ``rms_norm`` with
the residual's addition, ``rms_norm_int8`` and ``int8_quantize`` (rows as codes with a
scale each), ``int8_dequantize``, and ``int8_matmul``.

``quantized_matmul`` keeps activations in 16 bits and multiplies them with
dequantised weights; here both operands are codes, and the matrix cores multiply
them as they are, at twice the 16-bit rate.  The reference has no such product; its
norms are ``nn.RMSNorm`` (src/mflux/models/z_image/model/z_image_transformer/transformer_block.py).

The calls run on the current stream of their tensors' device and launch nothing
anywhere else; the same inputs give the same bits.  All can be captured into a graph.
``rms_norm`` has first derivatives in reverse mode, the others none: they refuse tensors
that want one.
"""
from __future__ import annotations

import torch

from . import _lib
from .core import _DTYPE_CODE, _require_hip

MAX_INNER = (1 << 17) - 1  # |x w| <= 2^14, and their sum fits 32 bits


def _check_rows(fn: str, x: torch.Tensor) -> None:
    if x.dtype not in _DTYPE_CODE:
        raise ValueError(f"[{fn}] x must be float32, float16 or bfloat16, got {x.dtype}")
    if x.ndim < 1 or not 0 < x.shape[-1] <= 1 << 28:
        raise ValueError(f"[{fn}] x must be [..., K] with 1 to 2^28 values a row, got {tuple(x.shape)}")
    if x.numel() // x.shape[-1] >= 2 ** 31:
        raise ValueError(f"[{fn}] fewer than 2^31 rows fit a call, got {tuple(x.shape)}")


def _check_norm(fn: str, x, weight, residual, eps) -> None:
    _check_rows(fn, x)
    if weight is not None:
        if tuple(weight.shape) != (x.shape[-1],) or weight.dtype != x.dtype:
            raise ValueError(f"[{fn}] weight must be a [{x.shape[-1]}] vector of {x.dtype}, got {tuple(weight.shape)} {weight.dtype}")
        if weight.device != x.device:
            raise ValueError(f"[{fn}] `weight` lives on {weight.device}, x on {x.device}")
    if residual is not None:
        if residual.shape != x.shape or residual.dtype != x.dtype:
            raise ValueError(f"[{fn}] residual must be as x, {tuple(x.shape)} {x.dtype}, got {tuple(residual.shape)} {residual.dtype}")
        if residual.device != x.device:
            raise ValueError(f"[{fn}] `residual` lives on {residual.device}, x on {x.device}")
    if not 0 <= eps <= 1e30:
        raise ValueError(f"[{fn}] eps must not be negative, got {eps!r}")
    _require_hip(fn, x, "x")


def _refuse_gradients(fn: str, *tensors) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise ValueError(f"[{fn}] codes have no gradient: detach the inputs, or call it under torch.no_grad()")


def rms_norm(x: torch.Tensor, weight: torch.Tensor | None = None, *, residual: torch.Tensor | None = None, eps: float = 1e-6):
    """``x / sqrt(mean(x^2) + eps) * weight`` over the last axis; with ``residual`` of ``x + residual``,
    returned as well: ``(y, sum)``, the two lines ``h = h + block(...)`` and ``norm(h)`` of a transformer
    block as one pass.

    ``x``: ``[..., K]`` of float32, float16 or bfloat16, any strides (a last axis that is not
    dense, or rows without one stride, are copied); ``weight`` ``[K]`` and ``residual`` of its type.  The sum is
    rounded to the type, and what is normalised is the rounded sum; everything else is
    float32 and rounded once, of any finite row (also one whose squares float32 does not hold).  Results are densely packed.

    Gradients for ``x``, ``residual`` (the same one) and ``weight``, through both results (the sum has none where
    the weight alone wants one)."""
    y = _lib.native().rms_norm(x, weight, residual, eps)
    if y is not None:
        return y
    _check_norm("rms_norm", x, weight, residual, eps)
    y, total = _lib.ops().rms_norm_call(x, weight, residual, eps)
    return y if residual is None else (y, total)


def rms_norm_int8(x: torch.Tensor, weight: torch.Tensor | None = None, *, residual: torch.Tensor | None = None, eps: float = 1e-6):
    """``int8_quantize(rms_norm(x, weight, residual=residual))`` without the 16-bit rounding in between:
    ``(codes, scales)``, with ``residual`` ``(codes, scales, sum)``.

    A code is ``rint(127 p / max|p|)`` of the row's products ``p = sum * weight``, ties to even (the root is a
    factor of the scale alone).  It is decided by the exact quotient for 16-bit types whose products float32 holds as
    normal numbers, and for float32 without a weight; float32 products and their quotient are float64, which may
    decide otherwise within 2^-45 of a border.  Products of 16-bit types are taken in
    float32: one beyond its range makes the row's scale NaN, as an infinity or NaN in the row does.
    No gradients."""
    rows = _lib.native().int8_rows(x, weight, residual, eps, True)
    if rows is not None:
        return rows
    fn = "rms_norm_int8"
    _check_norm(fn, x, weight, residual, eps)
    _refuse_gradients(fn, x, weight, residual)
    codes, scales, total = _lib.ops().rms_norm_int8(x, weight, residual, eps)
    return (codes, scales) if residual is None else (codes, scales, total)


def int8_quantize(x: torch.Tensor):
    """Rows in 8 bits: ``(codes, scales)`` with ``codes = rint(127 x / max|x|)`` int8 ``[..., K]``, ties to even,
    and ``scales = max|x| / 127`` float32 ``[...]``: activations with a scale for each token, or a
    weight ``[N, K]`` with one for each output feature.

    A row of zeros has codes and scale 0; one that holds an infinity or NaN has the scale NaN (and
    codes 0), so that its products are NaN.  Rows of codes begin at whole 16 bytes: where ``K`` is no
    multiple of 16 the codes are a view with a stride between rows.  No gradients."""
    rows = _lib.native().int8_rows(x, None, None, 0.0, False)
    if rows is not None:
        return rows
    fn = "int8_quantize"
    _check_rows(fn, x)
    _refuse_gradients(fn, x)
    _require_hip(fn, x, "x")
    return _lib.ops().int8_quantize(x)


def _check_codes(fn: str, name: str, codes: torch.Tensor, scales: torch.Tensor) -> None:
    if codes.dtype != torch.int8 or codes.ndim < 1 or codes.shape[-1] < 1:
        raise ValueError(f"[{fn}] {name} must be int8 [..., K], got {tuple(codes.shape)} {codes.dtype}")
    if scales.dtype != torch.float32 or scales.shape != codes.shape[:-1]:
        raise ValueError(f"[{fn}] the scales of {name} must be float32 {tuple(codes.shape[:-1])}, got {tuple(scales.shape)} {scales.dtype}")
    if scales.device != codes.device:
        raise ValueError(f"[{fn}] `{name}` lives on {codes.device}, its scales on {scales.device}")


def int8_dequantize(codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``codes * scales[..., None]`` in ``dtype``, rounded once.  No gradients."""
    values = _lib.native().int8_dequantize(codes, scales, _DTYPE_CODE.get(dtype))
    if values is not None:
        return values
    fn = "int8_dequantize"
    _check_codes(fn, "codes", codes, scales)
    if dtype not in _DTYPE_CODE:
        raise ValueError(f"[{fn}] dtype must be float32, float16 or bfloat16, got {dtype}")
    if codes.shape[-1] > 1 << 28 or codes.numel() // codes.shape[-1] >= 2 ** 31:
        raise ValueError(f"[{fn}] at most 2^28 values a row and fewer than 2^31 rows fit a call, got {tuple(codes.shape)}")
    _refuse_gradients(fn, scales)
    _require_hip(fn, codes, "codes")
    return _lib.ops().int8_dequantize(codes, scales, dtype)


def int8_matmul(x: torch.Tensor, x_scales: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor, *, bias: torch.Tensor | None = None,
                dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``(x @ w.T) * x_scales[..., None] * w_scales (+ bias)``: the product of a linear layer with 8-bit
    integers on both sides, ``x`` ``[..., K]`` with a scale for each row (``int8_quantize``, ``rms_norm_int8``) and
    ``w`` ``[N, K]`` with a scale for each output feature.

    The integer sum is exact (``K`` below 2^17); it times ``x_scales``, that times ``w_scales``, and the
    sum with ``bias`` ``[N]`` of ``dtype`` are float32, rounded once to ``dtype`` (float32, float16 or bfloat16).
    Any values from -128 to 127, any strides; rows that are not whole 16 bytes apart are copied,
    and so is an ``x`` whose ``K`` is no multiple of 16.  No gradients."""
    y = _lib.native().int8_matmul(x, x_scales, w, w_scales, bias, _DTYPE_CODE.get(dtype))
    if y is not None:
        return y
    fn = "int8_matmul"
    _check_codes(fn, "x", x, x_scales)
    _check_codes(fn, "w", w, w_scales)
    if w.ndim != 2 or x.shape[-1] != w.shape[-1]:
        raise ValueError(f"[{fn}] x [..., K] and w [N, K] must agree in K, got {tuple(x.shape)} and {tuple(w.shape)}")
    if x.shape[-1] > MAX_INNER - 15:
        raise ValueError(f"[{fn}] rows of up to {MAX_INNER - 15} codes fit a 32-bit sum, got {x.shape[-1]}")
    if w.device != x.device:
        raise ValueError(f"[{fn}] `w` lives on {w.device}, x on {x.device}")
    if dtype not in _DTYPE_CODE:
        raise ValueError(f"[{fn}] dtype must be float32, float16 or bfloat16, got {dtype}")
    if bias is not None:
        if tuple(bias.shape) != (w.shape[0],) or bias.dtype != dtype:
            raise ValueError(f"[{fn}] bias must be a [{w.shape[0]}] vector of {dtype}, got {tuple(bias.shape)} {bias.dtype}")
        if bias.device != x.device:
            raise ValueError(f"[{fn}] `bias` lives on {bias.device}, x on {x.device}")
    if x.numel() // x.shape[-1] > 2 ** 30 or w.shape[0] > 2 ** 30 or x.numel() // x.shape[-1] * w.shape[0] > 2 ** 42:
        raise ValueError(f"[{fn}] at most 2^30 rows of x and of w, and 2^42 results, fit a call")
    _refuse_gradients(fn, x_scales, w_scales, bias)
    _require_hip(fn, x, "x")
    return _lib.ops().int8_matmul(x, x_scales, w, w_scales, bias, dtype)
