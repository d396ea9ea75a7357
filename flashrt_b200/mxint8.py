"""Activations kept in 8 bits for a backward pass, in MXINT8 (8-bit integers in blocks of 32 with a shared power-of-two scale): rows to 8 bits and back, SwiGLU that
keeps its gate and up rows in the same pass, and its gradient from what was kept. Calls go to libfrx (include/frx.h, "MXINT8"); errors surface as ``FrxError``. The
products around them are in ``moe`` (``moe_matmul`` and its gradients). The gradients are calls of their own: nothing here takes part in torch.autograd.
"""
from __future__ import annotations

import torch

from . import lib as _l
from .lib import FrxError, check, fast
from .moe import DTYPES, _code, _matrix, _on, _on_device, _raw_stream, _typed

BLOCK = 32   # values that share a scale


def _blocks(name: str, n: int) -> None:
    if n % BLOCK:
        raise FrxError(_l.ERR_SHAPE, f"{name}: rows of {n} values are not whole blocks of {BLOCK}")


def _kept(codes: torch.Tensor, scales: torch.Tensor):
    """T, n of rows in 8 bits."""
    if codes.dim() != 2 or codes.dtype != torch.int8 or not codes.is_contiguous():
        raise FrxError(_l.ERR_ARG, "codes: a contiguous int8 tensor of [rows][n] is wanted")
    T, n = codes.shape
    _blocks("codes", n)
    _typed("scales", scales, torch.uint8, (T, n // BLOCK))
    return T, n


def quantize(x: torch.Tensor, stream=None):
    """x [T][n] float32, bfloat16 or float16 (n a multiple of 32) -> codes int8 [T][n], scales uint8 [T][n / 32]."""
    if stream is not None:
        return _on(stream, quantize, x)
    _on_device(x)
    ldx = _matrix("x", x)
    T, n = x.shape
    _blocks("x", n)
    codes, scales = x.new_empty(T, n, dtype=torch.int8), x.new_empty(T, n // BLOCK, dtype=torch.uint8)
    check(fast.mxint8_quantize(_raw_stream(stream), x.data_ptr(), ldx, DTYPES[x.dtype], T, n, codes.data_ptr(), scales.data_ptr()))
    return codes, scales


def dequantize(codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.float32, out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """The values that codes and scales stand for, [T][n] in `dtype` (or that of `out`): exact in float32 and bfloat16, rounded where float16 does not hold them."""
    if stream is not None and out is None:
        return _on(stream, dequantize, codes, scales, dtype=dtype, out=out)
    _on_device(codes, scales, out)
    T, n = _kept(codes, scales)
    if out is None:
        out, ldo = codes.new_empty(T, n, dtype=dtype), n
    else:
        ldo = _matrix("out", out, None, (T, n))
    check(fast.mxint8_dequantize(_raw_stream(stream), codes.data_ptr(), scales.data_ptr(), T, n, _code(out.dtype), out.data_ptr(), ldo))
    return out


def swiglu(gu: torch.Tensor, out: torch.Tensor | None = None, stream=None):
    """h = silu(g) * u of rows [g | u], gu [S][2 ff] -> h [S][ff] in its type (or `out`), and gu in 8 bits: codes int8 [S][2 ff], scales uint8 [S][2 ff / 32]. ff a
    multiple of 32."""
    if stream is not None:
        return _on(stream, swiglu, gu, out=out)
    _on_device(gu, out)
    ldgu = _matrix("gu", gu)
    S, ff = gu.shape[0], gu.shape[1] // 2
    _blocks("gu", gu.shape[1])
    _blocks("gu (half of it)", ff)
    codes, scales = gu.new_empty(S, 2 * ff, dtype=torch.int8), gu.new_empty(S, 2 * ff // BLOCK, dtype=torch.uint8)
    if out is None:
        out, ldo = gu.new_empty(S, ff), ff
    else:
        ldo = _matrix("out", out, gu.dtype, (S, ff))
    check(fast.mxint8_swiglu(_raw_stream(stream), gu.data_ptr(), ldgu, DTYPES[gu.dtype], S, ff, codes.data_ptr(), scales.data_ptr(), out.data_ptr(), ldo))
    return out, codes, scales


def swiglu_backward(gh: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, out: torch.Tensor | None = None, hidden: bool = True, stream=None):
    """From the gradient gh [S][ff] of h and what swiglu kept: the gradient [S][2 ff] of its rows (or `out`) and, with `hidden`, h again, [S][ff], which the gradient of the next
    matrix needs (else None). Both are those of the rows as they were kept, in the type of gh."""
    if stream is not None:
        return _on(stream, swiglu_backward, gh, codes, scales, out=out, hidden=hidden)
    _on_device(gh, codes, scales, out)
    ldgh = _matrix("gh", gh)
    S, ff = gh.shape
    _blocks("gh", ff)
    if _kept(codes, scales) != (S, 2 * ff):
        raise FrxError(_l.ERR_ARG, f"codes: {tuple(codes.shape)} for gradients of {(S, ff)}: {(S, 2 * ff)} is wanted")
    if out is None:
        out, ldo = gh.new_empty(S, 2 * ff), 2 * ff
    else:
        ldo = _matrix("out", out, gh.dtype, (S, 2 * ff))
    h = gh.new_empty(S, ff) if hidden else None
    check(fast.mxint8_swiglu_backward(_raw_stream(stream), gh.data_ptr(), ldgh, codes.data_ptr(), scales.data_ptr(), DTYPES[gh.dtype], S, ff, out.data_ptr(), ldo,
                                      None if h is None else h.data_ptr(), ff))
    return out, h
