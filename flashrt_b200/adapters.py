"""Low-rank adapters of many requests beside a shared projection (``mxfp4.matmul``, ``moe.moe_matmul``, or any other). The call goes to libfrx (include/frx.h,
"low-rank adapters"); errors surface as ``FrxError``.
"""
from __future__ import annotations

import torch

from . import lib as _l
from .lib import FrxError, check, fast
from .moe import _code, _half, _matrices, _matrix, _on, _on_device, _raw_stream, _typed


def add(y: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, offsets: torch.Tensor, which: torch.Tensor, scale: torch.Tensor | None = None,
        out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """out[t] = y[t] + scale[j] * B_j (A_j x[t]) for the tokens t = offsets[i] .. offsets[i + 1] - 1 of each request i, j = which[i]; y[t] alone where that is negative.

    y [T][rows]: what the shared projection of x [T][n] gave, float32, bfloat16 or float16; a [L][rank][n], b [L][rows][rank] and x bfloat16 or float16, rank up to 128 (adapters of
    a smaller one filled up with zeros); offsets int32 [R + 1], which int32 [R], scale float32 [L] or None for 1. Rows of x, a and b on 16-byte boundaries: a `b` of a rank that is not a
    multiple of 8 is the first columns of a wider one (`wide[:, :, :4]` of [L][rows][8]); contiguous it is refused. Rows of y and `out` that are not whole multiples of 32 bytes, 32 bytes aligned,
    are slow for requests of several tokens (ten times at 16,384 tokens). `out`: y itself, or another
    tensor of its shape and type, or None for a new one; tokens of no request are left as they were (in a new one: anything). A decode batch is R = T requests of a token each."""
    if stream is not None and out is None:
        return _on(stream, add, y, x, a, b, offsets, which, scale=scale, out=out)
    _on_device(y, x, a, b, offsets, which, scale, out)
    code = _half("x", x)
    try:
        (T, n), (L, rank, columns), (count, rows, inner) = x.shape, a.shape, b.shape
    except ValueError:
        raise FrxError(_l.ERR_ARG, f"x {tuple(x.shape)}, a {tuple(a.shape)}, b {tuple(b.shape)}: [T][n], [L][rank][n] and [L][rows][rank] are wanted") from None
    if columns != n or count != L or inner != rank or y.shape != (T, rows):
        raise FrxError(_l.ERR_ARG, f"adapters {tuple(a.shape)}, {tuple(b.shape)} for rows of {n} values and results {tuple(y.shape)}: [L][rank][n], [L][rows][rank] and [T][rows] are wanted")
    if a.dtype != x.dtype or b.dtype != x.dtype:
        raise FrxError(_l.ERR_ARG, f"adapters of {a.dtype} and {b.dtype} for rows of {x.dtype}")
    ldx, ldy = _matrix("x", x), _matrix("y", y)
    lda, stride_a = (n, rank * n) if a.is_contiguous() else _matrices("a", a)[3:]
    ldb, stride_b = (rank, rows * rank) if b.is_contiguous() else _matrices("b", b)[3:]
    R = which.numel()
    _typed("which", which, torch.int32)
    _typed("offsets", offsets, torch.int32, (R + 1,))
    if scale is not None:
        _typed("scale", scale, torch.float32, (L,))
    if out is None:
        out, ldo = y.new_empty(T, rows), rows
    else:
        ldo = _matrix("out", out, y.dtype, (T, rows))
    check(fast.adapter_add(_raw_stream(stream), x.data_ptr(), ldx, a.data_ptr(), lda, stride_a, b.data_ptr(), ldb, stride_b, code, L, rank, n, rows, offsets.data_ptr(), which.data_ptr(), R,
                           None if scale is None else scale.data_ptr(), T, y.data_ptr(), ldy, out.data_ptr(), ldo, _code(out.dtype)))
    return out
