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
    a smaller one filled up with zeros); offsets int32 [R + 1], which int32 [R], scale float32 [L] or None for 1. Rows of x, a and b on 16-byte boundaries. `out`: y itself, or another
    tensor of its shape and type, or None for a new one; tokens of no request are left as they were (in a new one: anything). A decode batch is R = T requests of a token each."""
    if stream is not None and out is None:
        return _on(stream, add, y, x, a, b, offsets, which, scale=scale, out=out)
    _on_device(y, x, a, b, offsets, which, scale, out)
    ldx, code = _matrix("x", x), _half("x", x)
    T, n = x.shape
    L, rank, _, lda, stride_a = _matrices("a", a, x.dtype)
    rows = y.shape[-1]
    ldy = _matrix("y", y, None, (T, rows))
    if a.shape[2] != n or b.shape != (L, rows, rank):
        raise FrxError(_l.ERR_ARG, f"adapters {tuple(a.shape)}, {tuple(b.shape)} for rows of {n} values and results of {rows}: [L][rank][n] and [L][rows][rank] are wanted")
    _, _, _, ldb, stride_b = _matrices("b", b, x.dtype)
    R = which.numel()
    _typed("which", which, torch.int32, (R,))
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
