"""Experts and dense layers in MXFP4 (4-bit floats in blocks of 32 with a shared power-of-two scale): quantizer, product,
and the expert layer. Calls go to libfrx (include/frx.h, "MXFP4"); errors surface as ``FrxError``. The routing and the
plan that sorts tokens by expert are in ``moe`` (``moe_route_topk``, ``moe_sort``).
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import lib as _l
from .lib import FrxError, check, fast, lib
from .moe import DTYPES, _code, _ids, _matrix, _on, _on_device, _raw_stream, _typed, _ws_span

BLOCK, UNIT = 32, 128       # values that share a scale; rows and columns of a unit of the packed layout
UNIT_BYTES = 8704           # of a unit: its codes and scales
ROWS_BF16 = 16              # FRX_ROWS_BF16


def quantize(x: torch.Tensor, stream=None):
    """x [T][n] float32, bfloat16 or float16 (n a multiple of 32) -> codes uint8 [T][n / 2], scales uint8 [T][n / 32]."""
    if stream is not None:
        return _on(stream, quantize, x)
    _on_device(x)
    ldx = _matrix("x", x)
    T, n = x.shape
    if n % BLOCK:
        raise FrxError(_l.ERR_SHAPE, f"quantize: rows of {n} values are not whole blocks of {BLOCK}")
    codes, scales = x.new_empty(T, n // 2, dtype=torch.uint8), x.new_empty(T, n // BLOCK, dtype=torch.uint8)
    check(fast.mxfp4_quantize(_raw_stream(stream), x.data_ptr(), ldx, DTYPES[x.dtype], T, n, codes.data_ptr(), scales.data_ptr()))
    return codes, scales


def _quantized(codes: torch.Tensor, scales: torch.Tensor):
    """T, n of quantized rows."""
    size = codes.shape
    if len(size) != 2 or codes.dtype != torch.uint8 or not codes.is_contiguous():
        raise FrxError(_l.ERR_ARG, "codes: a contiguous uint8 tensor of [rows][n / 2] is wanted")
    T, half = size
    _typed("scales", scales, torch.uint8, (T, 2 * half // BLOCK))
    return T, 2 * half


def dequantize(codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.float32, out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """The values that codes and scales stand for, float32 or bfloat16 [T][n]."""
    if stream is not None and out is None:
        return _on(stream, dequantize, codes, scales, dtype=dtype, out=out)
    _on_device(codes, scales, out)
    T, n = _quantized(codes, scales)
    if out is None:
        out, ldo = codes.new_empty(T, n, dtype=dtype), n
    else:
        ldo = _matrix("out", out, None, (T, n))
    check(fast.mxfp4_dequantize(_raw_stream(stream), codes.data_ptr(), scales.data_ptr(), T, n, _code(out.dtype), out.data_ptr(), ldo))
    return out


class Packed(NamedTuple):
    """E matrices [rows][n] in the layout that the product reads."""
    data: torch.Tensor
    E: int
    rows: int
    n: int


def _whole(w: Packed) -> None:
    """The matrices that a Packed names lie in its data (a slice of another one may not)."""
    data, E, rows, n = w
    if data.dtype != torch.uint8 or not data.is_contiguous() or data.numel() < E * (-(-rows // UNIT) * (n // UNIT) * UNIT_BYTES):
        raise FrxError(_l.ERR_ARG, f"a packed matrix: {E} of {rows} x {n} are not in {data.numel()} contiguous elements of {data.dtype}")


def packed_bytes(rows: int, n: int) -> int:
    return int(lib.frx_mxfp4_packed_bytes(rows, n))


def pack(codes: torch.Tensor, scales: torch.Tensor, stream=None) -> Packed:
    """codes uint8 [E][rows][n / 2], scales uint8 [E][rows][n / 32] (or one matrix without E) -> Packed; once, when weights are loaded."""
    if stream is not None:
        return _on(stream, pack, codes, scales)
    _on_device(codes, scales)
    if codes.dim() == 2:
        codes, scales = codes.unsqueeze(0), scales.unsqueeze(0)
    if codes.dim() != 3:
        raise FrxError(_l.ERR_ARG, "codes: uint8 [E][rows][n / 2] is wanted")
    E, rows, half = codes.shape
    _typed("codes", codes, torch.uint8)
    _typed("scales", scales, torch.uint8, (E, rows, 2 * half // BLOCK))
    data = codes.new_empty(E * packed_bytes(rows, 2 * half), dtype=torch.uint8)
    check(lib.frx_mxfp4_pack(_raw_stream(stream), codes.data_ptr(), scales.data_ptr(), E, rows, 2 * half, data.data_ptr()))
    return Packed(data, E, rows, 2 * half)


def unpack(w: Packed, stream=None):
    """codes and scales of a Packed (the inverse of pack)."""
    if stream is not None:
        return _on(stream, unpack, w)
    _on_device(w.data)
    _whole(w)
    codes, scales = w.data.new_empty(w.E, w.rows, w.n // 2), w.data.new_empty(w.E, w.rows, w.n // BLOCK)
    check(lib.frx_mxfp4_unpack(_raw_stream(stream), w.data.data_ptr(), w.E, w.rows, w.n, codes.data_ptr(), scales.data_ptr()))
    return codes, scales


def _columns(w: Packed, n: int) -> None:
    _whole(w)
    if w.n != n:
        raise FrxError(_l.ERR_ARG, f"a matrix of {w.n} columns for rows of {n} values")


def matmul(codes: torch.Tensor, scales: torch.Tensor, w: Packed, out: torch.Tensor | None = None, dtype: torch.dtype = torch.bfloat16, stream=None) -> torch.Tensor:
    """y[t] = W x[t] of quantized rows x and one packed matrix: [T][rows] in `dtype` (or that of `out`)."""
    if stream is not None and out is None:
        return _on(stream, matmul, codes, scales, w, out=out, dtype=dtype)
    _on_device(codes, scales, out, w.data)
    T, n = _quantized(codes, scales)
    _columns(w, n)
    if w.E != 1:
        raise FrxError(_l.ERR_ARG, f"matmul: {w.E} matrices: moe_matmul takes several")
    if out is None:
        out, ldo = codes.new_empty(T, w.rows, dtype=dtype), w.rows
    else:
        ldo = _matrix("out", out, None, (T, w.rows))
    check(fast.mxfp4_matmul(_raw_stream(stream), codes.data_ptr(), scales.data_ptr(), T, n, w.data.data_ptr(), w.rows, out.data_ptr(), ldo, _code(out.dtype)))
    return out


def moe_matmul(codes: torch.Tensor, scales: torch.Tensor, w: Packed, offsets: torch.Tensor, slot_of: torch.Tensor | None = None, K: int = 1,
               out: torch.Tensor | None = None, dtype: torch.dtype = torch.bfloat16, stream=None) -> torch.Tensor:
    """y[r] = W_e x[slot_of[r] / K] for the sorted rows r of each expert e (offsets, slot_of: moe.moe_sort); without slot_of W_e x[r]. Rows of `out`
    that no expert has are left as they were."""
    if stream is not None and out is None:
        return _on(stream, moe_matmul, codes, scales, w, offsets, slot_of=slot_of, K=K, out=out, dtype=dtype)
    _on_device(codes, scales, offsets, slot_of, out, w.data)
    T, n = _quantized(codes, scales)
    _columns(w, n)
    _typed("offsets", offsets, torch.int32, (w.E + 1,))
    if slot_of is not None:
        _typed("slot_of", slot_of, torch.int32)
    S = T if slot_of is None else slot_of.numel()
    if out is None:
        out, ldo = codes.new_empty(S, w.rows, dtype=dtype), w.rows
    else:
        ldo = _matrix("out", out, None, (S, w.rows))
    check(fast.mxfp4_moe_matmul(_raw_stream(stream), codes.data_ptr(), scales.data_ptr(), T, n, w.data.data_ptr(), w.E, w.rows, offsets.data_ptr(),
                                None if slot_of is None else slot_of.data_ptr(), K, S, out.data_ptr(), ldo, _code(out.dtype)))
    return out


def moe_layer_workspace_bytes(T: int, K: int, n: int, ff: int, E: int) -> int:
    return int(lib.frx_mxfp4_moe_layer_workspace_bytes(T, K, n, ff, E))


def moe_layer(x: torch.Tensor, ids: torch.Tensor, wts: torch.Tensor, w_gate: Packed, w_up: Packed, w_down: Packed, out: torch.Tensor | None = None,
              dtype: torch.dtype | None = None, ws: torch.Tensor | None = None, stream=None, rows: torch.dtype = torch.float32) -> torch.Tensor:
    """The expert layer in MXFP4 (frx_mxfp4_moe_layer): out[t] = sum over k of wts[t][k] * expert_{ids[t][k]}(x[t]), [T][n] in `dtype` (that of
    `out`, or of x). Slots with a negative id take no part. `rows`: what the experts' rows are kept in before their sum; bfloat16 for a bfloat16
    output moves half the bytes and rounds twice."""
    if stream is not None and (out is None or ws is None):
        return _on(stream, moe_layer, x, ids, wts, w_gate, w_up, w_down, out=out, dtype=dtype, ws=ws, rows=rows)
    gate, E, ff, gate_n = w_gate
    up, down = w_up[0], w_down[0]
    _on_device(x, ids, wts, out, ws, gate, up, down)
    ldx = _matrix("x", x)
    (T, n), shape = x.shape, ids.shape
    _ids("ids", ids)
    if shape[0] != T:
        raise FrxError(_l.ERR_ARG, f"ids: {shape[0]} tokens, x has {T}")
    K = shape[1]
    _typed("wts", wts, torch.float32, shape)
    if gate_n != n or w_up[1:] != (E, ff, n) or w_down[1:] != (E, n, ff):
        raise FrxError(_l.ERR_ARG, f"matrices (experts, rows, columns) {w_gate[1:]}, {w_up[1:]}, {w_down[1:]} for rows of {n} values: two of {(E, ff, n)} and {(E, n, ff)} are wanted")
    for w in (w_gate, w_up, w_down):
        _whole(w)
    if out is None:
        out, ldo = x.new_empty(T, n, dtype=dtype or x.dtype), n
    else:
        ldo = _matrix("out", out, None, (T, n))
    code = _code(out.dtype)
    if rows != torch.float32:
        if rows != torch.bfloat16 or out.dtype != torch.bfloat16:
            raise FrxError(_l.ERR_ARG, f"moe_layer: rows of {rows} for an output of {out.dtype}: float32, or bfloat16 for a bfloat16 output")
        code |= ROWS_BF16
    if ws is None:
        ws = x.new_empty(moe_layer_workspace_bytes(T, K, n, ff, E) + 256, dtype=torch.uint8)   # (nobody asks for its status)
    wp, wb = _ws_span(ws)
    check(fast.mxfp4_moe_layer(_raw_stream(stream), gate.data_ptr(), up.data_ptr(), down.data_ptr(), E, n, ff, x.data_ptr(), ldx, DTYPES[x.dtype],
                               ids.data_ptr(), wts.data_ptr(), T, K, out.data_ptr(), ldo, code, wp, wb))
    return out
