"""What the 16-bit products by expert, the adapters and MXINT8 refuse before they touch CUDA, what they answer without work to do, and where their Python calls allocate.
CPU only."""
import contextlib
import ctypes as C
import inspect

import pytest
import torch

from flashrt_b200 import adapters, moe, mxint8
from test_grid_wait_loads import kernels


@pytest.fixture(scope="module")
def L():
    from flashrt_b200 import lib
    return lib


P = C.c_void_p(4096)        # an address that no refused call reads


def refused(call, ok, cases):
    for i, v, rc in cases:
        args = list(ok)
        args[i] = v
        assert call(*args) == rc, (i, v)


def odd(n):
    return C.c_void_p(4096 + n)


def test_product_refusals(L):
    A, S = L.ERR_ARG, L.ERR_SHAPE
    # stream, x, ldx, w, ldw, lde, dtype, offsets, E, rows, n, S, y, ldy, out_dtype
    ok = [None, P, 64, P, 64, 64 * 32, 1, P, 4, 32, 64, 10, P, 32, 0]
    refused(L.lib.frx_moe_matmul, ok, ((1, None, A), (1, odd(8), A), (2, 56, A), (2, 68, A), (3, None, A), (3, odd(2), A), (4, 60, A), (4, 70, A), (5, 64 * 31, A), (5, 64 * 32 + 4, A), (6, 0, A), (6, 3, A),
                                       (7, None, A), (8, 0, S), (8, 4097, S), (9, 0, S), (9, 2 ** 20 + 1, S), (10, 0, S), (10, -8, S), (11, -1, A), (12, None, A), (12, odd(2), A), (13, 31, A), (14, 3, A),
                                       (14, -1, A)))
    assert L.lib.frx_moe_matmul(None, None, 64, None, 64, 2048, 1, None, 4, 32, 64, 0, None, 32, 0) == L.OK
    # stream, gy, ldgy, w, ldw, lde, dtype, offsets, E, rows, n, S, gx, ldgx, out_dtype
    ok = [None, P, 32, P, 64, 64 * 32, 2, P, 4, 32, 64, 10, P, 64, 1]
    refused(L.lib.frx_moe_matmul_backward_x, ok, ((1, None, A), (1, odd(4), A), (2, 24, A), (2, 36, A), (3, None, A), (4, 56, A), (5, 64 * 30, A), (6, 0, A), (7, None, A), (8, 5000, S), (9, 0, S), (10, 0, S),
                                                  (11, -1, A), (12, None, A), (12, odd(1), A), (13, 63, A), (14, 9, A)))
    assert L.lib.frx_moe_matmul_backward_x(None, None, 32, None, 64, 2048, 2, None, 4, 32, 64, 0, None, 64, 1) == L.OK
    # stream, gy, ldgy, x, ldx, dtype, offsets, E, rows, n, S, gw, ldgw, ldge, out_dtype, add
    ok = [None, P, 32, P, 64, 1, P, 4, 32, 64, 10, P, 64, 64 * 32, 0, 0]
    refused(L.lib.frx_moe_matmul_backward_w, ok, ((1, None, A), (1, odd(8), A), (2, 31, A), (2, 33, A), (3, None, A), (3, odd(8), A), (4, 63, A), (5, 0, A), (6, None, A), (7, 0, S), (8, 0, S), (9, 0, S),
                                                  (10, -1, A), (11, None, A), (11, odd(2), A), (12, 63, A), (13, 64 * 31, A), (14, 4, A)))


def test_adapter_refusals(L):
    A, S = L.ERR_ARG, L.ERR_SHAPE
    # stream, x, ldx, a, lda, stride_a, b, ldb, stride_b, dtype, L, rank, n, rows, offsets, which, R, scale, T, y, ldy, out, ldo, y_dtype
    ok = [None, P, 64, P, 64, 64 * 16, P, 16, 16 * 40, 1, 5, 16, 64, 40, P, P, 3, None, 7, P, 40, P, 40, 1]
    refused(L.lib.frx_adapter_add, ok, ((1, None, A), (1, odd(8), A), (2, 56, A), (2, 65, A), (3, None, A), (3, odd(2), A), (4, 63, A), (5, 64 * 15, A), (5, 64 * 16 + 1, A), (6, None, A), (6, odd(4), A),
                                        (7, 15, A), (7, 17, A), (8, 16 * 39, A), (9, 0, A), (10, 0, S), (11, 0, S), (11, 129, S), (12, 0, S), (13, 0, S), (13, 2 ** 20 + 1, S), (14, None, A), (15, None, A),
                                        (16, -1, A), (18, -1, A), (19, None, A), (19, odd(1), A), (20, 39, A), (21, None, A), (21, odd(1), A), (22, 39, A), (23, 5, A)))
    for i in (16, 18):                # no requests, no tokens: nothing is looked at
        args = list(ok)
        args[i] = 0
        for j in (1, 3, 6, 14, 15, 19, 21):
            args[j] = None
        assert L.lib.frx_adapter_add(*args) == L.OK


def test_mxint8_refusals(L):
    A, S = L.ERR_ARG, L.ERR_SHAPE
    ok = [None, P, 64, 0, 4, 64, P, P]
    refused(L.lib.frx_mxint8_quantize, ok, ((1, None, A), (1, odd(2), A), (2, 63, A), (3, 3, A), (4, -1, A), (5, -32, A), (5, 48, S), (6, None, A), (6, odd(4), A), (7, None, A)))
    assert L.lib.frx_mxint8_quantize(None, P, 2 ** 30, 0, 2 ** 20, 2 ** 20, P, P) == S
    assert L.lib.frx_mxint8_quantize(None, None, 64, 0, 0, 64, None, None) == L.OK
    back = [None, P, P, 4, 64, 2, P, 64]
    refused(L.lib.frx_mxint8_dequantize, back, ((1, None, A), (1, odd(4), A), (2, None, A), (3, -1, A), (4, 40, S), (5, 7, A), (6, None, A), (6, odd(1), A), (7, 60, A)))
    assert L.lib.frx_mxint8_dequantize(None, None, None, 4, 0, 0, None, 0) == L.OK
    up = [None, P, 128, 1, 4, 64, P, P, P, 64]
    refused(L.lib.frx_mxint8_swiglu, up, ((1, None, A), (1, odd(1), A), (2, 127, A), (3, 4, A), (4, -1, A), (5, 63, S), (6, None, A), (6, odd(4), A), (7, None, A), (8, None, A), (8, odd(1), A), (9, 63, A)))
    assert L.lib.frx_mxint8_swiglu(None, None, 128, 1, 0, 64, None, None, None, 64) == L.OK
    grad = [None, P, 64, P, P, 1, 4, 64, P, 128, P, 64]
    refused(L.lib.frx_mxint8_swiglu_backward, grad, ((1, None, A), (2, 63, A), (3, None, A), (3, odd(4), A), (4, None, A), (5, 8, A), (6, -1, A), (7, 33, S), (8, None, A), (9, 127, A), (10, odd(1), A), (11, 63, A)))
    args = list(grad)
    args[6] = 0
    assert L.lib.frx_mxint8_swiglu_backward(*args) == L.OK


class Side:
    cuda_stream, device_index = 77, 0


def calls():
    S, E, n, rows, ff, T, rank = 300, 4, 64, 96, 32, 40, 8
    x, gy, w, offsets = torch.zeros(S, n).half(), torch.zeros(S, rows).half(), torch.zeros(E, rows, n).half(), torch.zeros(E + 1, dtype=torch.int32)
    gu, codes, scales = torch.zeros(T, 2 * ff), torch.zeros(T, 2 * ff, dtype=torch.int8), torch.zeros(T, 2 * ff // 32, dtype=torch.uint8)
    y, a, b, which = torch.zeros(S, rows), torch.zeros(2, rank, n).half(), torch.zeros(2, rows, rank).half(), torch.zeros(3, dtype=torch.int32)
    return {"moe_matmul": (moe.moe_matmul, x, w, offsets), "moe_matmul_backward_x": (moe.moe_matmul_backward_x, gy, w, offsets),
            "moe_matmul_backward_w": (moe.moe_matmul_backward_w, gy, x, offsets), "quantize": (mxint8.quantize, gu), "dequantize": (mxint8.dequantize, codes, scales),
            "swiglu": (mxint8.swiglu, gu), "swiglu_backward": (mxint8.swiglu_backward, gu[:, :ff].contiguous(), codes, scales), "adapters.add": (adapters.add, y, x, a, b, offsets[:4], which)}


@pytest.fixture
def trace(monkeypatch):
    """The stream that is current at every allocation of a tensor from another one, and at every call of the library."""
    current, seen = [1], {"allocated": [], "called": []}

    @contextlib.contextmanager
    def under(stream):
        current.append(stream.cuda_stream)
        yield
        current.pop()

    class Library:
        def __getattr__(self, name):
            def call(*args):
                seen["called"].append(args[0])
                return 0
            return call

    class Allocations(torch.overrides.TorchFunctionMode):
        def __torch_function__(self, func, types, args=(), kwargs=None):
            if func in (torch.Tensor.new_empty, torch.empty, torch.zeros, torch.empty_like):
                seen["allocated"].append(current[-1])
            return func(*args, **(kwargs or {}))

    for module in (moe, mxint8, adapters):
        monkeypatch.setattr(module, "fast", Library())
        monkeypatch.setattr(module, "_on_device", lambda *ts: None)
        monkeypatch.setattr(module, "_raw_stream", lambda stream=None: current[-1] if stream is None else stream.cuda_stream)
    monkeypatch.setattr(moe, "_current_device", lambda: 0)
    monkeypatch.setattr(moe, "_current_raw_stream", lambda device: current[-1])
    monkeypatch.setattr(torch.cuda, "stream", under)
    return seen, Allocations


@pytest.mark.parametrize("name", sorted(calls()))
def test_a_call_on_a_stream_allocates_from_it(trace, name):
    seen, allocations = trace
    call, *args = calls()[name]
    with allocations():
        call(*args, stream=Side())
    assert seen["allocated"] and set(seen["allocated"]) == {Side.cuda_stream} and seen["called"] == [Side.cuda_stream]
    for key in seen:
        seen[key].clear()
    with allocations():
        call(*args)
    assert set(seen["allocated"]) == {1} and seen["called"] == [1]


def test_a_call_that_allocates_nothing_stays_as_it_is(trace, monkeypatch):
    seen, allocations = trace
    monkeypatch.setattr(torch.cuda, "stream", lambda stream: pytest.fail("the current stream was changed"))
    made = calls()
    x, w, offsets = made["moe_matmul"][1:]
    gy = made["moe_matmul_backward_x"][1]
    y, ax, a, b, ranges, which = made["adapters.add"][1:]
    codes, scales = made["dequantize"][1:]
    with allocations():
        moe.moe_matmul(x, w, offsets, out=gy, stream=Side())
        moe.moe_matmul_backward_x(gy, w, offsets, out=x, stream=Side())
        moe.moe_matmul_backward_w(gy, x, offsets, out=w, add=True, stream=Side())
        adapters.add(y, ax, a, b, ranges, which, out=y, stream=Side())
        mxint8.dequantize(codes, scales, out=made["quantize"][1], stream=Side())
    assert not seen["allocated"] and seen["called"] == [Side.cuda_stream] * 5


def test_every_argument_is_handed_on(trace, monkeypatch):
    """What a call passes to itself under its stream are all of its parameters, each in its place."""
    handed, checked = {}, 0
    for module in (mxint8, adapters):
        monkeypatch.setattr(module, "_on", lambda stream, call, *a, **k: handed.update(inspect.signature(call).bind(*a, **k).arguments))
        for f in vars(module).values():
            if not inspect.isfunction(f) or f.__module__ != module.__name__ or "stream" not in inspect.signature(f).parameters:
                continue
            handed.clear()
            given = {p: None if p == "out" else object() for p in inspect.signature(f).parameters}
            f(**given)
            assert handed == {p: v for p, v in given.items() if p != "stream"}, f.__qualname__
            checked += 1
    assert checked == 5


@pytest.mark.parametrize("source,least", [("frx_mxint8.cu", 4), ("frx_experts.cu", 1), ("frx_adapters.cu", 1)])
def test_loads_behind_the_wait_are_ordinary_ones(source, least):
    import re
    seen = 0
    for name, params, body in kernels(source):
        assert "pdl_wait()" in body, name
        seen += 1
        assert not re.search(r"\bconst\b[^,]*\*\s*__restrict__", params) and "__ldg(" not in body, name
    assert seen >= least


def test_places_are_free_before_the_second_product_fills_them():
    """Asynchronous copies have no order among themselves: those that the first product of a single token still has in flight (zeros from behind its depth) have to be waited for
    before the second product's rows go to the same places."""
    from pathlib import Path
    text = (Path(moe.__file__).parent / "csrc" / "frx_adapters.cu").read_text()
    body = text[text.index("void one_token_of_rank("):]
    last, first = body.index("fetch(at);"), body.index("fetch(mine + i * 2 * NB * kSlotBytes);")   # the first product's last, the second's first
    assert last < first and "fetch_wait<0>();" in body[last:first]


def test_adapter_result_in_place_has_the_rows_of_y(L):
    ok = [None, P, 64, P, 64, 64 * 16, P, 16, 16 * 40, 1, 5, 16, 64, 40, P, P, 3, None, 7, P, 40, P, 40, 1]
    refused(L.lib.frx_adapter_add, ok, ((20, 48, L.ERR_ARG), (22, 48, L.ERR_ARG)))


def test_timings_name_these_kernels(L):
    names, c = [], 0
    while name := L.lib.frx_profile_class_name(c):
        names.append(name.decode())
        c += 1
    assert len(set(names)) == len(names) and {"gate_up", "quant_q8", "moe_product", "adapter", "swiglu"} <= set(names) and L.lib.frx_profile_class_name(-1) == b""
