"""Calls that are given a stream allocate from it: what a call makes and drops (its workspace) must not be shared with the kernels of the stream that is
current meanwhile. The first part needs no GPU: the allocations and the library calls are looked at through stand-ins."""
import contextlib
import inspect

import pytest
import torch

from flashrt_b200 import moe, mxfp4


class Side:
    cuda_stream, device_index = 77, 0


@pytest.fixture
def trace(monkeypatch):
    """The stream that is current at every allocation of a tensor (from another one or through torch.empty / zeros), and at every call of the library."""
    current, seen = [1], {"allocated": [], "called": []}

    @contextlib.contextmanager
    def under(stream):
        current.append(stream.cuda_stream)
        yield
        current.pop()

    class Library:
        def __getattr__(self, name):
            def call(*args):
                seen["called"].append(current[-1])
                return 4096 if name.endswith("bytes") else 0
            return call

    class Allocations(torch.overrides.TorchFunctionMode):
        def __torch_function__(self, func, types, args=(), kwargs=None):
            if func in (torch.Tensor.new_empty, torch.empty, torch.zeros, torch.empty_like):
                seen["allocated"].append(current[-1])
                kwargs = {k: v for k, v in (kwargs or {}).items() if k != "device"}
            return func(*args, **(kwargs or {}))

    for module in (moe, mxfp4):
        monkeypatch.setattr(module, "fast", Library())
        monkeypatch.setattr(module, "lib", Library())
        monkeypatch.setattr(module, "_on_device", lambda *ts: None)
        monkeypatch.setattr(module, "_raw_stream", lambda stream=None: current[-1] if stream is None else stream.cuda_stream)
    monkeypatch.setattr(moe, "_dev", lambda *ts: None)
    monkeypatch.setattr(moe, "_current_device", lambda: 0)
    monkeypatch.setattr(moe, "_current_raw_stream", lambda device: current[-1])
    monkeypatch.setattr(torch.cuda, "stream", under)
    return seen, Allocations


def calls():
    T, K, E, n, ff = 600, 2, 4, 256, 128
    x, ids, wts, rows = torch.zeros(T, n), torch.zeros(T, K, dtype=torch.int32), torch.zeros(T, K), torch.zeros(T * K, n)
    codes, scales, plan = torch.zeros(T, n // 2, dtype=torch.uint8), torch.zeros(T, n // 32, dtype=torch.uint8), torch.zeros(E + 1, dtype=torch.int32)

    def packed(E, rows, n):
        return mxfp4.Packed(torch.zeros(E * -(-rows // 128) * (n // 128) * 8704, dtype=torch.uint8), E, rows, n)

    one, up, down = packed(1, ff, n), packed(E, ff, n), packed(E, n, ff)
    return {
        "sort": (moe.moe_sort, ids, E), "sort_rows": (moe.moe_sort_rows, x, ids), "sort_rows_backward": (moe.moe_sort_rows_backward, rows, ids),
        "unsort_rows": (moe.moe_unsort_rows, rows, wts, ids), "unsort_rows_backward": (moe.moe_unsort_rows_backward, x, rows, wts, ids),
        "route_topk_backward": (moe.moe_route_topk_backward, wts, wts, ids, E), "quantize": (mxfp4.quantize, x), "dequantize": (mxfp4.dequantize, codes, scales),
        "pack": (mxfp4.pack, codes, scales), "unpack": (mxfp4.unpack, one), "matmul": (mxfp4.matmul, codes, scales, one),
        "moe_matmul": (mxfp4.moe_matmul, codes, scales, up, plan, ids.view(-1), K), "mxfp4.moe_layer": (mxfp4.moe_layer, x, ids, wts, up, up, down),
        "route_topk": (moe.moe_route_topk, x, K), "router_logits": (moe.router_logits, x.bfloat16(), None, x), "quantize_q8": (moe.quantize_q8, x),
        "moe_decode": (moe.moe_decode, 4096, 4096, E, None, n, ff, x, ids, wts, None), "moe_layer": (moe.moe_layer, 4096, 4096, E, None, n, ff, x, wts, None, K),
        "moe_hits": (moe.moe_hits, ids.long(), ids[:, 0], K, x, n, ff, rows), "moe_q2.run": (moe.moe_q2.run, 4096, 4096, E, n, ff, x, ids),
        "moe_q2.run_ex": (moe.moe_q2.run_ex, 4096, 4096, E, n, ff, x, ids), "matvec": (moe.gemv.matvec, moe.Q2_0_TYPE, codes, x, 8),
        "tile_experts": (moe.tile_experts, codes, n, ff, 1),
    }


@pytest.mark.parametrize("name", sorted(calls()))
def test_a_call_on_a_stream_allocates_from_it(trace, name):
    seen, allocations = trace
    call, *args = calls()[name]
    with allocations():
        call(*args, stream=Side())
    assert seen["allocated"] and set(seen["allocated"]) == {Side.cuda_stream}
    assert seen["called"][-1] == Side.cuda_stream
    # and without one, or with the one that is current, from that
    for key in seen:
        seen[key].clear()
    with allocations():
        call(*args)
        Side1 = type("Side1", (), {"cuda_stream": 1, "device_index": 0})
        call(*args, stream=Side1())
    assert set(seen["allocated"]) == {1} and set(seen["called"]) == {1}


def test_every_argument_is_handed_on(trace, monkeypatch):
    """What a call passes to itself under its stream are all of its parameters, each in its place."""
    handed = {}
    monkeypatch.setattr(moe, "_on", lambda stream, call, *a, **k: handed.update(inspect.signature(call).bind(*a, **k).arguments))
    monkeypatch.setattr(mxfp4, "_on", moe._on)
    functions = [f for m in (moe, mxfp4) for f in vars(m).values() if inspect.isfunction(f) and f.__module__ == m.__name__]
    functions += [f.__func__ for c in (moe.moe_q2, moe.gemv, moe.gemm) for f in vars(c).values() if isinstance(f, staticmethod)]
    checked = 0
    for f in functions:
        if "stream" not in inspect.signature(f).parameters or "_on(stream" not in inspect.getsource(f):
            continue
        made = [p for p in inspect.signature(f).parameters if p in ("out", "yd", "ws", "scratch")]
        for absent in made or [None]:               # where the caller may give what a call would allocate: each of these left out
            handed.clear()
            given = {p: None if p == absent else object() for p in inspect.signature(f).parameters}
            f(**given)
            assert handed == {p: v for p, v in given.items() if p != "stream"}, f.__qualname__
            checked += 1
    assert checked >= 30


def test_a_call_that_allocates_nothing_stays_as_it_is(trace, monkeypatch):
    """With results and workspace given there is nothing to allocate: the call does not change the current stream, which costs microseconds."""
    seen, allocations = trace
    monkeypatch.setattr(torch.cuda, "stream", lambda stream: pytest.fail("the current stream was changed"))
    made = calls()
    x, ids, wts, up, _, down = made["mxfp4.moe_layer"][1:]
    ws, out, rows = torch.zeros(4096 + 256, dtype=torch.uint8), torch.zeros(600, 256), torch.zeros(1200, 256)
    with allocations():
        mxfp4.moe_layer(x, ids, wts, up, up, down, out=out, ws=ws, stream=Side())
        moe.moe_sort_rows(x, ids, out=rows, stream=Side())
        moe.moe_unsort_rows(rows, wts, ids, out=out, stream=Side())
        moe.moe_decode(*made["moe_decode"][1:], out=out, ws=ws, stream=Side())
        moe.moe_layer(*made["moe_layer"][1:], out=out, ws=ws, stream=Side())
    assert not seen["allocated"] and seen["called"]


@pytest.mark.gpu
def test_workspace_of_a_call_on_another_stream_is_its_own():
    """A sort and a layer on a side stream that is kept busy first, and tensors of the same sizes made and filled on the current stream right behind the calls: the results are
    those of the plain calls, and what the calls return lies in memory of the side stream."""
    T, K, E, n, ff = 3000, 4, 64, 512, 256
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    ids = torch.randint(-1, E, (T, K), generator=g, device="cuda", dtype=torch.int32)
    x, wts = torch.randn(T, n, generator=g, device="cuda"), torch.rand(T, K, generator=g, device="cuda")
    W = [mxfp4.pack(torch.randint(0, 256, (E, r, c // 2), generator=g, device="cuda", dtype=torch.uint8), torch.full((E, r, c // 32), 121, device="cuda", dtype=torch.uint8))
         for r, c in ((ff, n), (ff, n), (n, ff))]
    want, want_out = moe.moe_sort(ids, E), mxfp4.moe_layer(x, ids, wts, *W)
    torch.cuda.synchronize()
    side, busy = torch.cuda.Stream(), torch.randn(4096, 4096, device="cuda")
    sizes = [moe.moe_sort_workspace_bytes(T, K, E) + 256, mxfp4.moe_layer_workspace_bytes(T, K, n, ff, E) + 256]
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        with torch.cuda.stream(side):
            for _ in range(4):
                busy = torch.tanh(busy @ busy)
        got = moe.moe_sort(ids, E, stream=side)
        out = mxfp4.moe_layer(x, ids, wts, *W, stream=side)
        for size in sizes:
            torch.empty(size, dtype=torch.uint8, device="cuda").fill_(0x7f)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        assert torch.equal(out, want_out)
        owner = {}
        for segment in torch.cuda.memory_snapshot():
            owner[segment["address"]] = (segment["address"] + segment["total_size"], segment["stream"])
        for t in (*got, out):
            assert [s for a, (b, s) in owner.items() if a <= t.data_ptr() < b] == [side.cuda_stream]
