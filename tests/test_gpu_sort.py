"""Tokens sorted by expert, the way back, and their gradients, against plain forms in 64 bits. Every operator sums in
32 bits and rounds once, so a float output may be off by the bound of such a sum: for m terms m * 2^-24 of the sum of their
magnitudes, and half a step of the output's type."""
import numpy as np
import pytest
import torch

from flashrt_b200 import moe

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def make_ids(T, K, E, seed, drop=0.0):
    g = gen(seed)
    ids = torch.stack([torch.randperm(E, generator=g)[:K] for _ in range(T)]) if T else torch.zeros(0, K)
    ids = ids.to(torch.int32)
    if drop:
        ids[torch.rand(T, K, generator=g) < drop] = -1
        ids[-1] = -1                       # a token with no slot at all
    return ids


def plan(ids, E):
    """offsets, slot_of, row_of by a plain stable sort."""
    flat = ids.reshape(-1).long().numpy()
    live = (flat >= 0) & (flat < E)
    order = np.array(sorted(np.nonzero(live)[0], key=lambda s: (flat[s], s)), dtype=np.int64)
    slot_of = np.full(flat.size, -1, dtype=np.int32)
    row_of = np.full(flat.size, -1, dtype=np.int32)
    slot_of[:order.size] = order
    row_of[order] = np.arange(order.size)
    offsets = np.concatenate([[0], np.cumsum([(flat == e).sum() for e in range(E)])]).astype(np.int32)
    return offsets, slot_of, row_of.reshape(tuple(ids.shape))


@pytest.mark.parametrize("T,K,E,drop", [(0, 2, 8, 0), (1, 1, 1, 0), (1, 10, 512, 0), (37, 10, 512, 0.2), (102, 10, 300, 0), (103, 10, 300, 0.3), (1000, 8, 128, 0.05),
                                        (513, 32, 33, 0.5), (7000, 10, 512, 0.1), (2049, 1, 4096, 0), (100, 4, 4095, 0)])
def test_sort(T, K, E, drop):
    ids = make_ids(T, K, E, 11 * T + K + E, drop)
    offsets, slot_of, row_of = moe.moe_sort(ids.cuda(), E)
    want = plan(ids, E)
    for got, w in zip((offsets, slot_of, row_of), want):
        assert got.dtype == torch.int32 and np.array_equal(got.cpu().numpy(), w)


def test_sort_same_expert_twice_and_everything_on_one_expert():
    ids = torch.zeros(900, 3, dtype=torch.int32)       # every slot names expert 0, three times a token
    ids[5:9] = -1
    got = moe.moe_sort(ids.cuda(), 2)
    for a, b in zip(got, plan(ids, 2)):
        assert np.array_equal(a.cpu().numpy(), b)


def test_sort_reports_an_id_beyond_the_experts():
    for T in (5, 3000):
        ids = make_ids(T, 4, 16, 3)
        ids[T // 2, 1] = 16
        ws = moe.workspace(moe.moe_sort_workspace_bytes(T, 4, 16))
        got = moe.moe_sort(ids.cuda(), 16, ws=ws)
        for a, b in zip(got, plan(ids, 16)):           # the slot has no row; all others have theirs
            assert np.array_equal(a.cpu().numpy(), b)
        with pytest.raises(moe.FrxError, match=f"slot {T // 2 * 4 + 1}"):
            moe.workspace_status(ws)
        moe.workspace_status(ws)                       # reported once
        moe.moe_sort(make_ids(T, 4, 16, 4).cuda(), 16, ws=ws)
        moe.workspace_status(ws)


def rows(T, n, dtype, seed, layout="contiguous"):
    x = torch.randn(T, n, generator=gen(seed)).to(dtype).cuda()
    if layout == "apart":              # rows that lie apart, 16-byte aligned ones
        wide = torch.full((T, n + 16), float("nan"), dtype=dtype, device="cuda")
        wide[:, :n] = x
        return wide[:, :n]
    if layout == "odd":                # rows that lie an odd number of elements apart, from an odd start
        wide = torch.full((T * (n + 3) + 1,), float("nan"), dtype=dtype, device="cuda")
        view = wide[1:].view(T, n + 3)[:, :n]
        view.copy_(x)
        return view
    return x


def close(got, want, magnitude, terms, dtype):
    """|got - want| <= terms * 2^-24 * magnitude + half a step of dtype around the value (and of its smallest numbers)."""
    got, want, magnitude = got.double().cpu(), want.double(), magnitude.double()
    info = torch.finfo(dtype)
    bound = terms * 2.0 ** -24 * magnitude
    bound = bound + (want.abs() + bound) * info.eps / 2 + info.smallest_normal * info.eps
    assert got.shape == want.shape and bool(torch.isfinite(got).all())
    worst = float(((got - want).abs() - bound).max()) if got.numel() else -1
    assert worst <= 0, worst


SIZES = [(1, 1, 1), (1, 10, 2048), (37, 10, 2560), (5, 3, 7), (64, 8, 384), (9, 32, 130), (300, 2, 33), (3, 6, 5000)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,K,n", SIZES)
@pytest.mark.parametrize("layout", ["contiguous", "apart", "odd"])
def test_rows_there_and_back(T, K, n, dtype, layout):
    E = 48
    ids = make_ids(T, K, E, T + n, 0.25 if T > 2 else 0.0)
    _, _, row_of = plan(ids, E)
    row_of = torch.from_numpy(row_of)
    live, r = row_of >= 0, row_of.clamp(min=0).long()
    dr = row_of.cuda()
    S = T * K
    x, ys, gout = rows(T, n, dtype, 1, layout), rows(S, n, dtype, 2, layout), rows(T, n, dtype, 3, layout)
    gxs = rows(S, n, dtype, 4, layout)
    wts = torch.rand(T, K, generator=gen(5))
    # out: a copy, bit for bit; rows that no slot has keep what they held
    xs = rows(S, n, dtype, 6, layout)
    want = xs.clone().cpu()
    want[r[live]] = x.cpu().unsqueeze(1).expand(T, K, n)[live]
    assert torch.equal(moe.moe_sort_rows(x, dr, out=xs).cpu(), want)
    # back, with weights and without
    picked = torch.where(live.unsqueeze(2), ys.cpu().double()[r], 0.0)
    terms = picked * wts.double().unsqueeze(2)
    close(moe.moe_unsort_rows(ys, wts.cuda(), dr), terms.sum(1), terms.abs().sum(1), K, dtype)
    terms = torch.where(live.unsqueeze(2), gxs.cpu().double()[r], 0.0)
    close(moe.moe_sort_rows_backward(gxs, dr), terms.sum(1), terms.abs().sum(1), K, dtype)
    # the gradients of the way back
    gys = rows(S, n, dtype, 7, layout)
    want = gys.cpu().double()
    want[r[live]] = (wts.double().unsqueeze(2) * gout.cpu().double().unsqueeze(1))[live]
    got, gw = moe.moe_unsort_rows_backward(gout, ys, wts.cuda(), dr, gys=gys)
    assert got.data_ptr() == gys.data_ptr()
    close(got, want, want.abs(), 1, dtype)
    terms = torch.where(live.unsqueeze(2), picked * gout.cpu().double().unsqueeze(1), 0.0)
    close(gw, terms.sum(2), terms.abs().sum(2), n, torch.float32)
    assert bool((gw.cpu()[~live] == 0).all())


def test_rows_more_than_32_bits_apart():
    T, K, n, E = 3, 2, 64, 4
    far = 1_200_000_000                                  # elements between rows; the third begins at 2.4 * 10^9
    row_of = torch.tensor([[2, 0], [-1, 1], [0, -1]], dtype=torch.int32).cuda()
    wts = torch.rand(T, K, generator=gen(1)).cuda()
    flat = torch.empty(2 * far + n, dtype=torch.bfloat16, device="cuda")
    place = flat.as_strided((T, n), (far, 1))
    x = torch.randn(T, n, generator=gen(2)).bfloat16().cuda()
    near = torch.zeros(T, n, dtype=torch.bfloat16, device="cuda")
    place.zero_()
    plan_of = torch.tensor([[2, -1], [1, -1], [0, -1]], dtype=torch.int32).cuda()
    assert torch.equal(moe.moe_sort_rows(x, plan_of, out=place), moe.moe_sort_rows(x, plan_of, out=near))
    assert torch.equal(moe.moe_unsort_rows(place, wts, row_of), moe.moe_unsort_rows(near, wts, row_of))
    assert torch.equal(moe.moe_sort_rows_backward(place, row_of), moe.moe_sort_rows_backward(near, row_of))
    gys = torch.zeros_like(near)
    a = moe.moe_unsort_rows_backward(x, near, wts, plan_of, gys=gys)
    far_gys = torch.empty(2 * far + n, dtype=torch.bfloat16, device="cuda").as_strided((T, n), (far, 1))
    far_gys.zero_()
    b = moe.moe_unsort_rows_backward(x, place, wts, plan_of, gys=far_gys)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_rows_with_infinities_and_nan_in_rows_that_nobody_has():
    """A row without a slot may hold anything: nothing of it is read into a sum."""
    ids = make_ids(20, 4, 8, 1, 0.4)
    _, _, row_of = plan(ids, 8)
    n_live = int((row_of >= 0).sum())
    ys = torch.randn(80, 64, generator=gen(2)).cuda()
    wts = torch.rand(20, 4, generator=gen(3)).cuda()
    dr = torch.from_numpy(row_of).cuda()
    a = moe.moe_unsort_rows(ys, wts, dr)
    dirty = ys.clone()
    dirty[n_live:] = float("nan")
    wts2 = torch.where(dr < 0, float("inf"), wts)     # nor is the weight of such a slot
    assert torch.equal(moe.moe_unsort_rows(dirty, wts2, dr), a)
    assert torch.equal(moe.moe_sort_rows_backward(dirty, dr), moe.moe_sort_rows_backward(ys, dr))
    gout = torch.randn(20, 64, generator=gen(4)).cuda()
    _, gw = moe.moe_unsort_rows_backward(gout, dirty, wts2, dr)
    assert torch.equal(gw, moe.moe_unsort_rows_backward(gout, ys, wts, dr)[1])


def test_rows_that_the_buffer_does_not_have():
    """A plan made for more rows than a buffer holds: what has no row there is left out, nothing beyond the buffer is touched."""
    T, K, n, E = 30, 4, 64, 8
    ids = make_ids(T, K, E, 9)
    _, _, row_of = plan(ids, E)
    dr = torch.from_numpy(row_of).cuda()
    x, big = rows(T, n, torch.float32, 1), torch.full((T * K, n), 7.0, device="cuda")
    moe.moe_sort_rows(x, dr, out=big[:50])
    assert bool((big[50:] == 7).all())
    cut = torch.where(dr < 50, dr, -1)
    full = moe.moe_sort_rows(x, dr)
    assert torch.equal(big[:50], full[:50])
    wts = torch.rand(T, K, generator=gen(2)).cuda()
    assert torch.equal(moe.moe_unsort_rows(full[:50], wts, dr), moe.moe_unsort_rows(full, wts, cut))


@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 512, 10), (37, 512, 10), (293, 128, 8), (5, 33, 32), (9, 1023, 7), (64, 1024, 32)])
def test_route_backward(T, E, k):
    """Against the formula in 64 bits, and against differences of the router itself in 64 bits."""
    logits = torch.randn(T, E, generator=gen(T + E + k)).cuda() * 2
    ids, wts = moe.moe_route_topk(logits, k)
    gw = torch.randn(T, k, generator=gen(8)).cuda()
    got = moe.moe_route_topk_backward(gw, wts, ids, E).double().cpu()
    l, i, g = logits.double().cpu(), ids.long().cpu(), gw.double().cpu()
    w = torch.softmax(l.gather(1, i), 1)
    want = torch.zeros(T, E, dtype=torch.float64).scatter_(1, i, w * (g - (w * g).sum(1, keepdim=True)))
    # the weights are within 2^-20 of the softmax (a double sum, rounded), k products and sums of 2^-24 each, one more product
    bound = (k + 20) * 2.0 ** -24 * torch.zeros(T, E, dtype=torch.float64).scatter_(1, i, w * (g.abs() + (w * g).abs().sum(1, keepdim=True))) * 2
    assert bool(((got - want).abs() <= bound).all())
    # differences: loss = sum of gw * weights as the softmax of all logits, restricted to the chosen and renormalized
    p = lambda z: torch.softmax(z, 1)                                                    # noqa: E731
    loss = lambda z: (g * p(z).gather(1, i) / p(z).gather(1, i).sum(1, keepdim=True)).sum(1)   # noqa: E731
    h = 1e-5
    for e in {0, E - 1, int(i[0, 0]), int(i[0, -1])}:
        d = torch.zeros(1, E, dtype=torch.float64)
        d[0, e] = h
        slope = (loss(l + d) - loss(l - d)) / (2 * h)
        assert float((slope - got[:, e]).abs().max()) < 1e-5


def test_route_backward_ids_without_a_logit_and_named_twice():
    ids = torch.tensor([[3, 3, -1, 40], [0, 1, 0, 0]], dtype=torch.int32)
    wts, gw = torch.rand(2, 4, generator=gen(1)), torch.randn(2, 4, generator=gen(2))
    got = moe.moe_route_topk_backward(gw.cuda(), wts.cuda(), ids.cuda(), 40).cpu()
    term = (wts.double() * (gw.double() - (wts.double() * gw.double()).sum(1, keepdim=True)))
    want = torch.zeros(2, 40, dtype=torch.float64)
    want[0, 3] = term[0, 0] + term[0, 1]
    want[1, 0] = term[1, 0] + term[1, 2] + term[1, 3]
    want[1, 1] = term[1, 1]
    assert float((got - want).abs().max()) < 1e-6
    assert bool((got[want == 0] == 0).all())


@pytest.mark.parametrize("drop", [0.0, 0.3])
def test_training_step_around_experts_of_the_program(drop):
    """Logits -> router -> sort -> experts in torch -> back -> loss, forward and down to the gradients of x and of the logits, in
    float32; against torch.autograd in 64 bits. Tolerance: the longest sums have 96 terms and pass five operators, 5 * 96 * 2^-24 = 3e-5."""
    T, E, K, n = 50, 12, 3, 96
    g = gen(6)
    x, logits = torch.randn(T, n, generator=g), torch.randn(T, E, generator=g)
    w = torch.randn(E, n, n, generator=g) / n ** 0.5
    keep = torch.rand(T, K, generator=g) >= drop
    target = torch.randn(T, n, generator=g)
    # the library's operators
    ids, wts = moe.moe_route_topk(logits.cuda(), K)
    kept = torch.where(keep.cuda(), ids, -1)
    offsets, slot_of, row_of = moe.moe_sort(kept, E)
    xs = moe.moe_sort_rows(x.cuda(), row_of, out=torch.zeros(T * K, n, device="cuda"))
    at = offsets.tolist()
    ys = torch.zeros_like(xs)
    for e in range(E):
        ys[at[e]:at[e + 1]] = torch.tanh(xs[at[e]:at[e + 1]].double() @ w[e].double().cuda()).float()
    out = moe.moe_unsort_rows(ys, wts, row_of)
    gout = 2 * (out - target.cuda())
    gys, gw = moe.moe_unsort_rows_backward(gout, ys, wts, row_of, gys=torch.zeros_like(ys))
    gxs = torch.zeros_like(xs)
    for e in range(E):
        s = slice(at[e], at[e + 1])
        gxs[s] = ((gys[s].double() * (1 - ys[s].double() ** 2)) @ w[e].double().cuda().t()).float()
    gx = moe.moe_sort_rows_backward(gxs, row_of)
    gl = moe.moe_route_topk_backward(gw, wts, ids, E)
    # the same by torch in 64 bits
    xd, ld = x.double().requires_grad_(), logits.double().requires_grad_()
    top = ids.long().cpu()
    p = torch.softmax(ld, 1).gather(1, top)
    p = p / p.sum(1, keepdim=True)
    y = torch.tanh(torch.einsum("tn,tknm->tkm", xd, w.double()[top]))
    o = (torch.where(keep, p, 0.0).unsqueeze(2) * y).sum(1)
    ((o - target.double()) ** 2).sum().backward()
    for got, want in ((out, o.detach()), (gx, xd.grad), (gl, ld.grad)):
        scale = float(want.abs().max())
        assert float((got.cpu().double() - want).abs().max()) <= 3e-5 * scale


def test_sort_captured_and_on_another_stream():
    """A graph of the whole chain, replayed on new values, gives what the eager calls give."""
    T, K, E, n = 130, 8, 64, 256
    ids, x, wts = make_ids(T, K, E, 5, 0.1).cuda(), rows(T, n, torch.bfloat16, 1), torch.rand(T, K, generator=gen(2)).cuda()
    ws = moe.workspace(moe.moe_sort_workspace_bytes(T, K, E))
    xs = torch.zeros(T * K, n, dtype=torch.bfloat16, device="cuda")

    def chain():
        o, s, r = moe.moe_sort(ids, E, ws=ws)
        moe.moe_sort_rows(x, r, out=xs)
        return o, s, r, moe.moe_unsort_rows(xs, wts, r)

    chain()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = chain()
    for seed in (21, 22):
        ids.copy_(make_ids(T, K, E, seed, 0.1))
        x.copy_(rows(T, n, torch.bfloat16, seed))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        seen = [t.clone() for t in got]
        for a, b in zip(seen, chain()):
            assert torch.equal(a, b)


def test_refusals():
    ids = torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    x, w = torch.zeros(4, 8, device="cuda"), torch.zeros(4, 2, device="cuda")
    ys = torch.zeros(8, 8, device="cuda")
    bad = [lambda: moe.moe_sort(ids.long(), 8), lambda: moe.moe_sort(ids.cpu(), 8), lambda: moe.moe_sort(ids[:, :1], 8), lambda: moe.moe_sort(ids, 0),
           lambda: moe.moe_sort(ids, 4097), lambda: moe.moe_sort(torch.zeros(4, 33, dtype=torch.int32, device="cuda"), 64),
           lambda: moe.moe_sort(torch.zeros(600, 2, dtype=torch.int32, device="cuda"), 64, ws=torch.zeros(600, dtype=torch.uint8, device="cuda")),
           lambda: moe.moe_sort_rows(x.double(), ids), lambda: moe.moe_sort_rows(x.t(), ids), lambda: moe.moe_sort_rows(x, ids[:3]),
           lambda: moe.moe_sort_rows(x, ids, out=ys.half()), lambda: moe.moe_sort_rows(x, ids, out=ys[:, :7]), lambda: moe.moe_sort_rows(x.cpu(), ids),
           lambda: moe.moe_sort_rows(x.expand(4, 8)[:1].expand(4, 8), ids),
           lambda: moe.moe_unsort_rows(ys, w.half(), ids), lambda: moe.moe_unsort_rows(ys, w[:, :1], ids), lambda: moe.moe_unsort_rows(ys, w, ids, out=x[:3]),
           lambda: moe.moe_unsort_rows_backward(x.half(), ys, w, ids), lambda: moe.moe_unsort_rows_backward(x[:3], ys, w, ids),
           lambda: moe.moe_route_topk_backward(w, w, ids, 1), lambda: moe.moe_route_topk_backward(w, w, ids, 1025), lambda: moe.moe_route_topk_backward(w[:2], w, ids, 8)]
    for i, call in enumerate(bad):
        with pytest.raises(moe.FrxError):
            call()
            raise AssertionError(f"call {i} was not refused")


def test_sorts_of_several_threads_with_other_numbers_of_experts():
    """Threads that sort for 1,400, 2,500 and 4,096 experts at once, whose kernels take different amounts of shared memory: no call is refused, all plans are right."""
    import ctypes as C
    import threading

    from flashrt_b200.lib import lib
    T, K = 50, 4
    jobs = []
    for E in (1400, 2500, 4096):
        ids = make_ids(T, K, E, E)
        jobs.append((E, ids, ids.cuda(), [torch.empty(m, dtype=torch.int32, device="cuda") for m in (E + 1, T * K, T * K)], torch.cuda.Stream(), []))
    torch.cuda.synchronize()

    def run(E, ids, on_device, outs, stream, codes):
        ptr = [C.c_void_p(t.data_ptr()) for t in (on_device, *outs)]
        for _ in range(4000):
            codes.append(lib.frx_moe_sort(C.c_void_p(stream.cuda_stream), ptr[0], T, K, E, ptr[1], ptr[2], ptr[3], None, 0))

    threads = [threading.Thread(target=run, args=j) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for E, ids, _, outs, _, codes in jobs:
        assert set(codes) == {0}, (E, sum(c != 0 for c in codes))
        for got, want in zip(outs, plan(ids, E)):
            assert np.array_equal(got.cpu().numpy(), want.reshape(-1))


def test_calls_on_values_that_the_call_in_front_rewrites_in_place():
    """Chains of this library's own kernels, each of which lets the next one start early, over the same buffers with other values every time, without a wait: what every
    call gives when the GPU is waited for in between."""
    from flashrt_b200 import mxfp4
    T, K, E, n, steps = 600, 6, 24, 1024, 12
    S = T * K
    g = gen(4)
    codes = [torch.randint(0, 256, (S, n // 2), generator=g, dtype=torch.uint8).cuda() for _ in range(steps)]
    scales = torch.full((S, n // 32), 125, dtype=torch.uint8).cuda()
    logits = [torch.randn(T, E, generator=g).cuda() for _ in range(steps)]
    buffers = [torch.zeros(S, n, device="cuda") for _ in range(4)]

    def chain(wait):
        x, ys, gys, out = buffers
        results = []

        def do(call, *args, **kwargs):
            got = call(*args, **kwargs)
            if wait:
                torch.cuda.synchronize()
            return got

        for c, l in zip(codes, logits):
            ids, wts = do(moe.moe_route_topk, l, K)
            _, _, row_of = do(moe.moe_sort, ids, E)
            do(mxfp4.dequantize, c, scales, out=x)
            do(moe.moe_sort_rows, x[:T], row_of, out=ys)
            do(moe.moe_unsort_rows, ys, wts, row_of, out=out[:T])
            _, gw = do(moe.moe_unsort_rows_backward, out[:T], ys, wts, row_of, gys=gys)
            do(moe.moe_sort_rows_backward, gys, row_of, out=out[T:2 * T])
            gl = do(moe.moe_route_topk_backward, gw, wts, ids, E)
            q = do(mxfp4.quantize, out[:2 * T])
            results.append([t.clone() for t in (out[:2 * T], gys, gw, gl, *q)])
        torch.cuda.synchronize()
        return results

    want = chain(True)
    for _ in range(3):
        for a, b in zip(chain(False), want):
            for s, t in zip(a, b):
                assert torch.equal(s, t)
