"""Products of sorted rows with matrices of their experts in 16 bits, and both gradients, against plain forms in 64 bits.

Tolerance. A product of two 16-bit elements is exact in 32 bits, and a sum of m of them in 32 bits is off by at most m steps of 2^-23 of the sum of their
magnitudes, whatever the order and whether an addition rounds or cuts; then half a step of the output's type (for float16 also half its smallest subnormal)."""
import pytest
import torch

from flashrt_b200 import lib as L
from flashrt_b200 import moe

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def normal(g, *shape):
    return torch.randn(*shape, generator=g, dtype=torch.float32)


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def plan(counts, behind=0):
    """offsets of experts with so many rows, and how many rows there are with those that nobody has."""
    offsets = [0]
    for c in counts:
        offsets.append(offsets[-1] + c)
    return torch.tensor(offsets, dtype=torch.int32), offsets[-1] + behind


def bound(magnitudes, m, want, dtype):
    """What a result may be off by: magnitudes = the sums of the products' magnitudes, m = how many they are."""
    tiny = 2.0 ** -25 if dtype == F16 else 2.0 ** -150
    return m * 2.0 ** -23 * magnitudes + torch.finfo(dtype).eps / 2 * (want.abs() + m * 2.0 ** -23 * magnitudes) + tiny


def close(got, want, tol, live=None):
    got = got.double().cpu()
    if live is not None:
        got, want, tol = got[live], want[live], tol[live]
    off = (got - want).abs()
    assert torch.isfinite(got).all()
    assert (off <= tol).all(), f"off by {float((off / tol).max()):.2f} of what is allowed"


def apart(t, pad):
    """The same values with `pad` elements of NaN between the rows (a multiple of eight keeps them on 16-byte boundaries)."""
    wide = torch.full((*t.shape[:-1], t.shape[-1] + pad), float("nan"), dtype=t.dtype, device=t.device)
    wide[..., :t.shape[-1]] = t
    return wide[..., :t.shape[-1]]


def rows_of(offsets):
    at = offsets.tolist()
    return list(enumerate(zip(at, at[1:])))


COUNTS = {
    "one": [1], "none": [0, 0, 3, 0], "few": [1, 0, 2, 5, 0, 1], "around16": [15, 16, 17, 1, 31, 33], "around256": [255, 256, 257], "ragged": [700, 3, 0, 64, 65, 63, 1],
    "many": [(i * 37) % 11 for i in range(300)],
}


def case(counts, n, rows, dtype, seed, behind=5):
    g = gen(seed)
    offsets, S = plan(counts, behind)
    x, gy = normal(g, S, n).to(dtype), normal(g, S, rows).to(dtype)
    w = (normal(g, len(counts), rows, n) / n ** 0.5).to(dtype)
    live = int(offsets[-1])
    x[live:], gy[live:] = float("nan"), float("nan")           # rows that nobody has are not read into anything
    return offsets, x, w, gy, live


def aligned(t):
    """t in device memory, its rows on 16-byte boundaries."""
    pad = -t.shape[-1] % 8
    return apart(t.cuda(), pad) if pad else t.cuda()


def check_all(offsets, x, w, gy, live, out_dtype, place=aligned):
    S, E, rows, n = x.shape[0], *w.shape
    xd, wd, gyd, od = place(x), place(w), place(gy), offsets.cuda()
    y = torch.full((S, rows), 7.0, dtype=out_dtype, device="cuda")
    gx = torch.full((S, n), 7.0, dtype=out_dtype, device="cuda")
    gw = torch.full((E, rows, n), 7.0, dtype=out_dtype, device="cuda")
    assert moe.moe_matmul(xd, wd, od, out=y) is y
    moe.moe_matmul_backward_x(gyd, wd, od, out=gx)
    moe.moe_matmul_backward_w(gyd, xd, od, out=gw)
    x64, w64, gy64 = x.cuda().double(), w.cuda().double(), gy.cuda().double()
    wy, wx, ww = (torch.zeros_like(t, dtype=torch.float64) for t in (y, gx, gw))
    my, mx, mw = (torch.zeros_like(t) for t in (wy, wx, ww))
    mt = torch.zeros(E, 1, 1, dtype=torch.float64)
    for e, (a, b) in rows_of(offsets):
        wy[a:b], my[a:b] = x64[a:b] @ w64[e].T, x64[a:b].abs() @ w64[e].abs().T
        wx[a:b], mx[a:b] = gy64[a:b] @ w64[e], gy64[a:b].abs() @ w64[e].abs()
        ww[e], mw[e] = gy64[a:b].T @ x64[a:b], gy64[a:b].abs().T @ x64[a:b].abs()
        mt[e] = b - a
    wy, wx, ww, my, mx, mw = (t.cpu() for t in (wy, wx, ww, my, mx, mw))
    close(y, wy, bound(my, n, wy, out_dtype), slice(0, live))
    close(gx, wx, bound(mx, rows, wx, out_dtype), slice(0, live))
    close(gw, ww, bound(mw, mt, ww, out_dtype))
    assert (y[live:] == 7).all() and (gx[live:] == 7).all()    # left as they were


@pytest.mark.parametrize("counts", sorted(COUNTS))
@pytest.mark.parametrize("n,rows", [(64, 128), (200, 72), (2048, 1024)])
def test_products_and_gradients(counts, n, rows):
    if counts == "many" and n > 1000:
        n, rows = 512, 256
    check_all(*case(COUNTS[counts], n, rows, BF16, 3 * n + rows), F32)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("out", [F32, BF16, F16])
@pytest.mark.parametrize("n,rows", [(8, 8), (1, 1), (63, 65), (129, 130), (257, 3), (384, 1280)])
def test_types_and_odd_sizes(dtype, out, n, rows):
    check_all(*case([3, 0, 40, 130, 1], n, rows, dtype, n + rows), out)


@pytest.mark.parametrize("counts", [[1] * 4096, [0] * 4095 + [200], [2000] + [0] * 4095])
def test_many_experts(counts):
    check_all(*case(counts, 72, 40, BF16, 9), BF16)


def test_rows_and_matrices_apart():
    offsets, x, w, gy, live = case([5, 70, 0, 300], 192, 136, F16, 4)
    check_all(offsets, x, w, gy, live, F16, place=lambda t: apart(t.cuda(), 24))
    # what is written has any alignment of an element
    xd, wd, gyd, od = x.cuda(), w.cuda(), gy.cuda(), offsets.cuda()
    for out in (F32, BF16):
        buf = torch.full((x.shape[0] * 137 + 1,), 7.0, dtype=out, device="cuda")
        y = buf[1:].view(x.shape[0], 137)[:, :136]
        moe.moe_matmul(xd, wd, od, out=y)
        assert torch.equal(y[:live], moe.moe_matmul(xd, wd, od, dtype=out)[:live])
        assert (buf[1:].view(-1, 137)[:, 136] == 7).all() and buf[0] == 7 and (y[live:] == 7).all()
        buf = torch.full((4 * 141 * 193 + 1,), 7.0, dtype=out, device="cuda")
        gw = buf[1:].view(4, 141, 193)[:, :136, :192]
        moe.moe_matmul_backward_w(gyd, xd, od, out=gw)
        assert torch.equal(gw, moe.moe_matmul_backward_w(gyd, xd, od, dtype=out))
        assert (buf[1:].view(4, 141, 193)[:, 136:] == 7).all() and (buf[1:].view(4, 141, 193)[:, :, 192] == 7).all()


def test_nan_and_infinity_stay_with_their_expert():
    """Rows and matrices of one expert full of NaN and infinities, beside every border of a tile: the others' results are those without."""
    counts = [20, 17, 300, 1, 64]
    offsets, x, w, gy, live = case(counts, 136, 264, BF16, 8, behind=0)
    od = offsets.cuda()

    def run(x, w, gy):
        x, w, gy = x.cuda(), w.cuda(), gy.cuda()
        return moe.moe_matmul(x, w, od), moe.moe_matmul_backward_x(gy, w, od), moe.moe_matmul_backward_w(gy, x, od)
    want = run(x, w, gy)
    at = offsets.tolist()
    for e in range(len(counts)):
        x2, w2, gy2 = x.clone(), w.clone(), gy.clone()
        x2[at[e]:at[e + 1]], w2[e], gy2[at[e]:at[e + 1]] = float("nan"), float("inf"), float("-inf")
        y, gx, gw = run(x2, w2, gy2)
        others = [i for i in range(len(counts)) if i != e]
        for i in others:
            rows = slice(at[i], at[i + 1])
            assert torch.equal(y[rows], want[0][rows]) and torch.equal(gx[rows], want[1][rows]) and torch.equal(gw[i], want[2][i])
        assert y[at[e]:at[e + 1]].isnan().all() and gw[e].isnan().all()


@pytest.mark.parametrize("out", [F32, BF16, F16])
def test_gradient_added_to_what_is_there(out):
    offsets, x, w, gy, live = case([33, 0, 130], 72, 300, BF16, 6)
    xd, gyd, od = x.cuda(), gy.cuda(), offsets.cuda()
    gyd, xd = aligned(gy), aligned(x)
    old = (normal(gen(1), 3, 300, 72) * 4).to(out).cuda()
    gw = old.clone()
    moe.moe_matmul_backward_w(gyd, xd, od, out=gw, add=True)
    want, mag = old.double().cpu(), old.double().cpu().abs()
    for e, (a, b) in rows_of(offsets):
        want[e] += gy[a:b].double().T @ x[a:b].double()
        mag[e] += gy[a:b].double().abs().T @ x[a:b].double().abs()
    close(gw, want, bound(mag, 131, want, out))
    assert torch.equal(gw[1], old[1])


def test_gradients_are_those_of_differences():
    """For a linear map differences are exact: <gy, f(x + dx, w) - f(x, w)> = <gx, dx>, and the same for w, up to the roundings of sums of 32 bits."""
    offsets, x, w, gy, live = case([7, 0, 50, 19], 96, 80, F16, 12, behind=0)
    g = gen(5)
    dx, dw = normal(g, *x.shape).to(F16), normal(g, *w.shape).to(F16)
    od = offsets.cuda()
    f = lambda x, w: moe.moe_matmul(x.cuda(), w.cuda(), od, dtype=F32).double().cpu()   # noqa: E731
    gx = moe.moe_matmul_backward_x(gy.cuda(), w.cuda(), od, dtype=F32).double().cpu()
    gw = moe.moe_matmul_backward_w(gy.cuda(), x.cuda(), od, dtype=F32).double().cpu()
    G = gy.double()
    # both sides are sums of the same products; each is off by at most (n + rows + count) steps of 2^-23 of the sum of their magnitudes
    for lhs, rhs, mag in ((f(dx, w), gx * dx.double(), f(dx.abs(), w.abs())), (f(x, dw), gw * dw.double(), f(x.abs(), dw.abs()))):
        assert abs(float((G * lhs).sum() - rhs.sum())) <= (96 + 80 + 50) * 2.0 ** -23 * float((G.abs() * mag).sum()) * 1.01


def test_no_rows_at_all():
    w = torch.ones(3, 16, 24, dtype=BF16, device="cuda")
    none, od = torch.zeros(0, 24, dtype=BF16, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    assert moe.moe_matmul(none, w, od).shape == (0, 16)
    gy = torch.zeros(0, 16, dtype=BF16, device="cuda")
    assert moe.moe_matmul_backward_x(gy, w, od).shape == (0, 24)
    buf = torch.full((3, 17, 32), 7.0, device="cuda")
    gw = buf[:, :16, :24]
    moe.moe_matmul_backward_w(gy, none, od, out=gw)
    assert (gw == 0).all() and (buf[:, 16] == 7).all() and (buf[:, :, 24:] == 7).all()
    gw.fill_(3)
    moe.moe_matmul_backward_w(gy, none, od, out=gw, add=True)
    assert (gw == 3).all()
    # rows, none of which belongs to an expert
    gw = moe.moe_matmul_backward_w(torch.full((40, 16), float("nan"), dtype=BF16, device="cuda"), torch.full((40, 24), float("nan"), dtype=BF16, device="cuda"), od)
    assert (gw == 0).all()


def test_plans_that_are_none():
    """Offsets out of range or descending: nothing outside the result is touched, and rows of other experts are right or left out."""
    x, w = torch.randn(100, 64, device="cuda").to(BF16), torch.randn(4, 48, 64, device="cuda").to(BF16)
    for bad in ([-5, 10, 20, 30, 1000], [0, 50, 20, 70, 100], [2 ** 31 - 1, 0, 5, 5, -2 ** 31], [0, 100, 0, 100, 0]):
        od = torch.tensor(bad, dtype=torch.int32, device="cuda")
        buf = torch.full((102, 48), 7.0, dtype=BF16, device="cuda")
        moe.moe_matmul(x, w, od, out=buf[1:101])
        gw = torch.full((6, 48, 64), 7.0, dtype=BF16, device="cuda")
        moe.moe_matmul_backward_w(buf[1:101], x, od, out=gw[1:5])
        assert (buf[0] == 7).all() and (buf[101] == 7).all() and (gw[0] == 7).all() and (gw[5] == 7).all()


def test_same_bits_again_captured_and_on_a_stream():
    offsets, x, w, gy, live = case([70, 0, 600, 19], 256, 192, BF16, 2)
    xd, wd, gyd, od = x.cuda(), w.cuda(), gy.cuda(), offsets.cuda()
    live = slice(0, live)

    def run(stream=None):
        return (moe.moe_matmul(xd, wd, od, stream=stream)[live], moe.moe_matmul_backward_x(gyd, wd, od, stream=stream)[live], moe.moe_matmul_backward_w(gyd, xd, od, stream=stream))
    want = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = run(side)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        captured = run()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    for a, b, c in zip(want, got, captured):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_outputs_more_than_32_bits_apart():
    """Rows of the result so far apart that their distance passes 2^31 elements, and rows of x that do in bytes."""
    offsets = torch.tensor([0, 2, 5], dtype=torch.int32, device="cuda")
    w = torch.randn(2, 16, 64, device="cuda").to(BF16)
    x = torch.randn(5, 64, device="cuda").to(BF16)
    far = 2 ** 29 + 8
    buf = torch.empty(4 * far + 64, dtype=BF16, device="cuda")
    y = buf.as_strided((5, 16), (far, 1))
    want = moe.moe_matmul(x, w, offsets)
    moe.moe_matmul(x, w, offsets, out=y)
    assert torch.equal(y, want)
    x_far = buf.as_strided((5, 64), (far, 1), 0)
    x_far.copy_(x)
    assert torch.equal(moe.moe_matmul(x_far, w, offsets), want)


@pytest.mark.parametrize("out", [F32, BF16])
def test_a_wait_that_runs_out_leaves_nan(out):
    """An expert of half a million rows keeps the warp that zeroes what is behind the last of them waiting for a millisecond or two; with a limit of ten microseconds it gives up, and everyone
    else of its pair of blocks. Nothing hangs, no wrong number is left, and the next call is as if nothing had been."""
    S = 1 << 19
    gy, x, od = torch.randn(S, 64, device="cuda").to(BF16), torch.randn(S, 128, device="cuda").to(BF16), torch.tensor([0, S - 3], dtype=torch.int32, device="cuda")
    want = moe.moe_matmul_backward_w(gy, x, od, dtype=out)
    torch.cuda.synchronize()
    try:
        L.check(L.lib.frx_debug_set_wait_limit_ns(10_000))
        got = moe.moe_matmul_backward_w(gy, x, od, dtype=out)
        torch.cuda.synchronize()
    finally:
        L.check(L.lib.frx_debug_set_wait_limit_ns(0))
    lost = got.isnan()
    assert bool(lost.any()), "no wait ran out"
    assert bool((lost | (got == want)).all()) and torch.equal(moe.moe_matmul_backward_w(gy, x, od, dtype=out), want)


def test_refusals():
    x, w, od = torch.zeros(6, 64, dtype=BF16, device="cuda"), torch.zeros(2, 32, 64, dtype=BF16, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    gy = torch.zeros(6, 32, dtype=BF16, device="cuda")
    f, bx, bw = moe.moe_matmul, moe.moe_matmul_backward_x, moe.moe_matmul_backward_w
    for call in (lambda: f(x.float(), w.float(), od), lambda: f(x.half(), w, od), lambda: f(x[:, :56], w, od), lambda: f(x, w, od[:2]), lambda: f(x, w, od.long()),
                 lambda: f(x, w[0], od), lambda: f(x.t(), w, od), lambda: f(x, w, od, out=gy[:5]), lambda: f(x, w.transpose(1, 2), od), lambda: f(x.cpu(), w, od),
                 lambda: f(torch.zeros(6, 65, dtype=BF16, device="cuda")[:, 1:], w, od), lambda: f(x, w.expand(2, 32, 64)[:1].expand(2, 32, 64), od),
                 lambda: f(torch.zeros(6, 63, dtype=BF16, device="cuda"), torch.zeros(2, 32, 63, dtype=BF16, device="cuda"), od),
                 lambda: f(x, w, od, out=gy, dtype=F32), lambda: bx(x, w, od), lambda: bx(gy, w.half(), od), lambda: bw(gy, x[:5], od), lambda: bw(gy, x.half(), od),
                 lambda: bw(gy, x, od, add=True), lambda: bw(gy, x, od[:0]), lambda: bw(gy, x, od, out=torch.zeros(2, 32, 63, device="cuda")),
                 lambda: bw(gy, x, od, out=torch.zeros(1, 32, 64, device="cuda").expand(2, 32, 64))):
        with pytest.raises(L.FrxError):
            call()


def test_timings_are_kept_apart():
    """Each of these kernels is counted in a class of its own, not with the expert layer's gate and up product or its quantizer."""
    import ctypes as C

    from flashrt_b200 import adapters, mxint8
    x, w, od = torch.zeros(6, 64, dtype=BF16, device="cuda"), torch.zeros(2, 32, 64, dtype=BF16, device="cuda"), torch.tensor([0, 2, 6], dtype=torch.int32, device="cuda")
    gy, a, b = torch.zeros(6, 32, dtype=BF16, device="cuda"), torch.zeros(2, 16, 64, dtype=BF16, device="cuda"), torch.zeros(2, 32, 16, dtype=BF16, device="cuda")
    ms, launches = (C.c_float * 32)(), (C.c_int * 32)()
    L.check(L.lib.frx_profile_begin())
    try:
        moe.moe_matmul(x, w, od)
        moe.moe_matmul_backward_x(gy, w, od)
        moe.moe_matmul_backward_w(gy, x, od)
        adapters.add(gy, x, a, b, od, od[:2])
        h, codes, scales = mxint8.swiglu(x)
        mxint8.swiglu_backward(h, codes, scales)
        mxint8.dequantize(*mxint8.quantize(x))
    finally:
        L.check(L.lib.frx_profile_end(ms, launches, 32))
    counted = {L.lib.frx_profile_class_name(i).decode(): launches[i] for i in range(32) if launches[i]}
    assert counted == {"moe_product": 3, "adapter": 1, "swiglu": 2, "quant_q8": 2}
