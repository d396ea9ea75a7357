"""MXINT8: rows in 8 bits, and SwiGLU with its gradient from rows kept so, against plain forms in 64 bits.

Tolerances. Codes, scales and what they stand for are exact and compared for equality. SwiGLU and its gradient are computed in 32 bits: the sigmoid and its complement have a relative
error of at most (8 + 1.25 |g|) 2^-24 (exponential 2^-22 and |g| 1.25 * 2^-24 of its rounded argument, reciprocal 2^-23, a product), every other step one of 2^-24,
where exp(-|g|) is at least 2^-126; below, the sigmoid may be 0. Then half a step of the result's type."""
import pytest
import torch

from flashrt_b200 import lib as L
from flashrt_b200 import moe, mxint8

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def kept(x):
    """codes, scale bytes and values of finite rows x, in 64 bits."""
    v = x.double().reshape(x.shape[0], -1, 32)
    amax = v.abs().amax(2, keepdim=True)
    e = (torch.frexp(torch.where(amax > 0, amax, 2.0 ** -140)).exponent.long() - 1).clamp(min=-127)
    t = torch.ldexp(v, 6 - e)
    low = t.floor()
    q = (low + ((t - low > 0.5) | ((t - low == 0.5) & (low % 2 != 0)))).clamp(-127, 127)
    return q.view(x.shape).to(torch.int8), (e + 127).squeeze(2).to(torch.uint8), torch.ldexp(q, e - 6).view(x.shape)


def hard(T, n, dtype, seed):
    """Blocks of every magnitude of the type, with halves between codes, values next to 127.5 steps and to powers of two, zeros and the type's extremes."""
    g, info = gen(seed), torch.finfo(dtype)
    lo, hi = (-24, 15) if dtype == torch.float16 else (-148, 127)
    e = torch.randint(lo, hi + 1, (T, n // 32, 1), generator=g).double()
    x = torch.rand(T, n // 32, 32, generator=g, dtype=torch.float64) * 2 - 1
    steps = torch.randint(-255, 256, (T, n // 32, 32), generator=g).double() / 128       # multiples of half a step of the block below
    x = torch.where(torch.rand(T, n // 32, 1, generator=g) < 0.5, x, steps)
    x[:, :, 3] = torch.tensor([1.0, 255 / 128, 1.9999, 1.0])[torch.randint(0, 4, (T, n // 32), generator=g)].double()
    x = (x * torch.exp2(e)).clamp(-info.max, info.max).view(T, n).to(dtype)
    flat = x.view(-1)
    flat[:32] = 0
    if flat.numel() >= 160:
        flat[32:64] = info.tiny * info.eps          # the smallest subnormal
        flat[64], flat[96:128], flat[128] = info.max, -info.tiny, -info.max
    return x


def place(x, layout):
    x = x.cuda()
    if layout == "apart":
        wide = torch.full((x.shape[0], x.shape[1] + 16), float("nan"), dtype=x.dtype, device="cuda")
    elif layout == "odd":
        wide = torch.full((x.shape[0] * (x.shape[1] + 1) + 1,), float("nan"), dtype=x.dtype, device="cuda")[1:].view(x.shape[0], -1)
    else:
        return x
    wide[:, :x.shape[1]] = x
    return wide[:, :x.shape[1]]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,n", [(1, 32), (1, 2560), (3, 96), (37, 2048), (200, 640), (4097, 32), (2500, 2048)])
@pytest.mark.parametrize("layout", ["contiguous", "apart", "odd"])
def test_rows_in_8_bits(T, n, dtype, layout):
    x = hard(T, n, dtype, T + n)
    codes, scales = mxint8.quantize(place(x, layout))
    want_codes, want_scales, want = kept(x)
    assert torch.equal(scales.cpu(), want_scales) and torch.equal(codes.cpu(), want_codes)
    for out in TYPES:
        got = mxint8.dequantize(codes, scales, dtype=out)
        assert got.dtype == out and torch.equal(got.cpu(), want.to(out))           # the one rounding of float16; the others hold every value
        if out != torch.float16:
            assert torch.equal(got.cpu().double(), want)
        buf = place(torch.full((T, n), 7.0, dtype=out), layout)
        assert mxint8.dequantize(codes, scales, out=buf) is buf and torch.equal(buf.cpu(), want.to(out))


@pytest.mark.parametrize("dtype", TYPES)
def test_nan_infinity_and_what_is_around_them(dtype):
    x = torch.randn(6, 96, generator=gen(1)).to(dtype)
    x[0, 5], x[1, 40], x[2, 95], x[3, 0] = float("nan"), float("inf"), -float("inf"), float("nan")
    codes, scales = mxint8.quantize(x.cuda())
    bad = torch.zeros(6, 3, dtype=torch.bool)
    bad[0, 0] = bad[1, 1] = bad[2, 2] = bad[3, 0] = True
    assert torch.equal(scales.cpu() == 255, bad) and (codes.cpu().view(6, 3, 32)[bad] == 0).all()
    got = mxint8.dequantize(codes, scales).cpu().view(6, 3, 32)
    assert got[bad].isnan().all()
    clean = torch.where(bad.repeat_interleave(32, 1), torch.zeros((), dtype=dtype), x)
    assert torch.equal(got[~bad].double(), kept(clean)[2].view(6, 3, 32)[~bad])


def hidden(g, u):
    """g s(g) u and what it may be off by before it is rounded."""
    h = g * torch.sigmoid(g) * u
    return h, h.abs() * (16 + 1.25 * g.abs()) * 2.0 ** -24 + (g * u).abs() * 2.0 ** -126


def near(got, want, tol, dtype):
    tiny = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -149
    tol = tol + torch.finfo(dtype).eps / 2 * (want.abs() + tol) + tiny
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    off = (got - want).abs()
    assert (off <= tol).all(), f"off by {float((off / tol).max()):.2f} of what is allowed"


def gate_up(T, ff, dtype, seed):
    g = gen(seed)
    gu = torch.randn(T, 2 * ff, generator=g) * torch.exp2(torch.randint(-6, 4, (T, 1), generator=g).float())
    flat = gu.view(-1)
    special = torch.tensor([0.0, -0.0, -1.2784645, 30.0, -30.0, 87.0, -87.0, -88.5, 100.0, -100.0, -200.0, 1e-6, -1e-6])
    flat[:13 if flat.numel() >= 64 else 0] = special[:13 if flat.numel() >= 64 else 0]
    return gu.to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("S,ff", [(1, 32), (1, 512), (7, 96), (301, 640), (9000, 512)])
@pytest.mark.parametrize("layout", ["contiguous", "apart", "odd"])
def test_swiglu_and_its_gradient(S, ff, dtype, layout):
    gu = gate_up(S, ff, dtype, S + ff)
    gh = (torch.randn(S, ff, generator=gen(S))).to(dtype)
    h, codes, scales = mxint8.swiglu(place(gu, layout))
    v = gu.double()
    near(h, *hidden(v[:, :ff], v[:, ff:]), dtype)
    want_codes, want_scales, k = kept(gu)
    assert torch.equal(codes.cpu(), want_codes) and torch.equal(scales.cpu(), want_scales)
    buf = place(torch.full((S, ff), 7.0, dtype=dtype), layout)
    h2, codes2, scales2 = mxint8.swiglu(gu.cuda(), out=buf)
    assert h2 is buf and torch.equal(h2, h) and torch.equal(codes2, codes) and torch.equal(scales2, scales)

    g, u, d = k[:, :ff], k[:, ff:], gh.double()
    s, c = torch.sigmoid(g), torch.sigmoid(-g)
    want = torch.cat((d * u * s * (1 + g * c), d * g * s), 1)
    error = (24 + 2.5 * g.abs()) * 2.0 ** -24
    tol = torch.cat(((d * u * s).abs() * (1 + (g * c).abs()) * error, (d * g * s).abs() * error), 1) + torch.cat(((d * u).abs() * (1 + g.abs()), (d * g).abs()), 1) * 2.0 ** -126
    ggu, again = mxint8.swiglu_backward(place(gh, layout), codes, scales)
    near(ggu, want, tol, dtype)
    near(again, *hidden(g, u), dtype)
    buf = place(torch.full((S, 2 * ff), 7.0, dtype=dtype), layout)
    ggu2, none = mxint8.swiglu_backward(gh.cuda(), codes, scales, out=buf, hidden=False)
    assert ggu2 is buf and none is None and torch.equal(ggu2, ggu)


def test_gradient_is_that_of_differences():
    """(f(x + d) - f(x - d)) / 2d of the formula in 64 bits, at what was kept: off by its third derivative, d^2 / 6 of at most 2 |u| + 2, and what 32 bits leave."""
    gu = gate_up(64, 128, torch.float32, 5).clamp(-20, 20)
    _, codes, scales = mxint8.swiglu(gu.cuda())
    k = mxint8.dequantize(codes, scales).double().cpu()
    g, u = k[:, :128], k[:, 128:]
    one = torch.ones(64, 128, device="cuda")
    ggu, _ = mxint8.swiglu_backward(one, codes, scales)
    d = 2.0 ** -16
    f = lambda g, u: g * torch.sigmoid(g) * u   # noqa: E731
    dg, du = (f(g + d, u) - f(g - d, u)) / (2 * d), (f(g, u + d) - f(g, u - d)) / (2 * d)
    # 64-bit differences: 2^-52 of f over d
    tol = d * d * (2 * u.abs() + 2) + (f(g, u).abs() + 1) * 2.0 ** -52 / d + ((1 + g.abs()) * (1 + u.abs())) * (25 + 2.5 * g.abs()) * 2.0 ** -24
    got = ggu.double().cpu()
    assert ((got[:, :128] - dg).abs() <= tol).all() and ((got[:, 128:] - du).abs() <= tol).all()


def test_nan_reaches_the_gradient_of_its_block_alone():
    gu = torch.randn(4, 128, generator=gen(3))
    gu[1, 3], gu[2, 100] = float("nan"), float("inf")
    h, codes, scales = mxint8.swiglu(gu.cuda())
    ggu, again = mxint8.swiglu_backward(torch.ones(4, 64, device="cuda"), codes, scales)
    bad = torch.zeros(4, 64, dtype=torch.bool)
    bad[1, :32] = bad[2, 32:] = True
    assert torch.equal(again.cpu().isnan(), bad)
    assert torch.equal(ggu.cpu()[:, :64].isnan(), bad) and ggu.cpu()[1, 64:96].isnan().all() and torch.isfinite(ggu[0]).all() and torch.isfinite(ggu[3]).all()
    assert h[1, 3].isnan() and torch.isfinite(h[0]).all()


def test_nothing_to_do_captured_and_on_a_stream():
    for T, n in ((0, 64), (3, 0)):
        codes, scales = mxint8.quantize(torch.zeros(T, n, device="cuda"))
        assert codes.shape == (T, n) and scales.shape == (T, n // 32) and mxint8.dequantize(codes, scales).shape == (T, n)
    h, codes, scales = mxint8.swiglu(torch.zeros(0, 64, device="cuda"))
    assert h.shape == (0, 32) and mxint8.swiglu_backward(h, codes, scales)[0].shape == (0, 64)
    gu, gh = gate_up(300, 256, torch.bfloat16, 9).cuda(), torch.randn(300, 256, device="cuda").to(torch.bfloat16)

    def run(stream=None):
        h, codes, scales = mxint8.swiglu(gu, stream=stream)
        return (h, codes, scales, *mxint8.swiglu_backward(gh, codes, scales, stream=stream), mxint8.dequantize(*mxint8.quantize(gu, stream=stream), dtype=torch.bfloat16, stream=stream))
    want = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = run(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run()
    graph.replay()
    torch.cuda.synchronize()
    for a, b, c in zip(want, got, captured):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_refusals():
    x = torch.zeros(4, 64, device="cuda")
    codes, scales = mxint8.quantize(x)
    gh = torch.zeros(4, 32, device="cuda")
    for call in (lambda: mxint8.quantize(x[:, :40]), lambda: mxint8.quantize(x.double()), lambda: mxint8.quantize(x.cpu()), lambda: mxint8.quantize(x.t()),
                 lambda: mxint8.dequantize(codes, scales[:, :1]), lambda: mxint8.dequantize(codes.view(torch.uint8), scales), lambda: mxint8.dequantize(codes, scales, dtype=torch.float64),
                 lambda: mxint8.dequantize(codes, scales, out=x[:3]), lambda: mxint8.swiglu(torch.zeros(4, 96, device="cuda")), lambda: mxint8.swiglu(x, out=gh.half()),
                 lambda: mxint8.swiglu_backward(x, codes, scales), lambda: mxint8.swiglu_backward(gh, codes, scales, out=gh), lambda: mxint8.swiglu_backward(gh.cpu(), codes, scales)):
        with pytest.raises(L.FrxError):
            call()


def test_experts_are_trained_with_rows_kept_in_8_bits():
    """A step of an expert layer through all of its calls: sort, products, SwiGLU that keeps 8 bits, back to tokens, and the whole way back. Gradients against those of
    the same computation in 64 bits at the values that were kept."""
    T, K, E, n, ff = 75, 3, 6, 128, 96
    g, dt = gen(4), torch.bfloat16
    x, gout = torch.randn(T, n, generator=g).to(dt), torch.randn(T, n, generator=g).to(dt)
    w1, w2 = (torch.randn(E, 2 * ff, n, generator=g) / n ** 0.5).to(dt), (torch.randn(E, n, ff, generator=g) / ff ** 0.5).to(dt)
    logits = torch.randn(T, E, generator=g)
    xd, gd, w1d, w2d = x.cuda(), gout.cuda(), w1.cuda(), w2.cuda()
    ids, wts = moe.moe_route_topk(logits.cuda(), K)[:2]
    offsets, slot_of, row_of = moe.moe_sort(ids, E)
    xs = moe.moe_sort_rows(xd, row_of)
    x_kept = mxint8.quantize(xs)
    h, codes, scales = mxint8.swiglu(moe.moe_matmul(xs, w1d, offsets))
    ys = moe.moe_matmul(h, w2d, offsets)
    out = moe.moe_unsort_rows(ys, wts, row_of)
    gys, gwts = moe.moe_unsort_rows_backward(gd, ys, wts, row_of)
    gh = moe.moe_matmul_backward_x(gys, w2d, offsets)
    ggu, again = mxint8.swiglu_backward(gh, codes, scales)
    gw2 = moe.moe_matmul_backward_w(gys, again, offsets, dtype=torch.float32)
    gw1 = moe.moe_matmul_backward_w(ggu, mxint8.dequantize(*x_kept, dtype=dt), offsets, dtype=torch.float32)
    gx = moe.moe_sort_rows_backward(moe.moe_matmul_backward_x(ggu, w1d, offsets), row_of)
    glogits = moe.moe_route_topk_backward(gwts, wts, ids, E)

    # the same in 64 bits, without rounding or 8 bits, by automatic differentiation
    leaves = [t.double().requires_grad_() for t in (x, w1, w2, logits)]
    X, W1, W2, LG = leaves
    idc = ids.cpu().long()
    p = torch.softmax(LG.gather(1, idc), 1)
    gu = torch.einsum("tn,tkmn->tkm", X, W1[idc])
    hh = torch.nn.functional.silu(gu[..., :ff]) * gu[..., ff:]
    want = (p.unsqueeze(2) * torch.einsum("tkm,tknm->tkn", hh, W2[idc])).sum(1)
    want.backward(gout.double())

    def relative(got, want):
        return float((got.double().cpu() - want).norm() / want.norm())
    # forward: three roundings to bfloat16 in a chain (rows, h, y) of at most 2^-9 each in the root mean square, and that of the result
    assert relative(out, want.detach()) < 4 * 2.0 ** -9
    # gradients: as many roundings again, and what 8 bits leave of gate, up and x: half a step is at most 2^-7 of a block's largest value, 2^-7 / sqrt(3) of it in the root mean
    # square, which for normal values (the largest of 32 is about 2.5 of their deviation and a power of two or less above 2^e) is below 2.5 * 2^-7 / sqrt(3) = 0.0113 of their own root
    # mean square; each enters a gradient at most twice
    for got, leaf in zip((gx, gw1, gw2, glogits), leaves):
        assert relative(got, leaf.grad) < 8 * 2.0 ** -9 + 3 * 2 * 0.0113
