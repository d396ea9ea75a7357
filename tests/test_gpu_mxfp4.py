"""MXFP4: quantizer, layout, product and expert layer against plain forms in 64 bits.

Tolerances. The quantizer is exact: codes and scales are compared for equality. A product of two elements is exact, and a sum
of m of them in 32 bits is off by at most m steps of 2^-23 of the sum of their magnitudes, whatever the order and whether an
addition rounds or cuts; then half a step of the output's type."""
import pytest
import torch

from flashrt_b200 import moe, mxfp4

pytestmark = pytest.mark.gpu

GRID = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def scale_exponent(amax):
    """floor(log2(amax)) - 2, at least -127; amax float64."""
    e = torch.frexp(torch.where(amax > 0, amax, 2.0 ** -130)).exponent.to(torch.int64) - 1
    return (e - 2).clamp(min=-127)


def elements(v, e):
    """The element of v / 2^e: to nearest, ties to the even code."""
    a = torch.ldexp(v.abs(), -e)
    code = torch.zeros_like(a, dtype=torch.int64)
    for i in range(7):
        mid = (GRID[i] + GRID[i + 1]) / 2
        code += (a > mid) | ((a == mid) & (i % 2 == 1))
    return code


def quantized(x):
    """x [T][n] -> code magnitudes, exponents [T][n / 32], values, in 64 bits; x finite."""
    v = x.double().reshape(x.shape[0], -1, 32)
    e = scale_exponent(v.abs().amax(2)).unsqueeze(2)
    code = elements(v, e)
    return code.view(x.shape), e.squeeze(2), (torch.ldexp(GRID[code], e) * torch.where(v < 0, -1.0, 1.0)).view(x.shape)


def nibbles(codes):
    return torch.stack((codes & 15, codes >> 4), -1).view(*codes.shape[:-1], -1).long()


def values(codes, scales):
    n = nibbles(codes)
    s = torch.exp2(scales.double() - 127).repeat_interleave(32, -1)
    return GRID[n & 7] * torch.where(n > 7, -1.0, 1.0) * s


def check_quantized(x, codes, scales):
    mag, e, val = quantized(x.cpu())
    n = nibbles(codes.cpu())
    assert torch.equal(scales.cpu().long() - 127, e)
    assert torch.equal(n & 7, mag)
    assert torch.equal((n > 7) & (mag > 0), (x.cpu().double() < 0) & (mag > 0))
    return val


def hard_values(T, n, dtype, seed):
    """Blocks of many magnitudes, with midpoints between elements, powers of two and their neighbours, zeros and the type's extremes."""
    g = gen(seed)
    info = torch.finfo(dtype)
    lo, hi = (-14, 15) if dtype == torch.float16 else (-140, 127)
    x = torch.randn(T, n, generator=g, dtype=torch.float64)
    e = torch.randint(lo, hi - 3, (T, n // 32, 1), generator=g).double()
    x = (x.view(T, -1, 32) * torch.exp2(e)).view(T, n)
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 0.5, 6.0, 7.999, 4.0, 0.0], dtype=torch.float64)
    tie = mids[torch.randint(0, 12, (T, n // 32, 32), generator=g)] * torch.where(torch.rand(T, n // 32, 32, generator=g) < 0.5, -1.0, 1.0)
    tie[:, :, 0] = 4.0
    tie = (tie * torch.exp2(e)).view(T, n)
    x = torch.where(torch.rand(T, n // 32, 1, generator=g).repeat(1, 1, 32).view(T, n) < 0.5, x, tie)
    x = x.clamp(-info.max, info.max).to(dtype)
    flat = x.view(-1)
    flat[:32] = 0
    if n * T >= 128:
        flat[32:64] = info.tiny * info.eps          # the smallest subnormal
        flat[64] = info.max
        flat[96:128] = -info.tiny
    return x


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,n", [(1, 32), (1, 2048), (3, 96), (37, 2560), (200, 640), (1000, 32)])
@pytest.mark.parametrize("layout", ["contiguous", "apart", "odd"])
def test_quantize(T, n, dtype, layout):
    x = hard_values(T, n, dtype, T + n).cuda()
    if layout == "apart":
        wide = torch.full((T, n + 16), float("nan"), dtype=dtype, device="cuda")
        wide[:, :n] = x
        x = wide[:, :n]
    elif layout == "odd":
        wide = torch.full((T * (n + 1) + 1,), float("nan"), dtype=dtype, device="cuda")
        view = wide[1:].view(T, n + 1)[:, :n]
        view.copy_(x)
        x = view
    codes, scales = mxfp4.quantize(x)
    want = check_quantized(x, codes, scales)
    for out in (torch.float32, torch.bfloat16):
        got = mxfp4.dequantize(codes, scales, dtype=out)
        assert got.dtype == out and torch.equal(got.cpu().double(), want)


def test_quantize_nothing_and_nan():
    codes, scales = mxfp4.quantize(torch.zeros(0, 64, device="cuda"))
    assert codes.shape == (0, 32) and scales.shape == (0, 2) and mxfp4.dequantize(codes, scales).shape == (0, 64)
    for layout in (0, 1):
        for dtype in (torch.float32, torch.bfloat16, torch.float16):
            wide = torch.randn(5, 129, generator=gen(1)).to(dtype).cuda()
            x = wide[:, layout:layout + 128] if layout else wide[:, :128].contiguous()
            x[0, 3], x[1, 40], x[2, 127], x[4, 64] = float("nan"), float("inf"), -float("inf"), float("nan")
            codes, scales = mxfp4.quantize(x)
            bad = torch.zeros(5, 4, dtype=torch.bool)
            bad[0, 0] = bad[1, 1] = bad[2, 3] = bad[4, 2] = True
            assert torch.equal(scales.cpu() == 255, bad)
            got = mxfp4.dequantize(codes, scales).cpu().view(5, 4, 32)
            assert bool(got[bad].isnan().all()) and bool(got[~bad].isfinite().all())
            assert bool((codes.cpu().view(5, 4, 16)[bad] == 0).all())


def test_dequantize_every_code_and_scale():
    codes = torch.arange(256, dtype=torch.uint8).repeat(255, 1).view(255, 256)
    scales = torch.arange(255, dtype=torch.uint8).view(255, 1).repeat(1, 16).contiguous()
    want = values(codes, scales)
    want = torch.where(want.abs() >= 2.0 ** 128, want * float("inf"), want)     # 4 * 2^126 is beyond both types: infinity
    for dtype in (torch.float32, torch.bfloat16):
        for off in (0, 1):
            wide = torch.zeros(255, 512 + 8, dtype=dtype, device="cuda")
            got = mxfp4.dequantize(codes.cuda(), scales.cuda(), out=wide[:, off:off + 512])
            assert torch.equal(got.cpu().double(), want)
    nan = mxfp4.dequantize(codes[:1].cuda(), torch.full((1, 16), 255, dtype=torch.uint8, device="cuda"))
    assert bool(nan.isnan().all())


def random_quantized(shape, seed, spread=3):
    """codes [.., n / 2] and scales [.., n / 32]: every code, scales around 1."""
    g = gen(seed)
    codes = torch.randint(0, 256, (*shape[:-1], shape[-1] // 2), generator=g, dtype=torch.uint8)
    scales = torch.randint(127 - spread, 127 + spread + 1, (*shape[:-1], shape[-1] // 32), generator=g, dtype=torch.uint8)
    return codes, scales


@pytest.mark.parametrize("E,rows,n", [(1, 1, 128), (2, 128, 256), (3, 130, 384), (1, 1001, 640), (5, 640, 128)])
def test_pack(E, rows, n):
    codes, scales = random_quantized((E, rows, n), rows + n, 100)
    w = mxfp4.pack(codes.cuda(), scales.cuda())
    tiles, units = -(-rows // 128), n // 128
    assert w.data.numel() == E * mxfp4.packed_bytes(rows, n) == E * tiles * units * 8704
    back = mxfp4.unpack(w)
    assert torch.equal(back[0].cpu(), codes) and torch.equal(back[1].cpu(), scales)
    # byte for byte as the layout is described
    full_c, full_s = torch.zeros(E, tiles * 128, n // 2, dtype=torch.uint8), torch.full((E, tiles * 128, n // 32), 127, dtype=torch.uint8)
    full_c[:, :rows], full_s[:, :rows] = codes, scales
    c = full_c.view(E, tiles, 128, units, 4, 16).permute(0, 1, 3, 4, 2, 5).reshape(E, tiles, units, 8192)
    s = full_s.view(E, tiles, 4, 32, units, 4).permute(0, 1, 4, 3, 2, 5).reshape(E, tiles, units, 512)
    assert torch.equal(w.data.cpu().view(E, tiles, units, 8704), torch.cat((c, s), 3))


def sum_bound(want, magnitude, terms, dtype):
    info = torch.finfo(dtype)
    bound = (terms + 2) * 2.0 ** -23 * magnitude
    return bound + (want.abs() + bound) * info.eps / 2 + info.smallest_normal * info.eps


def check_product(got, x, w, dtype):
    """got [T][rows] against x [T][n] and w [rows][n] in 64 bits."""
    want, mag = x @ w.t(), x.abs() @ w.abs().t()
    assert got.dtype == dtype
    off = (got.cpu().double() - want).abs() - sum_bound(want, mag, x.shape[1], dtype)
    assert float(off.max()) <= 0, float(off.max())


DENSE = [(1, 128, 128), (1, 2560, 1001), (7, 256, 1), (16, 384, 130), (17, 128, 640), (113, 640, 384), (112, 2048, 129), (128, 512, 256), (300, 1152, 257), (1000, 384, 64)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,n,rows", DENSE)
def test_matmul(T, n, rows, dtype):
    xq, wq = random_quantized((T, n), 1 + T), random_quantized((rows, n), 2 + rows)
    if dtype == torch.float16:
        wq[1].sub_(5)                       # within the type's range
    w = mxfp4.pack(wq[0].cuda(), wq[1].cuda())
    dx = [t.cuda() for t in xq]
    got = mxfp4.matmul(*dx, w, dtype=dtype)
    check_product(got, values(*xq), values(*wq), dtype)
    # rows that lie apart, from an odd start: the same bits, and nothing beside them is written
    wide = torch.full((T * (rows + 3) + 1,), 77.0, dtype=dtype, device="cuda")
    view = wide[1:].view(T, rows + 3)[:, :rows]
    mxfp4.matmul(*dx, w, out=view)
    assert torch.equal(view, got)
    view.fill_(77.0)
    assert bool((wide == 77).all())


def test_matmul_scales_of_every_size_and_nan():
    """Scales from 2^-60 to 2^60 on both sides; a NaN scale reaches every output that its block takes part in, and no other."""
    T, n, rows = 40, 512, 200
    xq, wq = random_quantized((T, n), 5, 60), random_quantized((rows, n), 6, 60)
    w = mxfp4.pack(wq[0].cuda(), wq[1].cuda())
    got = mxfp4.matmul(xq[0].cuda(), xq[1].cuda(), w, dtype=torch.float32)
    check_product(got, values(*xq), values(*wq), torch.float32)
    xq[1][7, 3], wq[1][150, 9] = 255, 255
    bad = mxfp4.matmul(xq[0].cuda(), xq[1].cuda(), mxfp4.pack(wq[0].cuda(), wq[1].cuda()), dtype=torch.float32)
    nan = torch.zeros(T, rows, dtype=torch.bool)
    nan[7], nan[:, 150] = True, True
    assert torch.equal(bad.cpu().isnan(), nan)
    assert torch.equal(bad.cpu()[~nan], got.cpu()[~nan])


@pytest.mark.parametrize("n,rows", [(256, 300), (2048, 128), (640, 64)])
def test_matmul_of_operands_at_the_least_alignment(n, rows):
    """Codes on 16 bytes, scales on 4, y on one element: the same bits as on the widest."""
    T = 50
    xq, wq = random_quantized((T, n), 11), random_quantized((rows, n), 12)
    w = mxfp4.pack(wq[0].cuda(), wq[1].cuda())
    want = mxfp4.matmul(xq[0].cuda(), xq[1].cuda(), w)
    shifted = []
    for t, by in ((xq[0], 16), (xq[1], 4), (w.data, 16)):
        flat = torch.zeros(t.numel() + by, dtype=torch.uint8, device="cuda")
        flat[by:] = t.reshape(-1).cuda()
        shifted.append(flat[by:].view(t.shape))
    moved = mxfp4.Packed(shifted[2], 1, rows, n)
    assert torch.equal(mxfp4.matmul(shifted[0], shifted[1], moved), want)


def test_layers_in_a_stream_without_a_wait():
    """Calls that follow one another, each on values that the kernels in front have just made, with one workspace: what each gives alone."""
    E, n, ff, K = 24, 512, 256, 4
    raw = [random_quantized(s, i) for i, s in enumerate(((E, ff, n), (E, ff, n), (E, n, ff)))]
    W = [mxfp4.pack(c.cuda(), (s - 6).cuda()) for c, s in raw]
    sizes = [1, 700, 3, 64, 1500, 2, 300, 1]
    ws = moe.workspace(max(mxfp4.moe_layer_workspace_bytes(T, K, n, ff, E) for T in sizes))
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    seeds = [(torch.randn(T, n, generator=g, device="cuda"), torch.randn(T, E, generator=g, device="cuda")) for T in sizes]
    mix = torch.randn(n, n, generator=g, device="cuda") / n ** 0.5

    def inputs(x, logits):
        y = x
        for _ in range(3):
            y = torch.tanh(y @ mix)
        ids, wts = moe.moe_route_topk(logits, K)
        return y.contiguous(), torch.where(logits[:, :K] > 1.5, -1, ids), wts

    torch.cuda.synchronize()
    outs = []
    for r in range(3):
        for x, logits in seeds:
            outs.append(mxfp4.moe_layer(*inputs(x + r, logits + r * mix[0, :E]), *W, ws=ws))
    torch.cuda.synchronize()
    for r in range(3):
        for x, logits in seeds:
            made = inputs(x + r, logits + r * mix[0, :E])
            torch.cuda.synchronize()
            want = mxfp4.moe_layer(*made, *W)
            torch.cuda.synchronize()
            assert torch.equal(outs.pop(0), want)


def test_rows_more_than_32_bits_apart():
    """Rows whose distance passes 2^31 bytes and 2^31 elements: x and out of the layer, x of the quantizer, y of the product."""
    T, n, ff, E, K = 3, 256, 128, 4, 2
    far = 1_200_000_000                                  # elements between rows; the third begins at 2.4 * 10^9
    ids, wts = (t.cuda() for t in routed(T, K, E, 3))
    raw = [random_quantized(s, i) for i, s in enumerate(((E, ff, n), (E, ff, n), (E, n, ff)))]
    W = [mxfp4.pack(c.cuda(), (s - 6).cuda()) for c, s in raw]
    x = torch.randn(T, n, generator=gen(1)).bfloat16().cuda()
    place = torch.empty(2 * far + n, dtype=torch.bfloat16, device="cuda").as_strided((T, n), (far, 1))
    place.copy_(x)
    want_q, want = mxfp4.quantize(x), mxfp4.moe_layer(x, ids, wts, *W)
    for a, b in zip(mxfp4.quantize(place), want_q):
        assert torch.equal(a, b)
    assert torch.equal(mxfp4.dequantize(*want_q, out=place), mxfp4.dequantize(*want_q, dtype=torch.bfloat16))
    place.copy_(x)
    got = mxfp4.moe_layer(place, ids, wts, *W, out=place)     # in place: x is read before the first row of out is written
    assert torch.equal(got, want)
    w = mxfp4.pack(raw[0][0][0].cuda(), raw[0][1][0].cuda())
    assert torch.equal(mxfp4.matmul(*want_q, w, out=place[:, :ff]), mxfp4.matmul(*want_q, w))


def routed(T, K, E, seed, drop=0.0, skew=False):
    g = gen(seed)
    score = torch.randn(T, E, generator=g)
    if skew:
        score -= torch.arange(E) * 0.4
    ids = score.topk(K, 1).indices.to(torch.int32)
    if drop:
        ids[torch.rand(T, K, generator=g) < drop] = -1
    return ids, torch.softmax(torch.randn(T, K, generator=g), 1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,K,E,n,rows,drop,skew", [(1, 1, 1, 128, 128, 0, False), (1, 4, 64, 256, 130, 0, False), (37, 4, 16, 384, 257, 0.3, False), (300, 2, 5, 256, 128, 0.1, True),
                                                    (64, 8, 300, 128, 640, 0, False), (500, 3, 7, 640, 100, 0.5, True), (350, 2, 500, 2048, 256, 0, False), (90, 2, 40, 4224, 128, 0.1, False),
                                                    (256, 1, 2, 2176, 300, 0, True), (300, 2, 4096, 512, 128, 0, False), (40, 3, 2049, 128, 256, 0.2, False)])
def test_moe_matmul(T, K, E, n, rows, drop, skew, dtype):
    ids, _ = routed(T, K, E, T + E, drop, skew)
    xq, wq = random_quantized((T, n), 3), random_quantized((E, rows, n), 4)
    offsets, slot_of, _ = moe.moe_sort(ids.cuda(), E)
    w = mxfp4.pack(wq[0].cuda(), wq[1].cuda())
    dx = [t.cuda() for t in xq]
    y = torch.full((T * K, rows), 77.0, dtype=dtype, device="cuda")
    assert mxfp4.moe_matmul(*dx, w, offsets, slot_of, K, out=y) is y
    x, W, at, slots = values(*xq), values(*wq), offsets.tolist(), slot_of.cpu().long()
    for e in range(E):
        if at[e + 1] > at[e]:
            check_product(y[at[e]:at[e + 1]], x[slots[at[e]:at[e + 1]] // K], W[e], dtype)
    assert bool((y[at[-1]:] == 77).all())              # rows that no expert has are left as they were
    # the rows already in order, without slot_of: the same bits
    xs = [t[(slots.clamp(min=0) // K).cuda()].contiguous() for t in dx]
    again = torch.full_like(y, 77.0)
    mxfp4.moe_matmul(*xs, w, offsets, out=again)
    assert torch.equal(again, y)


def test_moe_matmul_plan_that_points_outside():
    """Offsets beyond the rows and slots beyond the tokens are left out: nothing outside the buffers is read or written."""
    T, K, E, n, rows = 20, 2, 4, 128, 128
    xq, wq = random_quantized((T, n), 3), random_quantized((E, rows, n), 4)
    w = mxfp4.pack(wq[0].cuda(), wq[1].cuda())
    dx = [t.cuda() for t in xq]
    slot_of = torch.arange(T * K, dtype=torch.int32)
    good = mxfp4.moe_matmul(*dx, w, torch.tensor([0, 10, 10, 30, 40], dtype=torch.int32).cuda(), slot_of.cuda(), K, dtype=torch.float32)
    y = torch.full((T * K, rows), 77.0, device="cuda")
    slot_of[3], slot_of[15] = 1 << 30, -5
    mxfp4.moe_matmul(*dx, w, torch.tensor([-7, 10, 9, 30, 1 << 30], dtype=torch.int32).cuda(), slot_of.cuda(), K, out=y)
    keep = torch.tensor([r not in (3, 15) and r != 9 for r in range(T * K)])
    assert torch.equal(y.cpu()[keep], good.cpu()[keep])
    # ranges that overlap, more of them than the rows allow: nothing is computed
    y.fill_(77.0)
    mxfp4.moe_matmul(*dx, w, torch.tensor([0, 40, 0, 40, 0], dtype=torch.int32).cuda(), slot_of.cuda(), K, out=y)
    torch.cuda.synchronize()


def layer_reference(x, ids, wts, W, E):
    """The layer in 64 bits and how far a layer in 32 bits may be from it: the hidden rows' codes may differ where the sums' error can take a
    value, or its block's largest, over a border."""
    T, n = x.shape
    wg, wu, wd = W
    xv = quantized(x)[2]
    out, slack, mag = torch.zeros(T, n, dtype=torch.float64), torch.zeros(T, n, dtype=torch.float64), torch.zeros(T, n, dtype=torch.float64)
    for e in range(E):
        t, k = (ids == e).nonzero(as_tuple=True)
        if not t.numel():
            continue
        xe, mg = xv[t], (n + 2) * 2.0 ** -23
        g, u = xe @ wg[e].t(), xe @ wu[e].t()
        eg, eu = mg * (xe.abs() @ wg[e].abs().t()), mg * (xe.abs() @ wu[e].abs().t())
        s = g * torch.sigmoid(g)
        h = s * u
        # silu's slope is at most 1.1; its own evaluation and the product add 16 steps
        eh = 1.1 * eg * (u.abs() + eu) + s.abs() * eu + 16 * 2.0 ** -24 * h.abs()
        blocks = lambda v: v.view(t.numel(), -1, 32)                                     # noqa: E731
        q = quantized(h)[2]
        far = torch.zeros_like(h)
        top, room = blocks(h.abs()), blocks(eh)
        for big in ((top + room).amax(2), (top - room).clamp(min=0).amax(2)):
            ex = scale_exponent(big).unsqueeze(2)
            for v in (h - eh, h, h + eh):
                far = torch.maximum(far, ((torch.ldexp(GRID[elements(blocks(v), ex)], ex) * torch.where(blocks(v) < 0, -1.0, 1.0)).view_as(h) - q).abs())
        y = q @ wd[e].t()
        w = wts[t, k].double().unsqueeze(1)
        ymag = (q.abs() + far) @ wd[e].abs().t()
        out.index_add_(0, t, w * y)
        slack.index_add_(0, t, w * (far @ wd[e].abs().t() + (h.shape[1] + 2) * 2.0 ** -23 * ymag))
        mag.index_add_(0, t, w * y.abs())
    return out, slack, mag


@pytest.mark.parametrize("x_dtype,out_dtype", [(torch.float32, torch.float32), (torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16)])
@pytest.mark.parametrize("T,K,E,n,ff,drop,skew", [(1, 1, 1, 128, 128, 0, False), (1, 4, 32, 256, 128, 0, False), (5, 2, 8, 384, 640, 0.3, False), (64, 4, 16, 512, 256, 0, True),
                                                  (300, 2, 3, 128, 384, 0.2, True), (130, 6, 40, 256, 256, 0.1, False),
                                                  (300, 3, 6, 512, 128, 0.1, False)])
def test_moe_layer(T, K, E, n, ff, drop, skew, x_dtype, out_dtype):
    ids, wts = routed(T, K, E, T + ff, drop, skew)
    if T > 2:
        ids[T // 2] = -1                               # a token that no expert has
    x = torch.randn(T, n, generator=gen(T)).to(x_dtype)
    raw = [random_quantized(s, i) for i, s in enumerate(((E, ff, n), (E, ff, n), (E, n, ff)))]
    for _, s in raw:
        s.sub_(6)
    W = [mxfp4.pack(c.cuda(), s.cuda()) for c, s in raw]
    ws = moe.workspace(mxfp4.moe_layer_workspace_bytes(T, K, n, ff, E))
    out = mxfp4.moe_layer(x.cuda(), ids.cuda(), wts.cuda(), *W, dtype=out_dtype, ws=ws)
    moe.workspace_status(ws)
    assert out.dtype == out_dtype
    want, slack, mag = layer_reference(x, ids, wts, [values(*r) for r in raw], E)
    row_eps = torch.finfo(torch.bfloat16).eps / 2 if out_dtype == torch.bfloat16 and T * n >= 65536 else 2.0 ** -24      # the experts' rows, rounded once
    info = torch.finfo(out_dtype)
    bound = slack * (1 + row_eps) + (row_eps + (K + 1) * 2.0 ** -24) * mag
    bound = bound + (want.abs() + bound) * info.eps / 2 + info.smallest_normal * info.eps
    off = (out.cpu().double() - want).abs() - bound
    assert float(off.max()) <= 0, float(off.max())
    assert T <= 2 or bool((out[T // 2] == 0).all())
    # the same call again, and with rows that lie apart: the same bits
    wide = torch.full((T, n + 1), 5.0, dtype=x_dtype, device="cuda")
    wide[:, 1:] = x.cuda()
    place = torch.full((T, n + 3), 5.0, dtype=out_dtype, device="cuda")
    mxfp4.moe_layer(wide[:, 1:], ids.cuda(), wts.cuda(), *W, out=place[:, :n], ws=ws)
    assert torch.equal(place[:, :n], out) and bool((place[:, n:] == 5).all())


def test_moe_layer_is_the_operators_in_a_row():
    """The layer's parts called one by one, with the plain SwiGLU in between: the same rows up to codes at a border, so nearly the same output."""
    T, K, E, n, ff = 90, 4, 24, 512, 256
    ids, wts = routed(T, K, E, 7, 0.1)
    x = torch.randn(T, n, generator=gen(1))
    raw = [random_quantized(s, i) for i, s in enumerate(((E, ff, n), (E, ff, n), (E, n, ff)))]
    W = [mxfp4.pack(c.cuda(), (s - 6).cuda()) for c, s in raw]
    layer = mxfp4.moe_layer(x.cuda(), ids.cuda(), wts.cuda(), *W)
    offsets, slot_of, row_of = moe.moe_sort(ids.cuda(), E)
    xq = mxfp4.quantize(x.cuda())
    g, u = (mxfp4.moe_matmul(*xq, w, offsets, slot_of, K, out=torch.zeros(T * K, ff, device="cuda")) for w in W[:2])
    h = mxfp4.quantize((g.double() * torch.sigmoid(g.double()) * u.double()).float())
    ys = mxfp4.moe_matmul(*h, W[2], offsets, out=torch.zeros(T * K, n, device="cuda"))
    parts = moe.moe_unsort_rows(ys, wts.cuda(), row_of)
    # a code at a border differs for fewer than one value in 10^4 (an error of about 2^-22 between elements that are 2^-3 apart): a few of the rows' 9 10^4
    # values, each less than 1 % of its row
    rel = float((layer - parts).norm() / parts.norm())
    assert rel < 2e-3, rel


def test_moe_layer_reports_an_id_beyond_the_experts():
    T, K, E, n, ff = 6, 2, 4, 128, 128
    ids, wts = routed(T, K, E, 1)
    raw = [random_quantized(s, i) for i, s in enumerate(((E, ff, n), (E, ff, n), (E, n, ff)))]
    W = [mxfp4.pack(c.cuda(), s.cuda()) for c, s in raw]
    x = torch.randn(T, n, generator=gen(1)).cuda()
    ws = moe.workspace(mxfp4.moe_layer_workspace_bytes(T, K, n, ff, E))
    ids[3, 1] = 4
    got = mxfp4.moe_layer(x, ids.cuda(), wts.cuda(), *W, ws=ws)
    with pytest.raises(moe.FrxError, match="slot 7"):
        moe.workspace_status(ws)
    ids[3, 1] = -1
    assert torch.equal(mxfp4.moe_layer(x, ids.cuda(), wts.cuda(), *W, ws=ws), got)
    moe.workspace_status(ws)
    empty = mxfp4.moe_layer(x[:0], ids[:0].cuda(), wts[:0].cuda(), *W)
    assert empty.shape == (0, n)


def test_moe_layer_infinite_activations_stay_with_their_token():
    T, K, E, n, ff = 40, 2, 4, 256, 128
    ids, wts = routed(T, K, E, 2)
    raw = [random_quantized(s, i) for i, s in enumerate(((E, ff, n), (E, ff, n), (E, n, ff)))]
    W = [mxfp4.pack(c.cuda(), (s - 6).cuda()) for c, s in raw]
    x = torch.randn(T, n, generator=gen(1))
    clean = mxfp4.moe_layer(x.cuda(), ids.cuda(), wts.cuda(), *W).cpu()
    x[5, 17], x[20, 255] = float("inf"), float("nan")
    got = mxfp4.moe_layer(x.cuda(), ids.cuda(), wts.cuda(), *W).cpu()
    bad = torch.zeros(T, dtype=torch.bool)
    bad[5] = bad[20] = True
    assert bool(got[bad].isnan().all()) and torch.equal(got[~bad], clean[~bad])


def test_moe_layer_captured_on_another_stream_and_two_at_once():
    """Two layers in two graphs with workspaces of their own, replayed at the same time on new values, against the eager calls."""
    T, K, E, n, ff = 70, 4, 16, 256, 256
    raw = [random_quantized(s, i) for i, s in enumerate(((E, ff, n), (E, ff, n), (E, n, ff)))]
    W = [mxfp4.pack(c.cuda(), (s - 6).cuda()) for c, s in raw]
    need = mxfp4.moe_layer_workspace_bytes(T, K, n, ff, E)
    sides = []
    for i in range(2):
        ids, wts = (t.cuda() for t in routed(T, K, E, i, 0.1))
        x, out, ws = torch.randn(T, n, generator=gen(i)).cuda(), torch.zeros(T, n, device="cuda"), moe.workspace(need)
        call = lambda x=x, ids=ids, wts=wts, out=out, ws=ws: mxfp4.moe_layer(x, ids, wts, *W, out=out, ws=ws)   # noqa: E731
        call()
        torch.cuda.synchronize()
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            call()
        sides.append((x, ids, wts, out, stream, graph))
    for step in range(3):
        want = []
        for i, (x, ids, wts, out, _, _) in enumerate(sides):
            new_ids, new_wts = routed(T, K, E, 10 * step + i, 0.1)
            ids.copy_(new_ids), wts.copy_(new_wts), x.copy_(torch.randn(T, n, generator=gen(step + i)))
            want.append(mxfp4.moe_layer(x, ids, wts, *W))
        torch.cuda.synchronize()
        for _ in range(5):
            for *_, stream, graph in sides:
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for (_, _, _, out, _, _), w in zip(sides, want):
            assert torch.equal(out, w)


def test_a_wait_that_runs_out_leaves_nan_and_is_reported():
    """A row of a million columns keeps the epilogue waiting for milliseconds; with a limit of ten microseconds it gives up. Nothing hangs, no wrong number is
    left, and the next call is right again."""
    from flashrt_b200.lib import check, lib
    n, rows, ff = 1 << 20, 128, 128
    xq, wq = random_quantized((3, n), 1, 0), random_quantized((rows, n), 2, 0)
    w, dx = mxfp4.pack(wq[0].cuda(), wq[1].cuda()), [t.cuda() for t in xq]
    x, ids, wts = torch.randn(3, n, generator=gen(3)).cuda(), torch.zeros(3, 1, dtype=torch.int32).cuda(), torch.ones(3, 1).cuda()
    down = mxfp4.pack(*(t.cuda() for t in random_quantized((1, n, ff), 4, 0)))
    ws = moe.workspace(mxfp4.moe_layer_workspace_bytes(3, 1, n, ff, 1))
    layer = mxfp4.moe_layer(x, ids, wts, w, w, down, ws=ws)
    moe.workspace_status(ws)
    try:
        check(lib.frx_debug_set_wait_limit_ns(10_000))
        y = mxfp4.matmul(*dx, w, dtype=torch.float32)
        torch.cuda.synchronize()
        assert bool(y.isnan().any()), "the wait did not run out"
        lost = mxfp4.moe_layer(x, ids, wts, w, w, down, ws=ws)
        with pytest.raises(moe.FrxError, match="ran out"):
            moe.workspace_status(ws)
        assert bool(lost.isnan().any())
    finally:
        check(lib.frx_debug_set_wait_limit_ns(0))
    check_product(mxfp4.matmul(*dx, w, dtype=torch.float32), values(*xq), values(*wq), torch.float32)
    assert torch.equal(mxfp4.moe_layer(x, ids, wts, w, w, down, ws=ws), layer)
    moe.workspace_status(ws)


def test_refusals():
    x, q = torch.zeros(4, 256, device="cuda"), random_quantized((4, 256), 1)
    dq = [t.cuda() for t in q]
    w = mxfp4.pack(dq[0].view(1, 4, 128), dq[1].view(1, 4, 8))
    two = mxfp4.pack(dq[0].view(2, 2, 128), dq[1].view(2, 2, 8))
    offsets = torch.zeros(3, dtype=torch.int32, device="cuda")
    ids, wts = torch.zeros(4, 2, dtype=torch.int32, device="cuda"), torch.zeros(4, 2, device="cuda")
    big = mxfp4.pack(torch.zeros(2, 128, 128, dtype=torch.uint8, device="cuda"), torch.zeros(2, 128, 8, dtype=torch.uint8, device="cuda"))
    down = mxfp4.pack(torch.zeros(2, 256, 64, dtype=torch.uint8, device="cuda"), torch.zeros(2, 256, 4, dtype=torch.uint8, device="cuda"))
    bad = [lambda: mxfp4.quantize(x.double()), lambda: mxfp4.quantize(x.cpu()), lambda: mxfp4.quantize(x[:, :40]), lambda: mxfp4.quantize(x.t()), lambda: mxfp4.quantize(x[0]),
           lambda: mxfp4.dequantize(dq[0].int(), dq[1]), lambda: mxfp4.dequantize(dq[0], dq[1][:, :7]), lambda: mxfp4.dequantize(*dq, dtype=torch.float16),
           lambda: mxfp4.dequantize(*dq, out=x[:3]), lambda: mxfp4.pack(dq[0][:, :48].contiguous(), dq[1][:, :3].contiguous()), lambda: mxfp4.pack(dq[0], dq[1][:3]),
           lambda: mxfp4.matmul(dq[0][:, :64].contiguous(), dq[1][:, :4].contiguous(), w), lambda: mxfp4.matmul(*dq, two), lambda: mxfp4.matmul(*dq, w, out=x),
           lambda: mxfp4.matmul(*dq, w, dtype=torch.float64), lambda: mxfp4.matmul(*q, w),
           lambda: mxfp4.moe_matmul(*dq, two, offsets[:2]), lambda: mxfp4.moe_matmul(*dq, two, offsets.long()), lambda: mxfp4.moe_matmul(*dq, two, offsets, None, 2),
           lambda: mxfp4.moe_matmul(*dq, two, offsets, ids.view(-1), 0),
           lambda: mxfp4.moe_layer(x, ids, wts, big, big, big), lambda: mxfp4.moe_layer(x[:3], ids, wts, big, big, down), lambda: mxfp4.moe_layer(x, ids.long(), wts, big, big, down),
           lambda: mxfp4.moe_layer(x, ids, wts.half(), big, big, down), lambda: mxfp4.moe_layer(x, ids, wts, big, big, down, dtype=torch.float64),
           lambda: mxfp4.moe_layer(x, ids, wts, big, big, down, ws=torch.zeros(1000, dtype=torch.uint8, device="cuda"))]
    for i, call in enumerate(bad):
        with pytest.raises(moe.FrxError):
            call()
            raise AssertionError(f"call {i} was not refused")
    mxfp4.moe_layer(x, ids, wts, big, big, down)


def layer_of(T, K, E, n, ff, seed=0):
    ids, wts = (t.cuda() for t in routed(T, K, E, seed))
    raw = [random_quantized(s, seed + i) for i, s in enumerate(((E, ff, n), (E, ff, n), (E, n, ff)))]
    return torch.randn(T, n, generator=gen(seed)).cuda(), ids, wts, [mxfp4.pack(c.cuda(), (s - 6).cuda()) for c, s in raw]


@pytest.mark.parametrize("T,n", [(1, 2048), (31, 2048), (32, 2048), (256, 256), (700, 512)])
def test_moe_layer_output_is_rounded_once(T, n):
    """A 16-bit output is the 32-bit one, rounded: the experts' rows lose nothing on their way to it, whatever the size."""
    x, ids, wts, W = layer_of(T, 3, 8, n, 256)
    full = mxfp4.moe_layer(x, ids, wts, *W, dtype=torch.float32)
    for dtype in (torch.bfloat16, torch.float16):
        assert torch.equal(mxfp4.moe_layer(x, ids, wts, *W, dtype=dtype), full.to(dtype))


def test_moe_layer_a_token_alone_and_in_a_batch():
    """The same bits whatever shares the batch."""
    x, ids, wts, W = layer_of(300, 4, 6, 1024, 128)
    for rows in (torch.float32, torch.bfloat16):
        full = mxfp4.moe_layer(x, ids, wts, *W, dtype=torch.bfloat16, rows=rows)
        for a, b in ((0, 1), (7, 8), (31, 63), (100, 300)):
            assert torch.equal(mxfp4.moe_layer(x[a:b], ids[a:b], wts[a:b], *W, dtype=torch.bfloat16, rows=rows), full[a:b])


@pytest.mark.parametrize("T", [5, 300])
def test_moe_layer_rows_in_bfloat16(T):
    """Where the caller asks for them: each of the K rows of a token is off by half a step (2^-8) of bfloat16, weighted, and the sum by its own."""
    x, ids, wts, W = layer_of(T, 3, 8, 512, 256)
    ws = moe.workspace(mxfp4.moe_layer_workspace_bytes(T, 3, 512, 256, 8))
    got = mxfp4.moe_layer(x, ids, wts, *W, dtype=torch.bfloat16, rows=torch.bfloat16, ws=ws)
    moe.workspace_status(ws)
    want = mxfp4.moe_layer(x, ids, wts, *W, dtype=torch.float32).double()
    mag = sum(mxfp4.moe_layer(x, ids[:, k:k + 1].contiguous(), wts[:, k:k + 1].contiguous(), *W, dtype=torch.float32).double().abs() for k in range(3))
    half = torch.finfo(torch.bfloat16).eps / 2
    bound = (half + 5 * 2.0 ** -24) * mag       # the rows' rounding, three products and additions of either side
    bound = bound + half * (want.abs() + bound)
    assert bool(((got.double() - want).abs() <= bound).all())
    assert not torch.equal(got, want.bfloat16())


def test_moe_layer_refuses_rows_that_no_kernel_has():
    x, ids, wts, W = layer_of(4, 2, 4, 128, 128)
    for dtype, rows in ((torch.float32, torch.bfloat16), (torch.float16, torch.bfloat16), (torch.bfloat16, torch.float16), (torch.float16, torch.float16)):
        with pytest.raises(moe.FrxError):
            mxfp4.moe_layer(x, ids, wts, *W, dtype=dtype, rows=rows)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_tiles_behind_a_wait_that_ran_out_are_nan_too(dtype):
    """Six tiles a block of some hundreds of microseconds each, and a limit of ten: every output is the right one or NaN, in the tiles behind the first lost one too."""
    from flashrt_b200.lib import check, lib
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    T, n, rows = 6 * 112 * sms, 1 << 17, 128
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    codes = torch.randint(0, 256, (T, n // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = torch.full((T, n // 32), 120, device="cuda", dtype=torch.uint8)
    wq = random_quantized((rows, n), 2, 0)
    w = mxfp4.pack(wq[0].cuda(), wq[1].cuda())
    want = mxfp4.matmul(codes, scales, w, dtype=dtype)
    assert not bool(want.isnan().any())
    try:
        check(lib.frx_debug_set_wait_limit_ns(10_000))
        y = mxfp4.matmul(codes, scales, w, dtype=dtype)
        torch.cuda.synchronize()
    finally:
        check(lib.frx_debug_set_wait_limit_ns(0))
    lost = y.isnan()
    assert bool(lost.any()), "no wait ran out"
    assert bool((lost | (y == want)).all())
    assert torch.equal(mxfp4.matmul(codes, scales, w, dtype=dtype), want)


def test_hidden_codes_of_exact_sums():
    """Gate and up sums of one and two terms, which 32 bits hold exactly, a down matrix that passes the hidden values on: what is left is the error of silu(g) * u,
    and every code must be that of a value within its bound. The bound, in steps of 2^-24 of the value: the exponential is 2^fl(-g * fl(log2 e)), a product rounded by 2^-24
    and a constant that is off by 2^-26, hence (1 + 0.25) |g|; 4 for ex2.approx (2^-22), 2 for rcp.approx (2^-23), one for each of the sum 1 + e and the two products: 9,
    taken as 16. From g = -87.3 down the reciprocal is a subnormal (2^-21), from -88.7 on it is 0, as in a plain form of 32 bits."""
    T, n, ff = 96, 128, 128
    g = gen(9)
    grid = GRID.float()

    def matrix(rows, columns, at):
        codes = torch.zeros(1, rows, columns, dtype=torch.uint8)
        for c in at:
            codes[0, :, c] = torch.randint(0, 16, (rows,), generator=g, dtype=torch.uint8)
        scales = torch.full((1, rows, columns // 32), 127, dtype=torch.uint8)
        packed = (codes[..., 0::2] | (codes[..., 1::2] << 4)).contiguous()
        return values(packed, scales)[0], mxfp4.pack(packed.cuda(), scales.cuda())

    wg, gate = matrix(ff, n, (0, 64))
    wu, up = matrix(ff, n, (32,))
    eye = torch.zeros(1, n, ff, dtype=torch.uint8)
    eye[0, range(n), range(ff)] = 2                       # 1.0
    down = mxfp4.pack((eye[..., 0::2] | (eye[..., 1::2] << 4)).contiguous().cuda(), torch.full((1, n, ff // 32), 127, dtype=torch.uint8).cuda())
    x = torch.zeros(T, n)
    x[:, 0] = grid[torch.randint(1, 8, (T,), generator=g)] * 2 * torch.where(torch.rand(T, generator=g) < 0.5, -1.0, 1.0)
    x[:, 64] = grid[torch.randint(1, 8, (T,), generator=g)] * 0.5
    x[:, 32] = grid[torch.randint(1, 8, (T,), generator=g)]
    assert torch.equal(quantized(x)[2], x.double())
    ids, wts = torch.zeros(T, 1, dtype=torch.int32).cuda(), torch.ones(T, 1).cuda()
    got = mxfp4.moe_layer(x.cuda(), ids, wts, gate, up, down, dtype=torch.float32).cpu().double()
    a, u = x.double() @ wg.t(), x.double() @ wu.t()
    assert float(a.min()) < -80 and float(a.max()) > 80
    h = a * torch.sigmoid(a) * u
    eh = (16 + 1.25 * a.abs()) * 2.0 ** -24 * h.abs()
    eh = torch.where(a < -87.3, 2.0 ** -20 * h.abs(), eh)
    eh = torch.where(a < -88.7, h.abs(), eh)
    blocks = lambda v: v.view(T, -1, 32)                                             # noqa: E731
    fits, first, single = torch.zeros(T, ff, dtype=torch.bool), None, torch.ones(T, ff, dtype=torch.bool)
    top, room = blocks(h.abs()), blocks(eh)
    for big in ((top - room).clamp(min=0).amax(2), (top + room).amax(2)):
        ex = scale_exponent(big).unsqueeze(2)
        for v in (h - eh, h, h + eh):
            one = (torch.ldexp(GRID[elements(blocks(v), ex)], ex) * torch.where(blocks(v) < 0, -1.0, 1.0)).view_as(h)
            fits |= got == one
            first = one if first is None else first
            single &= one == first
    assert bool(fits.all())
    assert float(single.double().mean()) > 0.98          # (nearly every code is settled by the bound)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,n,rows", [(300, 128, 6499), (300, 256, 6598), (450, 384, 6400), (1, 128, 19001), (120, 640, 12929)])
def test_matmul_of_two_row_tiles_a_tile(T, n, rows, dtype):
    """More row tiles than SMs, two a tile: odd and even numbers of them, the last one whole, partial, of odd and even rows."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert -(-rows // 128) * (T // 112 + 1) > sms
    xq, wq = random_quantized((T, n), 1 + T), random_quantized((rows, n), 2 + rows)
    if dtype == torch.float16:
        wq[1].sub_(5)
    w = mxfp4.pack(wq[0].cuda(), wq[1].cuda())
    dx = [t.cuda() for t in xq]
    got = mxfp4.matmul(*dx, w, dtype=dtype)
    check_product(got, values(*xq), values(*wq), dtype)
    for off, apart in ((1, 3), (2, 2), (0, 1)):           # rows that lie apart, by odd and even numbers, from odd and even starts: nothing beside them is written
        wide = torch.full((T * (rows + apart) + off,), 77.0, dtype=dtype, device="cuda")
        view = wide[off:].view(T, rows + apart)[:, :rows]
        mxfp4.matmul(*dx, w, out=view)
        assert torch.equal(view, got)
        view.fill_(77.0)
        assert bool((wide == 77).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,K,E,n,rows", [(200, 4, 40, 256, 1001), (700, 2, 9, 128, 1410), (50, 8, 300, 384, 130)])
def test_moe_matmul_of_two_row_tiles_a_tile(T, K, E, n, rows, dtype):
    """The same by expert: partial last row tiles beside whole ones, 16-bit rows of odd length, rows of y that no expert has."""
    ids, _ = routed(T, K, E, T + E, 0.1, True)
    xq, wq = random_quantized((T, n), 3), random_quantized((E, rows, n), 4)
    if dtype == torch.float16:
        wq[1].sub_(5)
    offsets, slot_of, _ = moe.moe_sort(ids.cuda(), E)
    y = torch.full((T * K, rows), 77.0, dtype=dtype, device="cuda")
    mxfp4.moe_matmul(*(t.cuda() for t in xq), mxfp4.pack(wq[0].cuda(), wq[1].cuda()), offsets, slot_of, K, out=y)
    x, W, at, slots = values(*xq), values(*wq), offsets.tolist(), slot_of.cpu().long()
    for e in range(E):
        if at[e + 1] > at[e]:
            check_product(y[at[e]:at[e + 1]], x[slots[at[e]:at[e + 1]] // K], W[e], dtype)
    assert at[-1] < T * K and bool((y[at[-1]:] == 77).all())


def test_moe_matmul_ranges_that_overlap():
    """More blocks of rows than any plan without overlaps has (12; 300 // 112 + 8 at most): nothing is computed."""
    T, E, n, rows = 300, 8, 128, 128
    xq, wq = random_quantized((T, n), 3), random_quantized((E, rows, n), 4)
    y = torch.full((T, rows), 77.0, device="cuda")
    offsets = torch.tensor([0, 300, 0, 300, 0, 300, 0, 300, 0], dtype=torch.int32).cuda()
    mxfp4.moe_matmul(*(t.cuda() for t in xq), mxfp4.pack(wq[0].cuda(), wq[1].cuda()), offsets, out=y)
    assert bool((y == 77).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,n", [(4032, 2080), (4033, 2080), (4099, 2080), (262145, 32), (131073, 96)])
@pytest.mark.parametrize("layout", ["contiguous", "apart"])
def test_quantize_many_values(T, n, dtype, layout):
    """Around and beyond the 2^23 values from which a thread has several loads in flight, with a last block that is not full: what the rows give a few at a time, which
    is tested above, and nothing written beside the results."""
    from flashrt_b200.lib import check, lib
    g = torch.Generator(device="cuda")
    g.manual_seed(T + n)
    x = (torch.randn(T, n, generator=g, device="cuda") * torch.exp2(torch.randint(-9, 9, (T, 1), generator=g, device="cuda").float())).to(dtype)
    if layout == "apart":
        wide = torch.full((T, n + 16), float("nan"), dtype=dtype, device="cuda")
        wide[:, :n] = x
        x = wide[:, :n]
    pad = 4096
    codes, scales = torch.full((T * n // 2 + pad,), 0x5a, dtype=torch.uint8, device="cuda"), torch.full((T * n // 32 + pad,), 0x5a, dtype=torch.uint8, device="cuda")
    check(lib.frx_mxfp4_quantize(moe._stream(), moe._ptr(x), x.stride(0), mxfp4.DTYPES[dtype], T, n, moe._ptr(codes), moe._ptr(scales)))
    assert bool((codes[-pad:] == 0x5a).all()) and bool((scales[-pad:] == 0x5a).all())
    codes, scales = codes[:-pad].view(T, n // 2), scales[:-pad].view(T, n // 32)
    few = max(1, (1 << 20) // n)                        # rows of a part: an eighth of the limit
    parts = [mxfp4.quantize(x[a:a + few]) for a in range(0, T, few)]
    assert torch.equal(codes, torch.cat([p[0] for p in parts])) and torch.equal(scales, torch.cat([p[1] for p in parts]))
    check_quantized(x[-7:], codes[-7:], scales[-7:])    # the end, by the plain form too
    if dtype == torch.float16:
        return
    flat = torch.full((T * (n + 16),), 77.0, dtype=dtype, device="cuda")
    back = flat.view(T, n + 16)[:, :n] if layout == "apart" else flat[:T * n].view(T, n)
    mxfp4.dequantize(codes, scales, out=back)
    assert torch.equal(back, torch.cat([mxfp4.dequantize(*p, dtype=dtype) for p in parts]))
    back.fill_(77.0)
    assert bool((flat == 77).all())
