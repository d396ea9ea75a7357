"""Low-rank adapters of many requests beside a shared projection, against a plain form in 64 bits.

Tolerance. A sum of m products of 16-bit elements in 32 bits is off by at most m steps of 2^-23 of the sum of their magnitudes: n of them in A x, and as many as 3 rank in B (A x), whose right
side is three 16-bit pieces (what they leave, and the scale's rounding, are a few steps of 2^-24). With M = |scale| |B| (|A| |x|) that is (n + 3 rank + 4) 2^-23 M; the addition to y and the
rounding to its type half a step each."""
import pytest
import torch

from flashrt_b200 import adapters, moe, mxfp4
from flashrt_b200 import lib as L

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def apart(t, pad):
    wide = torch.full((*t.shape[:-1], t.shape[-1] + pad), float("nan"), dtype=t.dtype, device=t.device)
    wide[..., :t.shape[-1]] = t
    return wide[..., :t.shape[-1]]


def aligned(t):
    """t in device memory, its rows on 16-byte boundaries."""
    pad = -t.shape[-1] % 8
    return apart(t.cuda(), pad) if pad else t.cuda()


class Case:
    def __init__(self, lengths, n, rows, rank, dtype=BF16, out=BF16, count=5, seed=0, before=0, behind=3, none=0.2):
        g = gen(seed + n + rows + rank)
        offsets = [before]
        for m in lengths:
            offsets.append(offsets[-1] + m)
        self.T = T = offsets[-1] + behind
        self.offsets = offsets
        self.which = torch.randint(0, count, (len(lengths),), generator=g, dtype=torch.int32)
        self.which[torch.rand(len(lengths), generator=g) < none] = -1
        self.x = torch.randn(T, n, generator=g).to(dtype)
        self.a = (torch.randn(count, rank, n, generator=g) / n ** 0.5).to(dtype)
        self.b = (torch.randn(count, rows, rank, generator=g) / rank ** 0.5).to(dtype)
        self.scale = torch.randn(count, generator=g)
        self.y = torch.randn(T, rows, generator=g).to(out)

    def reference(self, scaled=True):
        want, tol = self.y.double().cuda(), torch.zeros(self.y.shape, dtype=torch.float64, device="cuda")
        x, a, b = self.x.cuda().double(), self.a.cuda().double(), self.b.cuda().double()
        live = torch.zeros(self.T, dtype=torch.bool)
        for i, j in enumerate(self.which.tolist()):
            rows = slice(self.offsets[i], self.offsets[i + 1])
            live[rows] = True
            if 0 <= j < a.shape[0]:
                s = float(self.scale[j]) if scaled else 1.0
                want[rows] += (x[rows] @ a[j].T) @ b[j].T * s
                tol[rows] = (a.shape[2] + 3 * a.shape[1] + 4) * 2.0 ** -23 * abs(s) * ((x[rows].abs() @ a[j].abs().T) @ b[j].abs().T)
        tiny = 2.0 ** -25 if self.y.dtype == F16 else 2.0 ** -149
        tol = tol + 2.0 ** -24 * (want.abs() + tol)
        tol = tol + torch.finfo(self.y.dtype).eps / 2 * (want.abs() + tol) + tiny
        return want.cpu(), tol.cpu(), live

    def args(self, place=aligned):
        return (self.y.cuda(), place(self.x), place(self.a), place(self.b), torch.tensor(self.offsets, dtype=torch.int32, device="cuda"), self.which.cuda())

    def check(self, place=aligned, scaled=True):
        want, tol, live = self.reference(scaled)
        y, *rest = self.args(place)
        out = torch.full_like(y, 7.0)
        scale = self.scale.cuda() if scaled else None
        assert adapters.add(y, *rest, scale=scale, out=out) is out
        got = out.double().cpu()
        assert torch.isfinite(got).all() and (got[~live] == 7).all()
        off = (got - want).abs()
        assert (off <= tol)[live].all(), f"off by {float((off / tol)[live].max()):.2f} of what is allowed"
        for i, j in enumerate(self.which.tolist()):
            if j < 0:
                rows = slice(self.offsets[i], self.offsets[i + 1])
                assert torch.equal(out[rows], y[rows])
        again = y.clone()
        assert adapters.add(again, *rest, scale=scale, out=again) is again         # in place
        assert torch.equal(again[live.cuda()], out[live.cuda()]) and torch.equal(again[~live.cuda()], y[~live.cuda()])
        new = adapters.add(y, *rest, scale=scale)
        assert torch.equal(new[live.cuda()], out[live.cuda()])


LENGTHS = {"one": [1], "few": [1, 0, 3, 1], "around16": [15, 16, 17, 1], "around64": [63, 64, 65], "around128": [127, 128, 129, 0, 300], "decode": [1] * 64, "more": [1] * 200,
           "mixed": [1, 1, 250, 1, 0, 1, 700, 1], "many": [(i * 13) % 7 for i in range(400)], "long": [5000, 3000]}


@pytest.mark.parametrize("lengths", sorted(LENGTHS))
@pytest.mark.parametrize("n,rows,rank", [(64, 128, 16), (2048, 2560, 16), (2560, 640, 64), (200, 1000, 8)])
def test_adapters(lengths, n, rows, rank):
    Case(LENGTHS[lengths], n, rows, rank).check()


@pytest.mark.parametrize("rank", [1, 7, 15, 16, 17, 24, 32, 48, 63, 64, 65, 80, 100, 127, 128])
@pytest.mark.parametrize("lengths", ["few", "around128", "long"])
def test_ranks(rank, lengths):
    Case(LENGTHS[lengths], 384, 300, rank, before=4).check()


@pytest.mark.parametrize("rank", [3, 16, 17, 24, 32, 33, 48, 63, 64, 100])
@pytest.mark.parametrize("users,n,rows", [(1, 2048, 2048), (1, 8, 3), (5, 1000, 257), (40, 2560, 384), (150, 72, 1030), (300, 520, 64)])
def test_a_token_each(users, n, rows, rank):
    """A decode batch: as many requests as tokens, few and many blocks a tile."""
    dtype = BF16 if rank % 2 else F16
    Case([1] * users, n, rows, rank, dtype=dtype, out=(F32, dtype)[rows % 2], behind=0, before=2 if users > 4 else 0).check()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("out", [F32, BF16, F16])
@pytest.mark.parametrize("n,rows,rank", [(1, 1, 1), (8, 3, 8), (63, 129, 20), (1000, 257, 72), (512, 512, 16)])
def test_types_and_odd_sizes(dtype, out, n, rows, rank):
    for lengths in ("few", "around64", "more"):
        Case(LENGTHS[lengths], n, rows, rank, dtype=dtype, out=out).check()


def test_without_scale_and_rows_apart():
    c = Case(LENGTHS["mixed"], 192, 264, 40, out=F16, dtype=F16)
    c.check(scaled=False)
    c.check(place=lambda t: apart(t.cuda(), 24))
    for out in (F32, BF16):                       # y and out at any alignment of an element, rows of different distances
        c = Case(LENGTHS["mixed"], 192, 264, 40, out=out)
        y, *rest = c.args()
        want = adapters.add(y, *rest)
        T = c.T
        wide = torch.full((T * 267 + 1,), float("nan"), dtype=out, device="cuda")[1:].view(T, 267)[:, :264]
        wide.copy_(y)
        buf = torch.full((T * 265 + 3,), 7.0, dtype=out, device="cuda")
        view = buf[3:].view(T, 265)[:, :264]
        adapters.add(wide, *rest, out=view)
        live = c.offsets[-1]
        assert torch.equal(view[:live], want[:live]) and (buf[3:].view(T, 265)[:, 264] == 7).all() and (buf[:3] == 7).all() and (view[live:] == 7).all()


@pytest.mark.parametrize("lengths,rank", [([1, 40, 200], 16), ([1] * 30, 16), ([1] * 30, 40)])
@pytest.mark.parametrize("size", [2.0 ** -20, 2.0 ** 12])
def test_small_and_large_values_in_float16(size, lengths, rank):
    """A x far below and far above what float16 holds: it stays in 32 bits. (B takes the opposite size, so that the result is ordinary.)"""
    c = Case(lengths, 512, 256, rank, dtype=F16, out=F32, none=0.0)
    c.a = (c.a.double() * size).to(F16)          # (small: subnormals, exact as they are)
    c.x = (c.x.double() * (64 if size > 1 else 2.0 ** -4)).to(F16)
    c.b = (c.b.double() / 16).to(F16) if size > 1 else c.b
    c.check()


def test_nan_and_infinity_stay_with_their_tokens():
    c = Case([30, 1, 128, 70, 1], 256, 300, 24, none=0.0, behind=0)
    c.which = torch.tensor([0, 1, 2, 0, 3], dtype=torch.int32)
    y, x, a, b, offsets, which = c.args()
    want = adapters.add(y, x, a, b, offsets, which)
    for t in (0, 29, 30, 31, 100, 158, 159, 229):
        for bad in (float("nan"), float("inf")):
            x2, y2 = x.clone(), y.clone()
            x2[t, 5] = bad
            got = adapters.add(y, x2, a, b, offsets, which)
            others = torch.arange(c.T) != t
            assert torch.equal(got[others], want[others]) and not torch.isfinite(got[t]).any()
            y2[t, 7] = bad
            got = adapters.add(y2, x, a, b, offsets, which)
            assert not torch.isfinite(got[t, 7])
            got[t, 7] = want[t, 7]
            assert torch.equal(got, want)
    # an adapter full of NaN that no request names, and one that two requests name
    a2, b2 = a.clone(), b.clone()
    a2[4], b2[4] = float("nan"), float("nan")
    assert torch.equal(adapters.add(y, x, a2, b2, offsets, which), want)
    a2[0] = float("nan")
    got = adapters.add(y, x, a2, b2, offsets, which)
    assert got[:30].isnan().all() and got[159:229].isnan().all() and torch.equal(got[30:159], want[30:159]) and torch.equal(got[229:], want[229:])


@pytest.mark.parametrize("rank", [8, 40])
def test_nan_and_infinity_of_a_token_each(rank):
    c = Case([1] * 50, 264, 300, rank, none=0.0, behind=0, count=50)
    c.which = torch.arange(50, dtype=torch.int32)
    y, x, a, b, offsets, which = c.args()
    want = adapters.add(y, x, a, b, offsets, which)
    for t in (0, 7, 49):
        for bad in (float("nan"), float("inf")):
            for spoil in range(3):
                x2, a2, b2 = x.clone(), a.clone(), b.clone()
                if spoil == 0:
                    x2[t, 200] = bad
                elif spoil == 1:
                    a2[t, rank - 1, 3] = bad
                else:
                    b2[t, :, 2] = bad
                got = adapters.add(y, x2, a2, b2, offsets, which)
                others = torch.arange(c.T) != t
                assert torch.equal(got[others], want[others]) and not torch.isfinite(got[t]).any()


def test_nothing_to_do():
    c = Case([2, 3], 64, 32, 16, none=0.0)
    y, x, a, b, offsets, which = c.args()
    out = torch.full_like(y, 7.0)
    adapters.add(y, x, a, b, offsets[:1], which[:0], out=out)                       # no requests
    assert (out == 7).all()
    adapters.add(y[:0], x[:0], a, b, offsets[:1], which[:0])                       # no tokens
    adapters.add(y, x, a, b, torch.zeros_like(offsets), which, out=out)             # requests without tokens
    assert (out == 7).all()
    adapters.add(y, x, a, b, offsets, torch.tensor([9, -2 ** 31], dtype=torch.int32, device="cuda"), out=out)   # adapters that there are not
    assert torch.equal(out[:5], y[:5]) and (out[5:] == 7).all()


def test_ranges_that_are_none():
    """Ranges out of bounds or descending: nothing outside the result is touched."""
    c = Case([50, 50], 64, 48, 16, none=0.0, behind=0)
    _, x, a, b, _, which = c.args()
    which = which.repeat(2)
    for bad in ([-5, 10, 20, 30, 1000], [0, 50, 20, 70, 100], [2 ** 31 - 1, 0, 5, 5, -2 ** 31], [0, 100, 0, 100, 0]):
        buf = torch.full((102, 48), 7.0, dtype=BF16, device="cuda")
        adapters.add(c.y.cuda(), x, a, b, torch.tensor(bad, dtype=torch.int32, device="cuda"), which, out=buf[1:101])
        assert (buf[0] == 7).all() and (buf[101] == 7).all()


def test_rows_more_than_32_bits_apart():
    c = Case([2, 3], 64, 16, 16, none=0.0, behind=0)
    y, x, a, b, offsets, which = c.args()
    want = adapters.add(y, x, a, b, offsets, which)
    far = 2 ** 29 + 8
    buf = torch.empty(4 * far + 64, dtype=BF16, device="cuda")
    wide = buf.as_strided((5, 16), (far, 1))
    wide.copy_(y)
    adapters.add(wide, x, a, b, offsets, which, out=wide)
    assert torch.equal(wide, want)
    x_far = buf.as_strided((5, 64), (far, 1))
    x_far.copy_(x)
    assert torch.equal(adapters.add(y, x_far, a, b, offsets, which), want)


def test_beside_an_mxfp4_projection_captured_and_on_a_stream():
    """The whole projection of a batch: a shared matrix in MXFP4 and each request's adapter, as a decode step captures it; requests change between replays."""
    c = Case([1] * 40 + [100], 512, 384, 16, out=BF16, behind=0)
    _, x, a, b, offsets, which = c.args()
    W = mxfp4.pack(*mxfp4.quantize((torch.randn(384, 512, generator=gen(8)) / 512 ** 0.5).cuda()))

    def run(stream=None):
        y = mxfp4.matmul(*mxfp4.quantize(x, stream=stream), W, stream=stream)
        return y, adapters.add(y, x, a, b, offsets, which, stream=stream), adapters.add(y, x, a, b, offsets, which, out=y, stream=stream)
    want = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = run(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run()
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    for w, g, k in zip(want, got, captured):
        assert torch.equal(w, g) and torch.equal(w, k)
    which.copy_(which.roll(1))
    offsets[1:41] += 3                                        # the first request has four tokens now, the last one three fewer
    graph.replay()
    torch.cuda.synchronize()
    for w, k in zip(run(), captured):
        assert torch.equal(w, k)


def test_two_calls_at_once():
    """Two streams, each with calls of clusters of its own: results as alone."""
    cases = [Case([1] * 30, 1024, 1024, 16, seed=1), Case([700, 300], 1024, 1024, 64, seed=2)]
    args = [c.args() for c in cases]
    want = [adapters.add(*a) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(20):
        got = [adapters.add(*a, stream=s) for a, s in zip(args, streams)]
        torch.cuda.synchronize()
        for c, w, g in zip(cases, want, got):
            assert torch.equal(w[:c.offsets[-1]], g[:c.offsets[-1]])


def test_adapters_in_the_order_of_a_sort():
    """Tokens sorted by adapter with the framework's sort, as requests of one adapter each: the same outputs as token by token, up to the order of sums."""
    T, count = 90, 6
    c = Case([1] * T, 256, 128, 16, out=F32, count=count, behind=0)
    y, x, a, b, offsets, which = c.args()
    want, tol, _ = c.reference(scaled=False)
    offs, _, row_of = moe.moe_sort(which.view(T, 1), count)
    xs, ys = moe.moe_sort_rows(x, row_of), moe.moe_sort_rows(y, row_of)
    zs = adapters.add(ys, xs, a, b, offs, torch.arange(count, dtype=torch.int32, device="cuda"))
    back = moe.moe_sort_rows_backward(zs, row_of)             # a token has one row: its sum is the row
    live = which.cpu() >= 0
    assert ((back.double().cpu() - want).abs() <= tol)[live].all()


@pytest.mark.parametrize("lengths,rank", [([1], 8), ([20], 16), ([40, 1, 30], 64)])
def test_a_wait_that_runs_out_leaves_nan(lengths, rank):
    """A row of half a million values keeps the rest of a tile waiting, and the other blocks of its cluster; with a limit of one microsecond (a few tokens are quick) it gives up. Nothing
    hangs, no wrong number is left, and the next call is as if nothing had been."""
    T, n, rows = sum(lengths), 1 << 19, 400
    g = gen(3)
    x, a = torch.randn(T, n, generator=g).to(BF16).cuda(), (torch.randn(3, rank, n, generator=g) / n ** 0.5).to(BF16).cuda()
    b, y = torch.randn(3, rows, rank, generator=g).to(BF16).cuda(), torch.randn(T, rows, generator=g).cuda()
    offsets = torch.tensor([0, *torch.tensor(lengths).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
    which = torch.arange(len(lengths), dtype=torch.int32, device="cuda")
    want = adapters.add(y, x, a, b, offsets, which)
    torch.cuda.synchronize()
    lost = torch.zeros_like(y, dtype=torch.bool)
    try:
        L.check(L.lib.frx_debug_set_wait_limit_ns(1_000))
        for _ in range(5):
            got = adapters.add(y, x, a, b, offsets, which)
            torch.cuda.synchronize()
            lost |= got.isnan()
            assert bool((got.isnan() | (got == want)).all())
    finally:
        L.check(L.lib.frx_debug_set_wait_limit_ns(0))
    assert bool(lost.any()) or lengths == [1], "no wait ran out"
    assert torch.equal(adapters.add(y, x, a, b, offsets, which), want)


def test_refusals():
    c = Case([2, 3], 64, 32, 16)
    y, x, a, b, offsets, which = c.args()
    f = adapters.add
    for call in (lambda: f(y, x.float(), a, b, offsets, which), lambda: f(y, x, a.half(), b, offsets, which), lambda: f(y, x, a, b.half(), offsets, which),
                 lambda: f(y, x[:4], a, b, offsets, which), lambda: f(y[:, :31], x, a, b, offsets, which), lambda: f(y, x[:, :56], a, b, offsets, which),
                 lambda: f(y, x, a[:2], b, offsets, which), lambda: f(y, x, a, b, offsets[:2], which), lambda: f(y, x, a, b, offsets.long(), which),
                 lambda: f(y, x, a, b, offsets, which, scale=torch.ones(4, device="cuda")), lambda: f(y, x, a, b, offsets, which, scale=torch.ones(5, dtype=BF16, device="cuda")),
                 lambda: f(y, x, a, b, offsets, which, out=y.float()), lambda: f(y.cpu(), x, a, b, offsets, which), lambda: f(y, x, a.transpose(1, 2), b, offsets, which),
                 lambda: f(y, x, torch.zeros(5, 136, 64, dtype=BF16, device="cuda"), torch.zeros(5, 32, 136, dtype=BF16, device="cuda"), offsets, which),
                 lambda: f(y, x, torch.zeros(5, 12, 64, dtype=BF16, device="cuda"), torch.zeros(5, 32, 12, dtype=BF16, device="cuda"), offsets, which),
                 lambda: f(y, x, a[:1].expand(5, 16, 64), b, offsets, which)):
        with pytest.raises(L.FrxError):
            call()


@pytest.mark.parametrize("rank", [64, 128])
@pytest.mark.parametrize("lengths", [[64] * 3, [50] * 400])
def test_sums_are_read_before_their_columns_are_used_again(lengths, rank):
    """The first product's parts fill tensor memory (512 of depth: as many parts as there is room for) and the second product's sums take the same columns: a tile over a cluster and tiles of
    a block each give the same bits in every one of many launches, and the formula's values."""
    c = Case(lengths, 512, 256, rank, out=F32, behind=0)
    y, *rest = c.args()
    c.check(scaled=False)
    want = adapters.add(y, *rest)
    got = [adapters.add(y, *rest) for _ in range(40)]
    assert all(torch.equal(g, want) for g in got)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("tiles,rank,depths", [(18, 64, (86016, 92160, 94208, 96256, 98304, 100352)), (320, 16, (9728, 10752, 11264, 11776, 12288, 15872))])
def test_a_wait_that_runs_out_in_some_warps_leaves_no_wrong_number(tiles, rank, depths, dtype):
    """Depths at which the first product is done just as the warps that wait for it give up: in some the wait has run out, in others not. What these write is NaN too, or right: each of their
    outputs needs the whole of A x. (A wait ends at the earliest after some polls of a few microseconds each, so these depths are some tens of microseconds of work, with clusters and without.)"""
    g, most = torch.Generator(device="cuda").manual_seed(4), max(depths)
    x, a = torch.randn(64 * tiles, most, generator=g, device="cuda").to(dtype), (torch.randn(3, rank, most, generator=g, device="cuda") / most ** 0.5).to(dtype)
    b, y = torch.randn(3, 400, rank, generator=g, device="cuda").to(dtype), torch.randn(64 * tiles, 400, generator=g, device="cuda")
    offsets = torch.arange(tiles + 1, dtype=torch.int32, device="cuda") * 64
    which = (torch.arange(tiles, device="cuda") % 3).int()
    wrong = torch.zeros((), dtype=torch.int64, device="cuda")
    for n in depths:
        args = y, x[:, :n], a[:, :, :n], b, offsets, which
        want = adapters.add(*args)
        torch.cuda.synchronize()
        try:
            L.check(L.lib.frx_debug_set_wait_limit_ns(1))
            for _ in range(100):
                got = adapters.add(*args)
                wrong += (~got.isnan() & (got != want)).any()
            torch.cuda.synchronize()
        finally:
            L.check(L.lib.frx_debug_set_wait_limit_ns(0))
        assert torch.equal(adapters.add(*args), want)
    assert int(wrong) == 0, f"{int(wrong)} calls left a finite number that is wrong"
