"""How near results in 32 bits are to the formulas: sharper than the bounds that hold for any input.

Tolerances. The tensor cores cut off the sum that each instruction (16 of depth) adds to, towards zero: by half a step of it on average, which is 2^-24 of the power of two below it, 0.71 * 2^-24 of
it in the root mean square. Sums of random signs grow with the root of the depth, so a run of m instructions is off by 0.71 * 2^-24 (sum over k = 1 .. m of sqrt(k / m)) of its sum: 4.7e-7 for
the 16 of 256 of depth, and 1.3e-6, 2.1e-6 or more where runs are as long as a depth of 2,048 or 8,192. Runs are added rounded to nearest, 32 of them at most: 32 times a quarter of a step and less,
independent of one another, 1e-7. In the root of the squares' sum below 5e-7. The adapters' second product cuts the sums of its largest pieces up to four times, another 1.4e-7 at most: 6e-7."""
import pytest
import torch

from flashrt_b200 import adapters, moe

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def normal(seed, *shape, dtype=BF16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def rms(got, want):
    return float((got.double() - want).square().mean().sqrt() / want.square().mean().sqrt())


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("depth", [512, 2048, 8192])
def test_products_by_expert(depth, dtype):
    od = torch.tensor([0, 160, 300], dtype=torch.int32, device="cuda")
    x, w = normal(1, 300, depth, dtype=dtype), normal(2, 2, 256, depth, dtype=dtype)
    want = torch.cat([x[:160].double() @ w[0].double().T, x[160:].double() @ w[1].double().T])
    assert rms(moe.moe_matmul(x, w, od, dtype=F32), want) < 5e-7
    wt = w.transpose(1, 2).contiguous()
    assert rms(moe.moe_matmul_backward_x(x, wt, od, dtype=F32), want) < 5e-7
    od = torch.tensor([0, depth], dtype=torch.int32, device="cuda")
    gy, x = normal(3, depth, 128, dtype=dtype), normal(4, depth, 256, dtype=dtype)
    assert rms(moe.moe_matmul_backward_w(gy, x, od, dtype=F32)[0], gy.double().T @ x.double()) < 5e-7


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("lengths,rank", [([1] * 40, 16), ([1] * 40, 32), ([1] * 40, 64), ([64, 64, 30], 16), ([64, 64, 30], 64), ([64] * 310, 16)])
def test_adapters(lengths, rank, dtype):
    T = sum(lengths)
    x, a, b = normal(1, T, 2048, dtype=dtype), normal(2, 1, rank, 2048, dtype=dtype), normal(3, 1, 512, rank, dtype=dtype)
    y, offsets = torch.zeros(T, 512, device="cuda"), torch.tensor([0, *torch.tensor(lengths).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
    got = adapters.add(y, x, a, b, offsets, torch.zeros(len(lengths), dtype=torch.int32, device="cuda"))
    assert rms(got, (x.double() @ a[0].double().T) @ b[0].double().T) < 6e-7


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("lengths,rank", [([1] * 5, 16), ([1] * 200, 16), ([1] * 5, 32), ([1] * 200, 64), ([40, 1, 64], 16), ([40, 1, 64], 64), ([40, 1, 64], 128), ([64] * 310, 16)])
def test_what_is_between_the_products_has_32_bits(lengths, rank, dtype):
    """A x is whole numbers of 24 bits, from three products of whole numbers of eight bits each in different instructions, and every row of B has one power of two: there is nothing to round
    anywhere, if A x is kept whole. What is allowed is a step of 2^-23 for each of five additions, 6e-7 (the first product has two, the pieces of A x three); with its last eight bits left out A x is
    off by up to 2^-16 of it, 1.5e-5."""
    T, n, rows = sum(lengths), 256, 300
    g = torch.Generator().manual_seed(7)
    digits = torch.randint(1, 256, (rank, 3), generator=g)
    digits[:, 0] |= 128                                         # 24 bits, the first and the last of them set
    digits[:, 2] |= 1
    at, powers = (3, 100, 250), (2.0 ** 8, 1.0, 2.0 ** -8)
    a, x = torch.zeros(1, rank, n), torch.zeros(T, n)
    for c, p, d in zip(at, powers, digits.T):
        a[0, :, c], x[:, c] = d.float(), p
    sign = torch.randint(0, 2, (T, 1), generator=g) * 2.0 - 1
    x *= sign
    b = torch.zeros(1, rows, rank)
    of, size = torch.randint(0, rank, (rows,), generator=g), torch.exp2(torch.randint(-3, 4, (rows,), generator=g).float())
    b[0, torch.arange(rows), of] = size
    v = digits.double() @ torch.tensor(powers, dtype=torch.float64)
    want = sign.double() * (v[of] * size.double())
    offsets = torch.tensor([0, *torch.tensor(lengths).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
    for columns in (rows, 288):                                  # results whose rows are not whole accesses of 32 bytes, and that are
        got = adapters.add(torch.zeros(T, columns, device="cuda"), x.to(dtype).cuda(), a.to(dtype).cuda(), b[:, :columns].to(dtype).cuda(), offsets,
                           torch.zeros(len(lengths), dtype=torch.int32, device="cuda"))
        assert ((got.double().cpu() - want[:, :columns]).abs() <= 5 * 2.0 ** -23 * want[:, :columns].abs()).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_results_in_16_bits_are_rounded_once(dtype):
    """A result with an error of e lands on a neighbour of the value that the sum in 64 bits rounds to in e / (the type's step there) of all cases. Runs of 1,024 of depth leave 0.71 * 2^-24 (sum over
    k = 1 .. 64 of sqrt(k / 64)) = 1.83e-6 of the root mean square, s; the mean of magnitudes is 0.8 of that. A step at y is at least eps / 2 * |y|, and for normal y the mean of s / |y|, counted where
    |y| > s / 4, is 1.17: so no more than 0.8 * 1.83e-6 * 2 / eps * 1.17. (Runs as long as this depth leave 8e-6.)"""
    depth, rows = 8192, 1024
    od = torch.tensor([0, 256, 512], dtype=torch.int32, device="cuda")
    x, w = normal(5, 512, depth, dtype=dtype), (normal(6, 2, rows, depth, dtype=F32) / depth ** 0.5).to(dtype)
    wt, gy = w.transpose(1, 2).contiguous(), normal(7, depth, rows, dtype=dtype) * (1 / 64)
    want = torch.cat([x[:256].double() @ w[0].double().T, x[256:].double() @ w[1].double().T])
    xw = normal(8, depth, 512, dtype=dtype)
    for got, want in ((moe.moe_matmul(x, w, od), want), (moe.moe_matmul_backward_x(x, wt, od), want),
                      (moe.moe_matmul_backward_w(gy, xw, torch.tensor([0, depth], dtype=torch.int32, device="cuda"))[0], gy.double().T @ xw.double())):
        counted = want.abs() > want.square().mean().sqrt() / 4
        share = float((got != want.to(dtype))[counted].double().sum() / counted.numel())
        assert share < 0.8 * 1.83e-6 * 2 / torch.finfo(dtype).eps * 1.17
