"""Device-side waits that run out, in the products by expert and the adapters: nothing hangs, what is left is NaN or right, and the next call is as if
nothing had been. A wait gives up after some polls of a few microseconds each and its limit, so each of these has one of a hundred microseconds or so in its way."""
import pytest
import torch

from flashrt_b200 import adapters, moe
from flashrt_b200 import lib as L

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def normal(seed, *shape, dtype=BF16, size=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * size).to(dtype)


def until_lost(call, limit_ns, most):
    """Calls until a wait has run out, `most` at most; all of them leave what there is without limit, or NaN."""
    want = call()
    torch.cuda.synchronize()
    lost = torch.zeros_like(want, dtype=torch.bool)
    calls = 0
    try:
        L.check(L.lib.frx_debug_set_wait_limit_ns(limit_ns))
        while calls < most and not (calls >= 5 and bool(lost.any())):
            got = call()
            torch.cuda.synchronize()
            assert bool((got.isnan() | (got == want)).all()), "a finite number that is wrong"
            lost |= got.isnan()
            calls += 1
    finally:
        L.check(L.lib.frx_debug_set_wait_limit_ns(0))
    assert bool(lost.any()), "no wait ran out"
    assert torch.equal(call(), want)


@pytest.mark.parametrize("add", [False, True])
@pytest.mark.parametrize("out", [F32, BF16, F16])
def test_gradients_of_matrices(out, add):
    """Half a million rows of one expert between experts of few: the warp that zeroes what is behind its last row gives up, then the ones that load, multiply and write. (Of the other two forms no wait
    is for more than 512 of depth, a few microseconds: none of theirs can be made to run out like this. Their loops are the same code.)"""
    S = 1 << 19
    gy, x, offsets = normal(1, S, 64), normal(2, S, 128), torch.tensor([0, 5, 5, S - 3, S], dtype=torch.int32, device="cuda")
    old = normal(3, 4, 64, 128, dtype=out)
    until_lost(lambda: moe.moe_matmul_backward_w(gy, x, offsets, out=old.clone(), add=add), 10_000, 20)


@pytest.mark.parametrize("rank", [16, 32, 64])
def test_tokens_of_their_own(rank):
    """Clusters of eight blocks, some of which share their SMs with others and are late: the rest wait for their parts of A x."""
    users = 19
    x, a, b = normal(1, users, 1 << 20), normal(2, users, rank, 1 << 20, size=2.0 ** -10), normal(3, users, 400, rank)
    y, offsets = normal(4, users, 400, dtype=F32), torch.arange(users + 1, dtype=torch.int32, device="cuda")
    until_lost(lambda: adapters.add(y, x, a, b, offsets, offsets[:users]), 1, 60)
