"""Batches of adapters' requests that reach what the others do not: several tokens among single ones of a rank of 17 to 64, thousands of requests, depths that end before the copies do."""
import pytest
import torch

from flashrt_b200 import adapters
from test_gpu_adapters import BF16, F16, F32, Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rank", [24, 40, 64])
@pytest.mark.parametrize("lengths", [[1] * 40 + [2, 17, 0, 1], [3] + [1] * 150 + [64, 65], [1] * 70 + [40]])
def test_several_tokens_among_single_ones(lengths, rank, dtype):
    c = Case(lengths, 328, 272, rank, dtype=dtype, out=dtype, behind=2)
    assert c.T < 2 * len(lengths)
    c.check()
    Case(lengths, 328, 259, rank, dtype=dtype, out=F32, behind=2).check()


@pytest.mark.parametrize("rank", [8, 32, 100])
@pytest.mark.parametrize("lengths", [[1] * 4096, [(i * 7) % 3 for i in range(3001)], [0] * 5000 + [1, 0, 70] + [0] * 2000])
def test_thousands_of_requests(lengths, rank):
    Case(lengths, 72, 96, rank).check()


@pytest.mark.parametrize("rank", [17, 32, 48, 64])
@pytest.mark.parametrize("n", [8, 72, 160, 328])
def test_copies_from_behind_the_depth(n, rank):
    """Some warps have no part of such a depth, or fewer steps than copies in flight, which write zeros to the places of B's rows: the formula's values, in every one of many calls."""
    c = Case([1] * 200, n, 1040, rank, none=0.0, behind=0)
    c.check()
    args = c.args()
    want = adapters.add(*args)
    assert all(torch.equal(adapters.add(*args), want) for _ in range(50))
