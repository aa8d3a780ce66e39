"""Tokens that attention gives no weight: a score of -inf, as a mask kept in a key has, leaves nothing of a token's values, however large they are."""
import math

import pytest
import torch

from paged_cases import Cache, attend

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads, dim, page", [(1, 64, 16), (8, 128, 16), (20, 64, 16), (24, 128, 12), (3, 80, 16), (2, 256, 32)])
@pytest.mark.parametrize("left_out", [1, 2, 16, 70])
@pytest.mark.parametrize("n", [100, 3001])
def test_scores_of_minus_infinity(ops, dtype, heads, dim, page, left_out, n):
    """The first tokens of a sequence are left out by their keys.  In some columns they alone have a value: exactly 0 is theirs.  The rest is what the other tokens give."""
    cache = Cache([n], 1, page, dim, dtype, seed=n)
    q = torch.randn(1, heads, dim, generator=torch.Generator().manual_seed(2))
    q[..., 0] = q[..., 0].abs() + 0.5
    cache.v[..., [0, dim - 1]] = 0.0
    want, lse, bound, lse_bound = attend(cache, q.to(dtype), 1 / math.sqrt(dim), window=n - left_out)
    for j in range(left_out):
        p = int(cache.table[0, j // page])
        cache.k[p, 0, j % page, 0] = -math.inf
        cache.v[p, 0, j % page, [0, dim - 1]] = torch.tensor([1.0, -1.0]).to(dtype) * torch.finfo(dtype).max
        cache.v[p, 0, j % page, 1] = torch.finfo(dtype).max / 2
    table, lengths = cache.tensors(DEV)
    out, sums = cache.on(ops, DEV).attend(q.to(dtype).to(DEV), table, lengths, lse=True)
    out, sums = out.cpu().double(), sums.cpu().double()
    assert bool((out[..., [0, dim - 1]] == 0).all()), out[..., [0, dim - 1]]
    assert bool(((out - want).abs() <= bound).all()) and bool(((sums - lse).abs() <= lse_bound).all())
