"""A row whose sum is one large value and very many small ones."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("V,at", [(131072, 0), (131072, 77777), (120003, 120002), (8000, 5), (1024, 1000)])
def test_small_values_beside_a_large_one(ops, V, at):
    """Each small one is 0.7 of a step of fp32 at 1: added to the large one by itself each would be a whole step.  A thread's pieces are added
    up by themselves: a value goes through at most 7 additions in its piece, 2 of pieces, one for each 32 of a thread's values (4), 6 in the
    wavefront and 15 of wavefronts, each off by 2^-24 of at most the row's sum; the exponentials by (1 + |d|) 2^-23 of the small ones', the
    logarithm and the difference by 2^-23."""
    small = math.log(0.7 * 2.0**-23)
    x = torch.full((1, V), small)
    x[0, at] = 0
    logp, entropy = ops.token_log_probs(x.to(DEV), torch.tensor([at], device=DEV))
    d = x.double()
    rest = (V - 1) * math.exp(float(d[0, (at + 1) % V]))
    want = -math.log1p(rest)
    bound = (7 + 2 + 4 + 6 + 15) * 2.0**-24 * (1 + rest) + 17 * 2.0**-23 * rest + 2.0**-23 * abs(want)
    assert abs(float(logp) - want) <= bound
