"""Products with 4-bit weights at the ends of the scales' range: rows of the smallest and the largest codes, K that ends inside a unit."""
import pytest
import torch
from test_mx4_gpu import VALUES, check_product, power

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TOKENS = [1, 2, 5, 16, 33, 130, 300]


def matrix(ops, codes, K, seed=0):
    """(Mx4Tensor, its values in 64 bits) of rows with these scale codes in all blocks, any elements."""
    g = torch.Generator().manual_seed(seed + K)
    N, blocks = len(codes), -(-K // 32)
    packed = torch.randint(0, 256, (N, blocks * 16), generator=g, dtype=torch.uint8)
    scales = torch.tensor(codes, dtype=torch.uint8).unsqueeze(1).expand(N, blocks).contiguous()
    elements = torch.cat([VALUES, -VALUES])[torch.stack([packed & 15, packed >> 4], -1).view(N, -1).long()]
    return ops.Mx4Tensor(packed.to(DEV), scales.to(DEV), K), (elements * power(scales.int() - 127).repeat_interleave(32, 1))[:, :K]


@pytest.mark.parametrize("K", [31, 64, 96, 130, 200, 256, 777])
@pytest.mark.parametrize("M", TOKENS)
def test_fp16_rows_of_every_small_scale(ops, M, K):
    """Their products with fp16 tokens are far below fp16's range: zeros, whatever the row's largest code."""
    q, w = matrix(ops, list(range(40)), K)
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(M)).half()
    y = ops.mx4_linear(x.to(DEV), q)
    check_product(y, x, w, None, False)
    assert (y == 0).all()


@pytest.mark.parametrize("d_model,d_ff,M", [(64, 33, 1), (96, 100, 5), (96, 300, 40)])
def test_fp16_experts_of_every_small_scale(ops, d_model, d_ff, M):
    q1, _ = matrix(ops, [(i % 40) for i in range(d_ff)], d_model)
    q2, _ = matrix(ops, [(i % 40) for i in range(d_model)], d_ff, 1)
    plan = ops.MoeLayerPlan((torch.zeros(1, d_model, dtype=torch.float16, device=DEV), None), [q1], [q2], top_k=1, act_type="aten::relu")
    y = plan.forward(torch.randn(M, d_model, generator=torch.Generator().manual_seed(1)).half().to(DEV))[0]
    assert (y == 0).all()
