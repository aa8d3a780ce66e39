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


def check_finite(got, x, w):
    """check_product's bound where the magnitudes add up to less than 2^127: no sum of fp32, in whatever order, leaves its range there.  What
    is beyond may have met an infinity of either sign on the way, or both.  Returns where the bound was asked for."""
    want, size, eps = x.double() @ w.t(), x.double().abs() @ w.abs().t(), torch.finfo(got.dtype).eps / 2
    fine = size < 2.0**127
    bound = (x.size(-1) + 2) * 2.0**-24 * size * (1 + eps) + want.abs() * eps + 2.0**-134
    assert bool(((got.cpu().double() - want).abs() <= bound)[fine].all())
    return fine


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


@pytest.mark.parametrize("K", [96, 256, 777])
@pytest.mark.parametrize("M", TOKENS)
@pytest.mark.parametrize("scale", [0, 2.0**-125, 2.0**-30, 1, 2.0**60])
def test_bf16_rows_of_both_ends(ops, M, K, scale):
    """Every code from the smallest (2^-127, whose smallest elements are subnormal) to the largest (2^127, whose largest are beyond bfloat16)."""
    q, w = matrix(ops, [0, 1, 2, 3, 60, 126, 127, 128, 200, 251, 252, 253, 254], K)
    x = (torch.randn(M, K, generator=torch.Generator().manual_seed(M), dtype=torch.float64) * scale).bfloat16()
    fine = check_finite(ops.mx4_linear(x.to(DEV), q), x, w)
    assert fine[:, -1].all() or scale >= 1


@pytest.mark.parametrize("K", [96, 256, 777])
@pytest.mark.parametrize("M", TOKENS)
def test_bf16_rows_of_the_smallest_scales_meet_large_tokens(ops, M, K):
    q, w = matrix(ops, [0, 1, 2, 3, 4, 5, 8], K)
    x = (torch.randn(M, K, generator=torch.Generator().manual_seed(M), dtype=torch.float64) * 2.0**110).bfloat16()
    check_product(ops.mx4_linear(x.to(DEV), q), x, w, None, False)


@pytest.mark.parametrize("M", TOKENS)
def test_fp16_rows_of_the_largest_scales(ops, M):
    """What is not zero is beyond fp16, and zero tokens stay zero."""
    K = 200
    q, w = matrix(ops, [140, 200, 252, 253, 254], K)
    for x in (torch.zeros(M, K).half(), torch.randn(M, K, generator=torch.Generator().manual_seed(M)).half() * 2.0**-18):
        check_product(ops.mx4_linear(x.to(DEV), q), x, w, None, False)


@pytest.mark.parametrize("M", TOKENS)
def test_a_code_of_each_end_in_one_row(ops, M):
    """bfloat16, blocks of 2^127 beside blocks of 2^100 and of 2^-20; a token that only the small ones see."""
    K = 192
    q, w = matrix(ops, [127] * 20, K)
    codes = torch.tensor([254, 227, 107, 253, 1, 127], dtype=torch.uint8).expand(20, 6).contiguous()
    q = ops.Mx4Tensor(q.packed, codes.to(DEV), K)
    w = w * power(codes.int() - 127).repeat_interleave(32, 1)
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(M)).bfloat16() * 2.0**-20
    assert check_finite(ops.mx4_linear(x.to(DEV), q), x, w).all()
    x[:, :64], x[:, 96:160] = 0, 0
    assert check_finite(ops.mx4_linear(x.to(DEV), q), x, w).all()


@pytest.mark.parametrize("M", TOKENS)
def test_both_operands_in_4_bits_at_both_ends(ops, M):
    K = 200
    a, av = matrix(ops, [0, 1, 60, 127, 200, 253, 254] * 50, K, 1)
    a, av = ops.Mx4Tensor(a.packed[:M], a.scales[:M, :7], K), av[:M]
    b, bv = matrix(ops, [0, 1, 60, 127, 200, 253, 254], K, 2)
    for dtype in (torch.float32, torch.bfloat16):
        assert check_finite(ops.mx4_matmul(a, b, dtype), av, bv).any()


@pytest.mark.parametrize("M", [1, 5, 40])
def test_bf16_experts_of_the_largest_scales(ops, M):
    """Hidden values around 2^-100 meet weights of 2^127: fp32 sums over d_model, then over d_ff."""
    D, F = 96, 200
    q1, w1 = matrix(ops, [27] * F, D)
    q2, w2 = matrix(ops, [252, 253, 254] * (D // 3), F, 1)
    plan = ops.MoeLayerPlan((torch.zeros(1, D, dtype=torch.bfloat16, device=DEV), None), [q1], [q2], top_k=1, act_type="none")
    x = torch.randn(M, D, generator=torch.Generator().manual_seed(M)).bfloat16()
    y = plan.forward(x.to(DEV))[0].cpu().double()
    h, off = x.double() @ w1.t(), (D + 3) * 2.0**-24 * (x.double().abs() @ w1.abs().t())
    want, bound = h @ w2.t(), off @ w2.abs().t() + (F + 3) * 2.0**-24 * (h.abs() @ w2.abs().t())
    assert bool(((y - want).abs() <= bound * (1 + 2.0**-8) + want.abs() * 2.0**-8).all())
