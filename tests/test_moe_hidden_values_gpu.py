"""The expert layer's hidden values: as good as fp32 ones whatever their size, in every variant of the second product."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
INF = math.inf
# E, k, tokens, d_ff: one or two tokens, few and many pairs an expert, their values staged as a whole or not; many tokens of one expert
SHAPES = [(2, 2, 1, 16), (2, 2, 1, 8200), (2, 2, 2, 1040), (1, 1, 4, 4100), (2, 2, 5, 1040), (2, 2, 12, 16), (2, 2, 40, 16), (2, 2, 40, 3100), (32, 1, 40, 16), (32, 1, 40, 3100), (1, 1, 64, 520),
          (64, 32 // 2, 64, 100)]


def plan_of(ops, w1, w2, E, k, mx4, b1=None, **more):
    D = w1.size(1)
    each = lambda w: [ops.mx4_quantize(w.to(DEV)) for _ in range(E)] if mx4 else [w.to(DEV)] * E  # noqa: E731
    bias = [b1.to(DEV)] * E if b1 is not None else None
    return ops.MoeLayerPlan((torch.zeros(E, D, dtype=w1.dtype, device=DEV), None), each(w1), each(w2), bias, top_k=k, **more)


@pytest.mark.parametrize("E,k,M,F", SHAPES)
@pytest.mark.parametrize("dtype,mx4", [(torch.float16, False), (torch.float16, True), (torch.bfloat16, False), (torch.bfloat16, True)])
@pytest.mark.parametrize("size", ["small", "one", "large"])
def test_hidden_values_of_21_bits_cancel_exactly(ops, E, k, M, F, dtype, mx4, size):
    """Hidden values (1 + a 2^-9 + b 2^-18) u with a power of two u that takes them out of fp16's range: eight of them are added up, in pairs
    that leave a whole number of 2^-18 u.  Every sum on the way is a number of fp32, so the result is known to the bit; what a hidden
    value of fewer bits or of fp16's range drops is all of it."""
    g = torch.Generator().manual_seed(E + M + F)
    D = 32
    u = {"small": (-6, -6), "one": (0, 0), "large": (4, 13)}[size] if dtype == torch.float16 else {"small": (-20, -20), "one": (0, 0), "large": (20, 20)}[size]
    back = 2.0 ** -min(sum(u), 14) if dtype == torch.float16 else 2.0 ** -sum(u)
    x = torch.zeros(M, D, dtype=torch.float64)
    x[:, :4] = torch.tensor([1, 2.0**-9, 2.0**-18, 2.0 ** u[0]])
    values = torch.tensor([0, 1, 2, 3, 4, 6], dtype=torch.float64)   # (they are the same in 4 bits)
    w1 = torch.zeros(2 * F, D, dtype=torch.float64)
    w1[:F, 0] = 1
    w1[:F, 1:3] = values[torch.randint(6, (F, 2), generator=g)]
    w1[F:, 3] = 2.0 ** u[1]
    at = torch.randperm(F, generator=g)[:8].view(4, 2)
    w1[at[:, 1], 1] = w1[at[:, 0], 1]
    w2 = torch.zeros(D, F, dtype=torch.float64)
    sign = torch.randint(2, (D, 4), generator=g).double() * 2 - 1
    w2[:, at[:, 0]], w2[:, at[:, 1]] = sign * back, -sign * back
    want = ((w1[at[:, 0], 2] - w1[at[:, 1], 2]) * sign).sum(1) * 2.0**-18 * 2.0 ** sum(u) * back
    plan = plan_of(ops, w1.to(dtype), w2.to(dtype), E, k, mx4, act_type="none", gated=True)
    y, experts, shares = plan.forward(x.to(dtype).to(DEV))
    assert experts.cpu().tolist() == [list(range(k))] * M
    assert torch.equal(y.cpu().double(), want.expand(M, D))


@pytest.mark.parametrize("std,w2_std", [(0.003, 1.0), (1.0, 4096**-0.5), (200.0, 0.1 * 4096**-0.5)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("M", [2, 9])
def test_gated_layers_of_small_and_large_activations(ops, std, w2_std, dtype, M):
    """Against 64 bits: fp32 sums are within (n + 3) 2^-24 of the sum of magnitudes, SiLU within (8 + |v|) 2^-23 of its value, a hidden value
    loses at most 2^-22 of itself on the way into the second product, the result is rounded once."""
    g = torch.Generator().manual_seed(M)
    D, F = 1024, 4096
    x = (torch.randn(M, D, generator=g) * std).to(dtype)
    w1, w2 = (torch.randn(2 * F, D, generator=g) * D**-0.5).to(dtype), (torch.randn(D, F, generator=g) * w2_std).to(dtype)
    y = plan_of(ops, w1, w2, 1, 1, False, act_type="aten::silu", gated=True).forward(x.to(DEV))[0].cpu().double()
    x, w1, w2 = x.double(), w1.double(), w2.double()
    h, off = x @ w1.t(), (D + 3) * 2.0**-24 * (x.abs() @ w1.abs().t())
    a = h[:, :F] * torch.sigmoid(h[:, :F])
    off_a = 1.1 * off[:, :F] + a.abs() * (8 + h[:, :F].abs()) * 2.0**-23
    off_a = off_a * h[:, F:].abs() + a.abs() * off[:, F:] + off_a * off[:, F:]
    a = a * h[:, F:]
    off_a = off_a + a.abs() * 2.0**-22
    want = a @ w2.t()
    bound = off_a @ w2.abs().t() + (F + 3) * 2.0**-24 * (a.abs() @ w2.abs().t())
    half = torch.finfo(dtype).eps / 2
    bound = bound * (1 + half) + want.abs() * half + torch.finfo(dtype).tiny * half
    assert want.abs().max() < torch.finfo(dtype).max / 2
    assert bool(((y - want).abs() <= bound).all()), float(((y - want).abs() / bound).max())


@pytest.mark.parametrize("E,k,M,F", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_infinities_among_hidden_values_and_weights(ops, E, k, M, F, dtype):
    """An infinite hidden value is an infinite result of its weight's sign beside others that fp16 cannot hold; so is an infinite weight."""
    D = 16
    w1 = torch.zeros(2 * F, D, dtype=dtype)
    w1[:F, 0], w1[F:, 0] = 300.0, 300.0
    w2 = torch.ones(D, F, dtype=dtype) * -1
    w2[:8, F // 2] = 1
    b1 = torch.zeros(2 * F, dtype=dtype)
    x = torch.ones(M, D, dtype=dtype, device=DEV)
    b1[F // 2] = INF
    y = plan_of(ops, w1, w2, E, k, False, b1, act_type="none", gated=True).forward(x)[0].cpu()
    assert (y[:, :8] == INF).all() and (y[:, 8:] == -INF).all()
    w2[3, 0], w2[5, F - 1] = INF, -INF
    y = plan_of(ops, w1, w2, E, k, False, act_type="none", gated=True).forward(x)[0].cpu()
    assert (y[:, 3] == INF).all() and (y[:, 5] == -INF).all() and not y.isnan().any()


def test_a_pair_without_hidden_values(ops):
    """ReLU leaves nothing of one token, a little of another: neither takes the other's scale."""
    D, F = 64, 128
    w1, w2 = torch.zeros(F, D, dtype=torch.float16), torch.ones(D, F, dtype=torch.float16)
    w1[:, 0] = 1
    x = torch.zeros(3, D, dtype=torch.float16)
    x[:, 0] = torch.tensor([-5, 2.0**-24, 60000])
    y = plan_of(ops, w1, w2 * 2.0**-7, 1, 1, False, act_type="aten::relu").forward(x.to(DEV))[0].cpu().double()
    assert torch.equal(y, torch.tensor([0, 2.0**-24, 60000], dtype=torch.float64).half().double().unsqueeze(1).expand(3, D))
