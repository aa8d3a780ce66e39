"""Log probabilities, entropy and alternatives of rows of logits against 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.float16, torch.bfloat16, torch.float32]
INF = math.inf


def reference(x, tokens, top):
    """In 64 bits on the CPU: (logp, entropy, ids, top_logp) and what bounds the error of the fp32 statistics.

    A row's sum goes through c = pieces per thread, eight additions each, and sums over threads; each of its terms is exp(d), off by (2 + |d|) 2^-23
    relative, once at its own place and in all by (|d| + 2 c) 2^-23 more where the running maximum moves on.  So log s is off by
    rel = (8 c + 16) 2^-24 + (2 c + 4) 2^-23 + 2 sum p |d| 2^-23, and t / s by sum p |d| (rel + (4 + 2 |d|) 2^-23)."""
    x = x.double()
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    s = e.sum(-1, keepdim=True)
    d = torch.where(e > 0, x - m, 0.0)
    p = e / s
    logp = x - m - torch.log(s)
    entropy = -(p * torch.where(e > 0, logp, 0.0)).sum(-1)
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :top]
    V = x.size(-1)
    threads = 64 if V <= 1024 else 256 if V <= 8192 else 1024
    c = -(-(-(-V // 8)) // threads)
    mean = (p * d.abs()).sum(-1)
    rel = (8 * c + 16) * 2.0**-24 + (2 * c + 4) * 2.0**-23 + 2 * mean * 2.0**-23
    rel_t = (p * d.abs() * (rel.unsqueeze(-1) + (4 + 2 * d.abs()) * 2.0**-23)).sum(-1)
    picked = logp.gather(1, tokens.long().clamp(0, V - 1).unsqueeze(1)).squeeze(1)
    log_s = torch.log(s).squeeze(1)

    def bound(v):
        return rel.view(-1, *[1] * (v.dim() - 1)) + (v.abs() + log_s.abs().view(-1, *[1] * (v.dim() - 1)) * 2) * 2.0**-23 + 2.0**-23
    return (picked, bound(picked)), (entropy, rel + rel_t + (entropy.abs() + 2 * log_s.abs()) * 2.0**-23 + 2.0**-23), order, (logp.gather(1, order), bound(logp.gather(1, order)))


def near(got, want):
    got, (value, bound) = got.cpu().double(), want
    same = (got == value) | (got.isnan() & value.isnan())
    assert bool((same | ((got - value).abs() <= bound)).all()), float(((got - value).abs() / bound)[~same].max())


def check(ops, x, tokens, top):
    out = ops.token_log_probs(x.to(DEV), tokens.to(DEV), top=top)
    logp, entropy, order, top_logp = reference(x, tokens, top)
    near(out[0], logp)
    near(out[1], entropy)
    if top:
        assert out[3].dtype == torch.int32 and torch.equal(out[3].cpu().long(), order)
        near(out[2], top_logp)
    else:
        assert len(out) == 2


@pytest.mark.parametrize("V,rows,top", [(1, 3, 1), (2, 5, 2), (7, 4, 0), (8, 2, 8), (29, 40, 20), (64, 3, 5), (1000, 9, 32), (1024, 2, 1), (1025, 3, 20), (8192, 2, 32),
                                        (8193, 2, 8), (32000, 1, 8), (31999, 5, 20), (100003, 3, 32), (131073, 1, 32)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_logits(ops, V, rows, top, dtype):
    g = torch.Generator().manual_seed(V + rows)
    x = (3 * torch.randn(rows, V, generator=g)).to(dtype)
    x[torch.rand(rows, V, generator=g) < 0.05] = -INF
    x[:, V // 2] = 1.5   # (no row is left without anything)
    tokens = torch.randint(V, (rows,), generator=g)
    check(ops, x, tokens, top)
    check(ops, x, tokens.int(), 0)


@pytest.mark.parametrize("V", [5, 300, 5000, 40000])
@pytest.mark.parametrize("dtype", DTYPES)
def test_order_and_ties(ops, V, dtype):
    """Equal values by their index, -0 equal to 0, rising and falling rows (the running maximum moves on at every piece, or never)."""
    top = min(V, 32)
    ramp = torch.arange(V).float() * (40.0 / V)
    few = torch.randint(0, 4, (V,), generator=torch.Generator().manual_seed(V)).float()
    zeros = torch.zeros(V)
    zeros[::2] = -0.0
    x = torch.stack([torch.full((V,), 2.5), ramp, ramp.flip(0), few, zeros, -few]).to(dtype)
    check(ops, x, torch.tensor([0, V - 1, V // 2, 0, V - 1, 1]), top)


@pytest.mark.parametrize("V", [40, 3000, 30000])
@pytest.mark.parametrize("dtype", DTYPES)
def test_masks(ops, V, dtype):
    low = torch.finfo(dtype).min
    x = torch.zeros(6, V, dtype=dtype)
    x[0, :] = -INF                       # nothing is left
    x[1, :] = low                        # masks of the type's lowest value: all alike
    x[2, :], x[2, V - 1] = -INF, 3.0     # one token is left
    x[3, :], x[3, 7] = low, 3.0
    x[4, :], x[4, 5] = low, -low         # as far apart as the type goes
    x[5, :V // 2] = -INF
    tokens = torch.tensor([3, 3, V - 1, 7, 5, 0])
    top = min(V, 32)
    logp, entropy, top_logp, ids = (t.cpu() for t in ops.token_log_probs(x.to(DEV), tokens.to(DEV), top=top))
    assert logp[0] == -INF and entropy[0] == 0 and (top_logp[0] == -INF).all() and ids[0].tolist() == list(range(top))
    for r in (1,):
        assert abs(logp[r] + math.log(V)) < 1e-5 and abs(entropy[r] - math.log(V)) < 1e-5 and ids[r].tolist() == list(range(top))
    assert logp[2] == 0 and entropy[2] == 0 and ids[2, 0] == V - 1 and ids[2, 1:].tolist() == list(range(top - 1)) and (top_logp[2, 1:] == -INF).all()
    for r, at in ((3, 7), (4, 5)):
        assert logp[r] == 0 and entropy[r] == 0 and ids[r, 0] == at and ids[r, 1] == 0
    assert logp[5] == -INF and abs(entropy[5] - math.log(V - V // 2)) < 1e-5 and ids[5, 0] == V // 2


@pytest.mark.parametrize("V", [20, 2000, 20000])
@pytest.mark.parametrize("bad", [math.nan, INF])
def test_a_row_without_a_distribution(ops, V, bad):
    for dtype in DTYPES:
        x = torch.randn(3, V, generator=torch.Generator().manual_seed(1)).to(dtype)
        x[1, V - 3] = bad
        out = ops.token_log_probs(x.to(DEV), torch.tensor([0, 1, 2], device=DEV), top=3)
        good = ops.token_log_probs(x[[0, 2]].to(DEV), torch.tensor([0, 2], device=DEV), top=3)
        for a, b in zip(out, good):
            assert torch.equal(a[[0, 2]], b)
        assert out[0][1].isnan() and out[1][1].isnan() and out[2][1].isnan().all() and (out[3][1] == -1).all()


def test_more_values_reach_the_bound_than_there_is_room_for(ops):
    """Large values everywhere but in the last of the groups that share a row: the bound is a small value, and 190000 large ones reach it."""
    V = 400000
    piece = torch.arange(V) // 8
    x = torch.where((piece % 1024) // 16 < 31, 1.0, 0.0).expand(2, V).clone()
    x[1, 399000] = 2.0
    out = ops.token_log_probs(x.to(DEV), torch.zeros(2, dtype=torch.int64, device=DEV), top=32)
    assert out[3][0].tolist() == list(range(32)) and out[3][1].tolist() == [399000] + list(range(31))


def test_padding_and_tokens_out_of_range(ops):
    x = torch.randn(4, 50, generator=torch.Generator().manual_seed(1)).half().to(DEV)
    for dtype in (torch.int64, torch.int32):
        logp, _ = ops.token_log_probs(x, torch.tensor([-1, -100, 50, 49], dtype=dtype, device=DEV))
        assert logp[:2].tolist() == [0, 0] and logp[2].isnan() and logp[3] < 0


def test_shapes_strides_and_no_tokens(ops):
    g = torch.Generator().manual_seed(2)
    wide = torch.randn(6, 5, 700, generator=g).bfloat16().to(DEV)
    for x in (wide[:, :, 3:690], wide[::2, 1:4], wide[0, :, :11], wide.transpose(1, 2), wide[2, 3]):
        lead, V = x.shape[:-1], x.size(-1)
        tokens = torch.randint(V, lead, generator=g).to(DEV)
        got = ops.token_log_probs(x, tokens, top=5)
        want = ops.token_log_probs(x.contiguous().view(-1, V), tokens.view(-1), top=5)
        for a, b, shape in zip(got, want, (lead, lead, (*lead, 5), (*lead, 5))):
            assert a.shape == shape and torch.equal(a.reshape(b.shape), b)
        logp, entropy = ops.token_log_probs(x)
        assert logp is None and torch.equal(entropy, got[1])
    none = ops.token_log_probs(wide[:0], torch.zeros(0, 5, dtype=torch.int64, device=DEV), top=2)
    assert [tuple(t.shape) for t in none] == [(0, 5), (0, 5), (0, 5, 2), (0, 5, 2)]


def test_a_graph_replays(ops):
    x = torch.randn(3, 9000, generator=torch.Generator().manual_seed(3)).half().to(DEV)
    tokens = torch.tensor([1, 2, 3], device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.token_log_probs(x, tokens, top=4)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs = ops.token_log_probs(x, tokens, top=4)
    torch.cuda.synchronize()
    for _ in range(4):
        x.copy_(x.roll(17, 1))
        eager = ops.token_log_probs(x, tokens, top=4)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, eager))


def test_refusals_on_the_gpu(ops):
    x = torch.zeros(2, 40, device=DEV)
    t = torch.zeros(2, dtype=torch.int64, device=DEV)
    for call in (lambda: ops.token_log_probs(x, t, top=33), lambda: ops.token_log_probs(x[:, :3], t, top=4), lambda: ops.token_log_probs(x, t, top=-1),
                 lambda: ops.token_log_probs(x, t, top=1.0), lambda: ops.token_log_probs(x, t[:1]), lambda: ops.token_log_probs(x, t.float()),
                 lambda: ops.token_log_probs(x, t.cpu()), lambda: ops.token_log_probs(x.double(), t), lambda: ops.token_log_probs(x[:, :0], t),
                 lambda: ops.token_log_probs(x.clone().requires_grad_(), t)):
        with pytest.raises(ops.NNRuntimeException):
            call()


def test_more_rows_than_a_launch_holds_are_refused(ops):
    from pimaicompiler_amd import _lib as L
    x = torch.zeros(8, device=DEV)
    for rows, V in ((1 << 22, 9000), (1 << 24, 2000), (1 << 26, 64)):
        assert L.load().pimhip_token_log_probs(x.data_ptr(), L.PIMHIP_F32, V, rows, V, None, 0, 0, None, x.data_ptr(), None, None, None) == L.PIMHIP_ERR_UNSUPPORTED
