"""Sampling against the definition in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
INF, NAN = math.inf, math.nan
DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def f32(v):
    return float(torch.tensor(v, dtype=torch.float32))


def reference(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One row in 64 bits: (token, logp, how near the number is to the edge of its token, or top_p to the edge of what stays, relative to the whole).
    Settings are fp32."""
    x = x.double()
    temperature, top_p, min_p = f32(temperature), f32(top_p), f32(min_p)
    if bool((x.isnan() | (x == INF)).any()) or not 0 <= temperature < INF or any(v != v for v in (top_p, min_p, float(u))):
        return -1, NAN, 1.0
    if bool((x == -INF).all()):
        return -1, -INF, 1.0
    order = torch.sort(x, descending=True, stable=True).indices
    if temperature == 0:
        return int(order[0]), 0.0, 1.0
    w = torch.exp((x - x.max()) / temperature)
    kept, near = order[:top_k] if top_k > 0 else order, 1.0
    if top_p < 1:
        before = torch.cumsum(w[kept], 0) - w[kept]
        gap = (before - top_p * w[kept].sum()).abs() / w[kept].sum()
        near = float(torch.where(gap > 0, gap, 1.0).min())   # (an edge that is met exactly is one that both meet: sums of equal weights)
        n = max(1, int((before < top_p * w[kept].sum()).sum()))
        kept = kept[:n]
    if min_p > 0:
        kept = kept[w[kept] >= min(min_p, 1.0)]
    kept = torch.sort(kept).values
    edge = torch.cumsum(w[kept], 0)
    t = min(max(float(u), 0.0), 1 - 2.0**-24) * float(edge[-1])
    i = int(torch.searchsorted(edge, t, right=True))
    near = min(near, float((edge - t).abs().min() / edge[-1]))
    return int(kept[i]), float(torch.log(w[kept[i]] / edge[-1])) if float(w[kept[i]]) > 0 else -INF, near


def check(ops, x, u, **settings):
    """Tokens have to be the definition's; a number within 2^-28 of an edge (weights are good to 2^-38 of themselves and 2^-46 of the largest, and there are at
    most 2^17 of them here) may fall on either side of it, unless it is given that exactly.  logp is a difference of two numbers of 64 bits, rounded once."""
    on = {k: v.to(DEV) if isinstance(v, torch.Tensor) else v for k, v in settings.items()}
    tokens, logp = ops.sample_tokens(x.to(DEV), u.to(DEV), **on)
    assert tokens.dtype == torch.int64 and logp.dtype == torch.float32 and tokens.shape == logp.shape == x.shape[:-1]
    rows = x.reshape(-1, x.size(-1))
    for r in range(rows.size(0)):
        one = {k: v.reshape(-1)[r].item() if isinstance(v, torch.Tensor) else v for k, v in settings.items()}
        token, want, near = reference(rows[r], u.reshape(-1)[r], **one)
        got, lp = int(tokens.reshape(-1)[r]), float(logp.reshape(-1)[r])
        if near < 2.0**-28:
            continue
        assert got == token, (r, got, token, one)
        assert lp == want or (math.isnan(lp) and math.isnan(want)) or abs(lp - want) <= abs(want) * 2.0**-24 + 1e-9, (r, lp, want)


def logits(rows, V, dtype, seed=0, spread=2.5):
    g = torch.Generator().manual_seed(seed)
    x = spread * torch.randn(rows, V, generator=g)
    x = torch.where(torch.rand(rows, V, generator=g) < 0.002, x + 8, x)
    x[torch.rand(rows, V, generator=g) < 0.05] = -INF
    x[:, V // 2] = 1.5
    return x.to(dtype), torch.rand(rows, generator=g)


SETTINGS = [{}, {"temperature": 0.0}, {"temperature": 0.3}, {"temperature": 2.0, "top_k": 5}, {"top_k": 1}, {"top_k": 50, "top_p": 0.9}, {"top_p": 0.5}, {"top_p": 0.99, "min_p": 0.01},
            {"min_p": 0.2}, {"top_k": 300, "top_p": 0.7, "min_p": 0.05, "temperature": 1.5}, {"top_p": 0.0}, {"min_p": 1.0}, {"top_k": 10**9}]


@pytest.mark.parametrize("V", [1, 2, 7, 8, 29, 64, 511, 512, 513, 2048, 2049, 5000, 32000])
@pytest.mark.parametrize("dtype", DTYPES)
def test_settings(ops, V, dtype):
    for i, settings in enumerate(SETTINGS):
        x, u = logits(6, V, dtype, seed=V + i)
        check(ops, x, u, **settings)


@pytest.mark.parametrize("V", [70001, 131072])
@pytest.mark.parametrize("dtype", DTYPES)
def test_large_vocabularies(ops, V, dtype):
    for i, settings in enumerate(({}, {"top_p": 0.95}, {"top_k": 1000, "top_p": 0.9}, {"top_k": V // 2, "min_p": 1e-4}, {"temperature": 3.0, "top_p": 0.999})):
        x, u = logits(2, V, dtype, seed=i)
        check(ops, x, u, **settings)


def test_the_largest_vocabulary(ops):
    V = 1 << 21
    x, u = logits(1, V, torch.bfloat16)
    for settings in ({}, {"top_p": 0.9}, {"top_k": 100}, {"top_p": 0.9999, "temperature": 2.0}):
        token, logp = ops.sample_tokens(x.to(DEV), u.to(DEV), **settings)
        want, lp, near = reference(x[0], u[0], **settings)
        assert near < 2.0**-26 or int(token) == want and abs(float(logp) - lp) <= 1e-6 * abs(lp) + 1e-6
    with pytest.raises(ops.NNRuntimeException):
        ops.sample_tokens(torch.zeros(1, V + 1, device=DEV), u.to(DEV))


@pytest.mark.parametrize("V", [5, 300, 5000, 40000])
@pytest.mark.parametrize("dtype", DTYPES)
def test_ties(ops, V, dtype):
    """Equal values stay or go by their index, -0 equal to 0; all equal; two values; rising and falling rows."""
    g = torch.Generator().manual_seed(V)
    few = torch.randint(0, 3, (V,), generator=g).float()
    zeros = torch.zeros(V)
    zeros[torch.rand(V, generator=g) < 0.5] = -0.0
    ramp = torch.arange(V).float() * (20.0 / V)
    x = torch.stack([few, zeros, torch.full((V,), 3.0), ramp, -ramp, torch.where(torch.arange(V) == V - 1, 5.0, 1.0)]).to(dtype)
    for seed in range(3):
        u = torch.rand(6, generator=g)
        for settings in ({}, {"top_k": 2}, {"top_k": V // 2 + 1}, {"top_k": max(1, V - 1)}, {"top_p": 0.5}, {"top_p": 0.25, "top_k": V // 2 + 1}, {"min_p": 0.5}, {"top_p": 0.1, "min_p": 0.9},
                         {"temperature": 0.0}, {"top_k": 3, "top_p": 0.4}):
            check(ops, x, u, **settings)


def test_exact_borders(ops):
    """Four equal tokens: a sum that has reached top_p exactly takes no more, and a number on an edge goes to the token behind it."""
    x = torch.zeros(1, 4)
    for top_p, kept in ((0.25, 1), (0.26, 2), (0.5, 2), (0.75, 3), (0.76, 4)):
        for u in (0.0, 0.25, 0.5, 0.75, 0.999):
            token, logp = ops.sample_tokens(x.to(DEV), torch.tensor([u], device=DEV), top_p=top_p)
            assert int(token) == min(kept - 1, int(u * kept)) and abs(float(logp) + math.log(kept)) <= math.log(4) * 2.0**-24
    two = torch.tensor([[0.0, math.log(2.0)]]).double().float()
    for u, want in ((0.0, 0), (0.33, 0), (0.34, 1), (1 - 2.0**-24, 1)):
        assert int(ops.sample_tokens(two.to(DEV), torch.tensor([u], device=DEV))[0]) == want


def test_a_setting_for_each_row(ops):
    rows, V = 40, 3000
    x, u = logits(rows, V, torch.bfloat16, seed=5)
    g = torch.Generator().manual_seed(6)
    temperature = 2 * torch.rand(rows, generator=g)
    temperature[::5] = 0.0
    top_k = torch.randint(0, 100, (rows,), generator=g).int()
    top_k[1::4] = -3
    top_p, min_p = torch.rand(rows, generator=g) * 1.2, torch.rand(rows, generator=g) * 0.1 - 0.02
    check(ops, x, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    check(ops, x, u, temperature=0.7, top_k=top_k, top_p=0.9)
    check(ops, x.view(5, 8, V), u.view(5, 8), top_p=top_p.view(5, 8), min_p=0.01)


def test_rows_without_a_distribution(ops):
    V = 3000
    x = torch.randn(9, V)
    x[0, 5], x[1, V - 1] = NAN, INF
    x[2] = -INF
    x[3], x[3, 77] = -INF, 2.0
    u = torch.rand(9)
    u[4], u[5], u[6] = NAN, -3.0, 7.0
    temperature = torch.ones(9)
    for settings in ({}, {"top_k": 5}, {"top_p": 0.9}, {"temperature": 0.0}):
        check(ops, x, u, **settings)
    temperature[7], temperature[8], temperature[3] = -1.0, INF, NAN
    check(ops, x, u, temperature=temperature)
    bad = torch.ones(9)
    bad[7] = NAN
    check(ops, x, u, top_p=bad)
    check(ops, x, u, min_p=bad - 1)
    token, _ = ops.sample_tokens(x[:4].to(DEV), u[:4].to(DEV))
    assert token.tolist()[:3] == [-1, -1, -1] and int(token[3]) == 77


def test_temperatures_at_the_ends(ops):
    x, u = logits(4, 1000, torch.float32)
    for t in (1e-38, 1e-6, 1e3, 3e38):
        check(ops, x, u, temperature=t)
        check(ops, x, u, temperature=t, top_p=0.9)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [20000, 5003])
def test_exponents_out_of_range(ops, dtype, V):
    """Largest values whose power of two no 64 bits hold: sums are made relative to them."""
    x, u = logits(3, V, dtype, seed=V)
    for shift, t in ((0, 1e-3), (0, 0.004), (400, 0.3), (-700, 0.5)):
        for settings in ({}, {"top_p": 0.9}, {"top_k": 700, "top_p": 0.99}, {"min_p": 1e-3}, {"top_k": 20}):
            check(ops, (x.float() + shift).to(dtype), u, temperature=t, **settings)


@pytest.mark.parametrize("dtype", DTYPES)
def test_more_equal_values_than_a_count_holds(ops, dtype):
    """One value 100000 times in a row of 131072, or all of them: 16-bit counts pass their end."""
    V = 131072
    x = torch.full((2, V), 1.25)
    x[1, ::5] = 2.0
    x[1, 7::9] = -1.0
    x = x.to(dtype)
    for seed in range(2):
        u = torch.rand(2, generator=torch.Generator().manual_seed(seed))
        for settings in ({"top_p": 0.5}, {"top_k": 70000, "top_p": 0.75}, {"top_k": 3}, {"top_k": 1000}, {"min_p": 0.9}, {}):
            check(ops, x, u, **settings)


def test_many_rows(ops):
    """Rows of which two share a CU, and short ones by the thousand."""
    for rows, V, dtype in ((700, 9000, torch.float32), (3000, 300, torch.bfloat16), (600, 5000, torch.float16)):
        x, u = logits(rows, V, dtype, seed=rows)
        for settings in ({}, {"top_k": 30, "top_p": 0.9}, {"top_p": 0.8}):
            check(ops, x, u, **settings)


@pytest.mark.parametrize("rows, V", [(2, 24576), (2, 24577), (3, 32769), (257, 49152), (257, 49153), (513, 20000), (520, 33000)])
def test_rows_of_each_length_and_number(ops, rows, V):
    """What a row is worked out with depends on how long rows are and how many of them there are."""
    x, u = logits(rows, V, torch.bfloat16, seed=rows)
    some = torch.arange(0, rows, 1 + rows // 8)
    for settings in ({}, {"top_k": 40}, {"top_p": 0.9}, {"top_p": 0.6, "temperature": 0.3, "min_p": 0.01}, {"top_k": 2000, "top_p": 0.97}):
        tokens, logp = ops.sample_tokens(x.to(DEV), u.to(DEV), **settings)
        got = ops.sample_tokens(x[some].to(DEV), u[some].to(DEV), **settings)   # (few rows: other threads, the same tokens)
        assert torch.equal(tokens[some], got[0]) and bool(((logp[some] - got[1]).abs() <= logp[some].abs() * 2.0**-23 + 1e-9).all())
        check(ops, x[some], u[some], **settings)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, V", [(1, 49152), (1, 49153), (64, 49153), (65, 60000), (3, 131072), (128, 131080), (129, 131073), (2, 300007)])
def test_few_long_rows(ops, rows, V, dtype):
    """The first pass by all CUs for few rows: as each row by itself and as more of them."""
    x, u = logits(rows, V, dtype, seed=rows + V)
    some = torch.arange(0, rows, 1 + rows // 2)
    for settings in ({}, {"temperature": 0.0}, {"top_k": 40}, {"top_k": 900, "min_p": 1e-3}, {"top_p": 0.9}, {"top_p": 0.6, "temperature": 0.3}, {"top_k": 3000, "top_p": 0.97}, {"min_p": 0.05}):
        tokens, logp = ops.sample_tokens(x.to(DEV), u.to(DEV), **settings)
        got = ops.sample_tokens(x[some].to(DEV).repeat(300, 1), u[some].to(DEV).repeat(300), **settings)
        got = got[0].view(300, -1), got[1].view(300, -1)
        assert bool((got[0] == tokens[some]).all()) and bool(((got[1] - logp[some]).abs() <= logp[some].abs() * 2.0**-23 + 1e-9).all())
        if V < 2**17:
            check(ops, x[some], u[some], **settings)


def test_workspaces(ops):
    """A call that needs a workspace is refused without one; each call of two has its own."""
    import ctypes

    from pimaicompiler_amd import _lib as L
    x, u = torch.randn(2, 60000, device=DEV), torch.rand(2, device=DEV)
    tokens, logp, n = torch.full((2,), -7, device=DEV), torch.zeros(2, device=DEV), ctypes.c_uint64()
    settings = L.SampleSettings(temperature=1.0, top_k=5, top_p=1.0)
    lib = L.load()
    assert lib.pimhip_sample_workspace_bytes(L.PIMHIP_F32, 2, 60000, ctypes.byref(settings), ctypes.byref(n)) == L.PIMHIP_OK and n.value > 0
    call = [x.data_ptr(), L.PIMHIP_F32, 60000, 2, 60000, u.data_ptr(), ctypes.byref(settings), tokens.data_ptr(), logp.data_ptr()]
    workspace = torch.empty(n.value + 16, dtype=torch.uint8, device=DEV)
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.pimhip_sample_tokens(*call, None, stream) == L.PIMHIP_ERR_INVALID_ARGUMENT
    assert lib.pimhip_sample_tokens(*call, workspace.data_ptr() + 8, stream) == L.PIMHIP_ERR_INVALID_ARGUMENT
    assert tokens.tolist() == [-7, -7]
    assert lib.pimhip_sample_tokens(*call, workspace.data_ptr(), stream) == L.PIMHIP_OK
    assert torch.equal(tokens, ops.sample_tokens(x, u, top_k=5)[0])
    assert lib.pimhip_sample_workspace_bytes(L.PIMHIP_F32, 2, 1000, ctypes.byref(settings), ctypes.byref(n)) == L.PIMHIP_OK and n.value == 0
    assert lib.pimhip_sample_workspace_bytes(L.PIMHIP_F32, 2, 1000, ctypes.byref(settings), None) == L.PIMHIP_ERR_INVALID_ARGUMENT
    streams = [torch.cuda.Stream() for _ in range(2)]
    want = [ops.sample_tokens(v, u, top_p=0.5) for v in (x, -x)]
    torch.cuda.synchronize()
    for _ in range(5):
        got = [ops.sample_tokens(v, u, top_p=0.5, stream=s) for v, s in zip((x, -x), streams)]
        torch.cuda.synchronize()
        assert all(torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) for a, b in zip(got, want))


def test_two_captured_calls(ops):
    """Two graphs of calls that have workspaces, replayed in turn and at the same time with eager calls between, read logits, numbers and settings anew."""
    n, V = 3, 60000
    g = torch.Generator().manual_seed(1)
    xs = [torch.empty(n, V, dtype=t, device=DEV) for t in (torch.bfloat16, torch.float32)]
    us, ks = [torch.empty(n, device=DEV) for _ in xs], [torch.zeros(n, dtype=torch.int32, device=DEV) for _ in xs]
    streams, graphs, outs = [torch.cuda.Stream() for _ in xs], [torch.cuda.CUDAGraph() for _ in xs], []
    fill = lambda: [t.copy_(v) for x, u, k in zip(xs, us, ks) for t, v in ((x, 2.5 * torch.randn(n, V, generator=g)), (u, torch.rand(n, generator=g)),  # noqa: E731
                                                                          (k, torch.randint(0, 900, (n,), generator=g)))]
    fill()
    call = lambda i: ops.sample_tokens(xs[i], us[i], temperature=0.7, top_k=ks[i], top_p=0.9)  # noqa: E731
    for i in range(2):
        call(i)
    torch.cuda.synchronize()
    for graph, i in zip(graphs, range(2)):
        with torch.cuda.graph(graph):
            outs.append(call(i))
    for _ in range(4):
        fill()
        want = [call(i) for i in range(2)]
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        call(0)
        torch.cuda.synchronize()
        for out, w in zip(outs, want):
            assert torch.equal(out[0], w[0]) and torch.equal(out[1], w[1])


@pytest.mark.parametrize("V", [30001, 60001])
@pytest.mark.parametrize("dtype", DTYPES[:2])
def test_long_rows_at_the_ends(ops, dtype, V):
    """Rows that are counted: largest values out of range, no distribution, settings of their own."""
    x, u = logits(8, V, dtype, seed=3)
    for shift, t in ((0, 1e-3), (400, 0.3), (-700, 0.5)):
        for settings in ({"top_p": 0.9}, {"top_k": 700, "top_p": 0.99}, {"top_k": 5000, "min_p": 1e-3}):
            check(ops, (x.float() + shift).to(dtype), u, temperature=t, **settings)
    x[0, 5], x[1, V - 1] = NAN, INF
    x[2] = -INF
    x[3], x[3, 77] = -INF, 2.0
    x[4, ::2] = -INF
    u[5], u[6] = NAN, 7.0
    for settings in ({"top_p": 0.9}, {"top_k": 20000}, {"top_k": 20000, "top_p": 0.5}):
        check(ops, x, u, **settings)
    check(ops, x, u, top_k=torch.tensor([0, 900, 40, 0, 29000, 1, 600, 513]).int(), top_p=torch.tensor([0.9, 0.5, 0.9, 0.3, 0.999, 1.0, 1.0, 0.9]), temperature=0.8)


def test_shares(ops):
    """Evenly spread numbers draw each token as often as its share says, to one."""
    x, n = torch.tensor([0.5, 2.0, -1.0, 0.0, 1.0]), 4096
    u = (torch.arange(n) + 0.5) / n
    tokens, _ = ops.sample_tokens(x.expand(n, 5).to(DEV), u.to(DEV))
    got = torch.bincount(tokens.cpu(), minlength=5).double()
    assert bool(((got - n * torch.softmax(x.double(), 0)).abs() <= 1.0).all())


def test_views_and_shapes(ops):
    x, u = logits(6, 1001, torch.float16)
    want = ops.sample_tokens(x.to(DEV), u.to(DEV), top_p=0.9)
    wide = torch.zeros(6, 1010, dtype=torch.float16, device=DEV)
    wide[:, 3:1004] = x.to(DEV)
    for xx, uu in ((wide[:, 3:1004], u.to(DEV)), (x.to(DEV).t().contiguous().t(), torch.stack([u, u], 1).to(DEV)[:, 0])):
        got = ops.sample_tokens(xx, uu, top_p=0.9)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    one = ops.sample_tokens(x[0].to(DEV), u[0].to(DEV), top_p=0.9)
    assert one[0].shape == () and int(one[0]) == int(want[0][0])
    none = ops.sample_tokens(torch.zeros(0, 7, device=DEV), torch.zeros(0, device=DEV))
    assert none[0].shape == none[1].shape == (0,)


def test_refusals(ops):
    x, u = torch.zeros(2, 10, device=DEV), torch.zeros(2, device=DEV)
    ops.sample_tokens(x, u)
    for args, settings in (((x.double(), u), {}), ((x.cpu(), u), {}), ((x, u.double()), {}), ((x, u[:1]), {}), ((x, u.cpu()), {}), ((x[:, :0], u), {}), ((x.clone().requires_grad_(), u), {}),
                           ((x, u), {"temperature": -1.0}), ((x, u), {"temperature": NAN}), ((x, u), {"temperature": INF}), ((x, u), {"temperature": u.double()}), ((x, u), {"temperature": u[:1]}),
                           ((x, u), {"top_k": -1}), ((x, u), {"top_k": 1.5}), ((x, u), {"top_k": 2**31}), ((x, u), {"top_k": u}), ((x, u), {"top_p": 1.1}), ((x, u), {"top_p": -0.1}),
                           ((x, u), {"top_p": NAN}), ((x, u), {"min_p": 1.5}), ((x, u), {"min_p": -0.5}), ((x, u), {"min_p": u.cpu()}), ((x, u), {"temperature": "1"})):
        with pytest.raises(ops.NNRuntimeException):
            ops.sample_tokens(*args, **settings)
