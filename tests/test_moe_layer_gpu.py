"""The mixture-of-experts layer for a few tokens against the layer in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
INF = math.inf


class Layer:
    """A layer's tensors on the CPU, its plan, and its outputs in 64 bits with what bounds the error of the plan's."""

    def __init__(self, ops, seed, E, k, D, F, dtype=torch.float16, act="aten::relu", gated=False, bias=True, renormalize=True, mx4=False, stacked=False):
        g = torch.Generator().manual_seed(seed)
        rows = 2 * F if gated else F
        n = lambda *s, scale: (torch.randn(*s, generator=g) * scale).to(dtype)  # noqa: E731
        self.k, self.D, self.F, self.E, self.dtype, self.act, self.gated, self.renormalize = k, D, F, E, dtype, act, gated, renormalize
        self.wr, self.br = n(E, D, scale=D**-0.5), n(E, scale=0.1) if bias else None
        self.b1, self.b2 = (n(E, rows, scale=0.2), n(E, D, scale=0.2)) if bias else (None, None)
        w1, w2 = n(E, rows, D, scale=D**-0.5), n(E, D, F, scale=F**-0.5)
        dev = lambda t: t.to(DEV) if t is not None else None  # noqa: E731
        if mx4:
            q1, q2 = [ops.mx4_quantize(w.to(DEV)) for w in w1], [ops.mx4_quantize(w.to(DEV)) for w in w2]
            self.w1, self.w2 = (torch.stack([q.dequantize(torch.float32).cpu() for q in qs]).double() for qs in (q1, q2))
            weights = q1, q2
        else:
            self.w1, self.w2 = w1.double(), w2.double()
            weights = (w1.to(DEV), w2.to(DEV)) if stacked else ([w.to(DEV) for w in w1], [w.to(DEV) for w in w2])
        self.plan = ops.MoeLayerPlan((dev(self.wr), dev(self.br)), *weights, dev(self.b1), dev(self.b2), top_k=k, act_type=act, gated=gated,
                                     renormalize=renormalize)
        self.x = lambda M, s=0: torch.randn(M, D, generator=torch.Generator().manual_seed(seed + M + s)).to(dtype)

    def activation(self, v):
        return v if self.act == "none" else v.clamp(min=0) if self.act == "aten::relu" else v * torch.sigmoid(v)

    def reference(self, x):
        """y, its bound, experts, shares, and which tokens' choice is clear.  Products of fp32 sums: (n + 3) 2^-24 of the sum of magnitudes; the
        activation has a slope of at most 1.1 and, as SiLU, (8 + |v|) 2^-23 of its value from exp and the division; hidden values are kept
        in two pieces of their type, the second rounded by half a step of at most half a step of the first, y in one; shares are off by (2 + difference of logits) 2^-22."""
        x = x.double()
        logits = x @ self.wr.double().t()
        size = x.abs() @ self.wr.double().abs().t()
        if self.br is not None:
            logits, size = logits + self.br.double(), size + self.br.double().abs()
        order = torch.sort(logits, dim=-1, descending=True, stable=True)
        experts, picked = order.indices[:, :self.k], order.values[:, :self.k]
        off_logit = (self.D + 3) * 2.0**-24 * torch.nan_to_num(size, posinf=0).amax(-1)
        m = picked[:, :1]
        e = torch.where(torch.isinf(m) & (m < 0), 0.0, torch.exp(picked - m))
        full = torch.where(torch.isinf(m) & (m < 0), 0.0, torch.exp(logits - m)).sum(-1, keepdim=True)
        total = e.sum(-1, keepdim=True) if self.renormalize else full
        shares = torch.where(total > 0, e / total, 0.0)
        gaps = order.values[:, :-1] - order.values[:, 1:] if self.E > 1 else torch.full((x.size(0), 1), INF)
        clear = (gaps[:, :self.k] > 4 * off_logit.unsqueeze(1)).all(-1)
        half = torch.finfo(self.dtype).eps / 2
        y, bound = torch.zeros_like(x), torch.zeros_like(x)
        f32 = 2.0**-24
        for t in range(x.size(0)):
            for j in range(self.k):
                n, c = int(experts[t, j]), float(shares[t, j])
                if c == 0:
                    continue
                h, hs = x[t] @ self.w1[n].t(), x[t].abs() @ self.w1[n].abs().t()
                if self.b1 is not None:
                    h, hs = h + self.b1[n].double(), hs + self.b1[n].double().abs()
                off = (self.D + 3) * f32 * hs
                a = self.activation(h[:self.F])
                off_a = 1.1 * off[:self.F] + (a.abs() * (8 + h[:self.F].abs()) * 2.0**-23 if self.act == "aten::silu" else 0)
                if self.gated:
                    off_a = off_a * h[self.F:].abs() + a.abs() * off[self.F:] + off_a * off[self.F:]
                    a = a * h[self.F:]
                off_a = off_a + a.abs() * (half * half + 2.0**-23) + torch.finfo(self.dtype).tiny * half
                o, size_o = a @ self.w2[n].t(), a.abs() @ self.w2[n].abs().t()
                if self.b2 is not None:
                    o, size_o = o + self.b2[n].double(), size_o + self.b2[n].double().abs()
                off_o = off_a @ self.w2[n].abs().t() + (self.F + 3) * f32 * size_o
                off_c = c * ((2 + float(picked[t, 0] - picked[t, j])) * 2.0**-22 + 4 * float(off_logit[t]))
                y[t] += c * o
                bound[t] += c * off_o + off_c * (o.abs() + off_o)
        bound = bound * (1 + half) + y.abs() * (half + (self.k + 2) * f32) + torch.finfo(self.dtype).tiny * half
        return y, bound, experts, shares, clear, off_logit

    def check(self, x, out=None):
        y, experts, shares = (t.cpu() for t in (out or self.plan.forward(x.to(DEV))))
        want, bound, chosen, c, clear, off = self.reference(x)
        assert y.dtype == self.dtype and experts.dtype == torch.int32 and shares.dtype == torch.float32
        assert clear.double().mean() > 0.8 or x.size(0) < 3   # (tokens whose choice hangs on the last bits are left out)
        assert torch.equal(experts[clear].long(), chosen[clear])
        assert bool(((shares.double() - c).abs() <= 2.0**-20 + 4 * off.unsqueeze(1))[clear].all())
        far = (y.double() - want).abs()
        assert bool((far <= bound)[clear].all()), float((far / bound)[clear].max())


CASES = [
    # E, k, D, F, M
    (8, 2, 1024, 4096, 1), (8, 2, 256, 512, 5), (4, 1, 136, 520, 16), (1, 1, 8, 8, 3), (3, 3, 64, 24, 33), (60, 6, 200, 72, 13), (256, 16, 128, 64, 20),
    (2, 2, 264, 136, 64), (5, 4, 2048, 96, 40), (8, 2, 320, 1000, 65), (4, 2, 96, 160, 150),
    (32, 6, 1024, 520, 64), (3, 2, 128, 1032, 37),
    # hidden layers of sizes that are multiples of nothing
    (4, 2, 64, 65, 5), (8, 2, 136, 333, 40), (3, 1, 72, 1, 2), (60, 3, 200, 71, 13), (2, 1, 1160, 1615, 1), (8, 2, 64, 1027, 64),
]


@pytest.mark.parametrize("E,k,D,F,M", CASES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("gated,act,mx4", [(False, "aten::relu", False), (True, "aten::silu", False), (True, "aten::silu", True), (False, "none", True)])
def test_layer(ops, E, k, D, F, M, dtype, gated, act, mx4):
    layer = Layer(ops, E * D + F, E, k, D, F, dtype, act, gated, bias=(E + M) % 2 == 0, renormalize=M % 2 == 1, mx4=mx4, stacked=M % 3 == 0)
    layer.check(layer.x(M))


def test_every_token_wants_the_same_experts(ops):
    """64 tokens of one expert, and experts without any."""
    layer = Layer(ops, 5, 6, 2, 128, 256, bias=True)
    layer.br[:] = torch.tensor([0, 0, 50, 0, 40, 0]).half()
    layer.plan = ops.MoeLayerPlan((layer.wr.to(DEV), layer.br.to(DEV)), layer.w1.half().to(DEV), layer.w2.half().to(DEV), layer.b1.to(DEV), layer.b2.to(DEV),
                                  top_k=2, act_type="aten::relu")
    for M in (64, 17, 33):
        x = layer.x(M)
        out = layer.plan.forward(x.to(DEV))
        assert out[1].cpu().tolist() == [[2, 4]] * M
        layer.check(x, out)


def test_masked_experts(ops):
    """-inf in the router's bias takes experts out; where fewer are left than are chosen the rest have no share, also if they are broken."""
    layer = Layer(ops, 6, 4, 3, 64, 32, bias=True, act="aten::silu", gated=True)
    layer.br[:] = torch.tensor([-INF, 0, -INF, 0.1]).half()
    layer.w1[0] = math.nan
    make = lambda: ops.MoeLayerPlan((layer.wr.to(DEV), layer.br.to(DEV)), layer.w1.half().to(DEV), layer.w2.half().to(DEV), layer.b1.to(DEV),  # noqa: E731
                                    layer.b2.to(DEV), top_k=3, gated=True)
    x = layer.x(9)
    y, experts, shares = make().forward(x.to(DEV))
    assert (experts[:, 2] == 0).all() and (shares[:, 2] == 0).all() and torch.isfinite(y).all()
    want, bound, *_ = layer.reference(x)
    assert bool(((y.cpu().double() - want).abs() <= bound).all())
    layer.br[:] = -INF
    y, experts, shares = make().forward(x.to(DEV))
    assert (y == 0).all() and (shares == 0).all() and experts.cpu().tolist() == [[0, 1, 2]] * 9


def test_equal_logits_go_by_index_and_a_nan_spoils_its_token_alone(ops):
    layer = Layer(ops, 7, 10, 4, 72, 40, bias=False)
    x = layer.x(6)
    layer.plan = ops.MoeLayerPlan((torch.zeros_like(layer.wr).to(DEV), None), layer.w1.half().to(DEV), layer.w2.half().to(DEV), top_k=4, act_type="aten::relu")
    y, experts, shares = layer.plan.forward(x.to(DEV))
    assert experts.cpu().tolist() == [[0, 1, 2, 3]] * 6 and (shares == 0.25).all()
    x[2, 71] = math.nan
    z, experts, shares = layer.plan.forward(x.to(DEV))
    rest = [0, 1, 3, 4, 5]
    assert torch.equal(z[rest], y[rest]) and z[2].isnan().all() and shares[2].isnan().all() and experts[2].tolist() == [0, 1, 2, 3]


def test_shapes_and_strides(ops):
    layer = Layer(ops, 8, 4, 2, 40, 48, torch.bfloat16, "aten::silu", True)
    wide = torch.randn(4, 6, 49, generator=torch.Generator().manual_seed(1)).bfloat16().to(DEV)
    for x in (wide[:, :, 3:43], wide[1, :, 9:], wide[:, 2, :40], wide[0, 0, 5:45], wide[:, :, :40].transpose(0, 1)):
        y, experts, shares = layer.plan.forward(x)
        assert y.shape == x.shape and experts.shape == (*x.shape[:-1], 2)
        flat = layer.plan.forward(x.contiguous().view(-1, 40))
        assert torch.equal(y.view(-1, 40), flat[0]) and torch.equal(experts.view(-1, 2), flat[1]) and torch.equal(shares.view(-1, 2), flat[2])
    assert [tuple(t.shape) for t in layer.plan.forward(wide[:0, 0, :40])] == [(0, 40), (0, 2), (0, 2)]


def test_graphs_of_one_plan_keep_apart(ops):
    """Two captured forwards of one plan, replayed on two streams at a time, and eager calls between."""
    layer = Layer(ops, 9, 8, 2, 512, 1024, act="aten::silu", gated=True, bias=False)
    xs = [layer.x(3).to(DEV), layer.x(40).to(DEV)]
    streams, graphs, outs = [torch.cuda.Stream() for _ in xs], [], []
    for x, s in zip(xs, streams):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            layer.plan.forward(x)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                outs.append(layer.plan.forward(x))
            graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(6):
        for x in xs:
            x.copy_(x.roll(1, 1))
        eager = [layer.plan.forward(x) for x in xs]
        torch.cuda.synchronize()
        for _ in range(3):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
            layer.plan.forward(xs[0])
        torch.cuda.synchronize()
        for a, b in zip(outs, eager):
            assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_a_stream_of_the_caller_s(ops):
    layer = Layer(ops, 10, 4, 2, 64, 64)
    x = layer.x(5).to(DEV)
    want = layer.plan.forward(x)
    side = torch.cuda.Stream()
    for stream in (side, side.cuda_stream):
        side.wait_stream(torch.cuda.current_stream())
        got = layer.plan.forward(x, stream=stream)
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals_on_the_gpu(ops):
    z = lambda *s, dtype=torch.float16: torch.zeros(*s, dtype=dtype, device=DEV)  # noqa: E731
    E = ops.NNRuntimeException
    wr, w1, w2 = z(4, 64), z(4, 32, 64), z(4, 64, 32)
    q = [ops.mx4_quantize(w) for w in w1]
    bad = [dict(router=(z(3, 64), None)), dict(router=(wr.float(), None)), dict(w1=w1.bfloat16()), dict(w2=z(4, 64, 40)), dict(top_k=5), dict(top_k=0), dict(act_type="gelu"),
           dict(gated=True), dict(b1=z(4, 31)), dict(b2=z(4, 64).float()), dict(w1=q), dict(w1=w1.cpu()), dict(router=(wr, z(5))),
           dict(router=(z(4, 60), None), w1=z(4, 32, 60), w2=z(4, 60, 32)), dict(w1=w1.clone().requires_grad_()), dict(w1=z(4, 31, 64), gated=True)]
    for change in bad:
        with pytest.raises(E):
            ops.MoeLayerPlan(**{**dict(router=(wr, None), w1=w1, w2=w2), **change})
    plan = ops.MoeLayerPlan((wr, None), w1, w2)
    for x in (z(2, 63), z(2, 64).float(), z(2, 64).cpu(), z(2, 64).requires_grad_()):
        with pytest.raises(E):
            plan.forward(x)
    from pimaicompiler_amd import _lib as L
    import ctypes
    n = ctypes.c_uint64()
    assert L.load().pimhip_moe_layer_workspace_bytes(plan._handle, 65, ctypes.byref(n)) == L.PIMHIP_ERR_UNSUPPORTED
    assert L.load().pimhip_moe_layer_forward(plan._handle, None, 64, 1, None, None, None, None, None) == L.PIMHIP_ERR_INVALID_ARGUMENT


def test_a_destroyed_plan_is_refused(ops):
    from pimaicompiler_amd import _lib as L
    layer = Layer(ops, 3, 4, 2, 64, 32)
    x = layer.x(2).to(DEV)
    layer.plan.forward(x)
    assert L.load().pimhip_moe_layer_plan_destroy(layer.plan._handle) == L.PIMHIP_OK
    for stream in (None, torch.cuda.Stream()):
        with pytest.raises(ops.NNRuntimeException):
            layer.plan.forward(x, stream=stream)
    assert L.load().pimhip_moe_layer_plan_destroy(layer.plan._handle) == L.PIMHIP_ERR_INVALID_ARGUMENT
