"""A served model's step with a paged cache as a program runs it: prompts, then tokens one at a time through append, attend, a projection in 4 bits, log
probabilities and sampling; captured, on other streams, and without the native per-call path."""
import math
import sys
import warnings

import pytest
import torch

from paged_cases import FP8, Cache

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


class Model:
    """One attention layer and a classifier, its cache in pages that are handed out as sequences grow."""

    def __init__(self, P, held=torch.float16, heads=8, kv=2, dim=64, page=16, pages=40, vocab=1003, seed=0):
        g = torch.Generator().manual_seed(seed)
        r = lambda *s, scale=1.0, dtype=torch.float16: (scale * torch.randn(*s, generator=g)).to(dtype).to(DEV)  # noqa: E731
        self.P, self.heads, self.kv, self.dim, self.page, self.vocab = P, heads, kv, dim, page, vocab
        self.embed, self.qkv = r(vocab, heads * dim), r((heads + 2 * kv) * dim, heads * dim, scale=1 / math.sqrt(heads * dim))
        self.classifier = P.mx4_quantize(r(vocab, heads * dim, scale=3 / math.sqrt(heads * dim)))
        scales = [torch.full((kv,), 0.02, device=DEV) for _ in range(2)] if held == FP8 else [None, None]
        new = lambda: torch.zeros(pages, kv, page, dim, dtype=torch.float16, device=DEV).to(held)  # noqa: E731
        self.cache = P.PagedCache(new(), new(), *scales)
        self.angles = P.rotary_table(8 * page, dim, device=DEV)

    def project(self, tokens):
        x = (self.embed[tokens].float() @ self.qkv.float().t()).half().view(-1, self.heads + 2 * self.kv, self.dim)
        return x[:, :self.heads], x[:, self.heads:self.heads + self.kv], x[:, self.heads + self.kv:]

    def step(self, tokens, table, lengths, u, stream=None):
        """The next token of each sequence, with what led to it."""
        q, k, v = self.project(tokens)
        q = self.cache.append(k, v, table, lengths, q=q, rotary=self.angles, stream=stream)
        out, lse = self.cache.attend(q, table, lengths, lse=True, stream=stream)
        logits = self.P.mx4_linear(out.flatten(1), self.classifier, stream=stream)
        chosen, logp = self.P.sample_tokens(logits, u, temperature=0.8, top_k=40, top_p=0.95, stream=stream)
        return chosen, logp, self.P.token_log_probs(logits, chosen, stream=stream)[0], out, lse


def served(P, held=torch.float16, steps=5):
    """Three prompts at once, then steps of one token each; every step's results."""
    m = Model(P, held)
    prompts = [5, 33, 1]
    table = torch.randperm(40, generator=torch.Generator().manual_seed(1)).int()[:3 * 8].view(3, 8).to(DEV)
    lengths = torch.tensor(prompts, dtype=torch.int32, device=DEV)
    starts = torch.tensor([0, 5, 38, 39], dtype=torch.int32, device=DEV)
    tokens = torch.arange(39, device=DEV) * 7 % m.vocab
    q, k, v = m.project(tokens)
    m.cache.append(k, v, table, lengths, starts=starts, q=q, rotary=m.angles)
    tokens, out = tokens[starts[1:].long() - 1], []
    u = torch.rand(steps, 3, generator=torch.Generator().manual_seed(2)).to(DEV)
    for i in range(steps):
        lengths = lengths + 1
        result = m.step(tokens, table, lengths, u[i])
        tokens = result[0]
        out.append(result)
    return out, m, table, lengths


@pytest.mark.parametrize("held", [torch.float16, FP8])
def test_tokens_one_at_a_time_are_a_prompt_at_once(ops, held):
    """The cache after appending tokens one by one holds the bits of the cache that took them all at once, and attention reads the same."""
    m, n = Model(ops, held), Model(ops, held)
    table = torch.arange(8, dtype=torch.int32, device=DEV).view(1, 8)
    tokens = torch.arange(50, device=DEV) * 13 % m.vocab
    q, k, v = m.project(tokens)
    length = lambda x: torch.tensor([x], dtype=torch.int32, device=DEV)  # noqa: E731
    all_q = m.cache.append(k, v, table, length(50), starts=torch.tensor([0, 50], dtype=torch.int32, device=DEV), q=q, rotary=m.angles)
    one_q = [n.cache.append(k[i:i + 1], v[i:i + 1], table, length(i + 1), q=q[i:i + 1], rotary=n.angles) for i in range(50)]
    raw = torch.uint8 if held == FP8 else torch.int16
    assert torch.equal(torch.cat(one_q), all_q)
    assert torch.equal(m.cache.k_pages.view(raw), n.cache.k_pages.view(raw)) and torch.equal(m.cache.v_pages.view(raw), n.cache.v_pages.view(raw))
    assert torch.equal(m.cache.attend(all_q[-1:], table, length(50)), n.cache.attend(one_q[-1], table, length(50)))


def test_sampled_tokens_have_the_log_probabilities_that_scoring_gives(ops):
    """Of a distribution that nothing is cut from, both say the same: each has fp32's rounding of a difference, and the score its sums' of 1003 terms."""
    x = (3 * torch.randn(20, 1003)).half().to(DEV)
    token, logp = ops.sample_tokens(x, torch.rand(20, device=DEV))
    scored, _ = ops.token_log_probs(x, token)
    assert float((logp - scored).abs().max()) <= 1e-5


def test_steps_through_the_native_path_and_without_it(ops, monkeypatch):
    from pimaicompiler_amd import ops as O
    native, *_ = served(ops)
    monkeypatch.setitem(sys.modules, "pimaicompiler_amd._aten_ops_pimhip", None)
    monkeypatch.setattr(O, "_native_module", None)
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        bodies, *_ = served(ops)
        assert type(O._native()).__name__ == "_WithoutExtension"
    for a, b in zip(native, bodies):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("held", [torch.float16, FP8])
def test_a_captured_step_is_replayed(ops, held):
    """Replays with other tokens, lengths and numbers, eager work and synchronizations in between, each against the eager step's bits."""
    _, m, table, lengths = served(ops, held, steps=2)
    _, e, _, _ = served(ops, held, steps=2)
    tokens, u = torch.zeros(3, dtype=torch.int64, device=DEV), torch.zeros(3, device=DEV)
    now = lengths.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        m.step(tokens, table, now, u)
    torch.cuda.current_stream().wait_stream(side)
    e.step(tokens, table, lengths, u)   # (the step before the capture has stored its keys and values in the one cache: so has this in the other)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        result = m.step(tokens, table, now, u)
    for i in range(5):
        tokens.copy_(torch.tensor([i, 3 * i + 1, 500 + i]))
        u.copy_(torch.rand(3, generator=torch.Generator().manual_seed(i)))
        now.add_(1)
        graph.replay()
        torch.cuda.synchronize()
        want = e.step(tokens.clone(), table, now.clone(), u.clone())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(result, want)), i


def test_two_graphs_are_replayed_at_the_same_time(ops):
    """Each has a workspace of its own: long sequences whose parts are joined, on two streams."""
    cache = Cache([4000, 3000], 2, 16, 64, torch.float16)
    table, n = cache.tensors(DEV)
    c = cache.on(ops, DEV)
    q = [torch.randn(2, 8, 64).half().to(DEV) for _ in range(2)]
    want = [c.attend(x, table, n) for x in q]
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for x in q:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(c.attend(x, table, n))
        graphs.append(g)
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_calls_on_two_streams_at_the_same_time(ops):
    cache = Cache([4000, 1, 700], 2, 16, 64, torch.float16)
    table, n = cache.tensors(DEV)
    c = cache.on(ops, DEV)
    q = [torch.randn(3, 8, 64).half().to(DEV) for _ in range(2)]
    x, u = [(3 * torch.randn(5, 40000)).half().to(DEV) for _ in range(2)], torch.rand(5, device=DEV)
    want = [(c.attend(a, table, n), *ops.sample_tokens(b, u, top_p=0.99)) for a, b in zip(q, x)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for _ in range(10):
        for a, b, s in zip(q, x, streams):
            with torch.cuda.stream(s):
                got.append((c.attend(a, table, n), *ops.sample_tokens(b, u, top_p=0.99)))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(g, want[i % 2]))


def test_a_stream_that_is_asked_for(ops):
    """As an object and as its handle: the results are those of the current stream, and the inputs may be dropped at once."""
    want, *_ = served(ops, steps=1)
    for as_handle in (False, True):
        s = torch.cuda.Stream()
        m = Model(ops)
        table = torch.randperm(40, generator=torch.Generator().manual_seed(1)).int()[:3 * 8].view(3, 8).to(DEV)
        tokens = torch.arange(39, device=DEV) * 7 % m.vocab
        q, k, v = m.project(tokens)
        starts, lengths = torch.tensor([0, 5, 38, 39], dtype=torch.int32, device=DEV), torch.tensor([5, 33, 1], dtype=torch.int32, device=DEV)
        torch.cuda.synchronize()
        handle = s.cuda_stream if as_handle else s
        m.cache.append(k, v, table, lengths, starts=starts, q=q, rotary=m.angles, stream=handle)
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            got = m.step(tokens[starts[1:].long() - 1], table, lengths + 1, torch.rand(1, 3, generator=torch.Generator().manual_seed(2)).to(DEV)[0], stream=handle)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want[0]))


def test_a_padded_batch(ops):
    """Sequences of length 0 behind the last: nothing of theirs is stored, their results are zeros, and the others' are what they are without them."""
    _, m, table, lengths = served(ops, steps=1)
    _, e, _, _ = served(ops, steps=1)
    tokens, u = torch.tensor([4, 5, 6], device=DEV), torch.rand(3, device=DEV)
    want = e.step(tokens, table, lengths + 1, u)
    wide = torch.cat([table, torch.zeros(2, table.size(1), dtype=torch.int32, device=DEV)])
    got = m.step(torch.cat([tokens, tokens[:2]]), wide, torch.cat([lengths + 1, torch.zeros(2, dtype=torch.int32, device=DEV)]), torch.cat([u, u[:2]]))
    assert all(torch.equal(a[:3], b) for a, b in zip(got, want))
    assert bool((got[3][3:] == 0).all()) and bool((got[4][3:] == -math.inf).all())
    assert torch.equal(m.cache.k_pages, e.cache.k_pages) and torch.equal(m.cache.v_pages, e.cache.v_pages)


def test_tangents_are_refused(ops):
    import torch.autograd.forward_ad as fwd
    c = Cache([3, 4], 1, 16, 64, torch.float16)
    table, n = c.tensors(DEV)
    c = c.on(ops, DEV)
    x = torch.zeros(2, 1, 64, dtype=torch.float16, device=DEV)
    logits = torch.zeros(2, 10, device=DEV)
    with fwd.dual_level():
        d, l = fwd.make_dual(x, torch.ones_like(x)), fwd.make_dual(logits, torch.ones_like(logits))
        for call in (lambda: c.append(d, x, table, n), lambda: c.append(x, d, table, n), lambda: c.attend(d, table, n), lambda: ops.sample_tokens(l, torch.zeros(2, device=DEV))):
            with pytest.raises(ops.NNRuntimeException, match="derivative"):
                call()


def test_keys_and_values_in_the_same_memory(ops):
    """Attention may read such a cache; nothing is appended to it."""
    pages = torch.randn(3, 1, 16, 64).half().to(DEV)
    c = ops.PagedCache(pages, pages)
    table, n = torch.tensor([[2, 0]], dtype=torch.int32, device=DEV), torch.tensor([20], dtype=torch.int32, device=DEV)
    x = torch.randn(1, 1, 64).half().to(DEV)
    assert torch.equal(c.attend(x, table, n), ops.PagedCache(pages, pages.clone()).attend(x, table, n))
    with pytest.raises(ops.NNRuntimeException, match="same memory"):
        c.append(x, x, table, n)
    both = torch.zeros(3, 2, 1, 16, 64, dtype=torch.float16, device=DEV)   # beside one another they are not
    c = ops.PagedCache(both[:, 0], both[:, 1])
    c.append(x, 2 * x, table, n)
    assert torch.equal(both[0, 0, 0, 3], x[0, 0]) and torch.equal(both[0, 1, 0, 3], 2 * x[0, 0]) and int((both != 0).sum()) == int((x != 0).sum()) * 2
