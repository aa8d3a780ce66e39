"""Appending to a paged cache against 64 bits: what is stored, what is turned, and what stays as it was."""
import pytest
import torch

from paged_cases import FP8, Cache, step, turned

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def stored(got, want, sizes, dtype, before, written):
    """got [pages, heads, page, dim] against want where `written`; as before where not.  fp32 results of three roundings (two products, their sum), one
    rounding to the type; half a step of the subnormals at least."""
    got, before = got.cpu(), before.cpu()
    raw = (torch.uint8, got.view(torch.uint8), before.view(torch.uint8)) if dtype == FP8 else (torch.int16, got.view(torch.int16), before.view(torch.int16))
    assert torch.equal(raw[1][~written], raw[2][~written])
    g, w = got.double()[written], want[written]
    u = 2.0**-24
    bound = 3 * u * sizes[written] + (w.abs() * (1 + 2**-20) + 3 * u * sizes[written]) * step(dtype) + torch.finfo(dtype).smallest_normal * step(dtype)
    assert bool(((g - w).abs() <= bound).all()), float(((g - w).abs() / bound).max())


def run(P, lengths, counts, heads, kv, dim, rotary, interleaved, page, dtype, held, seed=0, layout="heads first", padding=0, with_q=True, extra_width=0):
    """One append of counts[s] tokens to sequences that are lengths[s] long with them."""
    g = torch.Generator().manual_seed(seed)
    cache = Cache(lengths, kv, page, dim, held, seed, extra_width=extra_width)
    c = cache.on(P, DEV, layout)
    table, n = cache.tensors(DEV)
    T = sum(counts) + padding
    q, k, v = (torch.randn(T, h, dim, generator=g).to(dtype) for h in (heads, kv, kv))
    angles = P.rotary_table(table.size(1) * page, rotary, device="cpu") if rotary else None
    decode = padding == 0 and all(x == 1 for x in counts)
    starts = torch.tensor([0] + list(torch.tensor(counts).cumsum(0)), dtype=torch.int32)
    before = [t.clone() for t in (c.k_pages.view(torch.uint8) if held == FP8 else c.k_pages, c.v_pages.view(torch.uint8) if held == FP8 else c.v_pages)]
    before = [t.view(held) for t in before]
    out = c.append(k.to(DEV), v.to(DEV), table, n, starts=None if decode else starts.to(DEV), q=q.to(DEV) if with_q and rotary else None,
                   rotary=angles.to(DEV) if rotary else None, interleaved=interleaved)
    # ---- the definition ----
    place = []
    for s, m in enumerate(counts):
        place += [(s, lengths[s] - m + j) for j in range(m)]
    place += [(-1, -1)] * padding
    positions = torch.tensor([p for _, p in place])
    ky, ks = turned(k, positions.clamp(min=0), angles, rotary, interleaved)
    written = torch.zeros(c.k_pages.shape, dtype=torch.bool)
    want = [torch.zeros(c.k_pages.shape, dtype=torch.float64) for _ in range(4)]
    for t, (s, p) in enumerate(place):
        if s < 0 or p < 0:
            continue
        at = int(cache.table[s, p // page]), slice(None), p % page
        written[at] = True
        for w, x in zip(want, (ky[t], ks[t], v[t].double(), v[t].double() * 0)):
            w[at] = x
    if held == FP8:
        for i, scale in ((0, cache.k_scale), (2, cache.v_scale)):
            scale = scale.double().view(1, -1, 1, 1)
            want[i + 1] = (want[i + 1] + want[i].abs()) / scale  # (one more rounding, of the quotient)
            want[i] = (want[i] / scale).clamp(-448, 448)
    stored(c.k_pages, want[0], want[1], held, before[0], written)
    stored(c.v_pages, want[2], want[3], held, before[1], written)
    if not (with_q and rotary):
        assert out is None
        return
    qy, qs = turned(q, positions.clamp(min=0), angles, rotary, interleaved)
    got = out.cpu().double()
    assert out.dtype == dtype and out.shape == q.shape
    nobody = torch.tensor([s < 0 or p < 0 for s, p in place])
    assert bool((got[nobody] == 0).all())
    u = 2.0**-24
    bound = 3 * u * qs + (qy.abs() + 3 * u * qs) * step(dtype) + torch.finfo(dtype).smallest_normal * step(dtype)
    assert bool(((got - qy).abs() <= bound)[~nobody].all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("heads,kv,dim,rotary,page", [(16, 16, 64, 64, 16), (8, 2, 128, 128, 64), (4, 1, 80, 40, 24), (7, 7, 96, 96, 1), (6, 2, 256, 2, 33), (3, 1, 16, 12, 5),
                                                      (5, 5, 112, 110, 256), (2, 2, 48, 0, 7)])
def test_a_token_for_each_sequence(ops, dtype, fp8, interleaved, heads, kv, dim, rotary, page):
    run(ops, [1, 2, 16, 17, 40, 333], [1] * 6, heads, kv, dim, rotary, interleaved, page, dtype, FP8 if fp8 else dtype, seed=dim)


@pytest.mark.parametrize("dtype,held", [(torch.float16, torch.float16), (torch.bfloat16, FP8)])
@pytest.mark.parametrize("counts", [[5], [1, 0, 7], [0, 0, 3, 0], [64, 1, 65, 2], [0, 0]])
@pytest.mark.parametrize("padding", [0, 3])
def test_prompts(ops, dtype, held, counts, padding):
    if sum(counts) + padding == 0:
        counts = counts + [1]
    run(ops, [n + 3 * i for i, n in enumerate(counts)], counts, 4, 2, 64, 64, False, 16, dtype, held, seed=len(counts), padding=padding, extra_width=2)


def test_many_sequences(ops):
    """More of them than are looked at in one step, or in two, some of no new tokens."""
    for S in (63, 64, 65, 200, 4500):
        counts = [(s * 7) % 3 for s in range(S)]
        run(ops, [n + s % 5 for s, n in enumerate(counts)], counts, 1, 1, 16, 16, True, 4, torch.float16, torch.float16, seed=S, padding=2)


@pytest.mark.parametrize("layout", ["heads first", "tokens first"])
@pytest.mark.parametrize("held", [torch.bfloat16, FP8])
def test_layouts_of_a_cache(ops, layout, held):
    run(ops, [100, 3, 17], [40, 3, 1], 8, 4, 64, 32, False, 16, torch.bfloat16, held, layout=layout)


def test_inputs_that_are_views(ops):
    """Queries, keys and values beside one another, at an odd element, and turned round."""
    cache = Cache([5, 9, 40], 2, 16, 64, torch.float16)
    table, n = cache.tensors(DEV)
    angles = ops.rotary_table(table.size(1) * 16, 64, device=DEV)
    g = torch.Generator().manual_seed(4)
    x = torch.randn(3, 8, 64, generator=g).half().to(DEV)
    q, k, v = x[:, :4], x[:, 4:6], x[:, 6:]
    a = cache.on(ops, DEV)
    want = a.append(k.contiguous(), v.contiguous(), table, n, q=q.contiguous(), rotary=angles)
    odd = torch.empty(3 * 2 * 64 + 1, dtype=torch.float16, device=DEV)
    odd[1:] = k.reshape(-1)
    wide = torch.zeros(3, table.size(1) + 3, dtype=torch.int32, device=DEV)
    wide[:, :table.size(1)] = table
    for kk, vv, qq, tt, nn, aa in ((k, v, q, table, n, angles), (odd[1:].view(3, 2, 64), v.transpose(0, 1).contiguous().transpose(0, 1), q, wide[:, :table.size(1)], n, angles),
                                   (k, v.transpose(1, 2).contiguous().transpose(1, 2), q, table, torch.stack([n, n], 1)[:, 0], torch.cat([angles, angles], 1)[:, :64])):
        b = cache.on(ops, DEV)
        got = b.append(kk, vv, tt, nn, q=qq, rotary=aa)
        assert torch.equal(got, want) and torch.equal(a.k_pages, b.k_pages) and torch.equal(a.v_pages, b.v_pages)


@pytest.mark.parametrize("held", [torch.float16, FP8])
def test_places_that_are_none(ops, held):
    """Pages outside of the cache, positions outside of the table, a sequence shorter than its tokens: nothing is stored, and the rest is."""
    cache = Cache([20, 20, 20, 20], 1, 8, 16, held, extra_width=1)
    good = cache.table.clone()
    c = cache.on(ops, DEV)
    table, _ = cache.tensors(DEV)
    table[0, 2], table[1, 2] = -5, c.k_pages.size(0)
    raw = torch.uint8 if held == FP8 else torch.int16
    before = [t.view(raw).clone() for t in (c.k_pages, c.v_pages)]
    k = torch.ones(8, 1, 16, dtype=torch.float16, device=DEV)
    lengths = torch.tensor([20, 20, 2**31 - 1, 1], dtype=torch.int32, device=DEV)   # the third ends behind its table, the last has one of its two tokens
    starts = torch.tensor([0, 1, 2, 6, 8], dtype=torch.int32, device=DEV)
    angles = ops.rotary_table(table.size(1) * 8, 16, device=DEV)
    q = c.append(k, k, table, lengths, starts=starts, q=k, rotary=angles)
    assert bool((q[2:7] == 0).all()) and bool((q[:2] != 0).any(-1).all()) and torch.equal(q[7], k[7])
    after = [t.view(raw) for t in (c.k_pages, c.v_pages)]
    page = int(good[3, 0])
    for a, b in zip(before, after):
        b = b.clone()
        assert not torch.equal(a[page, 0, 0], b[page, 0, 0])
        b[page, 0, 0] = a[page, 0, 0]
        assert torch.equal(a, b)


def test_values_of_eight_bits_at_the_ends(ops):
    """Borders between neighbours go to the even one, what is above saturates, a NaN stays one, and -0 is -0."""
    cache = Cache([1], 1, 16, 16, FP8)
    cache.k_scale = cache.v_scale = torch.ones(1)
    c = cache.on(ops, DEV)
    table, n = cache.tensors(DEV)
    x = torch.tensor([448.0, 464.0, 465.0, 1e4, -1e4, float("inf"), float("nan"), -0.0, 2.0**-9, 2.0**-10, 1.5 * 2.0**-9, 17.0, 19.0, 2.0**-11, 1.0625, 1.1875])
    want = [448.0, 448.0, 448.0, 448.0, -448.0, 448.0, float("nan"), -0.0, 2.0**-9, 0.0, 2 * 2.0**-9, 16.0, 20.0, 0.0, 1.0, 1.25]
    c.append(x.half().view(1, 1, 16).to(DEV), x.bfloat16().half().view(1, 1, 16).to(DEV), table, n)
    at = int(cache.table[0, 0])
    got = c.k_pages[at, 0, 0].cpu().float()
    want = torch.tensor(want)
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got[~got.isnan()], want[~want.isnan()]) and bool(torch.signbit(got[7]))


def test_no_tokens(ops):
    cache = Cache([3], 1, 4, 16, torch.float16)
    c = cache.on(ops, DEV)
    table, n = cache.tensors(DEV)
    before = c.k_pages.clone()
    none = torch.zeros(0, 1, 16, dtype=torch.float16, device=DEV)
    assert c.append(none, none, table, n, starts=torch.zeros(2, dtype=torch.int32, device=DEV)) is None
    assert c.append(none, none, table[:0], n[:0]) is None
    assert torch.equal(before, c.k_pages)


def test_refusals(ops):
    E = ops.NNRuntimeException
    h = lambda *s, t=torch.float16: torch.zeros(*s, dtype=t, device=DEV)  # noqa: E731
    pages = h(4, 2, 16, 64)
    for wrong in ((pages, pages[:3]), (pages, pages.bfloat16()), (pages.float(), pages.float()), (pages[..., :60], pages[..., :60]), (pages.transpose(2, 3), pages.transpose(2, 3)),
                  (h(1, 1, 16, 264), h(1, 1, 16, 264)), (pages[:1].expand(4, 2, 16, 64), pages), (pages[0], pages[0]), (pages[:0], pages[:0]),
                  (pages, pages, torch.ones(2, device=DEV), torch.ones(2, device=DEV)), (pages.to(FP8), pages.to(FP8)), (pages.to(FP8), pages.to(FP8), torch.ones(2, device=DEV)),
                  (pages.to(FP8), pages.to(FP8), torch.ones(1, device=DEV), torch.ones(2, device=DEV)), (pages.to(FP8)[..., :24], pages.to(FP8)[..., :24], torch.ones(2, device=DEV),
                                                                                                           torch.ones(2, device=DEV))):
        with pytest.raises(E):
            ops.PagedCache(*wrong)
    with pytest.raises(E):
        ops.PagedCache(pages.clone().requires_grad_(), pages)
    c = ops.PagedCache(pages, pages.clone())
    k, table, n = h(2, 2, 64), torch.zeros(2, 3, dtype=torch.int32, device=DEV), torch.ones(2, dtype=torch.int32, device=DEV)
    angles = ops.rotary_table(48, 64, device=DEV)
    good = dict(k=k, v=k, page_table=table, lengths=n)
    c.append(**good)
    for wrong in (dict(k=k[:, :1]), dict(v=k[:1]), dict(k=k.bfloat16(), v=k.bfloat16()), dict(v=k.bfloat16()), dict(k=k.cpu()), dict(k=k[..., :32]), dict(k=k.clone().requires_grad_()),
                  dict(page_table=table.long()), dict(page_table=table[:1]), dict(page_table=table[:, :0]), dict(lengths=n.long()), dict(lengths=n.cpu()), dict(starts=n),
                  dict(starts=torch.zeros(3, dtype=torch.int64, device=DEV)), dict(k=h(3, 2, 64), v=h(3, 2, 64)), dict(q=k), dict(q=h(3, 2, 64), rotary=angles), dict(q=k.bfloat16(), rotary=angles),
                  dict(rotary=angles[:47]), dict(rotary=angles.half()), dict(rotary=angles[:, :63]), dict(rotary=torch.cat([angles, angles], 1)), dict(rotary=angles.cpu())):
        with pytest.raises(E):
            c.append(**{**good, **wrong})
