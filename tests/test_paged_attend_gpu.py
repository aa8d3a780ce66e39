"""Attention of one new token over a paged cache against 64 bits."""
import copy
import math

import pytest
import torch

from paged_cases import FP8, Cache, attend

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
INF = math.inf


def near(got, want, bound):
    got = got.cpu().double()
    same = (got == want) | (got.isnan() & want.isnan())
    assert bool((same | ((got - want).abs() <= bound)).all()), float(((got - want).abs() / bound)[~same].max())


def run(P, lengths, heads, kv, dim, page, dtype, held, window=0, scale=None, seed=0, layout="heads first", rest=0.0, lse=True, extra_width=0, cache=None, q=None):
    cache = cache or Cache(lengths, kv, page, dim, held, seed, rest=rest, extra_width=extra_width)
    g = torch.Generator().manual_seed(seed + 1)
    q = torch.randn(len(lengths), heads, dim, generator=g).to(dtype) if q is None else q
    table, n = cache.tensors(DEV)
    got = cache.on(P, DEV, layout).attend(q.to(DEV), table, n, scale=scale, window=window, lse=lse)
    out, sums, out_bound, lse_bound = attend(cache, q, 1 / math.sqrt(dim) if scale is None else scale, window)
    if lse:
        near(got[1], sums, lse_bound)
        got = got[0]
    assert got.dtype == dtype and got.shape == q.shape
    near(got, out, out_bound)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dim", [16, 64, 80, 96, 128, 160, 192, 208, 256])
@pytest.mark.parametrize("heads,kv,page", [(4, 4, 16), (8, 2, 24)])
def test_heads_and_pages(ops, dtype, fp8, dim, heads, kv, page):
    run(ops, [0, 1, 15, 16, 17, 64, 65, 200], heads, kv, dim, page, dtype, FP8 if fp8 else dtype, seed=dim)


@pytest.mark.parametrize("dim", [8, 24, 72, 136, 200, 248])
def test_odd_head_sizes(ops, dim):
    run(ops, [1, 40, 130], 3, 1, dim, 16, torch.float16, torch.float16, seed=dim)
    run(ops, [1, 40, 130], 3, 1, dim, 3, torch.bfloat16, torch.bfloat16, seed=dim)


@pytest.mark.parametrize("heads,kv", [(1, 1), (7, 1), (14, 2), (16, 1), (17, 1), (24, 1), (32, 1), (33, 1), (64, 1), (71, 1), (40, 2)])
@pytest.mark.parametrize("dim,held", [(64, torch.float16), (128, FP8), (192, torch.float16)])
def test_query_heads_of_a_key_head(ops, heads, kv, dim, held):
    run(ops, [1, 33, 100], heads, kv, dim, 32, torch.float16, held, seed=heads)


@pytest.mark.parametrize("heads,kv", [(2, 2), (5, 1), (8, 1), (17, 1), (32, 1), (48, 2), (71, 1)])
@pytest.mark.parametrize("dim,page", [(64, 32), (128, 16), (192, 16), (72, 24)])
def test_query_heads_of_a_key_head_in_bfloat16(ops, heads, kv, dim, page):
    run(ops, [1, 33, 100, 400], heads, kv, dim, page, torch.bfloat16, torch.bfloat16, seed=heads)
    if dim % 16 == 0:
        run(ops, [1, 33, 100], heads, kv, dim, page, torch.bfloat16, FP8, seed=heads)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads", [1, 20])
def test_infinite_and_large_values(ops, dtype, heads):
    """A value that is infinite makes its columns so, also with a weight of exactly one, and large ones stay finite."""
    cache = Cache([1, 40, 200, 90], 1, 16, 64, dtype, seed=heads)
    for s, j, column, value in ((0, 0, 3, INF), (0, 0, 40, -INF), (1, 39, 63, INF), (2, 100, 0, -INF), (2, 150, 17, INF)):
        cache.v[int(cache.table[s, j // 16]), 0, j % 16, column] = value
    large = 2.0**100 if dtype == torch.bfloat16 else 2.0**14
    for page in cache.table[3][cache.table[3] >= 0].tolist():
        cache.v[page] *= large
    q = 0.05 * torch.randn(4, heads, 64, generator=torch.Generator().manual_seed(7))   # (weights that no type loses: an infinite value times 0 is NaN)
    table, n = cache.tensors(DEV)
    out = cache.on(ops, DEV).attend(q.to(dtype).to(DEV), table, n).cpu()
    want, _, bound, _ = attend(cache, q.to(dtype), 1 / 8)
    fixed = want.isfinite()
    assert torch.equal(out.double()[~fixed], want[~fixed]) and bool(out[fixed].isfinite().all())
    rest = fixed & bound.isfinite()
    assert bool(((out.double() - want).abs() <= bound)[rest].all())
    assert bool(out[3].isfinite().all()) and int((~fixed).sum()) == 5 * heads


@pytest.mark.parametrize("sequences,kv,longest", [(1, 1, 256), (1, 1, 257), (8, 8, 512), (8, 8, 513), (32, 8, 700), (128, 4, 512), (129, 4, 300), (70, 16, 100)])
@pytest.mark.parametrize("extra", [0, 60])
def test_sequences_that_are_not_cut(ops, sequences, kv, longest, extra):
    """Up to some length, which goes by the table's room and by the lengths, sequences are taken from end to end; windows are too."""
    g = torch.Generator().manual_seed(longest)
    lengths = torch.randint(0, longest + 1, (sequences,), generator=g).tolist()
    lengths[sequences // 2] = longest
    cache = Cache(lengths, kv, 64, 16, torch.bfloat16, seed=sequences, rest=float("nan"), extra_width=extra)
    run(ops, lengths, 2 * kv, kv, 16, 64, torch.bfloat16, torch.bfloat16, cache=cache)
    run(ops, lengths, 2 * kv, kv, 16, 64, torch.bfloat16, torch.bfloat16, cache=cache, window=100)


@pytest.mark.parametrize("page", [1, 2, 15, 16, 17, 32, 48, 100, 128, 1000])
@pytest.mark.parametrize("held", [torch.bfloat16, FP8])
def test_page_sizes(ops, page, held):
    """Pages that end inside a tile, and the places behind a sequence's end NaN."""
    run(ops, [1, 16, 31, 129, 300], 4, 2, 64, page, torch.bfloat16, held, seed=page, rest=float("nan"))


@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 64, 100, 299, 300, 301, 10**9])
@pytest.mark.parametrize("page", [16, 7])
def test_windows(ops, window, page):
    run(ops, [0, 1, 16, 100, 300], 2, 1, 64, page, torch.float16, torch.float16, window=window, seed=window % 1000, rest=float("nan"))


def test_what_lies_before_the_window_has_no_influence(ops):
    cache = Cache([300], 2, 16, 64, torch.float16)
    for j in range(300 - 37):
        p = int(cache.table[0, j // 16])
        cache.k[p, :, j % 16], cache.v[p, :, j % 16] = INF, float("nan")
    run(ops, [300], 4, 2, 64, 16, torch.float16, torch.float16, window=37, cache=cache)


@pytest.mark.parametrize("lengths", [[5000], [3000, 1, 0, 2999, 64, 7], [0, 0, 0], [700] * 40, [1] * 600])
@pytest.mark.parametrize("held", [torch.float16, FP8])
def test_lengths(ops, lengths, held):
    """Long sequences that many blocks share, many short ones that share a block."""
    run(ops, lengths, 4, 2, 64, 64, torch.float16, held, seed=len(lengths), extra_width=3)


@pytest.mark.parametrize("layout", ["heads first", "tokens first"])
@pytest.mark.parametrize("held", [torch.bfloat16, FP8])
def test_layouts_of_a_cache(ops, layout, held):
    run(ops, [77, 200, 3], 6, 3, 128, 16, torch.bfloat16, held, layout=layout)


@pytest.mark.parametrize("scale", [0.0, 1.0, -0.3, 3.0])
def test_scales(ops, scale):
    run(ops, [5, 150], 4, 2, 64, 16, torch.float16, torch.float16, scale=scale)
    run(ops, [5, 150], 4, 2, 64, 16, torch.bfloat16, FP8, scale=scale, lse=False)


@pytest.mark.parametrize("order", ["rising", "falling", "jump"])
def test_running_maximum(ops, order):
    """Scores that rise by hundreds along a sequence, fall, or jump at one token of a tile: the weights' reference moves on, once or often."""
    n, cache = 400, Cache([400], 1, 16, 64, torch.float16)
    ramp = torch.arange(n).float() if order == "rising" else torch.arange(n, 0, -1).float() if order == "falling" else torch.where(torch.arange(n) == 201, 400.0, 0.0)
    for j in range(n):
        p = int(cache.table[0, j // 16])
        cache.k[p, :, j % 16] = 0.0
        cache.k[p, :, j % 16, 0] = ramp[j]
    q = torch.zeros(1, 2, 64)
    q[0, 0, 0], q[0, 1, 0] = 4.0, 0.01
    run(ops, [n], 2, 1, 64, 16, torch.float16, torch.float16, scale=1.0, cache=cache, q=q.half())


def test_pages_that_are_none(ops):
    """A page outside of the cache is not seen; a sequence of nothing else has no result."""
    for page in (16, 12):
        cache = Cache([100, 50, 3 * page], 2, page, 64, torch.float16)
        cache.table[0, 1], cache.table[0, 3] = -7, cache.k.shape[0]
        cache.table[2, :3] = 2**31 - 1
        run(ops, [100, 50, 3 * page], 4, 2, 64, page, torch.float16, torch.float16, cache=cache)


def test_lengths_outside_of_the_table(ops):
    """A length below 0 is 0, one behind the table's end its end."""
    cache = Cache([64, 40], 1, 16, 64, torch.float16)
    q = torch.randn(2, 2, 64).half().to(DEV)
    table, n = cache.tensors(DEV)
    c = cache.on(ops, DEV)
    want, zero = c.attend(q, table, n), torch.zeros_like(q[1])
    got = c.attend(q, table, torch.tensor([2**31 - 1, -3], dtype=torch.int32, device=DEV))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], zero)


def test_infinities_and_nan_of_the_cache(ops):
    """A key of -inf in a product's sense leaves its token out; a NaN or +inf score makes its heads NaN and no others."""
    cache = Cache([40, 40], 2, 16, 64, torch.float16)
    q = torch.rand(2, 4, 64).half() + 0.5
    cache.k[int(cache.table[0, 0]), 0, 3] = -INF
    cache.k[int(cache.table[1, 1]), 1, 5] = float("nan")
    table, n = cache.tensors(DEV)
    c = cache.on(ops, DEV)
    out, lse = c.attend(q.to(DEV), table, n, lse=True)
    assert bool(out[1, 2:].isnan().all()) and bool(lse[1, 2:].isnan().all()) and bool(out[1, :2].isfinite().all()) and bool(out[0].isfinite().all())
    without = Cache([40, 40], 2, 16, 64, torch.float16)
    keep = [j for j in range(40) if j != 3]
    k, v = without.held(0)
    score = (q[0, :2].double() @ k[0][keep].t()) / 8
    want = torch.softmax(score, -1) @ v[0][keep]
    # fp16's rounding of values up to 4, and the fp32 sums' part
    assert float((out[0, :2].cpu().double() - want).abs().max()) <= 4 * 2.0**-12 + 1e-4
    cache.k[int(cache.table[0, 0]), 0, 3] = INF
    out = cache.on(ops, DEV).attend(q.to(DEV), table, n)
    assert bool(out[0, :2].isnan().all()) and bool(out[0, 2:].isfinite().all())


def test_large_and_small_magnitudes(ops):
    """Values at fp16's ends: products of 2^15 and 2^-14 in fp32 sums."""
    for size in (2.0**10, 2.0**-12):
        cache = Cache([100], 1, 16, 64, torch.float16)
        cache.v = (cache.v.float() * size).half()
        run(ops, [100], 4, 1, 64, 16, torch.float16, torch.float16, cache=cache)


def test_offsets_behind_32_bits(ops):
    """A cache of more than 4 GiB, its last pages used."""
    pages, kv, page, dim = 1100, 8, 1024, 256
    k = torch.zeros(pages, kv, page, dim, dtype=torch.float16, device=DEV)
    v = torch.zeros_like(k)
    assert k.numel() * 2 > 2**32
    g = torch.Generator().manual_seed(0)
    n = 1500
    kk, vv = torch.randn(kv, n, dim, generator=g).half(), torch.randn(kv, n, dim, generator=g).half()
    used = [pages - 1, pages - 2]
    for t, x in ((k, kk), (v, vv)):
        t[used[0]] = x[:, :page].to(DEV)
        t[used[1], :, :n - page] = x[:, page:].to(DEV)
    c = ops.PagedCache(k, v)
    table, lengths = torch.tensor([used], dtype=torch.int32, device=DEV), torch.tensor([n], dtype=torch.int32, device=DEV)
    q = torch.randn(1, kv, dim, generator=g).half()
    small = Cache([n], kv, page, dim, torch.float16, extra_width=0)
    small.k, small.v, small.table = torch.zeros(2, kv, page, dim).half(), torch.zeros(2, kv, page, dim).half(), torch.tensor([[0, 1]], dtype=torch.int32)
    for t, x in ((small.k, kk), (small.v, vv)):
        t[0], t[1, :, :n - page] = x[:, :page], x[:, page:]
    out, _, bound, _ = attend(small, q, 1 / 16)
    near(c.attend(q.to(DEV), table, lengths), out, bound)
    token = torch.full((1, kv, dim), 2.0, dtype=torch.float16, device=DEV)
    c.append(token, token, table, lengths + 1)
    assert bool((c.k_pages[used[1], :, n - page] == 2.0).all()) and bool((c.k_pages[:pages - 2] == 0).all())


def test_equal_calls_give_equal_bits(ops):
    cache = Cache([5000, 3, 700], 2, 16, 128, torch.bfloat16)
    table, n = cache.tensors(DEV)
    c, q = cache.on(ops, DEV), torch.randn(3, 8, 128).bfloat16().to(DEV)
    first = c.attend(q, table, n, lse=True)
    for _ in range(5):
        again = c.attend(q, table, n, lse=True)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_views_and_copies(ops):
    cache = Cache([50, 60], 2, 16, 64, torch.float16)
    table, n = cache.tensors(DEV)
    c = cache.on(ops, DEV)
    x = torch.randn(2, 9, 64).half().to(DEV)
    want = c.attend(x[:, :4].contiguous(), table, n)
    wide = torch.zeros(2, 9, dtype=torch.int32, device=DEV)
    wide[:, :table.size(1)] = table
    assert torch.equal(c.attend(x[:, :4], table, n), want)
    assert torch.equal(c.attend(x[:, :4].transpose(1, 2).contiguous().transpose(1, 2), wide[:, :table.size(1)], n), want)
    assert torch.equal(c.attend(x[:, :4], table.t().contiguous().t(), torch.stack([n, n], 1)[:, 0]), want)
    twin = copy.deepcopy(c)
    c.k_pages.zero_()
    assert torch.equal(twin.attend(x[:, :4], table, n), want)
    # every other page of a larger cache
    pages = torch.zeros(2 * twin.k_pages.size(0), 2, 16, 64, dtype=torch.float16, device=DEV)
    k, v = pages[::2], pages.clone()[1::2]
    k.copy_(twin.k_pages)
    v.copy_(twin.v_pages)
    assert torch.equal(ops.PagedCache(k, v).attend(x[:, :4], table, n), want)


def test_no_sequences(ops):
    c = Cache([3], 1, 4, 16, torch.float16).on(ops, DEV)
    none = torch.zeros(0, 2, 16, dtype=torch.float16, device=DEV)
    out, lse = c.attend(none, torch.zeros(0, 2, dtype=torch.int32, device=DEV), torch.zeros(0, dtype=torch.int32, device=DEV), lse=True)
    assert out.shape == (0, 2, 16) and lse.shape == (0, 2)


def test_refusals(ops):
    h = lambda *s, t=torch.float16: torch.zeros(*s, dtype=t, device=DEV)  # noqa: E731
    c = ops.PagedCache(h(4, 2, 16, 64), h(4, 2, 16, 64))
    good = dict(q=h(2, 4, 64), page_table=torch.zeros(2, 3, dtype=torch.int32, device=DEV), lengths=torch.ones(2, dtype=torch.int32, device=DEV))
    c.attend(**good)
    for wrong in (dict(q=h(2, 3, 64)), dict(q=h(3, 4, 64)), dict(q=h(2, 4, 32)), dict(q=h(2, 4, 64, t=torch.bfloat16)), dict(q=h(2, 4, 64).float()), dict(q=h(2, 0, 64)), dict(q=h(2, 4, 64).cpu()),
                  dict(q=h(2, 4, 64).requires_grad_()), dict(window=-1), dict(window=1.5), dict(window=2**31), dict(scale=INF), dict(scale=float("nan")),
                  dict(page_table=torch.zeros(2, 3, dtype=torch.int64, device=DEV)), dict(page_table=torch.zeros(3, 3, dtype=torch.int32, device=DEV)),
                  dict(lengths=torch.ones(2, device=DEV)), dict(page_table=torch.zeros(2, 0, dtype=torch.int32, device=DEV))):
        with pytest.raises(ops.NNRuntimeException):
            c.attend(**{**good, **wrong})
