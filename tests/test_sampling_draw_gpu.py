"""What a draw may be, asked of every row, near an edge or not: a token that stays, has a weight, and whose share holds the number."""
import math

import pytest
import torch

from test_sampling_gpu import DTYPES, f32

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
INF = math.inf


def kept_of(x, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(the tokens that stay in the order of indices, their weights) of one row, in 64 bits, and how near top_p is to the edge of what stays."""
    x = x.double()
    order = torch.sort(x, descending=True, stable=True).indices
    w, near = torch.exp((x - x.max()) / f32(temperature)), 1.0
    kept = order[:top_k] if top_k > 0 else order
    if top_p < 1:
        whole = w[kept].sum()
        before = torch.cumsum(w[kept], 0) - w[kept]
        near = float(((before - f32(top_p) * whole).abs() / whole).min())
        kept = kept[:max(1, int((before < f32(top_p) * whole).sum()))]
    if min_p > 0:
        kept = kept[w[kept] >= f32(min_p)]
    kept = torch.sort(kept).values
    return kept, w[kept], near


def unit_of(V):
    """What weights are rounded to, of the largest: V of them fit into 62 bits."""
    shift = 45
    while V > 1 << (62 - shift):
        shift -= 1
    return 2.0**-shift


def drawn(ops, x, u, some=None, **settings):
    """tokens and logp of a call, each looked at.  A running sum is off by 2^-36 of the whole (borders are moved by that), by 2^-38 of itself (weights) and by half a unit for
    each token; so is the whole.  Returns how many rows (all, or those of `some`) were compared: top_p may be as near as that to an edge of what stays."""
    tokens, logp = ops.sample_tokens(x.to(DEV), u.to(DEV), **{k: v.to(DEV) if isinstance(v, torch.Tensor) else v for k, v in settings.items()})
    compared, cache = 0, {}
    for r in range(x.size(0)) if some is None else some:
        one = {k: v[r].item() if isinstance(v, torch.Tensor) else v for k, v in settings.items()}
        same = (x[r].numpy().tobytes() if x.dtype != torch.bfloat16 else x[r].view(torch.int16).numpy().tobytes()), tuple(one.values())
        if same not in cache:
            cache[same] = kept_of(x[r], **one)
        kept, w, near = cache[same]
        whole = float(w.sum())
        off = 2.0**-36 + 2 * 2.0**-38 + x.size(1) * unit_of(x.size(1)) / 2 / whole
        token, lp = int(tokens[r]), float(logp[r])
        assert 0 <= token < x.size(1), (r, token)
        if near <= 2 * off:
            continue
        at = int(torch.searchsorted(kept, token))
        assert at < len(kept) and int(kept[at]) == token, (r, token, "does not stay")
        assert float(w[at]) > 0, (r, token, "has no weight")
        edge = float(w[:at + 1].sum())
        number = min(max(float(u[r]), 0.0), 1 - 2.0**-24)
        assert edge - float(w[at]) <= (number + 2 * off) * whole and edge >= (number - 2 * off) * whole, (r, token, number, edge / whole)
        want = math.log(float(w[at]) / whole)
        assert abs(lp - want) <= abs(want) * 2.0**-24 + 2 * off + 1e-9, (r, lp, want)
        compared += 1
    return compared


def low(V, at, gap, dtype, masked=()):
    """One token of weight 1 at `at`, the others `gap` below it, those of `masked` out."""
    x = torch.full((V,), -gap)
    x[list(masked)] = -INF
    x[at] = 0.0
    return x.to(dtype)


# (rows, V): 256, 512 and 1024 threads a row, many rows, 16-bit rows that may be counted, the first pass by all CUs, the largest
SIZES = [(6, 6147), (6, 3001), (6, 8196), (6, 32000), (2000, 8000), (300, 50000), (6, 60000), (6, 131072), (2, 300007)]


@pytest.mark.parametrize("rows, V", SIZES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_more_tokens_than_a_list_with_min_p_alone(ops, rows, V, dtype):
    """Nothing but min_p, which thousands of tokens pass: the list is given up and the row walked, with every wavefront's segments in the sum."""
    g = torch.Generator().manual_seed(V)
    x = torch.stack([torch.full((V,), 2.0), torch.randn(V, generator=g), torch.arange(V) * (3.0 / V), torch.where(torch.rand(V, generator=g) < 0.3, 1.0, -INF)]).to(dtype)
    x = x.repeat(-(-rows // 4), 1)[:rows]
    u = torch.rand(rows, generator=g)
    assert drawn(ops, x, u, min_p=1e-3) == rows
    on = x.to(DEV), u.to(DEV)
    first = ops.sample_tokens(*on, min_p=1e-3)
    for _ in range(20):
        again = ops.sample_tokens(*on, min_p=1e-3)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("rows, V", SIZES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_segments_whose_values_are_less_than_half_a_unit_each(ops, rows, V, dtype):
    """Tokens of 2^-47 to 2^-56 of the largest: one by one nothing, together some units.  A number that falls there draws one of them, never one that is out,
    nor one behind the row."""
    kinds = [low(V, V // 2 + 900, 32.5, dtype, masked=[0]), low(V, 0, 32.5, dtype), low(V, V - 1, 36.0, dtype, masked=range(3)), low(V, 2500, 38.0, dtype, masked=[0, 1, V - 1]),
             low(V, V // 2 + 900, 33.0, dtype, masked=range(1, min(V // 2, 5000), 2)), low(V, 2000, 32.0, dtype, masked=range(V - 3, V))]
    numbers = [0.0, 1.0 - 2.0**-24, 2.0**-60, 0.5, 2.0**-24, -1.0]
    for i, u in enumerate(numbers):
        x = torch.stack([kinds[(r + i) % 6] for r in range(min(rows, 12))])
        x = x.repeat(-(-rows // x.size(0)), 1)[:rows]
        for settings in ({}, {"top_k": V - 2}, {"min_p": 1e-17}, {"temperature": 0.5}, {"top_k": V - 5, "min_p": 1e-18}):
            scaled = (x.float() * settings.get("temperature", 1.0)).to(dtype)
            assert drawn(ops, scaled, torch.full((rows,), u), **settings) == rows


@pytest.mark.parametrize("rows, V", SIZES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_numbers_outside_of_their_range(ops, rows, V, dtype):
    """They count as the nearest in it, 0 and 1 - 2^-24: the last tokens, which together have less than 2^-24 of the whole, are not drawn by 1."""
    kinds = [low(V, V // 3, 20.0 + math.log(V), dtype, masked=[0]), low(V, 0, 20.0 + math.log(V), dtype), low(V, 5, 40.0, dtype, masked=range(V // 2, V)),
             2 * torch.randn(V, generator=torch.Generator().manual_seed(V)).to(dtype)]
    x = torch.stack([kinds[r % 4] for r in range(min(rows, 8))])
    for settings in ({}, {"top_k": 30}, {"top_k": 400}, {"top_k": V - 2}, {"min_p": 1e-13}, {"top_p": 0.97}):
        ends = [drawn_at(ops, x, u, settings) for u in (0.0, 1.0 - 2.0**-24)]
        for u in (1.0, 1.0 + 2.0**-23, 7.0, 1e30, INF):
            got = drawn_at(ops, x, u, settings)
            assert torch.equal(got[0], ends[1][0]) and torch.equal(got[1], ends[1][1])
        for u in (-0.0, -1e-30, -5.0, -INF):
            got = drawn_at(ops, x, u, settings)
            assert torch.equal(got[0], ends[0][0]) and torch.equal(got[1], ends[0][1])
        if settings.get("top_p", 1.0) == 1.0:
            assert drawn(ops, x, torch.full((x.size(0),), 1.0), **settings) == x.size(0)


def drawn_at(ops, x, u, settings):
    return ops.sample_tokens(x.to(DEV), torch.full((x.size(0),), u, device=DEV), **settings)


# (rows, V): around 2^17 tokens, up to which weights are whole numbers of 2^-45, and far above it; with the first pass by all CUs, and without
LONG = [(3, 131072), (3, 131073), (128, 131080), (129, 131073), (4, 300007), (3, 1 << 20), (3, (1 << 21) - 1), (3, 1 << 21)]


@pytest.mark.parametrize("rows, V", LONG)
@pytest.mark.parametrize("dtype", DTYPES)
def test_long_rows_against_the_definition(ops, rows, V, dtype):
    g = torch.Generator().manual_seed(V + rows)
    x = 2.5 * torch.randn(rows, V, generator=g)
    x = torch.where(torch.rand(rows, V, generator=g) < 0.001, x + 8, x)
    x[torch.rand(rows, V, generator=g) < 0.05] = -INF
    x, u = x.to(dtype), torch.rand(rows, generator=g)
    u[0] = 0.0
    some = [0, rows // 2, rows - 1]
    each = dict(temperature=0.3 + torch.rand(rows, generator=g), top_k=torch.randint(0, 2000, (rows,), generator=g).int(), top_p=0.5 + 0.5 * torch.rand(rows, generator=g),
                min_p=0.01 * torch.rand(rows, generator=g))
    whole, near = ({}, {"top_k": 40}, {"top_k": V // 2}, {"min_p": 0.03}, {"min_p": 1e-4, "top_k": 900}), ({"top_p": 0.9}, {"top_k": 3000, "top_p": 0.97}, {"top_p": 0.7, "temperature": 0.4}, each)
    for settings in whole:
        assert drawn(ops, x, u, some, **settings) == 3
    assert sum(drawn(ops, x, u, some, **settings) for settings in near) >= 10
