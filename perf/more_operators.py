"""What one step of a served language model runs around its layers, as measurable cases: keys and values appended to a paged cache with
the position rotation on the way, attention of each sequence's new token over that cache, and the next token sampled from the logits.

    own                    False: the operators in their plain form; True: the package's kernels
    listed()               the cases, each a dict of plain values
    draw(rng)              one more case of the same ranges
    prepare(case, seed)    what a program holds before the call: inputs, the cache and its page table
    run(state)             one pass, and its outputs
    work(case)             bytes and floating-point operations one pass cannot do without
    exact(case, seed)      the outputs from the definition in 64 bits
"""
import math

import torch

own = False

DEVICE = "cuda"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32, "fp8": torch.float8_e4m3fn}
SIZE = {"fp16": 2, "bf16": 2, "fp32": 4, "fp8": 1}
FP8_MOST = 448.0  # the largest finite value of the cache's 8-bit type


def listed():
    return [
        # One sequence's new token in a layer of 16 heads of 64 (1024 wide): the call is the cost.
        {"name": "append_token", "kind": "append", "sequences": 1, "tokens": 1, "heads": 16, "kv_heads": 16, "dim": 64, "rotary": 64, "interleaved": False,
         "page": 16, "context": 100, "dtype": "fp16", "cache": "fp16"},
        # A batch's decoding step into a cache in 8 bits, a layer 4096 wide with four query heads to a key head.
        {"name": "append_batch_64_fp8", "kind": "append", "sequences": 64, "tokens": 64, "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128,
         "interleaved": False, "page": 64, "context": 1000, "dtype": "bf16", "cache": "fp8"},
        # Seven prompts of together 8001 tokens, the first half of each head rotated by neighbouring pairs.
        {"name": "append_prompts_8001", "kind": "append", "sequences": 7, "tokens": 8001, "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 64,
         "interleaved": True, "page": 16, "context": 0, "dtype": "bf16", "cache": "bf16"},
        # One user's token after a page of text.
        {"name": "attend_one_1000", "kind": "attend", "sequences": 1, "shortest": 1000, "longest": 1000, "heads": 16, "kv_heads": 16, "dim": 64, "page": 16,
         "window": 0, "dtype": "fp16", "cache": "fp16", "lse": False},
        # One user's token at the end of a very long document: the work is split over the length.
        {"name": "attend_one_131071", "kind": "attend", "sequences": 1, "shortest": 131071, "longest": 131071, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "window": 0, "dtype": "fp16", "cache": "fp16", "lse": False},
        # A served batch of conversations of all lengths.
        {"name": "attend_64_ragged", "kind": "attend", "sequences": 64, "shortest": 1, "longest": 8192, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16,
         "window": 0, "dtype": "bf16", "cache": "bf16", "lse": False},
        # A larger batch over a cache in 8 bits.
        {"name": "attend_160_fp8", "kind": "attend", "sequences": 160, "shortest": 2000, "longest": 8000, "heads": 32, "kv_heads": 8, "dim": 128, "page": 32,
         "window": 0, "dtype": "bf16", "cache": "fp8", "lse": False},
        # All query heads on one key head, an odd head size, pages of no power of two, the last 1000 tokens only; the parts' sums are wanted too.
        {"name": "attend_31_window_odd", "kind": "attend", "sequences": 31, "shortest": 300, "longest": 5000, "heads": 24, "kv_heads": 1, "dim": 80, "page": 24,
         "window": 1000, "dtype": "fp16", "cache": "fp16", "lse": True},
        # One step of a decoder with 32000 words.
        {"name": "sample_token", "kind": "sample", "rows": 1, "vocab": 32000, "top_k": 50, "top_p": 0.9, "min_p": 0.0, "temperature": 0.8, "per_row": False,
         "dtype": "fp16"},
        # A served batch, each request with its own settings, over a large, odd vocabulary.
        {"name": "sample_64_requests", "kind": "sample", "rows": 64, "vocab": 100003, "top_k": 200, "top_p": 0.95, "min_p": 0.02, "temperature": 1.0,
         "per_row": True, "dtype": "bf16"},
        # Texts sampled with the nucleus alone: it holds thousands of words.
        {"name": "sample_256_nucleus", "kind": "sample", "rows": 256, "vocab": 131072, "top_k": 0, "top_p": 0.98, "min_p": 0.0, "temperature": 1.3,
         "per_row": False, "dtype": "bf16"},
        # Samples of the whole distribution, for a policy's training: nothing is cut off.
        {"name": "sample_512_whole", "kind": "sample", "rows": 512, "vocab": 32000, "top_k": 0, "top_p": 1.0, "min_p": 0.0, "temperature": 1.0, "per_row": False,
         "dtype": "fp32"},
    ]


# ---------------------------------------------------------------------------------------------------
# drawn cases
# ---------------------------------------------------------------------------------------------------
def _log_int(rng, lo, hi, multiple=1):
    hi = max(lo, hi)
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / multiple)) * multiple))


def _draw_heads(rng):
    kv = rng.choice([1, 2, 4, 8, 8, 16])
    group = rng.choice([1, 2, 4, 7, 8]) if kv > 1 else rng.choice([1, 8, 16, 24, 32])
    return kv * group, kv, rng.choice([64, 64, 80, 96, 128, 128, 128, 192, 256])


def _draw_append(rng):
    heads, kv, dim = _draw_heads(rng)
    most = 8001 * (2 * 32 + 4 * 8) * 128 // ((2 * heads + 4 * kv) * dim)
    decode = rng.random() < 0.5
    tokens = _log_int(rng, 1, min(512, most) if decode else most)
    dtype = rng.choice(["fp16", "bf16"])
    sequences = tokens if decode else rng.randint(1, min(16, tokens))
    context = rng.choice([0, _log_int(rng, 1, min(2000, 2**26 // (sequences * kv * dim)))])  # (the outputs are whole caches)
    return {"kind": "append", "sequences": sequences, "tokens": tokens, "heads": heads, "kv_heads": kv, "dim": dim, "rotary": rng.choice([dim, dim, dim // 2]),
            "interleaved": rng.random() < 0.3, "page": rng.choice([16, 32, 64, 128, _log_int(rng, 1, 256)]), "context": context, "dtype": dtype,
            "cache": rng.choice([dtype, dtype, "fp8"])}


def _draw_attend(rng):
    heads, kv, dim = _draw_heads(rng)
    dtype = rng.choice(["fp16", "bf16"])
    cache = rng.choice([dtype, dtype, "fp8"])
    most = 131071 * 8 * 128 * 2 // (kv * dim * SIZE[cache])  # tokens in all
    sequences = rng.choice([1, 1, _log_int(rng, 2, 256)])
    longest = _log_int(rng, 1, max(1, min(131071, most // sequences, 131071 * 32 * 128 // (heads * dim))))
    shortest = rng.choice([0, 1, longest, (longest + 1) // 2]) if sequences > 1 else longest
    return {"kind": "attend", "sequences": sequences, "shortest": shortest, "longest": longest, "heads": heads,
            "kv_heads": kv, "dim": dim, "page": rng.choice([16, 16, 32, 64, 128, _log_int(rng, 1, 256)]),
            "window": rng.choice([0, 0, 0, _log_int(rng, 1, 4096)]), "dtype": dtype, "cache": cache, "lse": rng.random() < 0.3}


def _draw_sample(rng):
    vocab = _log_int(rng, 29, 131072)
    dtype = rng.choice(["fp16", "bf16", "fp32"])
    return {"kind": "sample", "rows": _log_int(rng, 1, min(4096, 256 * 131072 // vocab // (2 if dtype == "fp32" else 1))), "vocab": vocab,
            "top_k": rng.choice([0, 0, 1, _log_int(rng, 2, 1000), vocab // 2]), "top_p": rng.choice([1.0, 1.0, 0.9, 0.99, round(rng.uniform(0.05, 0.999), 3)]),
            "min_p": rng.choice([0.0, 0.0, 0.05, round(rng.uniform(0.0001, 0.5), 4)]), "temperature": rng.choice([0.0, 1.0, 1.0, round(rng.uniform(0.3, 2.0), 2)]),
            "per_row": rng.random() < 0.4, "dtype": dtype}


def draw(rng):
    return rng.choice([_draw_append, _draw_attend, _draw_attend, _draw_sample, _draw_sample])(rng)


# ---------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------
class _Source:
    """Random tensors on the GPU from one seed."""

    def __init__(self, seed):
        self.g = torch.Generator(device=DEVICE).manual_seed(seed)

    def normal(self, *shape, dtype="fp16", scale=1.0):
        return torch.randn(*shape, generator=self.g, device=DEVICE, dtype=torch.bfloat16 if dtype == "fp8" else TYPES[dtype]).mul_(scale).to(TYPES[dtype])

    def shuffled(self, n):
        return torch.randperm(n, generator=self.g, device=DEVICE)

    def uniform(self, *shape):
        return torch.rand(*shape, generator=self.g, device=DEVICE)


def _lengths(case):
    """The sequences' lengths (what is in the cache after an append), spread evenly from the shortest to the longest."""
    n = case["sequences"]
    if case["kind"] == "append":
        counts = _counts(case)
        return [case["context"] + counts[i] for i in range(n)]
    return [case["shortest"] + (case["longest"] - case["shortest"]) * i // max(1, n - 1) for i in range(n)]


def _counts(case):
    """New tokens of each sequence."""
    n, total = case["sequences"], case["tokens"]
    if n == total:
        return [1] * n
    edges = [total * i * (i + 1) // (n * (n + 1)) for i in range(n + 1)]  # later sequences have more
    return [edges[i + 1] - edges[i] for i in range(n)]


def _inputs(case, seed):
    """The case's tensors, the same for the plain forms, the kernels and exact()."""
    s, d, kind = _Source(seed), dict(case), case["kind"]
    if kind == "sample":
        x = torch.randn(case["rows"], case["vocab"], generator=s.g, device=DEVICE) * 2.5
        x = torch.where(s.uniform(*x.shape) < 0.001, x + 8, x)  # a peaked distribution, with a few words that are not allowed
        x.masked_fill_(s.uniform(*x.shape) < 0.02, -math.inf)
        d["x"] = x.to(TYPES[case["dtype"]])
        d["u"] = s.uniform(case["rows"])
        if case["per_row"]:
            rows = case["rows"]
            spread = lambda v, lo, hi: (v * (lo + (hi - lo) * s.uniform(rows))).float()  # noqa: E731
            d["temperature"] = spread(case["temperature"], 0.5, 1.5)
            d["top_k"] = spread(case["top_k"], 0.2, 1.8).int()
            d["top_p"] = spread(case["top_p"], 0.8, 1.0)
            d["min_p"] = spread(case["min_p"], 0.0, 2.0)
        return d
    S, page, kv, dim = case["sequences"], case["page"], case["kv_heads"], case["dim"]
    order = s.shuffled(S).tolist()
    lengths = [_lengths(case)[i] for i in order]
    pages = [-(-n // page) for n in lengths]
    total, widest = sum(pages) + 1, max(1, max(pages))  # (one page is nobody's)
    place = s.shuffled(total).int().cpu()
    table = torch.full((S, widest), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(pages):
        table[i, :n] = place[at:at + n]
        at += n
    d["table"], d["lengths"] = table.to(DEVICE), torch.tensor(lengths, dtype=torch.int32, device=DEVICE)
    d["k_scale"] = d["v_scale"] = None
    if case["cache"] == "fp8":  # a head's largest key or value is about five times its spread
        d["k_scale"], d["v_scale"] = 0.01 + 0.02 * s.uniform(kv), 0.01 + 0.02 * s.uniform(kv)
    held = 60.0 if case["cache"] == "fp8" else 1.0
    d["k_pages"] = s.normal(total, kv, page, dim, dtype=case["cache"], scale=held)
    d["v_pages"] = s.normal(total, kv, page, dim, dtype=case["cache"], scale=held)
    if kind == "attend":
        d["q"] = s.normal(S, case["heads"], dim, dtype=case["dtype"])
        return d
    T = case["tokens"]
    d["q"] = s.normal(T, case["heads"], dim, dtype=case["dtype"])
    # A projection's result: queries, keys and values of a token lie beside one another.
    kv_rows = s.normal(T, 2 * kv, dim, dtype=case["dtype"])
    d["k"], d["v"] = kv_rows[:, :kv], kv_rows[:, kv:]
    counts = _counts(case)
    starts = [0]
    for i in order:
        starts.append(starts[-1] + counts[i])
    d["starts"] = None if T == S else torch.tensor(starts, dtype=torch.int32, device=DEVICE)
    d["position"] = torch.cat([torch.arange(lengths[i] - counts[j], lengths[i], dtype=torch.int32) for i, j in enumerate(order)]).to(DEVICE)
    d["sequence"] = torch.repeat_interleave(torch.arange(S, dtype=torch.int32), torch.tensor([counts[i] for i in order])).to(DEVICE)
    d["angles"] = _table(widest * page, case["rotary"])
    return d


def _table(positions, dim):
    """cos and sin of each position's angles, [positions, dim] in fp32: the cosines first."""
    frequency = 10000.0 ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=DEVICE) / dim)
    angle = torch.arange(positions, dtype=torch.float64, device=DEVICE).unsqueeze(1) * frequency
    return torch.cat([torch.cos(angle), torch.sin(angle)], 1).float()


def prepare(case, seed):
    d = _inputs(case, seed)
    if own:
        import pimaicompiler_amd as P
        P.initialize()
        d["P"] = P
        if case["kind"] != "sample":
            d["cache_of"] = P.PagedCache(d["k_pages"], d["v_pages"], d["k_scale"], d["v_scale"])
    return d


# ---------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------
def run(s):
    if own:
        return _own(s)
    return {"append": _plain_append, "attend": _plain_attend, "sample": _plain_sample}[s["kind"]](s)


def _own(s):
    if s["kind"] == "append":
        q = s["cache_of"].append(s["k"], s["v"], s["table"], s["lengths"], starts=s["starts"], q=s["q"], rotary=s["angles"], interleaved=s["interleaved"])
        return q, s["k_pages"], s["v_pages"]
    if s["kind"] == "attend":
        return s["cache_of"].attend(s["q"], s["table"], s["lengths"], window=s["window"], lse=s["lse"])
    return s["P"].sample_tokens(s["x"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])


def _plain_rotated(x, s):
    """x [T, heads, dim] in fp32 with the pairs of its first `rotary` values turned by their position's angles."""
    n = s["rotary"] // 2
    row = s["angles"][s["position"].long()].unsqueeze(1)
    c, w = row[..., :n], row[..., n:]
    head, rest = x[..., :2 * n], x[..., 2 * n:]
    if s["interleaved"]:
        a, b = head[..., 0::2], head[..., 1::2]
        return torch.cat([torch.stack([a * c - b * w, a * w + b * c], -1).flatten(-2), rest], -1)
    a, b = head[..., :n], head[..., n:]
    return torch.cat([a * c - b * w, a * w + b * c, rest], -1)


def _plain_append(s):
    page, at = s["page"], s["position"].long()
    where = s["table"][s["sequence"].long(), at // page].long()

    def put(pages, x, scale):
        if scale is None:
            pages[where, :, at % page] = x.to(pages.dtype)
        else:
            x = (x / scale.unsqueeze(1)).clamp(-FP8_MOST, FP8_MOST).to(pages.dtype)
            pages.view(torch.uint8)[where, :, at % page] = x.view(torch.uint8)

    put(s["k_pages"], _plain_rotated(s["k"].float(), s), s["k_scale"])
    put(s["v_pages"], s["v"].float(), s["v_scale"])
    return _plain_rotated(s["q"].float(), s).to(s["q"].dtype), s["k_pages"], s["v_pages"]


def _plain_held(pages, table, scale):
    """A cache's values [S, kv_heads, tokens, dim] in fp32, in the sequences' order."""
    x = pages.view(torch.uint8)[table].view(pages.dtype) if scale is not None else pages[table]
    x = x.transpose(1, 2).flatten(2, 3).float()
    return x if scale is None else x * scale.view(-1, 1, 1)


def _plain_attend(s):
    S, H, D = s["q"].shape
    kv, table = s["kv_heads"], s["table"].clamp(min=0).long()
    k = _plain_held(s["k_pages"], table, s["k_scale"])
    score = (s["q"].float().view(S, kv, H // kv, D) @ k.transpose(-1, -2)) / math.sqrt(D)
    at, length = torch.arange(k.shape[2], device=k.device), s["lengths"].view(-1, 1, 1, 1)
    seen = at < length
    if s["window"]:
        seen = seen & (at >= length - s["window"])
    score = torch.where(seen, score, -math.inf)
    m = score.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    e = torch.exp(score - m)
    z = e.sum(-1, keepdim=True)
    out = (e @ _plain_held(s["v_pages"], table, s["v_scale"])) / torch.where(z == 0, 1.0, z)
    out = out.view(S, H, D).to(s["q"].dtype)
    return (out, (m + torch.log(z)).view(S, H)) if s["lse"] else out


def _setting(v, x):
    """A row's setting as a column in 64 bits; numbers are fp32, like the tensors."""
    v = torch.as_tensor(v, device=x.device)
    return (v.float() if v.is_floating_point() else v).double().view(-1, 1)


def _plain_sample(s):
    x, V = s["x"].double(), s["x"].shape[1]  # (which word a number falls on hangs on the last bits)
    temperature, top_k, top_p, min_p = (_setting(s[name], x) for name in ("temperature", "top_k", "top_p", "min_p"))
    shifted = x - x.amax(-1, keepdim=True)
    greedy = temperature == 0
    w = torch.exp(shifted / torch.where(greedy, 1.0, temperature))
    order = torch.sort(s["x"].float(), dim=-1, descending=True, stable=True).indices
    rank = torch.arange(V, device=x.device)
    w = w.gather(1, order)
    w = torch.where(rank < torch.where(top_k > 0, top_k, V), w, 0.0)
    before = torch.cumsum(w, -1) - w
    kept = (top_p >= 1) | (before < top_p * w.sum(-1, keepdim=True)) | (rank == 0)
    kept = kept & ((min_p <= 0) | (w >= torch.clamp(min_p, max=1.0)))
    kept = kept & (~greedy | (rank == 0))
    w = torch.zeros_like(w).scatter_(1, order, torch.where(kept, w, 0.0))
    cum = torch.cumsum(w, -1)
    token = ((cum > s["u"].double().unsqueeze(1) * cum[:, -1:]) & (w > 0)).int().argmax(-1)
    logp = torch.log(w.gather(1, token.unsqueeze(1)).squeeze(1) / cum[:, -1])
    return token, logp.float()


# ---------------------------------------------------------------------------------------------------
# the work of a pass
# ---------------------------------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": SIZE[case["dtype"]] * n + 16 * case["rows"], "flops": 4 * n}
    H, kv, D, size, held = case["heads"], case["kv_heads"], case["dim"], SIZE[case["dtype"]], SIZE[case["cache"]]
    if kind == "append":
        T = case["tokens"]
        return {"bytes": T * (D * (2 * size * H + 2 * kv * (size + held)) + 4 * case["rotary"] + 4) + 4 * case["sequences"],
                "flops": 3 * T * (H + kv) * case["rotary"]}
    tokens = sum(min(n, case["window"] or n) for n in _lengths(case))
    return {"bytes": tokens * kv * 2 * D * held + 4 * tokens // case["page"] + case["sequences"] * (H * (2 * D * size + (4 if case["lse"] else 0)) + 4),
            "flops": 4 * tokens * H * D}


# ---------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------------
def _exact_append(d):
    """Every pair as a complex number times its position's; the rest as it is."""
    n = d["rotary"] // 2

    def turned(x):
        x = x.double().clone()
        row = d["angles"].double()[d["position"].long()]
        by = torch.complex(row[:, :n].contiguous(), row[:, n:].contiguous()).unsqueeze(1)
        first, second = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if d["interleaved"] else (slice(0, n), slice(n, 2 * n))
        z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * by
        x[..., first], x[..., second] = z.real, z.imag
        return x

    page = d["page"]
    slot = d["table"].long()[d["sequence"].long(), torch.div(d["position"].long(), page, rounding_mode="floor")] * page + d["position"].long() % page
    out = []
    for pages, x, scale in ((d["k_pages"], turned(d["k"]), d["k_scale"]), (d["v_pages"], d["v"].double(), d["v_scale"])):
        if scale is not None:
            x = torch.clamp(x / scale.double().unsqueeze(1), -FP8_MOST, FP8_MOST)
        flat = pages.double().transpose(1, 2).flatten(0, 1).index_copy(0, slot, x)  # [tokens of all pages, kv_heads, dim]
        out.append(flat.view(pages.shape[0], page, *flat.shape[1:]).transpose(1, 2))
    return (turned(d["q"]), *out)


def _exact_attend(d):
    S, H, D = d["q"].shape
    G = H // d["kv_heads"]
    out, sums = torch.zeros(S, H, D, dtype=torch.float64, device=DEVICE), torch.full((S, H), -math.inf, dtype=torch.float64, device=DEVICE)
    for i, n in enumerate(d["lengths"].tolist()):
        first = max(0, n - d["window"]) if d["window"] else 0
        if n == first:
            continue
        at = torch.arange(first, n, device=DEVICE)
        page, inside = d["table"][i].long()[at // d["page"]], at % d["page"]
        for h in range(d["kv_heads"]):
            k, v = (p[page.unique(), h].double() for p in (d["k_pages"], d["v_pages"]))
            where = torch.searchsorted(page.unique(), page)
            k, v = k[where, inside], v[where, inside]
            if d["k_scale"] is not None:
                k, v = k * d["k_scale"][h].double(), v * d["v_scale"][h].double()
            score = k @ d["q"][i, h * G:(h + 1) * G].double().t() / math.sqrt(D)
            total = torch.logsumexp(score, 0)
            out[i, h * G:(h + 1) * G] = torch.exp(score - total).t() @ v
            sums[i, h * G:(h + 1) * G] = total
    return (out, sums) if d["lse"] else out


def _exact_sample(d):
    """Row by row: the words in falling order, what each setting leaves of them, and the one the number falls on in the order of the words."""
    tokens, logps = [], []
    settings = [torch.as_tensor(d[name]).float().cpu().double().expand(d["rows"]).tolist() for name in ("temperature", "top_k", "top_p", "min_p")]
    for x, u, temperature, k, p, least in zip(d["x"].cpu().double(), d["u"].cpu().double().tolist(), *settings):
        at = torch.argsort(x, descending=True, stable=True)
        if temperature == 0:
            tokens.append(int(at[0]))
            logps.append(0.0)
            continue
        at = at[:int(k)] if k > 0 else at
        share = torch.softmax(x[at] / temperature, 0)
        if p < 1:
            n = int((torch.cumsum(share, 0) - share < p).sum())
            at, share = at[:max(1, n)], share[:max(1, n)]
        at = at[share >= least * share[0]] if least > 0 else at
        at = torch.sort(at).values
        logp = torch.log_softmax(x[at] / temperature, 0)
        edge = torch.cumsum(torch.exp(logp), 0)
        i = min(int(torch.searchsorted(edge, u * float(edge[-1]), right=True)), len(at) - 1)
        tokens.append(int(at[i]))
        logps.append(float(logp[i]))
    return torch.tensor(tokens), torch.tensor(logps, dtype=torch.float64)


def exact(case, seed):
    if case["kind"] == "sample" and case["rows"] * case["vocab"] > 4e7:
        return None
    d = _inputs(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "sample": _exact_sample}[case["kind"]](d)
