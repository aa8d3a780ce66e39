"""A paged cache's inputs on the CPU, and the definitions of append and attend in 64 bits."""
import math

import torch

FP8 = torch.float8_e4m3fn


def step(dtype):
    """Half the distance of neighbours, relative to the value."""
    return torch.finfo(dtype).eps / 2


class Cache:
    """A page table for sequences of `lengths` tokens (their pages shuffled, one page nobody's, entries behind a sequence's pages -1, the places nobody has
    filled holding `rest`) and random keys and values."""

    def __init__(self, lengths, heads, page, dim, dtype, seed=0, rest=0.0, extra_width=0):
        g = torch.Generator().manual_seed(seed)
        self.lengths, self.page, self.dtype = list(lengths), page, dtype
        counts = [-(-max(0, n) // page) for n in lengths]
        total, width = sum(counts) + 1, max([1] + counts) + extra_width
        order = torch.randperm(total, generator=g).int()
        self.table = torch.full((len(counts), width), -1, dtype=torch.int32)
        at = 0
        self.k, self.v = (torch.full((total, heads, page, dim), rest) for _ in range(2))
        for s, n in enumerate(counts):
            mine = order[at:at + n]
            self.table[s, :n] = mine
            at += n
            for j in range(lengths[s]):
                p, i = int(mine[j // page]), j % page
                self.k[p, :, i], self.v[p, :, i] = torch.randn(heads, dim, generator=g), torch.randn(heads, dim, generator=g)
        self.k_scale = self.v_scale = None
        if dtype == FP8:
            self.k_scale, self.v_scale = 0.01 + 0.02 * torch.rand(heads, generator=g), 0.01 + 0.02 * torch.rand(heads, generator=g)
            self.k, self.v = self.k / self.k_scale.view(1, -1, 1, 1), self.v / self.v_scale.view(1, -1, 1, 1)
            self.k, self.v = self.k.clamp(-448, 448), self.v.clamp(-448, 448)
        self.k, self.v = self.k.to(dtype), self.v.to(dtype)

    def on(self, P, device, layout="heads first"):
        """The package's cache of these values, [pages, heads, tokens, dim] in memory or [pages, tokens, heads, dim]."""
        def place(t):
            t = t.to(device)
            return t if layout == "heads first" else t.view(torch.uint8 if t.dtype == FP8 else t.dtype).transpose(1, 2).contiguous().transpose(1, 2).view(t.dtype)
        scales = [s.to(device) if s is not None else None for s in (self.k_scale, self.v_scale)]
        return P.PagedCache(place(self.k), place(self.v), *scales)

    def tensors(self, device):
        return self.table.to(device), torch.tensor(self.lengths, dtype=torch.int32, device=device)

    def held(self, s, first=0):
        """The values [heads, tokens, dim] of a sequence in 64 bits, whatever lies in pages outside of the cache left out (their tokens' numbers beside)."""
        n = min(self.lengths[s], self.table.shape[1] * self.page)
        seen = [j for j in range(max(0, first), n) if 0 <= int(self.table[s, j // self.page]) < self.k.shape[0]]
        rows = [(int(self.table[s, j // self.page]), j % self.page) for j in seen]
        if not rows:
            empty = torch.zeros(self.k.shape[1], 0, self.k.shape[3], dtype=torch.float64)
            return empty, empty
        out = []
        for t, scale in ((self.k, self.k_scale), (self.v, self.v_scale)):
            x = torch.stack([t[p, :, i].double() for p, i in rows], 1)
            out.append(x if scale is None else x * scale.double().view(-1, 1, 1))
        return out


def attend(cache, q, scale, window=0):
    """(out, lse, what bounds the error of out and of lse) in 64 bits.

    With u = 2^-24: a score is a sum of dim exact products in fp32, off by (dim + 1) u sum |q k|, and takes three more roundings (two factors of the scale, the
    product), relative to the score.  The difference to the running maximum and the power of two: u (|s| + |m|) + 2 u relative to the weight, and as much again
    wherever the maximum moves on and parts are joined, which leaves the same factor on sums and values unless it is rounded (4 u).  Sums over n
    tokens add up in some order, (n + 16) u of the sum of magnitudes; the last division and product 3 u.  Then one rounding to q's type."""
    u = 2.0**-24
    S, H, D = q.shape
    heads = cache.k.shape[1]
    out, lse = torch.zeros(S, H, D, dtype=torch.float64), torch.full((S, H), -math.inf, dtype=torch.float64)
    out_bound, lse_bound = torch.zeros_like(out), torch.zeros_like(lse)
    for s in range(S):
        n = min(cache.lengths[s], cache.table.shape[1] * cache.page)
        k, v = cache.held(s, n - window if window else 0)
        if k.shape[1] == 0:
            continue
        for h in range(H):
            kh, vh, x = k[h // (H // heads)], v[h // (H // heads)], q[s, h].double()
            score = scale * (kh @ x)
            total = torch.logsumexp(score, 0)
            p = torch.exp(score - total)
            off = abs(scale) * (D + 1) * u * (kh.abs() @ x.abs()).max() + 8 * u * score.abs().max() + 8 * u
            rel = 2 * off + (len(p) + 24) * u
            out[s, h], lse[s, h] = p @ vh, total
            size = p @ vh.abs()
            out_bound[s, h] = rel * 2 * size * (1 + 1e-3)
            lse_bound[s, h] = rel + 4 * u * total.abs() + 4 * u
    t = q.dtype
    out_bound = out_bound + (out.abs() + out_bound) * step(t) + torch.finfo(t).smallest_normal * step(t)
    return out, lse, out_bound, lse_bound


def turned(x, positions, angles, dim, interleaved):
    """x [tokens, heads, D] with its first `dim` values turned, in 64 bits, and sum of the magnitudes of the products of each."""
    y, size = x.double().clone(), x.double().abs()
    if not dim:
        return y, size * 0
    c, w = (t.double().unsqueeze(1) for t in angles[positions.long(), :dim].split(dim // 2, 1))
    first, second = (slice(0, dim, 2), slice(1, dim, 2)) if interleaved else (slice(0, dim // 2), slice(dim // 2, dim))
    a, b = x[..., first].double(), x[..., second].double()
    y[..., first], y[..., second] = a * c - b * w, a * w + b * c
    sizes = torch.zeros_like(y)
    sizes[..., first], sizes[..., second] = (a * c).abs() + (b * w).abs(), (a * w).abs() + (b * c).abs()
    return y, sizes
