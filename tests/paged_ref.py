"""Plain 64-bit forms of the paged cache's operators, and the bounds that their rounding errors keep to."""
import math

import torch

EPS = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}      # half a step, relative
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}   # half a step among the subnormals


def sequences(lens, news, page, gen, spare=3, width=2):
    """Page table (garbage behind every length), lens and starts for sequences of these lengths and new rows."""
    counts = [-(-n // page) for n in lens]
    pages = sum(counts) + spare
    order = torch.randperm(pages, generator=gen)
    table = torch.randint(-2 ** 31, 2 ** 31 - 1, (len(lens), max(counts) + width), generator=gen).to(torch.int32)
    at = 0
    for i, c in enumerate(counts):
        table[i, :c] = order[at:at + c].to(torch.int32)
        at += c
    starts = [0]
    for m in news:
        starts.append(starts[-1] + m)
    return pages, table, torch.tensor(lens, dtype=torch.int32), torch.tensor(starts, dtype=torch.int32)


def pool(pages, kv_heads, page, dim, dtype, inner, fill=float("nan")):
    """A pool [pages, kv_heads, page, dim] full of `fill`; inner: the heads lie inside the positions."""
    if inner:
        return torch.full((pages, page, kv_heads, dim), fill, dtype=dtype).transpose(1, 2)
    return torch.full((pages, kv_heads, page, dim), fill, dtype=dtype)


def store(p, table, b, first, rows):
    """rows [n, kv_heads, dim] at positions first.. of sequence b."""
    page = p.shape[2]
    pos = torch.arange(first, first + rows.shape[0])
    p[table[b, pos // page].long(), :, pos % page] = rows.to(p.dtype)


def load(p, table, b, n):
    """Positions 0 .. n - 1 of sequence b: [n, kv_heads, dim] in 64 bits."""
    pos = torch.arange(n)
    return p[table[b, pos // p.shape[2]].long(), :, pos % p.shape[2]].double()


def attend(q, k, v, positions, scale, window):
    """One sequence: q [m, H, D] at `positions` over k, v [n, Hk, D].  Returns out [m, H, D] and the bound of the error of a
    kernel that takes scores and sums in 32 bits and probabilities and results in q's type."""
    m, h, dim = q.shape
    n, hk, _ = k.shape
    eps, tiny, dtype = EPS[q.dtype], TINY[q.dtype], q.dtype
    q = q.double()
    out, bound = torch.zeros(m, h, dim, dtype=torch.float64), torch.zeros(m, h, dim, dtype=torch.float64)
    if n == 0:
        return out, bound, dtype
    at = torch.arange(n)[None]
    pos = positions[:, None]
    seen = at <= pos
    if window:
        seen = seen & (at > pos - window)
    some = seen.any(1)
    for head in range(h):
        kk, vv = k[:, head // (h // hk)], v[:, head // (h // hk)]
        s = (q[:, head] @ kk.T) * scale
        s = torch.where(seen, s, torch.full((), -math.inf, dtype=torch.float64))
        p = torch.softmax(s, 1)
        p = torch.where(some[:, None], p, torch.zeros((), dtype=torch.float64))
        o, mean = p @ vv, p @ vv.abs()
        # scores: dim products summed in 32 bits, each sum off by at most a step (tensor cores may cut); times log2 e and scale in
        # 32 bits: two more roundings of the score; exp within 2^-13 (the probabilities are rounded to 11 bits or fewer anyway)
        size = (torch.where(seen, (q[:, head].abs() @ kk.abs().T) * abs(scale), torch.zeros((), dtype=torch.float64))).amax(1)
        ds = size * (dim + 4) * 2.0 ** -23
        # probabilities rounded to the type; sums over n positions in 32 bits, numerator and denominator; both feel ds and exp
        rel = eps + 2 * (ds + 2.0 ** -13) + 2 * (n + 8) * 2.0 ** -23
        # probabilities below the type's normal range: half a subnormal step each, against a sum of at least one
        low = tiny * (seen.sum(1)[:, None] * torch.where(seen.any(0)[:, None], vv.abs(), torch.zeros((), dtype=torch.float64)).amax(0)[None])
        out[:, head] = o
        bound[:, head] = mean * rel[:, None] * (1 + eps) + low + eps * o.abs() + tiny
    return out, bound, dtype


def rotate(x, heads, kv_heads, dim, cos, sin, pos):
    """Rows x [n, (heads + 2 kv_heads) dim] -> q, k, v in 64 bits and the bound of their error in 32-bit arithmetic (before the
    rounding to the cache's type)."""
    x = x.double().view(x.shape[0], heads + 2 * kv_heads, dim)
    r = cos.shape[1]
    c, s = cos.double()[pos][:, None], sin.double()[pos][:, None]
    a, b = x[:, :heads + kv_heads, :r], x[:, :heads + kv_heads, r:2 * r]
    turned = torch.cat((a * c - b * s, b * c + a * s, x[:, :heads + kv_heads, 2 * r:]), 2)
    size = torch.cat(((a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs(), torch.zeros_like(x[:, :heads + kv_heads, 2 * r:])), 2)
    return turned[:, :heads], turned[:, heads:], x[:, heads + kv_heads:], size * 2.0 ** -23   # two products, one sum: 3 roundings of 2^-24 at most
