"""Plain 64-bit definitions of the operators over a paged KV cache, on the CPU,
and the small caches the tests use."""
import math

import numpy as np
import torch

HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half a step, relative
TINY = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}  # half the smallest step


def make_pages(gen, n_seqs, max_pages, page, heads, dim, dtype, spare=3, bad=None):
    """k, v pages with every sequence's pages scattered; `bad` fills all of both (a value that must
    never matter), else they are normal."""
    n = n_seqs * max_pages + spare
    k = torch.randn(n, page, heads, dim, generator=gen)
    v = torch.randn(n, page, heads, dim, generator=gen)
    if bad is not None:
        k.fill_(bad), v.fill_(bad)
    table = torch.randperm(n, generator=gen)[:n_seqs * max_pages].view(n_seqs, max_pages).to(torch.int32)
    return k.to(dtype), v.to(dtype), table


def rows(pages, table, s, slots):
    """[slots, heads, dim] of sequence s."""
    page = pages.shape[1]
    slots = torch.as_tensor(slots, dtype=torch.long)
    return pages[table[s].long()[slots // page], slots % page]


def put(pages, table, s, slot, value):
    page = pages.shape[1]
    pages[int(table[s, slot // page]), slot % page] = value


def rope(x, pos, freqs, style, mscale):
    """x [tokens, heads, dim] in 64 bits."""
    x = x.double().clone()
    half = len(freqs)
    ang = pos.double()[:, None] * freqs.double()
    c, s = (torch.cos(ang) * mscale)[:, None], (torch.sin(ang) * mscale)[:, None]
    ia = torch.arange(half) * (2 if style == 0 else 1)
    ib = ia + (1 if style == 0 else half)
    a, b = x[..., ia].clone(), x[..., ib].clone()
    x[..., ia], x[..., ib] = a * c - b * s, a * s + b * c
    return x


def rope_tolerance(x, freqs, style, mscale, dtype, want):
    """The angle: a fraction of a turn of at most 1/2 rounded to 24 bits, 2 pi 2^-26 rad; sine and cosine
    within 2 ulp of values up to 1, 2^-23; the factor, two products and a sum, 4 half steps of 2^-24;
    then the output's rounding."""
    half = len(freqs)
    ia = torch.arange(half) * (2 if style == 0 else 1)
    ib = ia + (1 if style == 0 else half)
    size = torch.zeros_like(want)
    both = (x.double()[..., ia].abs() + x.double()[..., ib].abs()) * mscale
    size[..., ia] = both
    size[..., ib] = both
    return size * (2 * math.pi * 2.0 ** -26 + 2.0 ** -23 + 4 * 2.0 ** -24) * 1.01 + want.abs() * HALF[dtype] + TINY[dtype]


def attention(q, k_pages, v_pages, table, lens, scale):
    """out [b, n, hq, d], weights [b, hk, slots], and per output element the sum of p |v| and per row the largest
    sum of |q k| scale, for the tolerance. NaN-free cached rows only are read."""
    b, n, hq, d = q.shape
    hk = k_pages.shape[2]
    g = hq // hk
    slots = table.shape[1] * k_pages.shape[1]
    out, size = torch.zeros(b, n, hq, d, dtype=torch.float64), torch.zeros(b, n, hq, d, dtype=torch.float64)
    big = torch.zeros(b, n, hq, dtype=torch.float64)
    weights = torch.zeros(b, hk, slots, dtype=torch.float64)
    for s in range(b):
        for j in range(n):
            sees = int(lens[s]) - (n - 1 - j)
            if sees <= 0:
                continue
            k = rows(k_pages, table, s, range(sees)).double()
            v = rows(v_pages, table, s, range(sees)).double()
            for h in range(hq):
                x = k[:, h // g] @ q[s, j, h].double() * scale
                p = torch.softmax(x, 0)
                out[s, j, h] = p @ v[:, h // g]
                size[s, j, h] = p @ v[:, h // g].abs()
                big[s, j, h] = (k[:, h // g].abs() @ q[s, j, h].double().abs()).max() * abs(scale)
                weights[s, h // g, :sees] += p
    return out, weights, size, big


def attention_tolerance(q_type, cache_type, d, longest, size, big, want):
    """Scores: q in parts that hold 2^-22 of it (or all of it) and an f32 sum of d products taken 16 at a time per part
    (3 parts at most), each step within 2^-23 of the sum of magnitudes; scale and base-2 exponent 4 half steps more.
    e^delta - 1 <= 1.1 delta each for the weight and for the sum it is divided by. Weights enter the product in parts
    that hold 2^-22 for f32 outputs, 2^-16 (two bf16 parts) for f16 outputs of a bf16 cache, else in one of the
    cache's type; exponentials are within 2^-21; sums over the positions, 16 at a time and 3 parts: 2^-23 a step (rescales included), and
    once more for the divisor."""
    delta = big * (2.0 ** -22 + (3 * d / 16 + 4) * 2.0 ** -23)
    enter = 2.0 ** -22 if q_type == torch.float32 else 2.0 ** -16 if HALF[q_type] < HALF[cache_type] else HALF[cache_type]
    rel = 2 * 1.1 * delta + enter + 2 * 2.0 ** -21 + 2 * (3 * longest / 16 + 40) * 2.0 ** -23
    return size * rel.unsqueeze(-1) + want.abs() * HALF[q_type] + TINY[q_type], delta


def evict(k_pages, v_pages, table, lens, weights, budget, recent, sinks):
    b, hk, slots = weights.shape
    kept = torch.full((b, hk, budget), -1, dtype=torch.int32)
    nw = torch.zeros_like(weights)
    k, v = k_pages.clone(), v_pages.clone()
    page = k.shape[1]
    for s in range(b):
        n = int(lens[s])
        for h in range(hk):
            w = weights[s, h].numpy()
            if n <= budget:
                keep = list(range(n))
            else:
                mid = list(range(sinks, n - recent))
                mid.sort(key=lambda t: (1, 0.0) if math.isnan(w[t]) else (0, -float(w[t])))  # stable: ties to the earlier
                keep = sorted(list(range(sinks)) + mid[:budget - recent - sinks] + list(range(n - recent, n)))
            for i, t in enumerate(keep):
                kept[s, h, i] = t
                nw[s, h, i] = weights[s, h, t]
                to, fr = (int(table[s, i // page]), i % page, h), (int(table[s, t // page]), t % page, h)
                k[to], v[to] = k_pages[fr], v_pages[fr]
    return kept, torch.tensor([min(int(n), budget) for n in lens], dtype=torch.int32), nw, k, v


def verify(p, q, draft, u, n_draft):
    b, n = draft.shape
    vocab = p.shape[2]
    p = p.double().numpy()
    q = None if q is None else q.double().numpy()
    u = u.double().numpy()
    tokens, accepted = np.full((b, n + 1), -1, np.int32), np.zeros(b, np.int32)
    for s in range(b):
        most = n if n_draft is None else min(max(int(n_draft[s]), 0), n)
        a = 0
        while a < most:
            x = int(draft[s, a])
            if not 0 <= x < vocab or not u[s, a] * (1.0 if q is None else q[s, a, x]) < p[s, a, x]:
                break
            tokens[s, a] = x
            a += 1
        row = np.where((p[s, a] > 0) & np.isfinite(p[s, a]), p[s, a], 0.0)
        left = row
        if a < most:
            sub = q[s, a] if q is not None else (np.arange(vocab) == int(draft[s, a])).astype(np.float64)
            with np.errstate(invalid="ignore"):
                d = np.where(np.isfinite(p[s, a]), p[s, a], 0.0) - sub
            left = np.where(d > 0, d, 0.0)
            if not (left > 0).any():
                left = row
        if (left > 0).any():
            c = np.cumsum(left)
            at = int(np.searchsorted(c, u[s, n] * c[-1], side="right"))
            tokens[s, a] = min(at, int(np.nonzero(left > 0)[0].max()))
        else:
            tokens[s, a] = 0
        accepted[s] = a
    return torch.from_numpy(tokens), torch.from_numpy(accepted)
