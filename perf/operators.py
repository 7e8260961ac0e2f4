"""The serving operators over a paged key-value cache, as they are measured.

Four operators that a serving loop runs one after the other:

  rope_append   rotary positions on the new tokens' q and k (pairs interleaved or in halves, the whole head or
                its first part, frequencies scaled for long contexts), k and v written into the cache's pages
  attn_paged    attention of each sequence's newest token (or newest few, when drafts are checked) over its
                pages; on request the weight that every cached position received is added up
  evict         the positions with the largest such sums kept, with the first and the latest ones, and the
                cache compacted in place
  verify_draft  drafted tokens taken or refused against the target's probabilities, and the token after them
                drawn, from given random numbers

Head counts and widths are those of nightrun_b200/configs.py, vocabularies too. A case is a dict of plain values;
`own` says whether run() makes the framework's calls or computes the plain forms below.
"""
import math

import torch

own = False

_T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}
# (query heads, KV heads, head width) of the framework's model configurations, small ones last.
_HEADS = [(32, 8, 64), (32, 8, 128), (40, 8, 64), (4, 2, 128), (2, 1, 128)]
_TYPES = [("f32", "f16"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "bf16")]
_VOCABS = [1000, 100352, 128256, 151936]


def listed():
    def rope(name, tokens, seqs, heads, rot, style, scaling, types, page, start):
        return {"name": name, "op": "rope_append", "tokens": tokens, "seqs": seqs, "heads": heads[0], "kv_heads": heads[1],
                "dim": heads[2], "rot": rot, "style": style, "scaling": scaling, "type": types[0], "cache": types[1],
                "page": page, "start": start}

    def attn(name, seqs, new, heads, types, page, shortest, longest, weights):
        return {"name": name, "op": "attn_paged", "seqs": seqs, "new": new, "heads": heads[0], "kv_heads": heads[1],
                "dim": heads[2], "type": types[0], "cache": types[1], "page": page, "shortest": shortest,
                "longest": longest, "weights": weights}

    def evict(name, seqs, heads, cache, page, shortest, longest, budget, recent, sinks):
        return {"name": name, "op": "evict", "seqs": seqs, "kv_heads": heads[1], "dim": heads[2], "cache": cache,
                "page": page, "shortest": shortest, "longest": longest, "budget": budget, "recent": recent, "sinks": sinks}

    def verify(name, seqs, draft, vocab, kind, sampled):
        return {"name": name, "op": "verify_draft", "seqs": seqs, "draft": draft, "vocab": vocab, "type": kind,
                "sampled": sampled}

    return [
        # One decode step of one sequence in the framework's own types: launch latency is all there is.
        rope("rope one token", 1, 1, _HEADS[0], 64, 0, "llama3", _TYPES[0], 16, 700),
        # A decode step of a ragged number of sequences far into a stretched context, a quarter of the head unrotated.
        rope("rope 203 sequences", 203, 203, _HEADS[1], 96, 1, "yarn", _TYPES[2], 24, 100000),
        # A prefill pass of several prompts.
        rope("rope prefill 8192", 8192, 5, _HEADS[1], 128, 1, "none", _TYPES[1], 64, 0),
        # The first steps of a chat with one user: a short context, the framework's types.
        attn("attn short one", 1, 1, _HEADS[0], _TYPES[0], 16, 77, 77, False),
        # One user with a very long document: the only parallelism is along the cache.
        attn("attn long one", 1, 1, _HEADS[1], _TYPES[1], 64, 131072, 131072, False),
        # A busy server: sequences of all ages in one batch.
        attn("attn ragged 64", 64, 1, _HEADS[1], _TYPES[2], 16, 200, 16384, False),
        # Checking four drafted tokens per sequence, with the weights that eviction goes by; pages of an odd size.
        attn("attn drafts 24", 24, 5, _HEADS[2], _TYPES[0], 24, 1000, 9001, True),
        # One sequence that outgrew a small budget.
        evict("evict one", 1, _HEADS[0], "f16", 16, 1500, 1500, 1024, 128, 4),
        # A server that halves its long sequences, the shorter ones of the batch stay whole.
        evict("evict 24", 24, _HEADS[1], "bf16", 64, 1000, 20000, 4096, 513, 4),
        # One user's four drafted tokens.
        verify("verify one", 1, 4, 128256, "f32", True),
        # A batch with drafts taken greedily (no draft distribution), half-precision probabilities, an odd batch.
        verify("verify greedy 37", 37, 3, 100352, "f16", False),
        # A large batch with seven drafts per sequence over the largest vocabulary.
        verify("verify 160", 160, 7, 151936, "f32", True),
    ]


def _log(rng, a, b):
    return max(a, min(b, int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))))


def draw(rng):
    op = rng.choice(["rope_append", "attn_paged", "evict", "verify_draft"])
    heads, kv_heads, dim = rng.choice(_HEADS)
    kind, cache = rng.choice(_TYPES)
    page = rng.choice([8, 16, 24, 32, 64, 100])
    if op == "rope_append":
        tokens = _log(rng, 1, 8192)
        return {"op": op, "tokens": tokens, "seqs": _log(rng, 1, min(tokens, 256)), "heads": heads, "kv_heads": kv_heads,
                "dim": dim, "rot": dim * rng.choice([4, 4, 3, 2, 1]) // 4, "style": rng.randrange(2),
                "scaling": rng.choice(["none", "llama3", "yarn"]), "type": kind, "cache": cache, "page": page,
                "start": _log(rng, 1, 120000)}
    if op == "attn_paged":
        new = rng.choice([1, 1, 1, 2, 3, 5, 8])
        seqs = _log(rng, 1, 128)
        longest = max(new, _log(rng, 1, min(131072, 230000 // seqs)))
        return {"op": op, "seqs": seqs, "new": new, "heads": heads, "kv_heads": kv_heads, "dim": dim, "type": kind,
                "cache": cache, "page": page, "shortest": max(1, longest // rng.choice([1, 3, 30])), "longest": longest,
                "weights": rng.random() < 0.25}
    if op == "evict":
        seqs = _log(rng, 1, 64)
        longest = _log(rng, 64, min(65536, 120000 // seqs))
        budget = max(16, int(longest * rng.uniform(0.15, 0.8)))
        return {"op": op, "seqs": seqs, "kv_heads": kv_heads, "dim": dim, "cache": cache, "page": page,
                "shortest": max(1, longest // rng.choice([1, 2, 10])), "longest": longest, "budget": budget,
                "recent": int(budget * rng.uniform(0.05, 0.5)), "sinks": rng.randrange(8)}
    draft = rng.randrange(1, 9)
    vocab = rng.choice(_VOCABS) - rng.choice([0, 0, 1, 5])
    return {"op": op, "seqs": _log(rng, 1, 160), "draft": draft, "vocab": vocab, "type": rng.choice(["f32", "f16", "bf16"]),
            "sampled": rng.random() < 0.7}


# ------------------------------------------------------------------------------------------------ inputs


def _lengths(case):
    """The sequences' lengths, from the shortest to the longest in equal ratios."""
    n, a, b = case["seqs"], case["shortest"], case["longest"]
    return [int(round(a * (b / a) ** (i / (n - 1)))) for i in range(n)] if n > 1 else [b]


def _freqs(dim, scaling):
    """Angle per position of each pair of `dim` rotated values, and the factor on cos and sin."""
    theta = 500000.0
    freq = theta ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    if scaling == "llama3":
        factor, low, high, orig = 32.0, 1.0, 4.0, 8192.0
        turns = orig * freq / (2 * math.pi)
        mix = ((turns - low) / (high - low)).clamp(0, 1)
        return (freq * mix + freq / factor * (1 - mix)).float(), 1.0
    if scaling == "yarn":
        factor, fast, slow, orig = 16.0, 32.0, 1.0, 8192.0
        at = lambda turns: dim * math.log(orig / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
        low, high = max(0, math.floor(at(fast))), min(dim - 1, math.ceil(at(slow)))
        keep = 1 - ((torch.arange(dim // 2, dtype=torch.float64) - low) / max(high - low, 1e-3)).clamp(0, 1)
        return (freq * keep + freq / factor * (1 - keep)).float(), 0.1 * math.log(factor) + 1
    return freq.float(), 1.0


def _pages(case, gen, seqs, slots):
    """Pages for `slots` positions per sequence, in no order, some unused, and the table that finds them."""
    per = -(-slots // case["page"])
    n = seqs * per + 3
    shape = (n, case["page"], case["kv_heads"], case["dim"])
    kv = [torch.randn(shape, generator=gen, device="cuda", dtype=_T[case["cache"]]) for _ in range(2)]
    table = torch.randperm(n, generator=gen, device="cuda")[:seqs * per].view(seqs, per).to(torch.int32)
    return kv[0], kv[1], table.contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    if op == "rope_append":
        t, s, hq, hk, d = (case[k] for k in ("tokens", "seqs", "heads", "kv_heads", "dim"))
        # One projection holds q, k and v side by side, as a fused linear layer leaves them.
        qkv = torch.randn(t, hq + 2 * hk, d, generator=gen, device="cuda").to(_T[case["type"]])
        counts = torch.full((s,), t // s, device="cuda")
        counts[: t % s] += 1
        seq = torch.repeat_interleave(torch.arange(s, device="cuda"), counts, output_size=t)
        begin = torch.cumsum(counts, 0) - counts
        nth = torch.arange(t, device="cuda") - begin[seq]
        base = torch.randint(0, 40, (s,), generator=gen, device="cuda")  # positions cached before
        k, v, table = _pages(case, gen, s, -(-t // s) + 40)
        freqs, mscale = _freqs(case["rot"], case["scaling"])
        return {"op": op, "q": qkv[:, :hq], "k": qkv[:, hq:hq + hk], "v": qkv[:, hq + hk:], "k_pages": k, "v_pages": v,
                "table": table, "freqs": freqs.cuda(), "mscale": mscale, "style": case["style"],
                "pos": (case["start"] + base[seq] + nth).to(torch.int32), "seq": seq.to(torch.int32),
                "slot": (base[seq] + nth).to(torch.int32),
                "q_out": torch.empty(t, hq, d, device="cuda", dtype=_T[case["type"]])}
    if op == "verify_draft":
        b, n, v, kind = case["seqs"], case["draft"], case["vocab"], _T[case["type"]]
        logits = torch.randn(b, n + 1, v, generator=gen, device="cuda") * 3
        p = torch.softmax(logits, -1)
        # The draft model's opinion: the target's, blurred; about two drafts of three are taken.
        q = torch.softmax(logits[:, :n] + torch.randn(b, n, v, generator=gen, device="cuda") * 0.8, -1)
        pick = torch.rand(b, n, 1, generator=gen, device="cuda", dtype=torch.float64)
        if case["sampled"]:
            draft = (torch.cumsum(q.double(), -1) <= pick).sum(-1).clamp(max=v - 1)
        else:
            draft = torch.where(pick[..., 0] < 0.6, p[:, :n].argmax(-1), q.argmax(-1))
        return {"op": op, "p": p.to(kind), "q": q.to(kind) if case["sampled"] else None, "draft": draft.to(torch.int32),
                "u": torch.rand(b, n + 1, generator=gen, device="cuda"),
                "n_draft": torch.randint(max(0, n - 1), n + 1, (b,), generator=gen, device="cuda", dtype=torch.int32),
                "tokens": torch.empty(b, n + 1, device="cuda", dtype=torch.int32),
                "accepted": torch.empty(b, device="cuda", dtype=torch.int32)}
    b, hk, d = case["seqs"], case["kv_heads"], case["dim"]
    order = torch.randperm(b, generator=gen, device="cuda")
    lens = torch.tensor(_lengths(case), device="cuda", dtype=torch.int32)[order]
    k, v, table = _pages(case, gen, b, case["longest"])
    slots = table.shape[1] * case["page"]
    state = {"op": op, "k_pages": k, "v_pages": v, "table": table, "lens": lens}
    if op == "attn_paged":
        shape, kind = (b, case["new"], case["heads"], d), _T[case["type"]]
        state |= {"q": (torch.randn(shape, generator=gen, device="cuda") * 2).to(kind), "scale": d ** -0.5,
                  "out": torch.empty(shape, device="cuda", dtype=kind), "weights": None}
        if case["weights"]:
            state["weights"] = torch.rand(b, hk, slots, generator=gen, device="cuda")
        return state
    # Summed attention weights: most positions got little, a few a great deal.
    w = torch.randn(b, hk, slots, generator=gen, device="cuda").mul_(2).exp_()
    return state | {"weights": w, "recent": case["recent"], "sinks": case["sinks"],
                    "kept": torch.empty(b, hk, case["budget"], device="cuda", dtype=torch.int32),
                    "new_lens": torch.empty_like(lens), "new_weights": torch.empty_like(w)}


# ------------------------------------------------------------------------------------------------ one pass


def _cache(state):
    """The framework's handle of the cache, made once as a program does."""
    from nightrun_b200 import kernels

    if "kv" not in state:
        state["kv"] = kernels.PagedKV(state["k_pages"], state["v_pages"], state["table"])
    return state["kv"]


def _own_rope(s):
    from nightrun_b200 import kernels

    kernels.rope_append(s["q_out"], s["q"], s["k"], s["v"], _cache(s), s["freqs"], s["pos"], s["seq"], s["slot"],
                        s["style"], mscale=s["mscale"])
    return s["q_out"], s["k_pages"], s["v_pages"]


def _own_attn(s):
    from nightrun_b200 import kernels

    if "workspace" not in s:
        s["workspace"] = kernels.attn_paged_workspace(s["q"], _cache(s), weights=s["weights"] is not None)
    kernels.attn_paged(s["out"], s["q"], _cache(s), s["lens"], s["scale"], weights=s["weights"], workspace=s["workspace"])
    return s["out"], s["weights"]


def _own_evict(s):
    from nightrun_b200 import kernels

    kernels.evict(s["kept"], s["new_lens"], s["new_weights"], _cache(s), s["lens"], s["weights"], s["recent"], s["sinks"])
    return s["kept"], s["new_lens"], s["new_weights"], s["k_pages"], s["v_pages"]


def _own_verify(s):
    from nightrun_b200 import kernels

    kernels.verify_draft(s["tokens"], s["accepted"], s["p"], s["q"], s["draft"], s["u"], s["n_draft"])
    return s["tokens"], s["accepted"]


def _rows(s, slot):
    """The row of each sequence's cached positions `slot` in the pages seen as [rows, heads, width]."""
    page = s["k_pages"].shape[1]
    return torch.gather(s["table"].long(), 1, slot // page) * page + slot % page


def _plain_rope(s):
    style, half = s["style"], s["freqs"].numel()
    angle = s["pos"].double()[:, None] * s["freqs"].double()
    cos, sin = ((f(angle) * s["mscale"]).float()[:, None] for f in (torch.cos, torch.sin))

    def turn(x):
        x = x.float()
        r, rest = x[..., :2 * half], x[..., 2 * half:]
        a, b = (r[..., 0::2], r[..., 1::2]) if style == 0 else (r[..., :half], r[..., half:])
        a, b = a * cos - b * sin, a * sin + b * cos
        return torch.cat([torch.stack([a, b], -1).flatten(-2) if style == 0 else torch.cat([a, b], -1), rest], -1)

    page = s["k_pages"].shape[1]
    at = s["slot"].long()
    row = s["table"].long()[s["seq"].long(), at // page] * page + at % page
    s["q_out"].copy_(turn(s["q"]))
    s["k_pages"].flatten(0, 1)[row] = turn(s["k"]).to(s["k_pages"].dtype)
    s["v_pages"].flatten(0, 1)[row] = s["v"].to(s["v_pages"].dtype)
    return s["q_out"], s["k_pages"], s["v_pages"]


def _plain_attn(s):
    b, n, hq, d = s["q"].shape
    hk = s["k_pages"].shape[2]
    k, v = (x[s["table"].long()].flatten(1, 2).float() for x in (s["k_pages"], s["v_pages"]))
    slots = k.shape[1]
    q = s["q"].float().view(b, n, hk, hq // hk, d).permute(0, 2, 1, 3, 4).reshape(b, hk, -1, d)
    x = torch.matmul(q, k.permute(0, 2, 3, 1)) * s["scale"]
    x = x.view(b, hk, n, hq // hk, slots)
    sees = s["lens"].long()[:, None] - (n - 1) + torch.arange(n, device=q.device)
    mask = torch.arange(slots, device=q.device) < sees[..., None]
    x = torch.where(mask[:, None, :, None], x, -torch.inf)
    e = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min))
    total = e.sum(-1, keepdim=True)
    e = e / torch.where(total > 0, total, 1.0)
    out = torch.matmul(e.view(b, hk, -1, slots), v.permute(0, 2, 1, 3))
    s["out"].copy_(out.view(b, hk, n, hq // hk, d).permute(0, 2, 1, 3, 4).reshape(b, n, hq, d))
    if s["weights"] is not None:
        s["weights"] += e.sum((2, 3))
    return s["out"], s["weights"]


def _plain_evict(s):
    b, hk, budget = s["kept"].shape
    slots = s["weights"].shape[2]
    at = torch.arange(slots, device=s["kept"].device)
    n = s["lens"].long()[:, None]
    must = (at < s["sinks"]) | (at >= n - s["recent"])
    w = torch.where(must[:, None], torch.inf, s["weights"])
    w = torch.where((at < n)[:, None], w, -torch.inf)
    best = torch.sort(w, dim=-1, descending=True, stable=True).indices[..., :budget]
    some = torch.arange(budget, device=at.device) < n  # [b, budget]
    best = torch.sort(torch.where(some[:, None], best, slots), dim=-1).values
    s["kept"].copy_(torch.where(some[:, None], best, -1))
    s["new_lens"].copy_(n[:, 0].clamp(max=budget))
    best = best.clamp(max=slots - 1)
    s["new_weights"].zero_()
    s["new_weights"][..., :budget] = torch.where(some[:, None], torch.gather(s["weights"], 2, best), 0.0)
    head = torch.arange(hk, device=at.device)[None, :, None]
    src = _rows(s, best.flatten(1)).view(b, hk, budget)
    dst = _rows(s, torch.arange(budget, device=at.device).expand(b, budget))[:, None].expand(b, hk, budget)
    heads = head.expand(b, hk, budget)
    put = some[:, None].expand(b, hk, budget)

    def move(x):
        x = x.flatten(0, 1)
        x[dst[put], heads[put]] = x[src[put], heads[put]]

    move(s["k_pages"])
    move(s["v_pages"])
    return s["kept"], s["new_lens"], s["new_weights"], s["k_pages"], s["v_pages"]


def _plain_verify(s):
    b, n = s["draft"].shape
    v = s["p"].shape[2]
    draft = s["draft"].long()[..., None]
    px = torch.gather(s["p"][:, :n], 2, draft)[..., 0].double()
    qx = torch.gather(s["q"], 2, draft)[..., 0].double() if s["q"] is not None else 1.0
    take = (s["u"][:, :n].double() * qx < px) & (torch.arange(n, device=px.device) < s["n_draft"][:, None])
    a = torch.cumprod(take.long(), 1).sum(1)
    each = torch.arange(b, device=px.device)
    p = s["p"][each, a].double()
    refused = a < s["n_draft"]
    last = a.clamp(max=n - 1)
    if s["q"] is not None:
        q = s["q"][each, last].double()
    else:
        q = (torch.arange(v, device=px.device) == draft[each, last]).double()
    r = torch.where(refused[:, None], (p - q).clamp(min=0), p)
    r = torch.where((r.amax(1) > 0)[:, None], r, p)
    c = torch.cumsum(r, 1)
    goal = s["u"][:, n].double() * c[:, -1]
    token = (c <= goal[:, None]).sum(1)
    last_one = torch.where(r > 0, torch.arange(v, device=px.device), 0).amax(1)
    token = torch.minimum(token, last_one)
    i = torch.arange(n + 1, device=px.device)
    out = torch.cat([s["draft"].long(), torch.full((b, 1), -1, device=px.device)], 1)
    out = torch.where(i < a[:, None], out, torch.where(i == a[:, None], token[:, None], -1))
    s["tokens"].copy_(out)
    s["accepted"].copy_(a)
    return s["tokens"], s["accepted"]


def run(state):
    op = state["op"]
    if own:
        return {"rope_append": _own_rope, "attn_paged": _own_attn, "evict": _own_evict, "verify_draft": _own_verify}[op](state)
    return {"rope_append": _plain_rope, "attn_paged": _plain_attn, "evict": _plain_evict, "verify_draft": _plain_verify}[op](state)


# ------------------------------------------------------------------------------------------------ floors, 64 bits


def work(case):
    op = case["op"]
    if op == "rope_append":
        t, hq, hk, d, z = case["tokens"], case["heads"], case["kv_heads"], case["dim"], _SIZE[case["type"]]
        moved = t * (2 * hq * d * z + 2 * hk * d * z + 2 * hk * d * 2)  # q in and out, k and v in, both cached
        return {"bytes": moved + t * 12 + t * 4 + case["rot"] * 2, "flops": 3 * t * (hq + hk) * case["rot"]}
    if op == "verify_draft":
        # A row of p to draw from, and where a draft was refused (in most sequences) the row of q beside it.
        z, b, v = _SIZE[case["type"]], case["seqs"], case["vocab"]
        rows = 2 if case["sampled"] else 1
        return {"bytes": b * (rows * v * z + case["draft"] * (2 * z + 4) + (case["draft"] + 1) * 8 + 8), "flops": b * v * 2}
    lens = _lengths(case)
    hk, d = case["kv_heads"], case["dim"]
    if op == "attn_paged":
        rows = case["heads"] * case["new"]
        moved = sum(lens) * hk * d * 2 * 2 + sum(-(-n // case["page"]) for n in lens) * 4
        moved += 2 * case["seqs"] * rows * d * _SIZE[case["type"]]
        if case["weights"]:
            moved += sum(lens) * hk * 8
        return {"bytes": moved, "flops": 4 * sum(lens) * rows * d}
    budget, over = case["budget"], [n for n in lens if n > case["budget"]]
    slots = -(-case["longest"] // case["page"]) * case["page"]
    moved = sum(lens) * hk * 4 + case["seqs"] * hk * (budget + slots) * 4  # weights in; kept and the new weights out
    moved += len(over) * hk * (budget - case["sinks"]) * d * 2 * 2 * 2  # rows of K and V in and out
    return {"bytes": moved, "flops": sum(lens) * hk}


def exact(case, seed):
    """What run() returns, from the definitions, in 64 bits, sequence by sequence."""

    def rope(s):
        f = s["freqs"].double().tolist()
        ang = torch.stack([s["pos"].double() * x for x in f], -1)
        z = torch.polar(torch.full_like(ang, s["mscale"]), ang)[:, None]

        def turn(x):
            x = x.double().clone()
            if s["style"] == 0:
                w = torch.complex(x[..., 0:2 * len(f):2], x[..., 1:2 * len(f):2]) * z
                x[..., 0:2 * len(f):2], x[..., 1:2 * len(f):2] = w.real, w.imag
            else:
                w = torch.complex(x[..., :len(f)], x[..., len(f):2 * len(f)]) * z
                x[..., :len(f)], x[..., len(f):2 * len(f)] = w.real, w.imag
            return x

        page = s["k_pages"].shape[1]
        k, v = s["k_pages"].double(), s["v_pages"].double()
        page_of = s["table"][s["seq"].long(), torch.div(s["slot"], page, rounding_mode="floor").long()].long()
        k[page_of, s["slot"].long() % page] = turn(s["k"])
        v[page_of, s["slot"].long() % page] = s["v"].double()
        return turn(s["q"]), k, v

    def attn(s):
        b, n, hq, d = s["q"].shape
        page, hk = s["k_pages"].shape[1:3]
        out = torch.zeros(b, n, hq, d, dtype=torch.float64, device="cuda")
        weights = None if s["weights"] is None else s["weights"].double()
        for i, length in enumerate(s["lens"].tolist()):
            ids = s["table"][i, :-(-length // page)].long()
            for h in range(hk):
                k, v = (x[ids, :, h].double().reshape(-1, d)[:length] for x in (s["k_pages"], s["v_pages"]))
                for j in range(n):
                    sees = length - (n - 1 - j)
                    if sees <= 0:
                        continue
                    heads = slice(h * (hq // hk), (h + 1) * (hq // hk))
                    p = torch.softmax(s["q"][i, j, heads].double() @ k[:sees].T * s["scale"], -1)
                    out[i, j, heads] = p @ v[:sees]
                    if weights is not None:
                        weights[i, h, :sees] += p.sum(0)
        return out, weights

    def evict(s):
        b, hk, budget = s["kept"].shape
        page = s["k_pages"].shape[1]
        kept = torch.full((b, hk, budget), -1, dtype=torch.int32)
        new_weights = torch.zeros(s["weights"].shape, dtype=torch.float64)
        w = s["weights"].double().cpu()
        k, v = s["k_pages"].clone(), s["v_pages"].clone()
        lens = s["lens"].tolist()
        for i, n in enumerate(lens):
            for h in range(hk):
                if n <= budget:
                    keep = torch.arange(n)
                else:
                    first, latest = torch.arange(s["sinks"]), torch.arange(n - s["recent"], n)
                    middle = w[i, h, s["sinks"]:n - s["recent"]]
                    more = torch.argsort(-middle, stable=True)[:budget - s["sinks"] - s["recent"]] + s["sinks"]
                    keep = torch.cat([first, more.sort().values, latest])
                kept[i, h, :len(keep)] = keep.to(torch.int32)
                new_weights[i, h, :len(keep)] = w[i, h, keep]
                src, dst = keep.cuda(), torch.arange(len(keep), device="cuda")
                ids = s["table"][i].long()
                for new, old in ((k, s["k_pages"]), (v, s["v_pages"])):
                    new[ids[dst // page], dst % page, h] = old[ids[src // page], src % page, h]
        return kept, torch.tensor([min(n, budget) for n in lens], dtype=torch.int32), new_weights, k, v

    def verify(s):
        p, u = s["p"], s["u"].double().cpu()
        b, n = s["draft"].shape
        tokens, accepted = torch.full((b, n + 1), -1, dtype=torch.int32), torch.zeros(b, dtype=torch.int32)
        for i in range(b):
            a, most = 0, int(s["n_draft"][i])
            while a < most:
                x = int(s["draft"][i, a])
                chance = 1.0 if s["q"] is None else float(s["q"][i, a, x])
                if not float(u[i, a]) * chance < float(p[i, a, x]):
                    break
                tokens[i, a] = x
                a += 1
            row = p[i, a].double().cpu()
            left = row.clone()
            if a < most:
                if s["q"] is None:
                    left[int(s["draft"][i, a])] -= 1
                else:
                    left -= s["q"][i, a].double().cpu()
                left.clamp_(min=0)
                if not bool((left > 0).any()):
                    left = row
            c = torch.cumsum(left, 0)
            at = int(torch.searchsorted(c, float(u[i, n]) * float(c[-1]), right=True))
            tokens[i, a] = min(at, int(torch.nonzero(left > 0).max()))
            accepted[i] = a
        return tokens, accepted

    s = prepare(case, seed)
    return {"rope_append": rope, "attn_paged": attn, "evict": evict, "verify_draft": verify}[case["op"]](s)
