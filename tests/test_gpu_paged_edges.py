"""Edges of the operators over a paged KV cache: long pieces of work with weights, infinities and NaN in the cache,
overlapping tensors, goals on the border of a running sum. Definitions in 64 bits as in tests/pagedref.py, or taken on the
GPU where they are large."""
import pytest
import torch

from nightrun_b200._lib import NrcError
from tests import pagedref as R

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
INF, NAN = float("inf"), float("nan")


@pytest.fixture(scope="module")
def K():
    from nightrun_b200 import kernels
    return kernels


@pytest.fixture(autouse=True)
def no_device_error(K):
    yield
    K.sync_check()


def gen(seed, device="cpu"):
    return torch.Generator(device).manual_seed(seed)


# ------------------------------------------------------------------ weights of long pieces

LONG = [  # sequences, shortest, longest, new, heads, kv heads, dim, type, cache, page
    (24, 1000, 9001, 5, 40, 8, 64, F32, F16, 24),     # 25 rows, tiles of 120
    (28, 700, 8189, 7, 40, 8, 64, F16, F16, 16),      # 35 rows: two row blocks one after the other
    (24, 2001, 7003, 3, 32, 8, 64, BF16, BF16, 64),
    (12, 3000, 9999, 4, 32, 8, 128, F32, BF16, 32)]


@pytest.mark.parametrize("seqs,shortest,longest,new,hq,hk,d,dt,ct,page", LONG, ids=[str(i) for i in range(len(LONG))])
def test_weights_of_long_pieces(K, seqs, shortest, longest, new, hq, hk, d, dt, ct, page):
    """Blocks of the tcgen05 kernel with dozens of tiles per piece of work and ends that cut a tile: every position's
    weight, the same bits in every call."""
    g = gen(seqs + new, "cuda")
    lens = torch.linspace(shortest, longest, seqs, device="cuda").int()
    per = -(-longest // page)
    n = seqs * per + 3
    k, v = (torch.randn(n, page, hk, d, generator=g, device="cuda").to(ct) for _ in range(2))
    table = torch.randperm(n, generator=g, device="cuda")[:seqs * per].view(seqs, per).int()
    q = (torch.randn(seqs, new, hq, d, generator=g, device="cuda") * 1.5).to(dt)
    w0 = torch.rand(seqs, hk, per * page, generator=g, device="cuda")
    kv = K.PagedKV(k, v, table)
    out, ws = torch.empty_like(q), K.attn_paged_workspace(q, kv, weights=True)
    first = None
    for _ in range(6):
        w = w0.clone()
        K.attn_paged(out, q, kv, lens, d ** -0.5, weights=w, workspace=ws)
        if first is None:
            first = w, out.clone()
        assert torch.equal(w, first[0]) and torch.equal(out, first[1])
    rows = new * hq // hk
    for s in range(seqs):
        m = int(lens[s])
        keys = k[table[s].long()].flatten(0, 1)[:m].double()
        qs = q[s].double().view(new, hk, hq // hk, d)
        x = torch.einsum("nhgd,lhd->hngl", qs, keys) * d ** -0.5
        big = (torch.einsum("nhgd,lhd->hngl", qs.abs(), keys.abs()).amax() * d ** -0.5).item()
        seen = torch.arange(m, device="cuda") < m - (new - 1) + torch.arange(new, device="cuda")[:, None]
        want = x.masked_fill(~seen[:, None], -INF).softmax(-1).sum((1, 2))
        # Scores as in R.attention_tolerance; the sum they are divided by and the row's own weight each follow them; the
        # exponentials; f32 sums of up to `m` and of `rows` values.
        delta = big * (2.0 ** -22 + (3 * d / 16 + 4) * 2.0 ** -23)
        rel = 2.2 * delta + 2.0 ** -20 + (3 * m / 16 + 40) * 2.0 ** -23 + rows * 2.0 ** -24
        whole = w0[s, :, :m].double() + want
        assert bool(((first[0][s, :, :m].double() - whole).abs() <= want * rel + whole * 2.0 ** -23).all())
        assert torch.equal(first[0][s, :, m:], w0[s, :, m:])


# ------------------------------------------------------------------ errors


def test_errors_of_several_kernels_are_all_reported(K):
    """A page outside the pool and a slot outside the table, then a wait that runs out: one report names all three."""
    from nightrun_b200._lib import lib
    k, v, table = R.make_pages(gen(1), 2, 2, 4, 1, 32, F16)
    table[0, 1] = 10 ** 6
    kv = K.PagedKV(k.cuda(), v.cuda(), table.cuda())
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    x, freqs = torch.zeros(2, 1, 32, device="cuda"), torch.tensor(K.rope_freqs(32, 10000.0), device="cuda")
    K.rope_append(x, x, x.clone(), x.clone(), kv, freqs, i32(0, 1), i32(0, 1), i32(4, 8))
    assert lib().nrc_wait_selftest(0, 20_000_000, None) == -4
    message = lib().nrc_last_error().decode()
    assert "wait expired" in message and "page id" in message and "slot" in message
    K.sync_check()  # reported once


# ------------------------------------------------------------------ infinities and NaN in the cache


def expected(q, k_pages, v_pages, table, lens, scale):
    """out, weights and their tolerances, in 64 bits and by IEEE's rules: a score of -inf has weight 0, one of +inf or NaN
    leaves NaN in its row, an infinite value at a position of weight above 0 is the output's.

    Scores: d products, summed in f32 one after the other at worst, (d + 8) 2^-24 of the sum of magnitudes, and operands
    that hold 2^-22 of theirs. Weights enter in two parts of the cache's type at least: two roundings of 2^-11 or 2^-8, and
    f16's smallest step, 2^-25 off where the row's sum is 2^8 or more. Sums as in R.attention_tolerance, but that tcgen05 adds
    128 tile sums of 16-bit calls, cut by 2^-23 each, before one to nearest: 2^-16."""
    b, n, hq, d = q.shape
    hk, slots = k_pages.shape[2], table.shape[1] * k_pages.shape[1]
    g = hq // hk
    out, tol = torch.zeros(b, n, hq, d, dtype=torch.float64), torch.zeros(b, n, hq, d, dtype=torch.float64)
    weights, wtol = torch.zeros(b, hk, slots, dtype=torch.float64), torch.zeros(b, hk, slots, dtype=torch.float64)
    enter = 2.0 ** -22 if q.dtype == F32 or k_pages.dtype == F16 else 2.0 ** -16  # f32: three parts over bf16; else two
    for s in range(b):
        m = int(lens[s])
        keys, values = (R.rows(x, table, s, range(m)).double() for x in (k_pages, v_pages))
        for j in range(n):
            sees = m - (n - 1 - j)
            if sees <= 0:
                continue
            for h in range(hq):
                kk, vv, qq = keys[:sees, h // g], values[:sees, h // g], q[s, j, h].double()
                x = (kk * qq).sum(1) * scale
                p = torch.softmax(x, 0)
                out[s, j, h] = (p[:, None] * vv).sum(0)
                big = ((kk * qq).abs().sum(1) * abs(scale)).nan_to_num(0.0, 0.0, 0.0).max()
                delta = big * ((d + 8) * 2.0 ** -24 + 2.0 ** -22)
                sums = (3 * sees / 16 + 40) * 2.0 ** -23
                size = (p[:, None] * vv.abs()).nan_to_num(0.0, 0.0, 0.0).sum(0)
                enters = enter + sees * 2.0 ** -33 + (0 if q.dtype == F32 else 2.0 ** -16)
                tol[s, j, h] = (size * (2.2 * delta + enters + 2.0 ** -20 + 2 * sums)
                                + out[s, j, h].abs().nan_to_num(0.0, 0.0, 0.0) * R.HALF[q.dtype] + R.TINY[q.dtype])
                weights[s, h // g, :sees] += p
                wtol[s, h // g, :sees] += p * (2.2 * delta + 2.0 ** -20 + sums + 2.0 ** -21)
    return out, tol, weights, wtol


def same(got, want, tol):
    """Finite where `want` is and within `tol` there, the same infinities, NaN where NaN."""
    got = got.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    at = torch.isinf(want)
    assert torch.equal(torch.isinf(got), at) and torch.equal(got[at], want[at])
    fine = torch.isfinite(want)
    assert bool(((got - want).abs()[fine] <= tol[fine]).all())


ODD = [  # lens, new, heads, kv heads, dim, type, cache, page
    ([70, 48], 1, 8, 2, 64, F16, F16, 16), ([70, 48], 1, 8, 2, 64, F32, F16, 16),         # unsplit; 4 of 8 columns
    ([700, 301], 1, 10, 2, 128, BF16, BF16, 16), ([700, 301], 1, 8, 2, 128, F32, BF16, 7),  # split and joined
    ([400], 3, 8, 2, 96, F16, BF16, 24), ([333, 90], 3, 6, 2, 32, F32, F16, 9),             # 12 and 9 rows off tcgen05
    ([700, 513], 3, 8, 2, 64, F32, F16, 16), ([640, 300], 4, 6, 2, 64, F16, F16, 24),       # tcgen05
    ([700, 400], 3, 8, 2, 128, F16, BF16, 64), ([650], 4, 20, 2, 128, BF16, BF16, 32)]


def odd_case(K, case, seed):
    lens, new, hq, hk, d, dt, ct, page = case
    g = gen(seed)
    k, v, table = R.make_pages(g, len(lens), -(-max(lens) // page) + 1, page, hk, d, ct)
    q = torch.randn(len(lens), new, hq, d, generator=g).to(dt)
    return q, k, v, table, torch.tensor(lens, dtype=torch.int32)


def run_odd(K, q, k, v, table, lens, scale):
    kv = K.PagedKV(k.cuda(), v.cuda(), table.cuda())
    w = torch.zeros(len(lens), k.shape[2], table.shape[1] * k.shape[1], device="cuda")
    out = torch.empty_like(q, device="cuda")
    K.attn_paged(out, q.cuda(), kv, lens.cuda(), scale, weights=w)
    alone = torch.empty_like(out)
    K.attn_paged(alone, q.cuda(), kv, lens.cuda(), scale)
    assert torch.equal(alone.isnan(), out.isnan()) and torch.equal(alone.nan_to_num(7.0), out.nan_to_num(7.0))
    return out, w


FINE = [c for c in ODD if c[5] != F32] + [
    ([2, 3, 5], 1, 8, 2, 64, F16, F16, 16), ([2, 3, 5], 1, 8, 2, 128, BF16, BF16, 16), ([900, 40], 1, 8, 2, 64, BF16, F16, 16),
    ([900, 40], 1, 24, 2, 64, BF16, BF16, 7), ([500, 333], 5, 8, 2, 64, BF16, BF16, 16), ([500, 333], 5, 8, 2, 128, F16, F16, 16)]


@pytest.mark.parametrize("case", FINE, ids=[str(i) for i in range(len(FINE))])
def test_16_bit_outputs_are_rounded_once(K, case):
    """16-bit outputs against 64 bits: the output's own rounding, and next to it only what two parts of a weight leave (one
    part would add a rounding of the cache's type to every weight)."""
    q, k, v, table, lens = odd_case(K, case, 35)
    want, tol, ww, wtol = expected(q, k, v, table, lens, 0.3)
    out, w = run_odd(K, q, k, v, table, lens, 0.3)
    same(out, want, tol)
    same(w, ww, wtol + 1e-30)


@pytest.mark.parametrize("case", ODD, ids=[str(i) for i in range(len(ODD))])
def test_infinite_keys_that_count_for_nothing(K, case):
    """Keys that are infinite where every query is below zero: their scores are -inf, their weights 0, and nothing else
    changes, whatever columns of a tile are no rows."""
    q, k, v, table, lens = odd_case(K, case, 31)
    q[..., 5] = -q[..., 5].abs().clamp(min=0.01)
    for s, n in enumerate(lens.tolist()):
        for t in (0, 17, n // 2, n - 1):
            row = R.rows(k, table, s, [t])[0].clone()
            row[:, 5] = INF
            R.put(k, table, s, t, row)
    want, tol, ww, wtol = expected(q, k, v, table, lens, 0.2)
    assert torch.isfinite(want).all() and torch.isfinite(ww).all()
    out, w = run_odd(K, q, k, v, table, lens, 0.2)
    same(w, ww, wtol + 1e-30)
    same(out, want, tol)


@pytest.mark.parametrize("case", ODD, ids=[str(i) for i in range(len(ODD))])
def test_infinite_values_are_the_outputs(K, case):
    """Infinite values, some at positions whose weight is far below a 16-bit number's: infinite outputs in their places, NaN
    where both signs meet, everything else as it was; the weights do not change. One infinity is at the last position,
    which only the last new token sees."""
    q, k, v, table, lens = odd_case(K, case, 32)
    for s, n in enumerate(lens.tolist()):
        far = n // 2  # a key against the queries: a weight of about e^-40
        mean = q[s].double().mean((0, 1))
        R.put(k, table, s, far, (-mean / mean.norm() * 3).to(k.dtype).expand(k.shape[2], -1))
        for t, at, x in ((3, 1, INF), (n // 3, 7, -INF), (far, 11, INF), (5, 20, INF), (n // 4, 20, -INF), (n - 1, 30, -INF),
                         (n // 5, 9, NAN)):
            row = R.rows(v, table, s, [t])[0].clone()
            row[:, at] = x
            R.put(v, table, s, t, row)
    want, tol, ww, wtol = expected(q, k, v, table, lens, 0.3)
    out, w = run_odd(K, q, k, v, table, lens, 0.3)
    same(w, ww, wtol + 1e-30)
    same(out, want, tol)


@pytest.mark.parametrize("case", ODD, ids=[str(i) for i in range(len(ODD))])
def test_infinite_and_nan_keys_reach_their_rows_only(K, case):
    """Keys of both signs of infinity and NaN: the rows that see a score of +inf or NaN are NaN, those of the other KV head,
    the other sequence and the tokens before are not."""
    q, k, v, table, lens = odd_case(K, case, 33)
    n = int(lens[0])
    for t, at, x in ((n - 2, 3, INF), (n - 1, 4, NAN), (n // 2, 6, -INF)):
        row = R.rows(k, table, 0, [t])[0].clone()
        row[1, at] = x
        R.put(k, table, 0, t, row)
    q[0, 0, :, 6] = q[0, 0, :, 6].abs() + 0.01  # the first token's scores at n // 2 are -inf
    want, tol, ww, wtol = expected(q, k, v, table, lens, 0.2)
    out, w = run_odd(K, q, k, v, table, lens, 0.2)
    same(out, want, tol)
    same(w, ww, wtol + 1e-30)


@pytest.mark.parametrize("case", [ODD[1], ODD[5], ODD[6], ODD[8]], ids=["unsplit", "mma", "tcgen05 64", "tcgen05 128"])
def test_scores_of_minus_infinity_count_alike_everywhere(K, case):
    """A score of -inf among the newest positions, which only some tokens see, as anywhere else: 0 times an infinite value is
    NaN, and in a row that is NaN the position's weight is too."""
    q, k, v, table, lens = odd_case(K, case, 36)
    q[..., 5] = -q[..., 5].abs().clamp(min=0.01)
    for s, n in enumerate(lens.tolist()):
        for t in (n - 2, n // 2):
            row = R.rows(k, table, s, [t])[0].clone()
            row[:, 5] = INF
            R.put(k, table, s, t, row)
        row = R.rows(v, table, s, [n - 2])[0].clone()
        row[0, 9] = INF
        R.put(v, table, s, n - 2, row)
        row = R.rows(k, table, s, [3])[0].clone()
        row[1, 7] = NAN
        R.put(k, table, s, 3, row)
    want, tol, ww, wtol = expected(q, k, v, table, lens, 0.2)
    out, w = run_odd(K, q, k, v, table, lens, 0.2)
    same(out, want, tol)
    same(w, ww, wtol + 1e-30)


@pytest.mark.parametrize("case", ODD, ids=[str(i) for i in range(len(ODD))])
def test_rows_of_nothing_but_minus_infinity_get_zeros(K, case):
    """Every score of a KV head's rows is -inf: zeros, as where a row sees nothing, and no weight."""
    q, k, v, table, lens = odd_case(K, case, 37)
    g = q.shape[2] // k.shape[2]
    q[:, :, :g, 5] = -q[:, :, :g, 5].abs().clamp(min=0.01)
    k[:, :, 0, 5] = INF
    out, w = run_odd(K, q, k, v, table, lens, 0.2)
    assert not out[:, :, :g].any() and not w[:, 0].any()
    want, tol, ww, wtol = expected(q, k, v, table, lens, 0.2)
    same(out[:, :, g:], want[:, :, g:], tol[:, :, g:])
    same(w[:, 1:], ww[:, 1:], wtol[:, 1:] + 1e-30)


@pytest.mark.parametrize("case", [ODD[1], ODD[6]], ids=["few", "many"])
def test_nan_queries_reach_their_rows_only(K, case):
    q, k, v, table, lens = odd_case(K, case, 34)
    q[0, 0, 1, 9] = NAN
    want, tol, ww, wtol = expected(q, k, v, table, lens, 0.2)
    out, w = run_odd(K, q, k, v, table, lens, 0.2)
    same(out, want, tol)
    same(w, ww, wtol + 1e-30)


# ------------------------------------------------------------------ drawn tokens


@pytest.mark.parametrize("seqs", [16, 64])
def test_drawn_tokens_hold_something_where_the_goal_meets_a_sum(K, seqs):
    """The two halves of a row hold the same values in another order, spread over 70 binary orders, and u is a half: the goal
    lies within a rounding of the sum over the first half, and zeros follow there. The drawn token has a probability, and
    the sums before it and with it enclose the goal up to the roundings of 64-bit sums of 128 values (128 halves of a step)."""
    import math

    import numpy as np
    vocab, drawn = 65536, 0
    tokens, accepted = (torch.empty(seqs, *x, dtype=torch.int32, device="cuda") for x in ((1,), ()))
    draft, u = torch.empty(seqs, 0, dtype=torch.int32, device="cuda"), torch.full((seqs, 1), 0.5, device="cuda")
    for seed in range(384 // seqs):
        r = np.random.default_rng(seed)
        rows = np.zeros((seqs, 1, vocab), np.float32)
        for s in range(seqs):
            h = (r.random(64) * 2.0 ** -r.integers(0, 70, 64)).astype(np.float32)
            w = r.permutation(h)
            if s % 2:
                w = np.concatenate([np.zeros(2, np.float32), np.delete(w, np.argsort(w)[:2])])
            rows[s, 0, 511::512] = np.concatenate([h, w])
        K.verify_draft(tokens, accepted, torch.from_numpy(rows).cuda(), None, draft, u)
        for s, t in enumerate(tokens[:, 0].tolist()):
            row = rows[s, 0].astype(np.float64)[511::512]
            assert rows[s, 0, t] > 0, (seed, s, t)
            i, goal = t // 512, math.fsum(row) / 2
            slack = 128 * 2.0 ** -53 * math.fsum(row)
            assert math.fsum(row[:i]) <= goal + slack and math.fsum(row[:i + 1]) >= goal - slack
            drawn += 1
    assert drawn == 384 and not accepted.any()


def test_draft_probabilities_below_every_number_count_as_nothing(K):
    """A draft distribution that holds -inf or NaN at a token: nothing is left there, as with any infinity."""
    vocab = 3000
    p = torch.zeros(3, 2, vocab)
    p[:, 0, 100:200] = 0.01
    q = torch.zeros(3, 1, vocab)
    q[:, 0, 7], q[0, 0, 150], q[1, 0, 2000], q[2, 0, 150] = 1.0, -INF, -INF, NAN
    tokens, accepted = torch.empty(3, 2, dtype=torch.int32, device="cuda"), torch.empty(3, dtype=torch.int32, device="cuda")
    u = torch.tensor([[0.5, 0.501], [0.5, 0.501], [0.5, 0.501]])
    K.verify_draft(tokens, accepted, p.cuda(), q.cuda(), torch.full((3, 1), 7, dtype=torch.int32, device="cuda"), u.cuda())
    # What is left: 100 tokens of 0.01 less the odd one; the goal 0.501 of the sum lies in the 50th or the 51st of them.
    assert accepted.tolist() == [0, 0, 0] and tokens.tolist() == [[149, -1], [150, -1], [149, -1]]


# ------------------------------------------------------------------ tensors beside one another


def test_interleaved_and_in_place_tensors(K):
    """What lies between one another's rows without touching them is taken, and so are the in-place forms: q, k, v and q's
    output in one projection, queries and outputs in alternate rows, K's and V's pages in turn, drafts in the tokens' place."""
    g = gen(3)
    hq, hk, d, page = 4, 2, 64, 8
    lens = torch.tensor([33, 20], dtype=torch.int32)
    both = torch.randn(12, 2, page, hk, d, generator=g).to(F16)
    table = torch.randperm(12, generator=g)[:10].view(2, 5).int()
    gb = both.cuda()
    kv = K.PagedKV(gb[:, 0], gb[:, 1], table.cuda())
    x = torch.randn(2, hq + 2 * hk, d, generator=g)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    freqs = torch.tensor(K.rope_freqs(d, 10000.0), device="cuda")
    gx = x.cuda()
    K.rope_append(gx[:, :hq], gx[:, :hq], gx[:, hq:hq + hk], gx[:, hq + hk:], kv, freqs, i32(32, 19), i32(0, 1), i32(32, 19))
    pos = torch.tensor([32, 19])
    want = R.rope(x[:, :hq], pos, freqs.cpu(), 1, 1.0)
    assert bool(((gx[:, :hq].double().cpu() - want).abs() <= R.rope_tolerance(x[:, :hq], freqs.cpu(), 1, 1.0, F32, want)).all())
    assert torch.equal(gx[:, hq:].cpu(), x[:, hq:])
    both = gb.cpu()
    for s, t in ((0, 32), (1, 19)):
        assert torch.equal(R.rows(both[:, 1], table, s, [t])[0], x[s, hq + hk:].to(F16))
    pair = torch.zeros(2, 1, hq, 2, d, device="cuda")  # a head's queries, then its output
    pair[:, :, :, 0] = gx[:, None, :hq]
    K.attn_paged(pair[:, :, :, 1], pair[:, :, :, 0], kv, lens.cuda(), 0.125)
    want, _, size, big = R.attention(gx[:, None, :hq].cpu(), both[:, 0], both[:, 1], table, lens, 0.125)
    tol, _ = R.attention_tolerance(F32, F16, d, 33, size, big, want)
    assert bool(((pair[:, :, :, 1].double().cpu() - want).abs() <= tol).all())
    p = torch.rand(1, 4, 500, generator=g)
    q, u = torch.rand(1, 3, 500, generator=g), torch.rand(1, 4, generator=g)
    draft = torch.randint(0, 500, (1, 3), generator=g, dtype=torch.int32)
    tokens = torch.cat([draft, draft[:, :1]], 1).cuda()
    number = i32(2)
    K.verify_draft(tokens, number, p.cuda(), q.cuda(), tokens[:, :3], u.cuda(), number)
    want_t, want_a = R.verify(p, q, draft, u, torch.tensor([2]))
    assert torch.equal(tokens.cpu(), want_t) and torch.equal(number.cpu(), want_a)
    shifted = gb.view(-1).as_strided((11, page, hk, d), gb[:, 0].stride(), 8)  # V's rows 16 bytes behind K's
    one_pool = K.PagedKV(gb[:11, 0], shifted, table.cuda() % 11)
    with pytest.raises(NrcError):
        K.rope_append(gx[:, :hq], gx[:, :hq], gx[:, hq:hq + hk], gx[:, hq + hk:], one_pool, freqs, i32(1, 1), i32(0, 1), i32(1, 1))
    with pytest.raises(NrcError):
        K.PagedKV(*(gb[:, i].as_strided(gb[:, i].shape, (gb.stride(0), gb.stride(2), 32, 1)) for i in (0, 1)), table.cuda())
