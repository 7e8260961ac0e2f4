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
