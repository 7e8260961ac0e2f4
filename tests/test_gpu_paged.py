"""The operators over a paged KV cache against their 64-bit definitions
(tests/pagedref.py): sizes and masks where each can go wrong, then the calls
that a serving loop makes of them together, captured and replayed too."""
import pytest
import torch

from nightrun_b200._lib import NrcError
from tests import pagedref as R

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
NAN = float("nan")


@pytest.fixture(scope="module")
def K():
    from nightrun_b200 import kernels
    return kernels


@pytest.fixture(autouse=True)
def no_device_error(K):
    yield
    K.sync_check()


def gen(seed):
    return torch.Generator().manual_seed(seed)


def cuda_kv(K, k, v, table):
    return K.PagedKV(k.cuda(), v.cuda(), table.cuda())


def worst(got, want, tol):
    """The largest error in units of its tolerance."""
    d = (got.double().cpu() - want).abs()
    assert torch.equal(torch.isfinite(got).cpu(), torch.isfinite(want))
    return float((d / tol.clamp(min=1e-300)).nan_to_num(0.0).max()) if d.numel() else 0.0


# ------------------------------------------------------------------ rope_append

ROPE = [  # tokens, heads, kv heads, dim, rot, style, type, cache, page
    (1, 32, 8, 64, 64, 0, F32, F16, 16), (1, 4, 2, 128, 128, 1, F16, F16, 1), (7, 3, 1, 32, 32, 1, BF16, BF16, 5),
    (33, 5, 5, 96, 72, 0, F32, BF16, 24), (200, 32, 8, 128, 32, 1, BF16, BF16, 64), (65, 40, 8, 64, 20, 1, F16, F16, 7),
    (19, 4, 2, 64, 2, 0, F16, BF16, 16), (12, 4, 2, 64, 0, 1, F32, F16, 16), (513, 2, 1, 128, 96, 1, F32, F16, 16),
    (9, 6, 3, 96, 6, 1, BF16, F16, 3)]


@pytest.mark.parametrize("tokens,hq,hk,d,rot,style,dt,ct,page", ROPE, ids=[str(i) for i in range(len(ROPE))])
def test_rope_append(K, tokens, hq, hk, d, rot, style, dt, ct, page):
    g = gen(tokens)
    seqs = 1 + tokens // 9
    k_pages, v_pages, table = R.make_pages(g, seqs, -(-(12 + 9) // page) + 2, page, hk, d, ct)
    qkv = torch.randn(tokens, hq + 2 * hk, d, generator=g).to(dt)
    seq = (torch.arange(tokens) // 9).to(torch.int32)
    slot = (torch.arange(tokens) % 9 + 3 * (seq % 3)).to(torch.int32)
    slot[tokens // 2] = -1  # a padding token: its q turns, nothing is cached
    pos = (slot + 1000003 * (seq % 5)).clamp(min=0).to(torch.int32)
    freqs = torch.tensor(K.rope_freqs(rot, 500000.0, (32.0, 1.0, 4.0, 8192.0)) if rot else [], dtype=F32)
    mscale = 1.25 if rot % 3 == 0 else 1.0
    x = qkv.cuda()
    kv = cuda_kv(K, k_pages, v_pages, table)
    out = torch.empty(tokens, hq, d, dtype=dt, device="cuda")
    K.rope_append(out, x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:], kv, freqs.cuda(), pos.cuda(), seq.cuda(), slot.cuda(),
                  style, mscale)
    want = R.rope(qkv[:, :hq], pos, freqs, style, mscale)
    assert worst(out, want, R.rope_tolerance(qkv[:, :hq], freqs, style, mscale, dt, want)) <= 1
    kx, vx = qkv[:, hq:hq + hk], qkv[:, hq + hk:]
    want_k = R.rope(kx, pos, freqs, style, mscale)
    tol = R.rope_tolerance(kx, freqs, style, mscale, ct, want_k)
    got_k, got_v = kv.k_pages.cpu(), kv.v_pages.cpu()
    seen_k, seen_v = k_pages.clone(), v_pages.clone()
    for t in range(tokens):
        if slot[t] < 0:
            continue
        at = (int(table[seq[t], slot[t] // page]), int(slot[t]) % page)
        assert worst(got_k[at], want_k[t], tol[t]) <= 1
        assert torch.equal(got_v[at], vx[t].to(ct))
        seen_k[at], seen_v[at] = got_k[at], got_v[at]
    assert torch.equal(got_k, seen_k) and torch.equal(got_v, seen_v)  # every other row as it was
    # In place, and from contiguous heads: the same bits.
    q2, k2, v2 = (t.contiguous() for t in (x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:]))
    kv2 = cuda_kv(K, k_pages, v_pages, table)
    K.rope_append(q2, q2, k2, v2, kv2, freqs.cuda(), pos.cuda(), seq.cuda(), slot.cuda(), style, mscale)
    assert torch.equal(q2, out) and torch.equal(kv2.k_pages, kv.k_pages) and torch.equal(kv2.v_pages, kv.v_pages)


def test_rope_append_odd_strides(K):
    """Heads behind one another per token, a head stride that is no multiple of 16 bytes, a shifted base."""
    g = gen(5)
    tokens, hq, hk, d, page = 11, 3, 2, 64, 4
    k_pages, v_pages, table = R.make_pages(g, 1, 4, page, hk, d, F16)
    flat = torch.randn(1 + hq * tokens * (d + 3), generator=g).to(F16)
    q = flat[1:].view(hq, tokens, d + 3)[:, :, :d].transpose(0, 1)
    kvx = torch.randn(tokens, hk, d + 1, generator=g).to(F16)[..., :d]
    pos = torch.arange(tokens, dtype=torch.int32) + 5
    seq, slot = torch.zeros(tokens, dtype=torch.int32), torch.arange(tokens, dtype=torch.int32)
    freqs = torch.tensor(K.rope_freqs(d, 10000.0), dtype=F32)
    gq = flat.cuda()[1:].view(hq, tokens, d + 3)[:, :, :d].transpose(0, 1)
    gkv = torch.randn(tokens, hk, d + 1).cuda().to(F16)[..., :d].copy_(kvx.cuda())
    for style in (0, 1):
        kv = cuda_kv(K, k_pages, v_pages, table)
        out = torch.zeros(hq, tokens, d + 5, dtype=F16, device="cuda")[:, :, :d].transpose(0, 1)
        K.rope_append(out, gq, gkv, gkv, kv, freqs.cuda(), pos.cuda(), seq.cuda(), slot.cuda(), style)
        want = R.rope(q, pos, freqs, style, 1.0)
        assert worst(out, want, R.rope_tolerance(q, freqs, style, 1.0, F16, want)) <= 1
        got = R.rows(kv.v_pages.cpu(), table, 0, range(tokens))
        assert torch.equal(got, kvx)


def test_rope_append_bad_slots_are_reported(K):
    g = gen(6)
    k_pages, v_pages, table = R.make_pages(g, 2, 2, 4, 1, 32, F16)
    table[1, 1] = 10 ** 6  # outside the pool
    x = torch.randn(4, 1, 32, generator=g)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    freqs = torch.tensor(K.rope_freqs(32, 10000.0), dtype=F32, device="cuda")
    for seq, slot in ((i32(0, 1, 0, 2), i32(0, 1, 2, 0)), (i32(0, 1, 0, -1), i32(0, 1, 2, 0)),
                      (i32(0, 1, 0, 0), i32(0, 1, 2, 8)), (i32(0, 1, 0, 1), i32(0, 1, 2, 4))):
        kv = cuda_kv(K, k_pages, v_pages, table)
        out = torch.empty(4, 1, 32, device="cuda")
        K.rope_append(out, x.cuda(), x.cuda(), x.cuda(), kv, freqs, i32(0, 1, 2, 3), seq, slot, 1)
        with pytest.raises(NrcError) as e:
            K.sync_check()
        assert e.value.name == "DEVICE"
        K.sync_check()  # reported once
        got = kv.v_pages.cpu()
        want = v_pages.clone()
        for t in range(3):  # the good tokens are cached, nothing else is touched
            R.put(want, table, int(seq[t]), int(slot[t]), x[t].to(F16))
        assert torch.equal(got, want)


# ------------------------------------------------------------------ attn_paged

ATTN = [  # lens, new, heads, kv heads, dim, type, cache, page, weights
    ([1], 1, 32, 8, 64, F32, F16, 16, True), ([0, 1, 2, 3], 1, 4, 2, 128, F16, F16, 4, True),
    ([77, 0, 15, 16, 17], 1, 8, 2, 64, F32, F16, 16, False), ([500], 1, 5, 1, 96, BF16, BF16, 24, True),
    ([63, 64, 65, 129, 255, 256, 257], 1, 3, 3, 32, F32, BF16, 1, True), ([1000, 3], 5, 40, 8, 64, F32, F16, 24, True),
    ([4, 0, 1, 2, 3, 5], 4, 4, 2, 32, F16, BF16, 3, True), ([2000], 8, 6, 2, 128, BF16, F16, 100, True),
    ([3000, 1200, 40], 2, 9, 3, 128, F32, F16, 64, False), ([333], 64, 2, 1, 64, F16, F16, 7, True),
    ([129] * 9, 1, 16, 1, 128, F32, BF16, 32, True), ([700, 20], 3, 33, 3, 64, BF16, BF16, 48, True),
    # 9 rows and more per KV head over longer tables: the tcgen05 kernel
    ([600], 3, 8, 2, 64, F16, F16, 16, False), ([128, 129, 127, 700, 1], 4, 12, 4, 128, F16, F16, 64, True),
    ([1500, 2, 0, 515], 16, 4, 2, 64, F32, F16, 9, True), ([999], 5, 16, 4, 128, F32, BF16, 16, True),
    ([2100, 300], 2, 20, 2, 64, F16, BF16, 24, False), ([5000, 17, 640], 1, 40, 4, 128, BF16, BF16, 128, True),
    ([1300], 7, 36, 3, 128, F32, F16, 20, True),
    ([1111, 500, 64], 3, 8, 2, 64, F32, F16, 8, True), ([2000], 2, 12, 2, 128, F16, F16, 40, True),
    ([700, 480, 481], 4, 6, 2, 64, BF16, BF16, 160, False), ([900, 256], 3, 14, 2, 128, BF16, BF16, 256, True),
    ([1200], 6, 4, 2, 64, F16, F16, 56, False)]


@pytest.mark.parametrize("lens,new,hq,hk,d,dt,ct,page,weights", ATTN, ids=[str(i) for i in range(len(ATTN))])
def test_attn_paged(K, lens, new, hq, hk, d, dt, ct, page, weights):
    g = gen(len(lens) * 1000 + new)
    b = len(lens)
    # Rows behind the sequences' ends hold NaN: they must never matter.
    k_pages, v_pages, table = R.make_pages(g, b, max(1, -(-max(lens) // page)) + 1, page, hk, d, ct, bad=NAN)
    for s, n in enumerate(lens):
        kr, vr = torch.randn(n, hk, d, generator=g).to(ct), torch.randn(n, hk, d, generator=g).to(ct)
        for t in range(n):
            R.put(k_pages, table, s, t, kr[t]), R.put(v_pages, table, s, t, vr[t])
    q = (torch.randn(b, new, hq, d, generator=g) * 1.5).to(dt)
    lens_t = torch.tensor(lens, dtype=torch.int32)
    slots = table.shape[1] * page
    w0 = torch.rand(b, hk, slots, generator=g)
    want, want_w, size, big = R.attention(q, k_pages, v_pages, table, lens_t, d ** -0.5)
    tol, delta = R.attention_tolerance(dt, ct, d, max(lens), size, big, want)
    kv = cuda_kv(K, k_pages, v_pages, table)
    out = torch.full((b, new, hq, d), NAN, dtype=dt, device="cuda")
    w = w0.cuda() if weights else None
    K.attn_paged(out, q.cuda(), kv, lens_t.cuda(), d ** -0.5, weights=w)
    assert worst(out, want, tol) <= 1
    if weights:
        # Every row's weight within 2.2 delta, the exponential, the running sum; then `rows` sums of f32.
        rows = new * hq // hk
        rel = 2.2 * float(delta.max()) + 2.0 ** -20 + (3 * max(lens) / 16 + 40) * 2.0 ** -23
        tol_w = want_w * (rel + rows * 2.0 ** -24) + (w0.double() + want_w) * 2 * 2.0 ** -24
        assert worst(w, w0.double() + want_w, tol_w) <= 1
        unseen = torch.arange(slots)[None] >= lens_t[:, None]
        assert torch.equal(w.cpu()[unseen[:, None].expand_as(w0)], w0[unseen[:, None].expand_as(w0)])
    # The same call with a workspace kept, twice: the same bits.
    ws = K.attn_paged_workspace(q.cuda(), kv, weights=weights)
    for _ in range(2):
        again = torch.empty_like(out)
        K.attn_paged(again, q.cuda(), kv, lens_t.cuda(), d ** -0.5, weights=None if w is None else w0.cuda(), workspace=ws)
        assert torch.equal(again, out)


def cache_of(K, lens, hk, d, page, ct, seed, extra=0):
    g = gen(seed)
    k, v, table = R.make_pages(g, len(lens), -(-max(lens) // page) + extra, page, hk, d, ct)
    return k, v, table, torch.tensor(lens, dtype=torch.int32), cuda_kv(K, k, v, table)


def check_attn(K, q, k, v, table, lens, kv, out, scale):
    want, _, size, big = R.attention(q, k, v, table, lens, scale)
    tol, _ = R.attention_tolerance(q.dtype, k.dtype, q.shape[-1], int(lens.max()), size, big, want)
    assert worst(out, want, tol) <= 1


@pytest.mark.parametrize("power", [-60, -20, 12, 40])
def test_attn_paged_far_scales(K, power):
    """q far from 1 with the scale that undoes it: no part of a split q under- or overflows."""
    k, v, table, lens, kv = cache_of(K, [150, 33], 2, 64, 16, F16, 3)
    q = torch.randn(2, 1, 8, 64, generator=gen(4)) * 2.0 ** power
    out = torch.empty(2, 1, 8, 64, device="cuda")
    K.attn_paged(out, q.cuda(), kv, lens.cuda(), 0.125 * 2.0 ** -power)
    check_attn(K, q, k, v, table, lens, kv, out, 0.125 * 2.0 ** -power)


@pytest.mark.parametrize("heads", [4, 12])
@pytest.mark.parametrize("ct,dt", [(F16, F32), (BF16, BF16)])
def test_attn_paged_steep_scores(K, ct, dt, heads):
    """Scores hundreds apart: one position takes nearly all of a row, wherever it lies."""
    k, v, table, lens, kv = cache_of(K, [700, 699, 64, 2], 1, 64, 16, ct, 8)
    q = (torch.randn(4, 1, heads, 64, generator=gen(9)) * 12).to(dt)
    for s, t in ((0, 0), (1, 698), (2, 17), (3, 1)):
        R.put(k, table, s, t, (q[s, 0, :1].double() / 2).to(ct))
    kv = cuda_kv(K, k, v, table)
    out = torch.empty(4, 1, heads, 64, dtype=dt, device="cuda")
    K.attn_paged(out, q.cuda(), kv, lens.cuda(), 0.5)
    check_attn(K, q, k, v, table, lens, kv, out, 0.5)


def test_attn_paged_masked_rows_with_infinities(K):
    """A draft token's own row is infinite or NaN: the tokens before it, which do not see it, are unharmed."""
    g = gen(11)
    k, v, table, lens, _ = cache_of(K, [70, 48, 5], 2, 64, 16, F16, 12)
    q = torch.randn(3, 4, 4, 64, generator=g)
    clean = R.attention(q, k, v, table, lens, 0.125)
    tol, _ = R.attention_tolerance(F32, F16, 64, 70, clean[2], clean[3], clean[0])
    for value in (float("inf"), NAN):
        for which in (0, 1):
            k2, v2 = k.clone(), v.clone()
            for s in range(3):
                R.put((k2, v2)[which], table, s, int(lens[s]) - 1, torch.full((2, 64), value).to(F16))
            kv = cuda_kv(K, k2, v2, table)
            out = torch.empty(3, 4, 4, 64, device="cuda")
            w = torch.zeros(3, 2, table.shape[1] * 16, device="cuda")
            K.attn_paged(out, q.cuda(), kv, lens.cuda(), 0.125, weights=w)
            assert worst(out[:, :3], clean[0][:, :3], tol[:, :3]) <= 1
            if which == 1:  # a value row: the last token's outputs carry it, the weights do not
                assert not torch.isfinite(out[:, 3]).any() and torch.isfinite(w).all()


def test_attn_paged_many_rows_with_infinities(K):
    """The same on the tcgen05 kernel, the infinite rows at the end of a tile, at its start and in the middle; a bad page."""
    g = gen(17)
    k, v, table, lens, _ = cache_of(K, [640, 513, 300], 2, 64, 16, F16, 18)
    q = torch.randn(3, 4, 12, 64, generator=g)
    clean = R.attention(q, k, v, table, lens, 0.125)
    tol, _ = R.attention_tolerance(F32, F16, 64, 640, clean[2], clean[3], clean[0])
    for value in (float("inf"), NAN):
        for which in (0, 1):
            k2, v2 = k.clone(), v.clone()
            for s in range(3):
                for back in (1, 2):
                    R.put((k2, v2)[which], table, s, int(lens[s]) - back, torch.full((2, 64), value).to(F16))
            kv = cuda_kv(K, k2, v2, table)
            out = torch.empty(3, 4, 12, 64, device="cuda")
            K.attn_paged(out, q.cuda(), kv, lens.cuda(), 0.125)
            assert worst(out[:, :2], clean[0][:, :2], tol[:, :2]) <= 1
            if which == 1:
                assert not torch.isfinite(out[:, 2:]).any()
    broken = table.clone()
    broken[0, 3] = 10 ** 6
    out = torch.empty(3, 4, 12, 64, device="cuda")
    K.attn_paged(out, q.cuda(), cuda_kv(K, k, v, broken), lens.cuda(), 0.125)
    with pytest.raises(NrcError):
        K.sync_check()
    assert worst(out[1:], clean[0][1:], tol[1:]) <= 1
    keep = [t for t in range(640) if not 48 <= t < 64]
    kk, vv = (R.rows(x, table, 0, keep).double() for x in (k, v))
    p = torch.softmax(q[0, 3, 0].double() @ kk[:, 0].T * 0.125, -1)
    assert torch.allclose(out[0, 3, 0].double().cpu(), p @ vv[:, 0], atol=1e-5)


@pytest.mark.parametrize("new,d,ct", [(1, 64, F16), (5, 64, F16), (3, 96, F16), (2, 128, BF16)])
def test_attn_paged_long_sums_lean_to_no_side(K, new, d, ct):
    """Products on the tensor cores are cut towards zero, so sums of many of them would lean that way. Positive values,
    scores well below 1: the errors' mean has to stay below what 8 products cut, each up to 2^-23 of a sum that grows to
    the whole (4.5 of 2^-23 together, under 2^-20); roundings to nearest have no mean."""
    g = torch.Generator(device="cuda").manual_seed(new)
    n, page, hq, hk, seqs = 16000, 64, 40, 8, 32
    k_pages, v_pages = (torch.randn(n // page, page, hk, d, generator=g, device="cuda").to(ct) for _ in range(2))
    v_pages = v_pages.abs()
    table = torch.randperm(n // page, generator=g, device="cuda").int().repeat(seqs, 1)  # all read the same pages
    q = (torch.randn(1, new, hq, d, generator=g, device="cuda") * 0.2).repeat(seqs, 1, 1, 1)
    lens = torch.full((seqs,), n, dtype=torch.int32, device="cuda")
    out = torch.empty_like(q)
    K.attn_paged(out, q, K.PagedKV(k_pages, v_pages, table), lens, d ** -0.5)
    keys, values = (x[table[0].long()].reshape(n, hk, d).double() for x in (k_pages, v_pages))
    s = torch.einsum("nhgd,lhd->hgnl", q[0].double().view(new, hk, hq // hk, d), keys) * d ** -0.5
    seen = torch.arange(n, device="cuda") < n - (new - 1) + torch.arange(new, device="cuda")[:, None]
    p = s.masked_fill(~seen, -float("inf")).softmax(-1)
    want = torch.einsum("hgnl,lhd->nhgd", p, values).reshape(1, new, hq, d)
    assert float(((out.double() - want).mean((1, 2, 3)) / want.mean()).abs().max()) < 2 ** -20


def test_attn_paged_strides_and_shapes(K):
    """q and out inside wider tensors, one token without its dimension, pages laid out by head, a narrow slice of a table."""
    g = gen(13)
    b, hq, hk, d, page = 3, 8, 2, 64, 8
    k = torch.randn(40, hk, page, d, generator=g).to(F16)
    v = torch.randn(40, hk, page, d, generator=g).to(F16)
    wide = torch.randperm(40, generator=g)[:33].view(b, 11).to(torch.int32)
    lens = torch.tensor([40, 33, 1], dtype=torch.int32)
    kv = K.PagedKV(k.cuda().transpose(1, 2), v.cuda().transpose(1, 2), wide.cuda()[:, 2:7])
    q = torch.randn(b, 1, hq, d, generator=g)
    want, _, size, big = R.attention(q, k.transpose(1, 2), v.transpose(1, 2), wide[:, 2:7], lens, 0.1)
    tol, _ = R.attention_tolerance(F32, F16, d, 40, size, big, want)
    qw = torch.zeros(b, 3, hq + 1, d + 1, device="cuda")
    qw[:, 1:2, 1:, 1:] = q.cuda()
    ow = torch.zeros(b, 2, hq, d + 3, device="cuda")
    K.attn_paged(ow[:, 1:, :, :d], qw[:, 1:2, 1:, 1:], kv, lens.cuda(), 0.1)
    assert worst(ow[:, 1:, :, :d], want, tol) <= 1
    assert not ow[:, :1].any() and not ow[..., d:].any()
    flat = torch.empty(b, hq, d, device="cuda")
    K.attn_paged(flat, q[:, 0].cuda(), kv, lens.cuda(), 0.1, max_len=40)
    assert torch.equal(flat, ow[:, 1, :, :d])


@pytest.mark.parametrize("heads", [4, 24])
def test_attn_paged_page_layouts(K, heads):
    """K and V interleaved in one pool, and pages that lie head by head, for few and for many rows."""
    g = gen(19)
    hk, d, page, per = 2, 64, 16, 30
    table = torch.randperm(64, generator=g)[:60].view(2, per).to(torch.int32)
    lens = torch.tensor([470, 333], dtype=torch.int32)
    q = torch.randn(2, 1, heads, d, generator=g)
    both = torch.randn(64, 2, page, hk, d, generator=g).to(F16)
    by_head = [torch.randn(64, hk, page, d, generator=g).to(F16) for _ in range(2)]
    gb = both.cuda()
    gh = [t.cuda().transpose(1, 2) for t in by_head]
    for k, v, gk, gv in ((both[:, 0], both[:, 1], gb[:, 0], gb[:, 1]),
                         (by_head[0].transpose(1, 2), by_head[1].transpose(1, 2), *gh)):
        kv = K.PagedKV(gk, gv, table.cuda())
        out = torch.empty(2, 1, heads, d, device="cuda")
        w = torch.zeros(2, hk, per * page, device="cuda")
        K.attn_paged(out, q.cuda(), kv, lens.cuda(), 0.125, weights=w)
        check_attn(K, q, k, v, table, lens, kv, out, 0.125)
        assert torch.allclose(w.sum(-1).cpu(), torch.full((2, hk), heads / hk), atol=1e-4)


def test_attn_paged_errors_are_reported(K):
    k, v, table, lens, kv = cache_of(K, [30, 20], 1, 32, 8, F16, 14)
    q = torch.randn(2, 1, 2, 32, generator=gen(15))
    out = torch.empty(2, 1, 2, 32, device="cuda")
    # A page outside the pool: its positions are left out.
    for page in (10 ** 6, -1):
        broken = table.clone()
        broken[0, 1] = page
        K.attn_paged(out, q.cuda(), cuda_kv(K, k, v, broken), lens.cuda(), 0.2)
        with pytest.raises(NrcError) as e:
            K.sync_check()
        assert e.value.name == "DEVICE" and "page" in str(e.value)
        keep = [t for t in range(30) if not 8 <= t < 16]
        kk, vv = (R.rows(x, table, 0, keep)[:, 0].double() for x in (k, v))
        p = torch.softmax(q[0, 0].double() @ kk.T * 0.2, -1)
        assert torch.allclose(out[0, 0].double().cpu(), p @ vv, atol=1e-5)
    # A length beyond the table, or beyond max_len: cut there.
    K.attn_paged(out, q.cuda(), kv, torch.tensor([1000, 20], dtype=torch.int32, device="cuda"), 0.2)
    with pytest.raises(NrcError):
        K.sync_check()
    check_attn(K, q, k, v, table, torch.tensor([32, 20]), kv, out, 0.2)
    K.attn_paged(out, q.cuda(), kv, lens.cuda(), 0.2, max_len=20)
    with pytest.raises(NrcError):
        K.sync_check()
    check_attn(K, q, k, v, table, torch.tensor([20, 20]), kv, out, 0.2)
    K.attn_paged(out, q.cuda(), kv, torch.tensor([-5, 20], dtype=torch.int32, device="cuda"), 0.2)
    with pytest.raises(NrcError):
        K.sync_check()
    assert not out[0].any()


def test_attn_paged_long_cache_past_32_bit_offsets(K):
    """Rows behind the 2^32-byte mark of the pool, and pages in descending order."""
    page, hk, d = 64, 8, 128
    n_pages = 36000  # 4.7 GB each of K and V
    k = torch.zeros(n_pages, page, hk, d, dtype=F16, device="cuda")
    v = torch.zeros(n_pages, page, hk, d, dtype=F16, device="cuda")
    used = 20
    table = torch.arange(n_pages - 1, n_pages - 1 - used, -1, dtype=torch.int32).view(1, used)
    g = gen(16)
    small_k, small_v = (torch.randn(used, page, hk, d, generator=g).to(F16) for _ in range(2))
    k[-used:], v[-used:] = small_k.cuda(), small_v.cuda()
    q = torch.randn(1, 1, 16, d, generator=g)
    out = torch.empty(1, 1, 16, d, device="cuda")
    lens = torch.tensor([used * page - 5], dtype=torch.int32)
    K.attn_paged(out, q.cuda(), K.PagedKV(k, v, table.cuda()), lens.cuda(), d ** -0.5)
    small_table = torch.arange(used - 1, -1, -1, dtype=torch.int32).view(1, used)
    check_attn(K, q, small_k, small_v, small_table, lens, None, out, d ** -0.5)


# ------------------------------------------------------------------ evict

EVICT = [  # lens, kv heads, dim, cache, page, budget, recent, sinks
    ([40], 1, 32, F16, 8, 16, 4, 2), ([0, 1, 15, 16, 17, 100], 2, 64, BF16, 5, 16, 5, 3), ([1500, 1024], 3, 64, F16, 16, 1024, 128, 4),
    ([3000, 2999, 10], 2, 128, F16, 24, 777, 0, 0), ([64], 2, 96, BF16, 1, 33, 33, 0), ([64, 65], 1, 128, F16, 64, 64, 0, 64),
    ([5000], 1, 32, F16, 7, 4100, 1, 1), ([90, 91], 4, 64, F16, 10, 1, 1, 0), ([50], 2, 64, F16, 10, 0, 0, 0)]


@pytest.mark.parametrize("kind", ["plain", "ties", "odd"])
@pytest.mark.parametrize("lens,hk,d,ct,page,budget,recent,sinks", EVICT, ids=[str(i) for i in range(len(EVICT))])
def test_evict(K, lens, hk, d, ct, page, budget, recent, sinks, kind):
    k, v, table, lens_t, kv = cache_of(K, lens, hk, d, page, ct, sum(lens) + budget, extra=1)
    slots = table.shape[1] * page + 3  # wider than the table
    g = gen(budget)
    w = torch.randn(len(lens), hk, slots, generator=g).mul(3).exp()
    if kind == "ties":
        w = w.clamp(0.5, 1.5).mul(4).round()
    if kind == "odd":
        pick = torch.randint(0, 12, w.shape, generator=g)
        for i, x in enumerate((NAN, float("inf"), -float("inf"), 0.0, -0.0, 1e-42, -1e-42, torch.finfo(F32).min, -1.0)):
            w[pick == i] = x
    kept, nl, nw, k2, v2 = R.evict(k, v, table, lens_t, w, budget, recent, sinks)
    got = torch.full((len(lens), hk, budget), -7, dtype=torch.int32, device="cuda")
    got_l, got_w = torch.full_like(lens_t, -7).cuda(), torch.full_like(w, -7).cuda()
    K.evict(got, got_l, got_w, kv, lens_t.cuda(), w.cuda(), recent, sinks)
    assert torch.equal(got.cpu(), kept) and torch.equal(got_l.cpu(), nl)
    assert torch.equal(got_w.cpu().view(torch.int32), nw.view(torch.int32))
    assert torch.equal(kv.k_pages.cpu().view(torch.int16), k2.view(torch.int16))
    assert torch.equal(kv.v_pages.cpu().view(torch.int16), v2.view(torch.int16))
    # Lengths and weights updated in place.
    kv = cuda_kv(K, k, v, table)
    ll, ww = lens_t.cuda(), w.cuda()
    K.evict(got, ll, ww, kv, ll, ww, recent, sinks)
    assert torch.equal(ll.cpu(), nl) and torch.equal(ww.cpu().view(torch.int32), nw.view(torch.int32))
    assert torch.equal(kv.k_pages.cpu().view(torch.int16), k2.view(torch.int16)) and torch.equal(got.cpu(), kept)


def test_evict_errors_are_reported(K):
    k, v, table, lens, kv = cache_of(K, [40, 40], 1, 32, 8, F16, 21)
    w = torch.rand(2, 1, 40, generator=gen(22))
    kept = torch.empty(2, 1, 16, dtype=torch.int32, device="cuda")
    nl, nw = torch.empty(2, dtype=torch.int32, device="cuda"), torch.empty_like(w).cuda()
    K.evict(kept, nl, nw, kv, torch.tensor([41, -3], dtype=torch.int32, device="cuda"), w.cuda(), 4, 2)
    with pytest.raises(NrcError):
        K.sync_check()
    assert nl.tolist() == [16, 0] and int(kept[1].max()) == -1
    broken = table.clone()
    broken[1] = 9999
    kv = cuda_kv(K, k, v, broken)
    K.evict(kept, nl, nw, kv, lens.cuda(), w.cuda(), 4, 2)
    with pytest.raises(NrcError):
        K.sync_check()
    _, _, _, k2, v2 = R.evict(k, v, table, [40, 0], w, 16, 4, 2)
    assert torch.equal(kv.k_pages.cpu(), k2) and torch.equal(kv.v_pages.cpu(), v2)


# ------------------------------------------------------------------ verify_draft


def verify_inputs(b, n, vocab, dt, seed, spread=3.0):
    g = gen(seed)
    logits = torch.randn(b, n + 1, vocab, generator=g) * spread
    p = torch.softmax(logits, -1).to(dt)
    q = torch.softmax(logits[:, :n] + torch.randn(b, n, vocab, generator=g), -1).to(dt)
    draft = torch.where(torch.rand(b, n, generator=g) < 0.7, p[:, :n].argmax(-1), torch.randint(0, vocab, (b, n), generator=g))
    return p, q, draft.to(torch.int32), torch.rand(b, n + 1, generator=g)


def check_verify(K, p, q, draft, u, n_draft, gp=None, gq=None):
    want_t, want_a = R.verify(p, q, draft, u, n_draft)
    b, n = draft.shape
    tokens = torch.full((b, n + 1), -7, dtype=torch.int32, device="cuda")
    accepted = torch.full((b,), -7, dtype=torch.int32, device="cuda")
    K.verify_draft(tokens, accepted, p.cuda() if gp is None else gp, gq if gq is not None else None if q is None else q.cuda(),
                   draft.cuda(), u.cuda(), None if n_draft is None else n_draft.cuda())
    assert torch.equal(accepted.cpu(), want_a) and torch.equal(tokens.cpu(), want_t)


VERIFY = [(1, 4, 1000, F32), (5, 1, 1, F32), (4, 3, 2, F16), (7, 7, 33, BF16), (3, 2, 100352, F16), (2, 3, 151936, F32),
          (3, 8, 4097, BF16), (300, 2, 257, F32), (2, 0, 5000, F32), (2, 63, 300, F16), (1, 2, 300001, F32)]


@pytest.mark.parametrize("b,n,vocab,dt", VERIFY, ids=[str(i) for i in range(len(VERIFY))])
def test_verify_draft(K, b, n, vocab, dt):
    for seed in range(3):
        p, q, draft, u = verify_inputs(b, n, vocab, dt, 100 * seed + b)
        n_draft = torch.randint(-1, n + 2, (b,), generator=gen(seed), dtype=torch.int32)
        check_verify(K, p, q, draft, u, None)
        check_verify(K, p, q, draft, u, n_draft)
        check_verify(K, p, None, draft, u, n_draft)


def test_verify_draft_edges(K):
    vocab, n = 2000, 3
    p, q, draft, u = verify_inputs(9, n, vocab, F32, 31)
    q[0], draft[0] = p[0, :n], p[0, :n].argmin(-1)  # the same distribution: every draft is taken
    u[1, 0], p[1, 0], q[1, 0] = 0.5, 0.0, 0.0       # nothing left, and nothing in p: token 0
    u[1, 0], draft[1, 0] = 0.5, 7
    p[2, 0] = q[2, 0]                               # refused although nothing is left: drawn from p
    draft[2, 0] = 11
    p[2, 0, 11], q[2, 0, 11] = 0.0, 0.0
    draft[3, 0], draft[4, 1] = -1, vocab            # ids outside the vocabulary
    p[5, 0, ::3], q[5, 0, 1::3] = NAN, NAN
    draft[5, 0] = 3
    p[6, 0] = -p[6, 0]
    p[6, 1:, 5], q[6, 1:, 9], p[8, 0, 40] = float("inf"), float("inf"), float("inf")
    u[7], u[8] = 0.0, 1.0 - 2.0 ** -24
    check_verify(K, p, q, draft, u, None)
    check_verify(K, p, None, draft, u, None)
    one = torch.zeros(2, 2, vocab)
    one[0, :, 1234], one[1, :, vocab - 1] = 1.0, 1.0  # all of it on one token, the last one too
    check_verify(K, one, one[:, :1].roll(1, -1).contiguous(), torch.tensor([[1235], [0]], dtype=torch.int32), torch.rand(2, 2), None)


def test_verify_draft_borders(K):
    """Running sums that are exact in binary and a goal on their border: the first index that exceeds it."""
    vocab = 1 << 14
    p = torch.full((vocab, 1, vocab), 1.0 / vocab)
    u = (torch.arange(vocab, dtype=F32) / vocab).view(vocab, 1)
    gp = p[:1].cuda().expand(vocab, 1, vocab)
    tokens = torch.empty(vocab, 1, dtype=torch.int32, device="cuda")
    accepted = torch.empty(vocab, dtype=torch.int32, device="cuda")
    K.verify_draft(tokens, accepted, gp, None, torch.empty(vocab, 0, dtype=torch.int32, device="cuda"), u.cuda())
    assert torch.equal(tokens[:, 0].cpu(), torch.arange(vocab, dtype=torch.int32)) and not accepted.any()


def test_verify_draft_strides(K):
    p, q, draft, u = verify_inputs(3, 4, 999, F16, 41)
    gp = torch.zeros(5, 3, 1003, dtype=F16, device="cuda")[:, :, 3:1002].transpose(0, 1).copy_(p.cuda())
    gq = torch.zeros(3, 6, 1001, dtype=F16, device="cuda")[:, 1:5, 1:1000].copy_(q.cuda())
    check_verify(K, p, q, draft, u, None, gp, gq)


# ------------------------------------------------------------------ together


def serving_loop(K, steps, graph):
    """Two sequences decode with three drafted tokens a step: append, attention with weights, verification; every third
    step the caches shrink. Against the same loop in 64 bits on the kernels' own q and caches."""
    g = gen(51)
    b, new, hq, hk, d, page, vocab, budget = 2, 4, 4, 2, 64, 8, 500, 40
    k, v, table = R.make_pages(g, b, 9, page, hk, d, F16, bad=NAN)
    kv = cuda_kv(K, k, v, table)
    freqs = torch.tensor(K.rope_freqs(d, 10000.0), dtype=F32, device="cuda")
    slots = 9 * page
    dev = dict(device="cuda")
    st = dict(x=torch.empty(b * new, hq + 2 * hk, d, **dev), q=torch.empty(b * new, hq, d, **dev),
              pos=torch.zeros(b * new, dtype=torch.int32, **dev), slot=torch.zeros(b * new, dtype=torch.int32, **dev),
              lens=torch.zeros(b, dtype=torch.int32, **dev), out=torch.empty(b, new, hq, d, **dev),
              w=torch.zeros(b, hk, slots, **dev), p=torch.empty(b, new, vocab, **dev), pq=torch.empty(b, new - 1, vocab, **dev),
              draft=torch.empty(b, new - 1, dtype=torch.int32, **dev), u=torch.empty(b, new, **dev),
              tokens=torch.empty(b, new, dtype=torch.int32, **dev), acc=torch.empty(b, dtype=torch.int32, **dev),
              kept=torch.empty(b, hk, budget, dtype=torch.int32, **dev))
    seq = torch.arange(b, dtype=torch.int32, **dev).repeat_interleave(new)
    ws = K.attn_paged_workspace(st["out"], kv, weights=True)

    def step():
        x = st["x"]
        K.rope_append(st["q"], x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:], kv, freqs, st["pos"], seq, st["slot"], 1)
        K.attn_paged(st["out"], st["q"].view(b, new, hq, d), kv, st["lens"], 0.125, weights=st["w"], workspace=ws)
        K.verify_draft(st["tokens"], st["acc"], st["p"], st["pq"], st["draft"], st["u"])

    captured = None
    if graph:
        captured = torch.cuda.CUDAGraph()
        with torch.cuda.graph(captured):
            step()
    lens = torch.zeros(b, dtype=torch.long)  # cached positions
    turned = torch.zeros(b, dtype=torch.long)  # rotary position of the next token
    results = []
    for i in range(steps):
        st["x"].copy_(torch.randn(b * new, hq + 2 * hk, d, generator=g))
        at = torch.arange(new).repeat(b)
        st["slot"].copy_((lens.repeat_interleave(new) + at))
        st["pos"].copy_((turned.repeat_interleave(new) + at))
        st["lens"].copy_(lens + new)
        p, pq, draft, u = verify_inputs(b, new - 1, vocab, F32, 60 + i)
        for name, t in (("p", p), ("pq", pq), ("draft", draft), ("u", u)):
            st[name].copy_(t)
        before = st["w"].cpu().double()
        captured.replay() if graph else step()
        K.sync_check()
        q = st["q"].cpu().view(b, new, hq, d)
        want_q = R.rope(st["x"].cpu()[:, :hq], st["pos"].cpu(), freqs.cpu(), 1, 1.0)
        assert worst(st["q"], want_q, R.rope_tolerance(st["x"].cpu()[:, :hq], freqs.cpu(), 1, 1.0, F32, want_q)) <= 1
        kc, vc = kv.k_pages.cpu(), kv.v_pages.cpu()
        want, want_w, size, big = R.attention(q, kc, vc, table, lens + new, 0.125)
        tol, delta = R.attention_tolerance(F32, F16, d, int(lens.max()) + new, size, big, want)
        assert worst(st["out"], want, tol) <= 1
        assert torch.allclose(st["w"].cpu().double(), before + want_w, atol=1e-4)
        want_t, want_a = R.verify(p, pq, draft, u, None)
        assert torch.equal(st["tokens"].cpu(), want_t) and torch.equal(st["acc"].cpu(), want_a)
        lens += want_a.long() + 1
        turned += want_a.long() + 1
        # Positions of refused drafts are forgotten: the next step overwrites them, their weights go.
        live = (torch.arange(slots)[None] < lens[:, None])[:, None]
        st["w"].mul_(live.cuda())
        if i % 3 == 2:
            ll = lens.to(torch.int32).cuda()
            kept, nl, nw, k2, v2 = R.evict(kc, vc, table, ll.cpu(), st["w"].cpu(), budget, 8, 2)
            K.evict(st["kept"], ll, st["w"], kv, ll, st["w"], 8, 2)
            assert torch.equal(st["kept"].cpu(), kept) and torch.equal(ll.cpu(), nl) and torch.equal(st["w"].cpu(), nw)
            for s in range(b):
                for got, exp in ((kv.k_pages, k2), (kv.v_pages, v2)):
                    assert torch.equal(R.rows(got.cpu(), table, s, range(int(nl[s]))), R.rows(exp, table, s, range(int(nl[s]))))
            lens = ll.cpu().long()
        results += [st["out"].clone(), st["tokens"].clone(), st["w"].clone()]
    assert int(lens.max()) <= budget + 3 * new and int(turned.max()) > budget
    return results


def test_serving_loop_eager_and_captured(K):
    eager = serving_loop(K, 24, graph=False)
    captured = serving_loop(K, 24, graph=True)
    assert all(torch.equal(a, b) for a, b in zip(eager, captured))


def test_other_streams(K):
    """Two calls at once on two streams, each with its own workspace, and a stream handed over explicitly."""
    k, v, table, lens, kv = cache_of(K, [900, 40, 1300], 2, 128, 16, BF16, 71)
    q = torch.randn(3, 1, 8, 128, generator=gen(72)).to(BF16).cuda()
    l_dev = lens.cuda()
    want = torch.empty_like(q)
    K.attn_paged(want, q, kv, l_dev, 0.09)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[torch.empty_like(q) for _ in range(20)] for _ in streams]
    torch.cuda.synchronize()
    for i in range(20):
        for s, o in zip(streams, outs):
            if i % 2:
                K.attn_paged(o[i], q, kv, l_dev, 0.09, stream=s)
            else:
                with torch.cuda.stream(s):
                    K.attn_paged(o[i], q, kv, l_dev, 0.09)
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for o in outs for x in o)


FIRST_CALL = """
import torch
from nightrun_b200 import kernels as K
torch.manual_seed(1)
c = dict(device="cuda")
kp, vp = (torch.randn(40, 16, 2, 64, **c).half() for _ in range(2))
kv = K.PagedKV(kp, vp, torch.randperm(40, **c).view(2, 20).int())
freqs = torch.tensor(K.rope_freqs(64, 10000.0), **c)
i = torch.arange(2, dtype=torch.int32, **c)
lens = torch.tensor([300, 211], dtype=torch.int32, **c)
x = torch.randn(2, 8, 64, **c)
few, many = torch.randn(2, 1, 4, 64, **c), torch.randn(2, 3, 8, 64, **c)
o1, o2 = torch.empty_like(few), torch.empty_like(many)
w = torch.rand(2, 2, 320, **c)
kept, nl, nw = torch.empty(2, 2, 100, dtype=torch.int32, **c), torch.empty_like(lens), torch.empty_like(w)
p, q = torch.rand(2, 4, 5000, **c), torch.rand(2, 3, 5000, **c)
draft, u = torch.randint(0, 5000, (2, 3), **c).int(), torch.rand(2, 4, **c)
tokens, accepted = torch.empty(2, 4, dtype=torch.int32, **c), torch.empty(2, dtype=torch.int32, **c)
def step():
    K.rope_append(x[:, :4], x[:, :4], x[:, 4:6], x[:, 6:], kv, freqs, i, i, i)
    K.attn_paged(o1, few, kv, lens, 0.125, weights=w)
    K.attn_paged(o2, many, kv, lens, 0.125)
    K.evict(kept, nl, nw, kv, lens, w, 20, 2)
    K.verify_draft(tokens, accepted, p, q, draft, u)
state = [t.clone() for t in (x, kp, vp, w)]
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    step()
def result(run):
    for t, s in zip((x, kp, vp, w), state):
        t.copy_(s)
    run()
    K.sync_check()
    return [t.clone() for t in (x, kp, vp, w, o1, o2, kept, nl, nw, tokens, accepted)]
a, b = result(g.replay), result(step)
assert all(torch.equal(m, n) for m, n in zip(a, b))
print("same")
"""


def test_first_calls_may_be_captured():
    """Every operator's first call in a process is made while a stream is captured."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST_CALL], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "same" in r.stdout, r.stderr[-2000:]


def test_python_refusals(K):
    k, v, table, lens, kv = cache_of(K, [30, 20], 2, 64, 8, F16, 81)
    c = dict(device="cuda")
    q = torch.zeros(2, 1, 4, 64, **c)
    ok = dict(out=torch.zeros_like(q), q=q, kv=kv, lens=lens.cuda(), scale=1.0)
    w = torch.zeros(2, 2, 32, **c)
    for bad in (dict(out=torch.zeros(2, 1, 4, 64, dtype=F16, **c)), dict(out=torch.zeros(2, 1, 2, 64, **c)),
                dict(q=q.double(), out=q.double()), dict(q=q[..., :32], out=q[..., :32]), dict(q=q[:1], out=q[:1]),
                dict(q=q[..., ::2].repeat(1, 1, 1, 2).transpose(2, 3), out=q.transpose(2, 3)), dict(lens=lens.long().cuda()),
                dict(lens=lens.cuda()[:1]), dict(weights=w[:, :1]), dict(weights=w.half()), dict(weights=w.transpose(1, 2)),
                dict(q=torch.zeros(2, 1, 3, 64, **c), out=torch.zeros(2, 1, 3, 64, **c)), dict(scale=NAN)):
        with pytest.raises(NrcError):
            K.attn_paged(**{**ok, **bad})
    need = K.attn_paged_workspace(q, kv).nbytes
    if need:
        with pytest.raises(NrcError):
            K.attn_paged(**ok, workspace=torch.zeros(need - 1, dtype=torch.uint8, **c))
    with pytest.raises(NrcError):
        K.attn_paged(**{**ok, "out": torch.zeros(2, 1, 1, 64, **c).expand(2, 1, 4, 64)})
    with pytest.raises(ValueError):
        K.attn_paged(**{**ok, "lens": lens})
    for bad in ((k.cuda(), v.cuda()[:-1], table.cuda()), (k.cuda().float(), v.cuda().float(), table.cuda()),
                (k.cuda(), v.cuda(), table.cuda().long()), (k.cuda()[..., :48], v.cuda()[..., :48], table.cuda()),
                (k.cuda(), v.cuda(), table.cuda().t().contiguous().t())):
        with pytest.raises(NrcError):
            K.PagedKV(*bad)
    i = torch.zeros(2, 2, dtype=torch.int32, **c)
    p, u = torch.zeros(2, 2, 10, **c), torch.zeros(2, 2, **c)
    for bad in (dict(p=p.transpose(1, 2)), dict(q=p), dict(q=p[:, :1].half()), dict(draft=i), dict(u=u.double()),
                dict(tokens=i[:, :1]), dict(accepted=i), dict(n_draft=i[:1, 0])):
        a = dict(tokens=i, accepted=i[:, 0].contiguous(), p=p, q=p[:, :1], draft=i[:, :1].contiguous(), u=u) | bad
        with pytest.raises(NrcError):
            K.verify_draft(**a)
    kept, nl = torch.zeros(2, 2, 8, dtype=torch.int32, **c), lens.cuda()
    for bad in (dict(recent=9), dict(recent=-1), dict(sinks=9), dict(weights=w[..., ::2]), dict(new_weights=w[..., :8].contiguous()),
                dict(kept=kept[:, :1]), dict(kept=torch.zeros(2, 2, 40, dtype=torch.int32, **c)), dict(new_lens=nl.long())):
        with pytest.raises(NrcError):
            K.evict(**(dict(kept=kept, new_lens=nl, new_weights=w, kv=kv, lens=nl, weights=w, recent=2) | bad))
    x = torch.zeros(3, 4, 64, **c)
    one = torch.zeros(3, dtype=torch.int32, **c)
    f = torch.zeros(32, **c)
    for bad in (dict(q_out=x[:2]), dict(k=x), dict(v=x[:, :2].half()), dict(freqs=f.double()), dict(freqs=torch.zeros(33, **c)),
                dict(pos=one[:2]), dict(seq=one.long()), dict(style=3), dict(q=x.transpose(1, 2))):
        a = dict(q_out=x, q=x, k=x[:, :2], v=x[:, :2], kv=kv, freqs=f, pos=one, seq=one, slot=one) | bad
        with pytest.raises(NrcError):
            K.rope_append(**a)
