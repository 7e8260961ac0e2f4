"""Refusals of the operators over a paged KV cache, and their host-side arithmetic: nothing here
reaches a device call, so it runs without a GPU."""
import ctypes as C
import math

import pytest
import torch

from nightrun_b200 import _lib, kernels, paged
from nightrun_b200._lib import NrcError, PagedKVDesc

FAKE = 0x10000  # never read: every call below is refused before a launch


@pytest.fixture(scope="module")
def L():
    return _lib.lib()


def desc(**kw):
    d = dict(k=FAKE, v=FAKE, table=FAKE, n_pages=8, page_stride=16 * 2 * 64, pos_stride=2 * 64, head_stride=64,
             page_size=16, n_kv_heads=2, head_dim=64, n_seqs=3, max_pages=2, table_stride=2, dtype=1)
    d.update(kw)
    return C.byref(PagedKVDesc(**d))


BAD_CACHES = [dict(dtype=0), dict(dtype=7), dict(head_dim=48), dict(head_dim=160), dict(head_dim=0), dict(page_size=0),
              dict(n_kv_heads=0), dict(n_seqs=70000), dict(max_pages=2 ** 28, table_stride=2 ** 28), dict(table_stride=1),
              dict(k=FAKE + 8), dict(v=FAKE + 2), dict(page_stride=2052), dict(pos_stride=132), dict(head_stride=68),
              dict(n_pages=2 ** 31), dict(k=None), dict(table=None), dict(table=FAKE + 2), dict(n_kv_heads=16385),
              dict(page_stride=0), dict(pos_stride=0), dict(head_stride=0)]


def rope(L, kv, dtype=0, tokens=4, heads=4, rot=64, style=1, q=FAKE, freqs=FAKE, pos=FAKE):
    args = paged._ROPE_ARGS.pack(FAKE, 256, 64, q or 0, 256, 64, FAKE, 128, 64, FAKE, 128, 64, freqs or 0, pos or 0, FAKE,
                                 FAKE, tokens, heads, rot, dtype, style, 1.0)
    return L.nrc_rope_append(kv, args, None)


def attn(L, kv, dtype=0, new=1, heads=4, scale=0.125, weights=None, wlen=0, ws=None, wsb=0, q=FAKE, lens=FAKE, out=2 * FAKE):
    args = paged._ATTN_ARGS.pack(out, 256, 256, 64, q or 0, 256, 256, 64, lens or 0, weights or 0, ws or 0, wsb, wlen, 0,
                                 new, heads, dtype, scale)
    return L.nrc_attn_paged(kv, args, None)


def evict(L, kv, wlen=32, budget=8, recent=2, sinks=1, kept=FAKE, weights=FAKE):
    return L.nrc_kv_evict(kv, kept, FAKE, FAKE, FAKE, weights, wlen, budget, recent, sinks, None)


def verify(L, dtype=0, seqs=2, n=3, vocab=100, p=FAKE, draft=FAKE):
    return L.nrc_verify_draft(FAKE, FAKE, p, 400, 100, FAKE, 300, 100, dtype, seqs, n, vocab, draft, FAKE, None, None)


@pytest.mark.parametrize("bad", BAD_CACHES, ids=[str(b) for b in BAD_CACHES])
def test_every_operator_refuses_a_bad_cache(L, bad):
    for call in (rope, attn, evict):
        assert call(L, desc(**bad)) == -1, call.__name__
    assert rope(L, None) == -1 and attn(L, None) == -1 and evict(L, None) == -1


def test_rope_append_refusals(L):
    for kw in (dict(dtype=3), dict(dtype=-1), dict(style=2), dict(rot=63), dict(rot=66), dict(q=None), dict(freqs=None),
               dict(pos=None), dict(tokens=2 ** 31), dict(heads=70000), dict(q=FAKE + 2), dict(q=FAKE + 1, dtype=1),
               dict(pos=FAKE + 1), dict(freqs=FAKE + 2)):
        assert rope(L, desc(), **kw) == -1, kw
        assert L.nrc_last_error()
    assert L.nrc_rope_append(desc(), None, None) == -1
    assert rope(L, desc(), tokens=0) == 0  # nothing to do, nothing launched


def test_attn_paged_refusals(L):
    need = C.c_size_t()
    assert L.nrc_attn_paged_workspace(desc(), 1, 4, 0, 0, C.byref(need)) == 0
    for kw in (dict(new=0), dict(new=65), dict(heads=3), dict(heads=0), dict(dtype=5), dict(scale=math.nan),
               dict(scale=math.inf), dict(weights=FAKE, wlen=0), dict(weights=FAKE, wlen=2 ** 31), dict(q=None),
               dict(lens=None), dict(lens=FAKE + 2), dict(q=FAKE + 2), dict(weights=FAKE + 2, wlen=32)):
        kw = dict(ws=FAKE, wsb=1 << 40) | kw
        assert attn(L, desc(), **kw) == -1, kw
    if need.value:
        assert attn(L, desc(), ws=FAKE, wsb=need.value - 1) == -1
        assert attn(L, desc(), ws=FAKE + 4, wsb=need.value) == -1
        assert attn(L, desc(), ws=None, wsb=need.value) == -1
    assert L.nrc_attn_paged(desc(), None, None) == -1
    assert L.nrc_attn_paged_workspace(desc(), 1, 4, 0, 0, None) == -1
    assert L.nrc_attn_paged_workspace(desc(), 1, 5, 0, 0, C.byref(need)) == -1
    assert attn(L, desc(n_seqs=0), ws=FAKE, wsb=1 << 40) == 0


def test_attn_paged_refuses_queries_as_its_output(L):
    assert attn(L, desc(), ws=FAKE, wsb=1 << 40, out=FAKE, q=FAKE) == -1
    assert b"overlap" in L.nrc_last_error()


def test_evict_refusals(L):
    for kw in (dict(budget=33), dict(wlen=4), dict(recent=9), dict(recent=8, sinks=1), dict(sinks=7), dict(kept=None),
               dict(weights=None), dict(wlen=2 ** 31, budget=2), dict(kept=FAKE + 1), dict(weights=FAKE + 2)):
        assert evict(L, desc(), **kw) == -1, kw
    assert evict(L, desc(), wlen=64, budget=40) == -1  # more than the table's 32 positions
    assert evict(L, desc(n_seqs=0)) == 0


def test_verify_draft_refusals(L):
    for kw in (dict(dtype=4), dict(n=64), dict(vocab=0), dict(vocab=2 ** 31), dict(p=None), dict(draft=None),
               dict(p=FAKE + 1, dtype=2), dict(p=FAKE + 2), dict(draft=FAKE + 2), dict(seqs=2 ** 28)):
        assert verify(L, **kw) == -1, kw
    assert verify(L, seqs=0) == 0


def test_yarn_frequencies(L):
    dim, theta, factor, orig = 128, 500000.0, 16.0, 8192.0
    freqs, mscale = kernels.rope_freqs_yarn(dim, theta, factor, orig)
    assert abs(mscale - (0.1 * math.log(factor) + 1)) < 1e-6
    plain = kernels.rope_freqs(dim, theta)
    for i, f in enumerate(freqs):
        turns = orig * theta ** (-2 * i / dim) / (2 * math.pi)
        ratio = f / theta ** (-2 * i / dim)
        assert 1 / factor - 1e-6 <= ratio <= 1 + 1e-6
        if turns > 32 * 1.25:  # a pair index is a whole number: the borders are rounded outwards
            assert abs(ratio - 1) < 1e-6
        if turns < 1 / 1.25:
            assert abs(ratio - 1 / factor) < 1e-6
    assert all(abs(a / b - 1) < 2e-6 for a, b in zip(kernels.rope_freqs_yarn(dim, theta, 1.0, orig)[0], plain))
    assert kernels.rope_freqs_yarn(dim, theta, 1.0, orig)[1] == 1.0
    for bad in ((0, theta, 4.0, orig), (7, theta, 4.0, orig), (8, 1.0, 4.0, orig), (8, theta, 0.0, orig),
                (8, theta, 4.0, 0.0), (8, theta, 4.0, orig, 1.0, 2.0), (8, math.nan, 4.0, orig)):
        with pytest.raises(NrcError):
            kernels.rope_freqs_yarn(*bad)


def test_tensors_off_the_gpu_are_refused():
    with pytest.raises(ValueError):
        kernels.PagedKV(torch.zeros(2, 4, 1, 64, dtype=torch.float16), torch.zeros(2, 4, 1, 64, dtype=torch.float16),
                        torch.zeros(1, 2, dtype=torch.int32))
    i = torch.zeros(1, 2, dtype=torch.int32)
    with pytest.raises(ValueError):
        kernels.verify_draft(i, i[0, :1], torch.zeros(1, 2, 8), None, i[:, :1], torch.zeros(1, 2))
