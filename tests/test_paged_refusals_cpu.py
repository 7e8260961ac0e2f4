"""Calls of the paged operators that are refused before a launch, so without a GPU: rows that overlap though no stride is 0,
tensors that overlap one another, workspaces that do not fit."""
import ctypes as C

import pytest

from nightrun_b200 import _lib, paged
from nightrun_b200._lib import PagedKVDesc

FAKE = 1 << 20  # never read: every call below is refused, or has nothing to do
INVALID = -1


@pytest.fixture(scope="module")
def L():
    return _lib.lib()


def desc(**kw):
    """8 pages of 16 positions, 2 KV heads of 64, f16; 3 sequences."""
    d = dict(k=FAKE, v=FAKE << 1, table=FAKE << 2, n_pages=8, page_stride=16 * 2 * 64, pos_stride=2 * 64, head_stride=64,
             page_size=16, n_kv_heads=2, head_dim=64, n_seqs=3, max_pages=2, table_stride=2, dtype=1)
    d.update(kw)
    return C.byref(PagedKVDesc(**d))


def rope(L, kv, tokens=4, heads=4, dtype=0, out=(FAKE << 3, 256, 64), q=(FAKE << 4, 256, 64), k=(FAKE << 5, 128, 64),
         v=(FAKE << 6, 128, 64)):
    args = paged._ROPE_ARGS.pack(*out, *q, *k, *v, FAKE << 7, FAKE << 8, FAKE << 9, FAKE << 10, tokens, heads, 64, dtype, 1, 1.0)
    return L.nrc_rope_append(kv, args, None)


def attn(L, kv, new=1, heads=4, out=(FAKE << 3, 256, 256, 64), q=(FAKE << 4, 256, 256, 64), weights=0, wlen=0, ws=FAKE << 8,
         wsb=1 << 40, max_len=0, dtype=0, lens=FAKE << 9):
    args = paged._ATTN_ARGS.pack(*out, *q, lens, weights, ws, wsb, wlen, max_len, new, heads, dtype, 0.125)
    return L.nrc_attn_paged(kv, args, None)


def evict(L, kv, kept=FAKE << 3, new_lens=FAKE << 4, new_weights=FAKE << 5, lens=FAKE << 6, weights=FAKE << 7, wlen=32, budget=8):
    return L.nrc_kv_evict(kv, kept, new_lens, new_weights, lens, weights, wlen, budget, 2, 1, None)


def verify(L, tokens=FAKE << 3, accepted=FAKE << 4, p=FAKE << 5, q=FAKE << 6, draft=FAKE << 7, u=FAKE << 8, n_draft=FAKE << 9,
           seqs=2, n=3, vocab=100):
    return L.nrc_verify_draft(tokens, accepted, p, (n + 1) * vocab, vocab, q, n * vocab, vocab, 0, seqs, n, vocab, draft, u,
                              n_draft, None)


def said(L, rc, word):
    return rc == INVALID and word in L.nrc_last_error().decode()


OVERLAPPING = [dict(head_stride=8), dict(pos_stride=64), dict(pos_stride=96), dict(page_stride=128), dict(page_stride=15 * 128),
               dict(head_stride=16 * 64, pos_stride=56), dict(page_stride=64, pos_stride=8 * 64, head_stride=8 * 64),
               dict(head_stride=-8), dict(n_kv_heads=1, pos_stride=56), dict(page_size=1, page_stride=64, n_pages=2)]
APART = [dict(), dict(head_stride=16 * 64, pos_stride=64),  # head by head
         dict(page_stride=64, pos_stride=2 * 8 * 64, head_stride=8 * 64),  # pages innermost
         dict(page_stride=2 * 16 * 2 * 64, v=FAKE + 2 * 16 * 2 * 64),  # K and V pages in turn
         dict(n_kv_heads=1, head_stride=0), dict(n_pages=1, page_stride=0), dict(pos_stride=-128, k=FAKE + 15 * 256, v=FAKE * 2 + 15 * 256)]


@pytest.mark.parametrize("bad", OVERLAPPING, ids=[str(b) for b in OVERLAPPING])
def test_pages_whose_rows_overlap(L, bad):
    for call in (rope, attn, evict):
        assert said(L, call(L, desc(**bad)), "overlap"), call.__name__


@pytest.mark.parametrize("good", APART, ids=[str(b) for b in APART])
def test_pages_whose_rows_lie_apart(L, good):
    assert rope(L, desc(**good), tokens=0) == 0
    assert L.nrc_kv_evict(desc(**dict(good, n_seqs=0)), None, None, None, None, None, 0, 0, 0, 0, None) == 0


def test_k_and_v_in_the_same_memory(L):
    """Written by rope_append and evict, so refused there; attention may read one pool as both."""
    half = 16 * 2 * 64 * 2  # bytes of a page
    for v in (FAKE, FAKE + 16, FAKE + 128, FAKE + 3 * half, FAKE - half + 32):
        assert said(L, rope(L, desc(v=v)), "overlap") and said(L, evict(L, desc(v=v)), "overlap"), v


def test_rope_append_outputs_that_overlap(L):
    at = FAKE << 3
    for kw in (dict(out=(at, 256, 32)), dict(out=(at, 64, 64)), dict(out=(at, 200, 64)), dict(out=(at, 256, 64), q=(at, 512, 64)),
               dict(out=(at, 256, 64), q=(at + 4, 256, 64)), dict(out=(at, 256, 64), q=(at + 256 * 4, 256, 64)),
               dict(out=(at, 256, 64), k=(at + 3 * 256 * 4 + 8, 128, 64)), dict(out=(at, 256, 64), v=(at - 64 * 4, 128, 64))):
        assert said(L, rope(L, desc(), **kw), "overlap"), kw


def test_attn_paged_outputs_that_overlap(L):
    at = FAKE << 3
    for kw in (dict(out=(at, 256, 256, 32)), dict(out=(at, 128, 256, 64)), dict(new=2, out=(at, 512, 64, 64)),
               dict(out=(at, 256, 256, 64), q=(at, 512, 512, 64)), dict(out=(at, 256, 256, 64), q=(at + 4, 256, 256, 64)),
               dict(out=(at, 256, 256, 64), q=(at - 2 * 256 * 4, 256, 256, 64)),
               dict(out=(at, 256, 256, 64), q=(at + 63 * 4, 512, 512, 128))):
        assert said(L, attn(L, desc(), **kw), "overlap"), kw
    w = dict(weights=FAKE << 5, wlen=32)
    for kw in (dict(weights=at + 64), dict(weights=(FAKE << 4) - 4), dict(weights=(FAKE << 9) - 8), dict(ws=FAKE << 5), dict(ws=at),
               dict(ws=FAKE << 9), dict(lens=at + 1020)):
        assert said(L, attn(L, desc(), **{**w, **kw}), "overlap"), kw


def test_evict_tensors_that_overlap(L):
    a = dict(kept=FAKE << 3, new_lens=FAKE << 4, new_weights=FAKE << 5, lens=FAKE << 6, weights=FAKE << 7)
    for one, two in (("kept", "new_lens"), ("kept", "new_weights"), ("kept", "lens"), ("kept", "weights"),
                     ("new_lens", "new_weights"), ("new_lens", "weights"), ("new_weights", "lens")):
        assert said(L, evict(L, desc(), **{**a, one: a[two]}), "overlap"), (one, two)
    assert said(L, evict(L, desc(), **{**a, "new_weights": a["weights"] + 4}), "overlap")
    assert said(L, evict(L, desc(), **{**a, "new_weights": a["weights"] - 4 * 32 * 2 * 3 + 4}), "overlap")
    assert said(L, evict(L, desc(), **{**a, "new_lens": a["lens"] + 8}), "overlap")


def test_verify_draft_tensors_that_overlap(L):
    a = dict(tokens=FAKE << 3, accepted=FAKE << 4, p=FAKE << 5, q=FAKE << 6, draft=FAKE << 7, u=FAKE << 8, n_draft=FAKE << 9)
    for one, two in (("tokens", "accepted"), ("tokens", "draft"), ("tokens", "u"), ("tokens", "n_draft"), ("accepted", "draft"),
                     ("accepted", "u"), ("tokens", "p"), ("tokens", "q"), ("accepted", "p"), ("accepted", "q")):
        assert said(L, verify(L, **{**a, one: a[two]}), "overlap"), (one, two)
    assert said(L, verify(L, **{**a, "accepted": a["n_draft"] + 4}), "overlap")
    assert said(L, verify(L, **{**a, "tokens": a["draft"] - 8}), "overlap")
    assert said(L, verify(L, seqs=1, **{**a, "tokens": a["draft"] - 4}), "overlap")


BIG = dict(max_pages=64, table_stride=64, n_pages=256)  # 1024 positions a sequence: split and joined


@pytest.mark.parametrize("with_weights", [0, 1])
@pytest.mark.parametrize("new", [1, 5])
def test_workspaces_that_do_not_fit(L, with_weights, new):
    def need(max_len=0, weights=with_weights):
        out = C.c_size_t()
        assert L.nrc_attn_paged_workspace(desc(**BIG), new, 4, weights, max_len, C.byref(out)) == 0
        return out.value

    kw = dict(new=new, out=(FAKE << 3, 256 * new, 256, 64), q=(FAKE << 4, 256 * new, 256, 64))
    if with_weights:
        kw |= dict(weights=FAKE << 5, wlen=1024)
    assert need() > 0
    for bad in (dict(wsb=need() - 1), dict(wsb=0), dict(ws=0), dict(ws=(FAKE << 8) + 4), dict(wsb=need(max_len=200))):
        assert said(L, attn(L, desc(**BIG), **{**kw, "wsb": need(), **bad}), "workspace"), bad
    assert need(max_len=200) < need() and need(weights=1) > need(weights=0)
    if with_weights:
        assert said(L, attn(L, desc(**BIG), **{**kw, "wsb": need(weights=0)}), "workspace")


def test_the_workspace_is_sized_for_the_tensors_device(monkeypatch):
    """Its size goes by the number of SMs: asked for on the device of the pages, whatever the current one is."""
    import torch
    current, seen = [0], []

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, current[0] = current[0], self.index

        def __exit__(self, *_):
            current[0] = self.before

    class Lib:
        def nrc_attn_paged_workspace(self, ref, new, heads, weights, max_len, out):
            seen.append((current[0], new, heads, weights))
            out._obj.value = 512
            return 0

    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(paged, "lib", Lib)
    kv = type("KV", (), dict(index=1, _ref=None, device=torch.device("cpu")))()
    assert paged.attn_paged_workspace(torch.empty(2, 3, 4, 64), kv, weights=True).nbytes == 512
    assert seen == [(1, 3, 4, 1)] and current == [0]
