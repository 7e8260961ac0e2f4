"""Serving over a paged KV cache: rotary append, attention of new tokens,
eviction, and the verification of drafted tokens (include/nrcuda.h, "serving
over a paged KV cache"). Re-exported by `kernels`, with its conventions:
outputs first, asynchronous on the current torch stream (or `stream=`).

Where the tensors live on another device than the current one, the call is
made on theirs. Shapes, types, strides and devices that do not fit raise
NrcError (INVALID); tensors that are not on a GPU raise ValueError.
"""
import ctypes as C

import torch

from ._lib import NRC_ERR_INVALID, NrcError, PagedKVDesc, check, lib

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def _need(ok, what):
    if not ok:
        raise NrcError(NRC_ERR_INVALID, what)


def _type(t):
    d = _DTYPES.get(t.dtype)
    if d is None:
        raise NrcError(NRC_ERR_INVALID, f"type {t.dtype}: float32, float16 or bfloat16")
    return d


def _on(device, *tensors):
    for t in tensors:
        if t.device != device:
            if not t.is_cuda:
                raise ValueError("nrcuda kernels take CUDA tensors")
            raise NrcError(NRC_ERR_INVALID, f"tensors on {device} and {t.device}")


def _ints(t, shape, what):
    if t.dtype != torch.int32 or t.shape != shape or not t.is_contiguous():
        raise NrcError(NRC_ERR_INVALID, f"{what}: contiguous int32 of shape {tuple(shape)}")


def _call(device, stream, fn, *args):
    """fn(*args, stream) on `device` and `stream` (None: the device's current one)."""
    index = device.index
    if stream is not None:
        _need(stream.device == device, f"a stream of {stream.device} for tensors on {device}")
        handle = stream.cuda_stream
    else:
        handle = torch._C._cuda_getCurrentRawStream(index)
    if torch.cuda.current_device() == index:
        rc = fn(*args, handle)
    else:
        with torch.cuda.device(index):
            rc = fn(*args, handle)
    if rc:
        check(rc)


class PagedKV:
    """A paged cache: k_pages and v_pages [n_pages, page_size, n_kv_heads, head_dim] (float16 or
    bfloat16, the same strides, the last dimension contiguous, 16-byte aligned rows) and the table,
    int32 [n_seqs, max_pages], whose entry [s, j] is the page of sequence s's positions from
    j * page_size on. A handle only: the tensors stay the caller's, and what is written to them
    (the table's entries too) is seen by the next call."""

    def __init__(self, k_pages, v_pages, table):
        if not (k_pages.is_cuda and v_pages.is_cuda and table.is_cuda):
            raise ValueError("nrcuda kernels take CUDA tensors")
        _on(k_pages.device, v_pages, table)
        _need(k_pages.dim() == 4 and k_pages.shape == v_pages.shape and k_pages.stride() == v_pages.stride()
              and k_pages.dtype == v_pages.dtype, "k_pages and v_pages: two alike [pages, page size, KV heads, head dim]")
        _need(k_pages.dtype in (torch.float16, torch.bfloat16), "pages are float16 or bfloat16")
        _need(k_pages.shape[3] in (32, 64, 96, 128), "head dim 32, 64, 96 or 128")
        _need(k_pages.stride(3) == 1, "the head dimension of the pages is contiguous")
        _need(table.dtype == torch.int32 and table.dim() == 2 and (table.stride(1) == 1 or table.shape[1] < 2),
              "table: int32 [sequences, pages], rows contiguous")
        self.k_pages, self.v_pages, self.table = k_pages, v_pages, table
        self.device = k_pages.device
        self.n_pages, self.page_size, self.n_kv_heads, self.head_dim = k_pages.shape
        self.n_seqs, self.max_pages = table.shape
        ps, rs, hs, _ = k_pages.stride()
        _need(self.page_size > 0 and self.n_kv_heads > 0, "empty pages")
        _need(not any(x % 8 for x in (ps, rs, hs)) and k_pages.data_ptr() % 16 == 0 and v_pages.data_ptr() % 16 == 0,
              "pages and their strides must be multiples of 16 bytes")
        _need(self.n_pages < 2 ** 31 and self.max_pages * self.page_size < 2 ** 31 and self.n_seqs < 65536
              and self.n_kv_heads <= 16384, "cache too large")
        self.desc = PagedKVDesc(k_pages.data_ptr(), v_pages.data_ptr(), table.data_ptr(), self.n_pages, ps, rs, hs,
                                self.page_size, self.n_kv_heads, self.head_dim, self.n_seqs, self.max_pages,
                                table.stride(0) if self.n_seqs > 1 else self.max_pages, _DTYPES[k_pages.dtype])
        self._ref = C.byref(self.desc)


def _heads(t, lead, kv, what):
    """Strides of [*lead, heads, head_dim], the last dimension contiguous."""
    s = t.stride()
    if t.dim() != lead + 2 or t.shape[-1] != kv.head_dim or s[-1] != 1:
        raise NrcError(NRC_ERR_INVALID, f"{what}: [..., heads, {kv.head_dim}] with a contiguous head dimension")
    return s


def rope_freqs_yarn(rot_dim, theta, factor, original_context, beta_fast=32.0, beta_slow=1.0):
    """Frequencies of a context stretched by `factor` (YaRN), and the factor on cos and sin."""
    out, mscale = (C.c_float * max(1, rot_dim // 2))(), C.c_float()
    check(lib().nrc_rope_freqs_yarn(out, C.byref(mscale), rot_dim, theta, factor, beta_fast, beta_slow, original_context))
    return list(out), mscale.value


def rope_append(q_out, q, k, v, kv, freqs, pos, seq, slot, style=1, mscale=1.0, stream=None):
    """rope::apply (rope.rs:49-65) of new tokens at their own positions and the append of
    infer.rs:536-551: q [tokens, heads, head_dim] rotated into q_out (q itself is allowed), k rotated
    and v [tokens, KV heads, head_dim] cached at `slot` of sequence `seq` of kv (slot < 0: not
    cached). freqs: float32 CUDA tensor, one value per rotated pair (the head's first 2 * numel
    values turn); pos, seq, slot: int32 [tokens]; style 0 = Adjacent, 1 = Neox. No two tokens of a
    call share (seq, slot)."""
    dev, dt = kv.device, _type(q)
    _on(dev, q_out, q, k, v, freqs, pos, seq, slot)
    n = (q.shape[0],)
    qs, ks, vs, os_ = _heads(q, 1, kv, "q"), _heads(k, 1, kv, "k"), _heads(v, 1, kv, "v"), _heads(q_out, 1, kv, "q_out")
    if q_out.shape != q.shape or k.shape != v.shape or k.shape[0] != n[0] or k.shape[1] != kv.n_kv_heads or not (
            k.dtype == v.dtype == q_out.dtype == q.dtype):
        raise NrcError(NRC_ERR_INVALID, "q, q_out [tokens, heads, head_dim] and k, v [tokens, KV heads, head_dim] of one type")
    _need(freqs.dtype == torch.float32 and freqs.dim() == 1 and freqs.is_contiguous(), "freqs: contiguous float32")
    _ints(pos, n, "pos"), _ints(seq, n, "seq"), _ints(slot, n, "slot")
    _call(dev, stream, lib().nrc_rope_append, kv._ref, q_out.data_ptr(), os_[0], os_[1], q.data_ptr(), qs[0], qs[1],
          k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1], dt, n[0], q.shape[1], freqs.data_ptr(),
          2 * freqs.numel(), mscale, style, pos.data_ptr(), seq.data_ptr(), slot.data_ptr())


def _attn_shape(q, kv):
    """q [seqs, new, heads, head_dim], or [seqs, heads, head_dim] for one new token each."""
    if q.dim() == 3:
        q = q.unsqueeze(1)
    _heads(q, 2, kv, "q")
    return q


def attn_paged_workspace(q, kv, weights=False, max_len=0):
    """The workspace of attn_paged calls of this shape: keep it, and use it in one call at a time."""
    q = _attn_shape(q, kv)
    need = C.c_size_t()
    check(lib().nrc_attn_paged_workspace(kv._ref, q.shape[1], q.shape[2], int(weights), max_len, C.byref(need)))
    return torch.empty(need.value, dtype=torch.uint8, device=kv.device)


def attn_paged(out, q, kv, lens, scale, weights=None, max_len=0, workspace=None, stream=None):
    """Attention (infer.rs:553-572) of the newest tokens of every sequence over its pages: q and out
    [seqs, new, heads, head_dim] ([seqs, heads, head_dim] for one token each), lens int32 [seqs]
    counting the new tokens too; token i of `new` sees the positions before lens - (new - 1 - i), one
    that sees nothing gets zeros. weights (float32 [seqs, KV heads, slots]): what every position
    received is added to it. max_len: no sequence is longer (0: the table's width). Without a
    workspace one is allocated for the call."""
    dev, dt = kv.device, _type(q)
    _on(dev, out, q, lens)
    if out.shape != q.shape or out.dtype != q.dtype:
        raise NrcError(NRC_ERR_INVALID, "out is like q")
    q, o = _attn_shape(q, kv), _attn_shape(out, kv)
    n, new, heads, _ = q.shape
    _need(n == kv.n_seqs, "q, lens and the table hold the same sequences")
    _ints(lens, (n,), "lens")
    wp, wl = None, 0
    if weights is not None:
        _on(dev, weights)
        _need(weights.dtype == torch.float32 and weights.dim() == 3 and weights.is_contiguous()
              and weights.shape[:2] == (n, kv.n_kv_heads), "weights: contiguous float32 [seqs, KV heads, slots]")
        wp, wl = weights.data_ptr(), weights.shape[2]
    if workspace is None:
        if stream is None:
            workspace = attn_paged_workspace(q, kv, weights is not None, max_len)
        else:
            with torch.cuda.stream(stream):  # the allocator hands it out again behind this call
                workspace = attn_paged_workspace(q, kv, weights is not None, max_len)
    else:
        _on(dev, workspace)
        _need(workspace.is_contiguous(), "the workspace is contiguous")
    qs, os_ = q.stride(), o.stride()
    _call(dev, stream, lib().nrc_attn_paged, kv._ref, o.data_ptr(), os_[0], os_[1], os_[2], q.data_ptr(), qs[0], qs[1],
          qs[2], dt, new, heads, lens.data_ptr(), scale, wp, wl, max_len, workspace.data_ptr(), workspace.nbytes)


def evict(kept, new_lens, new_weights, kv, lens, weights, recent, sinks=0, stream=None):
    """Shrinks every sequence longer than kept.shape[2] to that many positions, for each KV head the
    first `sinks`, the latest `recent` and those of largest weight (ties: the earlier one), and
    compacts its pages in place. kept: int32 [seqs, KV heads, budget], the old slots in ascending
    order, -1 behind a shorter sequence's; new_lens int32 [seqs]; weights, new_weights: float32
    [seqs, KV heads, slots]. new_lens may be lens, new_weights may be weights."""
    dev = kv.device
    _on(dev, kept, new_lens, new_weights, lens, weights)
    n = (kv.n_seqs,)
    _ints(lens, n, "lens"), _ints(new_lens, n, "new_lens")
    _need(kept.dim() == 3 and kept.shape[:2] == (kv.n_seqs, kv.n_kv_heads), "kept: [seqs, KV heads, budget]")
    _ints(kept, kept.shape, "kept")
    for t in (weights, new_weights):
        if (t.dtype != torch.float32 or t.dim() != 3 or not t.is_contiguous() or t.shape != weights.shape
                or t.shape[0] != kv.n_seqs or t.shape[1] != kv.n_kv_heads):
            raise NrcError(NRC_ERR_INVALID, "weights, new_weights: contiguous float32 [seqs, KV heads, slots]")
    _need(recent >= 0 and sinks >= 0, "negative counts")
    _call(dev, stream, lib().nrc_kv_evict, kv._ref, kept.data_ptr(), new_lens.data_ptr(), new_weights.data_ptr(),
          lens.data_ptr(), weights.data_ptr(), weights.shape[2], kept.shape[2], recent, sinks)


def verify_draft(tokens, accepted, p, q, draft, u, n_draft=None, stream=None):
    """Drafted tokens against the target, beside Sampler: p [seqs, n + 1, vocab], q [seqs, n, vocab]
    (None: each draft was certain), draft int32 [seqs, n], u float32 [seqs, n + 1] in [0, 1), n_draft
    int32 [seqs] (None: n). Draft i is taken while u[i] * q_i(draft) < p_i(draft); the token after the
    taken ones is drawn with u[n] from max(p - q, 0) at a refusal, else from p. tokens int32
    [seqs, n + 1]: taken drafts, the drawn token, -1; accepted int32 [seqs]: how many were taken."""
    if not p.is_cuda:
        raise ValueError("nrcuda kernels take CUDA tensors")
    dev, dt = p.device, _type(p)
    _on(dev, tokens, accepted, draft, u)
    _need(p.dim() == 3 and p.shape[1] > 0 and p.stride(2) == 1, "p: [seqs, n + 1, vocab], rows contiguous")
    b, m, vocab = p.shape
    ps, qp, qs = p.stride(), None, (0, 0)
    if q is not None:
        _on(dev, q)
        _need(q.dtype == p.dtype and q.shape == (b, m - 1, vocab) and q.stride(2) == 1,
              "q: [seqs, n, vocab] of p's type, rows contiguous")
        qp, qs = q.data_ptr(), q.stride()
    _ints(tokens, (b, m), "tokens"), _ints(accepted, (b,), "accepted"), _ints(draft, (b, m - 1), "draft")
    _need(u.dtype == torch.float32 and u.shape == (b, m) and u.is_contiguous(), "u: contiguous float32 [seqs, n + 1]")
    if n_draft is not None:
        _on(dev, n_draft)
        _ints(n_draft, (b,), "n_draft")
    _call(dev, stream, lib().nrc_verify_draft, tokens.data_ptr(), accepted.data_ptr(), p.data_ptr(), ps[0], ps[1], qp,
          qs[0], qs[1], dt, b, m - 1, vocab, draft.data_ptr(), u.data_ptr(),
          None if n_draft is None else n_draft.data_ptr())
