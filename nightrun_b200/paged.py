"""Serving over a paged KV cache: rotary append, attention of new tokens,
eviction, and the verification of drafted tokens (include/nrcuda.h, "serving
over a paged KV cache"). Re-exported by `kernels`, with its conventions:
outputs first, asynchronous on the current torch stream (or `stream=`).

Where the tensors live on another device than the current one, the call is
made on theirs. Shapes, types, strides and devices that do not fit, and
outputs that overlap one another or an input (but for the in-place forms
named below), raise NrcError (INVALID); tensors that are not on a GPU raise
ValueError.
"""
import ctypes as C
import struct

import torch

from ._lib import NRC_ERR_INVALID, NrcError, PagedKVDesc, check, lib

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_I32 = torch.int32
# nrc_rope_args and nrc_attn_args, packed in one step: a ctypes structure takes three times as long to fill.
_ROPE_ARGS = struct.Struct("QqqQqqQqqQqqQQQQQQQiif4x")
_ATTN_ARGS = struct.Struct("QqqqQqqqQQQQQQQQif")


def _need(ok, what):
    if not ok:
        raise NrcError(NRC_ERR_INVALID, what)


def _type(t):
    d = _DTYPES.get(t.dtype)
    if d is None:
        raise NrcError(NRC_ERR_INVALID, f"type {t.dtype}: float32, float16 or bfloat16")
    return d


def _elsewhere(device, *tensors):
    """Raises for the tensor that is not on `device`."""
    for t in tensors:
        if not t.is_cuda:
            raise ValueError("nrcuda kernels take CUDA tensors")
        _need(t.device == device, f"tensors on {device} and {t.device}")


def _ints(t, shape, what):
    if t.dtype is not _I32 or t.shape != shape or not t.is_contiguous():
        raise NrcError(NRC_ERR_INVALID, f"{what}: contiguous int32 of shape {tuple(shape)}")


def _on(index, fn, *args):
    """fn(*args) with device `index` the current one."""
    if torch.cuda.current_device() == index:
        return fn(*args)
    with torch.cuda.device(index):
        return fn(*args)


def _call(device, stream, fn, *args):
    """fn(*args, stream) on `device` and `stream` (None: the device's current one)."""
    index = device.index
    if stream is not None:
        _need(stream.device == device, f"a stream of {stream.device} for tensors on {device}")
        handle = stream.cuda_stream
    else:
        handle = torch._C._cuda_getCurrentRawStream(index)  # current_stream() takes 3 us to wrap it
    rc = _on(index, fn, *args, handle)
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
        _elsewhere(k_pages.device, v_pages, table)
        _need(k_pages.dim() == 4 and k_pages.shape == v_pages.shape and k_pages.stride() == v_pages.stride()
              and k_pages.dtype == v_pages.dtype, "k_pages and v_pages: two alike [pages, page size, KV heads, head dim]")
        _need(k_pages.dtype in (torch.float16, torch.bfloat16), "pages are float16 or bfloat16")
        _need(k_pages.shape[3] in (32, 64, 96, 128), "head dim 32, 64, 96 or 128")
        _need(k_pages.stride(3) == 1, "the head dimension of the pages is contiguous")
        _need(table.dtype == torch.int32 and table.dim() == 2 and (table.stride(1) == 1 or table.shape[1] < 2),
              "table: int32 [sequences, pages], rows contiguous")
        self.k_pages, self.v_pages, self.table = k_pages, v_pages, table
        self.device, self.index = k_pages.device, k_pages.device.index
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
        check(lib().nrc_attn_paged_workspace(self._ref, 1, self.n_kv_heads, 0, 0, C.byref(C.c_size_t())))  # rows that overlap


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
    i = kv.index
    if not (q.get_device() == i == k.get_device() == v.get_device() == q_out.get_device() == freqs.get_device()
            == pos.get_device() == seq.get_device() == slot.get_device()):
        _elsewhere(kv.device, q_out, q, k, v, freqs, pos, seq, slot)
    qz, kz, dt, d = q.shape, k.shape, q.dtype, kv.head_dim
    if (len(qz) != 3 or q_out.shape != qz or qz[2] != d or kz != (qz[0], kv.n_kv_heads, d) or v.shape != kz
            or k.dtype is not dt or v.dtype is not dt or q_out.dtype is not dt):
        raise NrcError(NRC_ERR_INVALID, f"q, q_out [tokens, heads, {d}] and k, v [tokens, {kv.n_kv_heads}, {d}] of one type")
    (qt, qh, a), (kt, kh, b), (vt, vh, c), (ot, oh, e) = q.stride(), k.stride(), v.stride(), q_out.stride()
    if not a == b == c == e == 1:
        raise NrcError(NRC_ERR_INVALID, "the head dimension is contiguous")
    if freqs.dtype is not torch.float32 or freqs.dim() != 1 or not freqs.is_contiguous():
        raise NrcError(NRC_ERR_INVALID, "freqs: contiguous float32")
    n = qz[:1]
    if (pos.dtype is not _I32 or seq.dtype is not _I32 or slot.dtype is not _I32 or not pos.shape == seq.shape == slot.shape == n
            or not (pos.is_contiguous() and seq.is_contiguous() and slot.is_contiguous())):
        raise NrcError(NRC_ERR_INVALID, "pos, seq, slot: contiguous int32 [tokens]")
    _call(kv.device, stream, lib().nrc_rope_append, kv._ref, _ROPE_ARGS.pack(
        q_out.data_ptr(), ot, oh, q.data_ptr(), qt, qh, k.data_ptr(), kt, kh, v.data_ptr(), vt, vh, freqs.data_ptr(),
        pos.data_ptr(), seq.data_ptr(), slot.data_ptr(), n[0], qz[1], 2 * freqs.numel(),
        _DTYPES[dt] if dt in _DTYPES else _type(q), style, mscale))


def attn_paged_workspace(q, kv, weights=False, max_len=0):
    """The workspace of attn_paged calls of this shape: keep it, and use it in one call at a time."""
    _need(q.dim() in (3, 4), "q: [seqs, new, heads, head_dim] or [seqs, heads, head_dim]")
    need = C.c_size_t()
    check(_on(kv.index, lib().nrc_attn_paged_workspace, kv._ref, q.shape[1] if q.dim() == 4 else 1, q.shape[-2], int(weights),
              max_len, C.byref(need)))  # its size goes by the device's SMs
    return torch.empty(need.value, dtype=torch.uint8, device=kv.device)


def attn_paged(out, q, kv, lens, scale, weights=None, max_len=0, workspace=None, stream=None):
    """Attention (infer.rs:553-572) of the newest tokens of every sequence over its pages: q and out
    [seqs, new, heads, head_dim] ([seqs, heads, head_dim] for one token each; not the same memory), lens int32 [seqs]
    counting the new tokens too; token i of `new` sees the positions before lens - (new - 1 - i), one
    that sees nothing gets zeros. weights (float32 [seqs, KV heads, slots]): what every position
    received is added to it. max_len: no sequence is longer (0: the table's width). Without a
    workspace one is allocated for the call."""
    i = kv.index
    if not q.get_device() == i == out.get_device() == lens.get_device():
        _elsewhere(kv.device, out, q, lens)
    z, dt, n = q.shape, q.dtype, kv.n_seqs
    if out.shape != z or out.dtype is not dt:
        raise NrcError(NRC_ERR_INVALID, "out is like q")
    if len(z) == 4:
        _, new, heads, d = z
        (qs, qt, qh, a), (os_, ot, oh, b) = q.stride(), out.stride()
    elif len(z) == 3:
        new, (_, heads, d) = 1, z
        (qs, qh, a), (os_, oh, b) = q.stride(), out.stride()
        qt = ot = 0
    else:
        raise NrcError(NRC_ERR_INVALID, "q: [seqs, new, heads, head_dim] or [seqs, heads, head_dim]")
    if z[0] != n or d != kv.head_dim or not a == b == 1:
        raise NrcError(NRC_ERR_INVALID, f"q: [{n} sequences as in the table, ..., heads, {kv.head_dim}], the last contiguous")
    _ints(lens, (n,), "lens")
    wp = wl = 0
    if weights is not None:
        if weights.get_device() != i:
            _elsewhere(kv.device, weights)
        if (weights.dtype is not torch.float32 or weights.dim() != 3 or not weights.is_contiguous()
                or weights.shape[:2] != (n, kv.n_kv_heads)):
            raise NrcError(NRC_ERR_INVALID, "weights: contiguous float32 [seqs, KV heads, slots]")
        wp, wl = weights.data_ptr(), weights.shape[2]
    _need(max_len >= 0, "negative max_len")
    if workspace is None:
        if stream is None:
            workspace = attn_paged_workspace(q, kv, weights is not None, max_len)
        else:
            with torch.cuda.stream(stream):  # the allocator hands it out again behind this call
                workspace = attn_paged_workspace(q, kv, weights is not None, max_len)
    else:
        if workspace.get_device() != i:
            _elsewhere(kv.device, workspace)
        if not workspace.is_contiguous():
            raise NrcError(NRC_ERR_INVALID, "the workspace is contiguous")
    _call(kv.device, stream, lib().nrc_attn_paged, kv._ref, _ATTN_ARGS.pack(
        out.data_ptr(), os_, ot, oh, q.data_ptr(), qs, qt, qh, lens.data_ptr(), wp, workspace.data_ptr(), workspace.nbytes,
        wl, max_len, new, heads, _DTYPES[dt] if dt in _DTYPES else _type(q), scale))


def evict(kept, new_lens, new_weights, kv, lens, weights, recent, sinks=0, stream=None):
    """Shrinks every sequence longer than kept.shape[2] to that many positions, for each KV head the
    first `sinks`, the latest `recent` and those of largest weight (ties: the earlier one), and
    compacts its pages, which belong to it alone, in place. kept: int32 [seqs, KV heads, budget], the old slots in ascending
    order, -1 behind a shorter sequence's; new_lens int32 [seqs]; weights, new_weights: float32
    [seqs, KV heads, slots]. new_lens may be lens, new_weights may be weights."""
    i = kv.index
    if not (kept.get_device() == i == new_lens.get_device() == new_weights.get_device() == lens.get_device()
            == weights.get_device()):
        _elsewhere(kv.device, kept, new_lens, new_weights, lens, weights)
    n, kz, wz = (kv.n_seqs,), kept.shape, weights.shape
    _ints(lens, n, "lens")
    _ints(new_lens, n, "new_lens")
    if len(kz) != 3 or kz[:2] != (n[0], kv.n_kv_heads):
        raise NrcError(NRC_ERR_INVALID, "kept: [seqs, KV heads, budget]")
    _ints(kept, kz, "kept")
    if (len(wz) != 3 or wz[:2] != kz[:2] or new_weights.shape != wz or weights.dtype is not torch.float32
            or new_weights.dtype is not torch.float32 or not (weights.is_contiguous() and new_weights.is_contiguous())):
        raise NrcError(NRC_ERR_INVALID, "weights, new_weights: contiguous float32 [seqs, KV heads, slots]")
    _need(recent >= 0 and sinks >= 0, "negative counts")
    _call(kv.device, stream, lib().nrc_kv_evict, kv._ref, kept.data_ptr(), new_lens.data_ptr(), new_weights.data_ptr(),
          lens.data_ptr(), weights.data_ptr(), wz[2], kz[2], recent, sinks)


def verify_draft(tokens, accepted, p, q, draft, u, n_draft=None, stream=None):
    """Drafted tokens against the target, beside Sampler: p [seqs, n + 1, vocab], q [seqs, n, vocab]
    (None: each draft was certain), draft int32 [seqs, n], u float32 [seqs, n + 1] in [0, 1), n_draft
    int32 [seqs] (None: n). Draft i is taken while u[i] * q_i(draft) < p_i(draft); the token after the
    taken ones is drawn with u[n] from max(p - q, 0) at a refusal, else from p. tokens int32
    [seqs, n + 1]: taken drafts, the drawn token, -1; accepted int32 [seqs]: how many were taken. accepted
    may be n_draft, and for one sequence tokens may begin where draft does."""
    i, dt = p.get_device(), p.dtype
    if i < 0 or not i == tokens.get_device() == accepted.get_device() == draft.get_device() == u.get_device():
        _elsewhere(p.device, p, tokens, accepted, draft, u)
    z = p.shape
    _need(len(z) == 3 and z[1] > 0, "p: [seqs, n + 1, vocab]")
    b, m, vocab = z
    (ps, pt, one), qp, qs, qt = p.stride(), 0, 0, 0
    if q is not None:
        if q.get_device() != i:
            _elsewhere(p.device, q)
        _need(q.dtype is dt and q.shape == (b, m - 1, vocab), "q: [seqs, n, vocab] of p's type")
        qp, (qs, qt, two) = q.data_ptr(), q.stride()
        one = one if two == 1 else two
    _need(one == 1 or vocab == 1, "the rows of p and q are contiguous")
    _ints(tokens, (b, m), "tokens")
    _ints(accepted, (b,), "accepted")
    _ints(draft, (b, m - 1), "draft")
    if u.dtype is not torch.float32 or u.shape != (b, m) or not u.is_contiguous():
        raise NrcError(NRC_ERR_INVALID, "u: contiguous float32 [seqs, n + 1]")
    if n_draft is not None:
        if n_draft.get_device() != i:
            _elsewhere(p.device, n_draft)
        _ints(n_draft, (b,), "n_draft")
    _call(p.device, stream, lib().nrc_verify_draft, tokens.data_ptr(), accepted.data_ptr(), p.data_ptr(), ps, pt, qp, qs, qt,
          _DTYPES[dt] if dt in _DTYPES else _type(p), b, m - 1, vocab, draft.data_ptr(), u.data_ptr(),
          None if n_draft is None else n_draft.data_ptr())
