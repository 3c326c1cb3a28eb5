"""Attention over a prompt's own keys and values, before (or beside) their being quantised into the cache.

A first chunk of a prompt has its bf16 or fp16 keys and values at hand: attending them as they are needs no store first and
loses nothing to the 4-bit codes, which only later steps then read. One HIP kernel (`qp_prompt`) serves packed sequences of
different lengths, with grouped heads, causal or not, keys that begin before the queries (the next turn of a conversation)
and single tokens over long contexts, whose keys are split over workgroups and merged.
"""
from __future__ import annotations

import torch

from .. import _hip

HEAD_SIZES = (64, 128, 256, 512)
_DTYPES = {torch.bfloat16: _hip.DTYPE_BF16, torch.float16: _hip.DTYPE_F16}
_PACK = _hip.Packer(_hip.PromptArgs)


def _check(q, k, v, out, cu_q, cu_k, lse):
    """What the kernel's indexing rests on (shapes and types; nothing is copied)."""
    if q.dtype not in _DTYPES:
        raise NotImplementedError(f"prompt_attention: bf16 or fp16 tensors, got {q.dtype}")
    if q.dim() != 3 or k.dim() != 3 or v.shape != k.shape or k.shape[2] != q.shape[2] or out.shape != q.shape:
        raise ValueError(f"prompt_attention: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)} and out "
                         f"{tuple(out.shape)} do not belong together: [tokens, heads, head size] each")
    if k.dtype != q.dtype or v.dtype != q.dtype or out.dtype != q.dtype:
        raise ValueError(f"prompt_attention: k {k.dtype}, v {v.dtype} and out {out.dtype} must have q's type {q.dtype}")
    if q.stride(2) != 1 or k.stride(2) != 1 or v.stride(2) != 1 or out.stride(2) != 1:
        raise ValueError("prompt_attention: channels must be contiguous")
    for name, t in (("cu_seqlens_q", cu_q), ("cu_seqlens_k", cu_k)):
        if t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous() or t.shape[0] < 1:
            raise ValueError(f"prompt_attention: {name} must be a contiguous int32 vector of sequences + 1 offsets")
    if cu_q.shape != cu_k.shape:
        raise ValueError("prompt_attention: cu_seqlens_q and cu_seqlens_k are of different batches")
    if lse is not None and (lse.dtype != torch.float32 or lse.shape != q.shape[:2]):
        raise ValueError(f"prompt_attention: lse must be fp32 {tuple(q.shape[:2])}")
    _hip.no_derivatives("prompt_attention", q, k, v, out, lse)


def _check_out(q, k, v, out):
    """Row blocks are written while others are at work: out lies in q's place, row for row, or apart from all three. (Their
    extents meet, or out has a stride of 0.)"""
    if _hip.repeats(out, out.stride()):
        raise ValueError("prompt_attention: rows of out share memory with each other")
    same = out.data_ptr() == q.data_ptr() and all(n == 1 or x == y for n, x, y in zip(q.shape, q.stride(), out.stride()))
    if not same and _hip.share_memory(out, q):
        raise ValueError("prompt_attention: out shares memory with q but is not q")
    for name, t in (("k", k), ("v", v)):
        if _hip.share_memory(out, t):
            raise ValueError(f"prompt_attention: out shares memory with {name}")


def _check_device(q, k, v, out, cu_q, cu_k, lse):
    index = q.get_device()
    if not (index == k.get_device() == v.get_device() == out.get_device() == cu_q.get_device() == cu_k.get_device()) or \
            index < 0 or (lse is not None and lse.get_device() != index):
        _hip.same_device("prompt_attention", q, k=k, v=v, out=out, cu_seqlens_q=cu_q, cu_seqlens_k=cu_k, lse=lse)


def prompt_attention(q, k, v, out=None, *, cu_seqlens_q, cu_seqlens_k=None, max_seqlen_k=None, max_seqlen_q=None,
                     softmax_scale=None, causal=True, lse=None, num_splits=0) -> torch.Tensor:
    """Attention of packed sequences: q [T, NQ, hs] over k and v [K, NKV, hs], bf16 or fp16, hs one of HEAD_SIZES, NQ a
    multiple of NKV; sequence i has the rows cu_seqlens_q[i] .. cu_seqlens_q[i + 1] of q and the rows cu_seqlens_k[i] ..
    of k and v (int32 on the GPU; cu_seqlens_k None: the same as the queries'). Its last query is at its last key: with
    causal, query t sees the keys j <= t + keys - queries. softmax_scale (hs ** -0.5 when None) multiplies q.k.

    Writes and returns out (made when None; it may be q itself, else it shares no memory with q, k and v); a query that
    sees no key gets zeros. lse (optional, fp32 [T, NQ]) receives the natural-log sum of the row's exponentials, -inf for
    such a query. Rows of q past the last sequence are not written. Keys and values that no query sees are never used,
    whatever they hold.

    Strides are free as long as channels are contiguous and rows 16-byte aligned, so q, k and v may be views of one
    projection's output. max_seqlen_k, the longest sequence's keys (K when None), is what the work is laid out by: the
    automatic key splits (num_splits 0) of batches with few rows, and the order of the row blocks. max_seqlen_q is accepted
    for symmetry and not used. The partials of a split come from torch's caching allocator; no host synchronisation."""
    del max_seqlen_q
    if cu_seqlens_k is None:
        cu_seqlens_k = cu_seqlens_q
    given = out is not None
    if not given:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    _check(q, k, v, out, cu_seqlens_q, cu_seqlens_k, lse)
    hs = q.shape[2]
    qs, ks, vs, os = q.stride(), k.stride(), v.stride(), out.stride()
    ls = (0, 0) if lse is None else lse.stride()
    if lse is not None and 0 in ls and _hip.repeats(lse, ls):
        raise ValueError("prompt_attention: lse must have a place for every row")
    q_at, k_at, v_at, out_at = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
    if given:
        (T, nq, _), (K, nkv, _) = q.shape, k.shape
        end = out_at + 2 * ((T - 1) * os[0] + (nq - 1) * os[1] + hs)
        if (0 in os or (out_at < q_at + 2 * ((T - 1) * qs[0] + (nq - 1) * qs[1] + hs) and q_at < end) or
                (out_at < k_at + 2 * ((K - 1) * ks[0] + (nkv - 1) * ks[1] + hs) and k_at < end) or
                (out_at < v_at + 2 * ((K - 1) * vs[0] + (nkv - 1) * vs[1] + hs) and v_at < end)):
            _check_out(q, k, v, out)
    _check_device(q, k, v, out, cu_seqlens_q, cu_seqlens_k, lse)
    args = _hip.PromptArgs()
    _PACK.pack(args, q_at, qs[0], qs[1], k_at, ks[0], ks[1], v_at, vs[0], vs[1],
               cu_seqlens_q.data_ptr(), cu_seqlens_k.data_ptr(), cu_seqlens_q.shape[0] - 1, q.shape[0], k.shape[0],
               q.shape[1], k.shape[1], hs, _DTYPES[q.dtype],
               int(k.shape[0] if max_seqlen_k is None else min(max_seqlen_k, k.shape[0])), int(num_splits), int(causal),
               float(hs ** -0.5 if softmax_scale is None else softmax_scale), out_at, os[0], os[1],
               0 if lse is None else lse.data_ptr(), ls[0], ls[1], 0, 0)
    lib = _hip.lib()
    with _hip.on_device_of(q):
        need = lib.qp_prompt_workspace_size(args)
        if need > 0:
            ws = torch.empty(need, dtype=torch.uint8, device=q.device)
            args.workspace = ws.data_ptr()
            args.workspace_bytes = need
        _hip.check(lib.qp_prompt(args, _hip.stream_of(q)), "prompt_attention")
    return out
