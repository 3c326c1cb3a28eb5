"""The attention weight that cached keys receive: what an eviction policy goes by.

`key_weights` reads the key half of an int4 or k8v4 paged cache and adds up, per KV head, the softmax probabilities that a
sequence's query tokens give each of its keys: after a decode step with that step's queries (with the weights so far as
`previous`), or once with the last tokens of a prompt. Attention itself keeps no probabilities, so this is a pass of its own
over the keys (`qp_key_weights`), about half of the cache.
"""
from __future__ import annotations

import torch

from .. import _hip

HEAD_SIZES = (64, 128, 256, 512)
_PACK = _hip.Packer(_hip.KeyWeightsArgs)


def _vector(name, t, length=None):
    if t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous() or (length is not None and t.shape[0] != length):
        raise ValueError(f"key_weights: {name} must be a contiguous int32 vector" +
                         ("" if length is None else f" of {length} entries"))


def _check_previous(previous, out, ps, os, length):
    """Weights are written while others are read: previous lies in out's place, entry for entry, or apart from it."""
    start, first = out.data_ptr(), previous.data_ptr()
    if start >= _hip.end_of(previous, ps) or first >= _hip.end_of(out, os):
        return
    if first == start and all(n == 1 or x == y for n, x, y in zip(out.shape, ps, os)):
        return
    if _hip.share_memory(previous[..., :max(length, 0)], out[..., :max(length, 0)]):
        raise ValueError("key_weights: previous shares memory with out but is not out")


def key_weights(q, k_cache, k_scale_cache, out, *, cu_seqlens_q, seqused_k, block_table, max_seqlen_q, max_seqlen_k=None,
                softmax_scale, query_signs=None, previous=None, decay=1.0) -> torch.Tensor:
    """out[i, g, j] = decay * previous[i, g, j] + the sum over sequence i's query tokens and the query heads of KV head g of
    the softmax probability of key j < seqused_k[i]; returns out. Entries from seqused_k[i] on are left as they are.

    q bf16 [T, NQ, hs] in the cache's domain, or unrotated with query_signs (`rht.signs`), which rotates each row as it
    loads; k_cache (blocks, bs, NKV, bytes) uint8 nibble pairs or int8 with its scale words k_scale_cache (the views of
    `k8v4_kv`; an int4 view's bytes past the codes are not read); out fp32 [sequences, NKV, L] with max_seqlen_k <= L (L
    when None); previous: None, or weights of the same shape (out itself for an update in place, else apart from it).
    softmax_scale multiplies q.k in the cache's domain, as in `prefill_attention`. A sequence's query tokens are the last of
    its positions and see the keys up to their own; the first max_seqlen_q of them are counted.

    A token that sees no key adds nothing, a sequence without tokens keeps its decayed weights, and a key on a page outside
    the cache gets none. The workspace comes from torch's caching allocator; no host synchronisation."""
    if q.dtype != torch.bfloat16:
        raise NotImplementedError(f"key_weights: bf16 queries only, got {q.dtype}")
    if q.dim() != 3 or q.stride(2) != 1:
        raise ValueError("key_weights: q must be [tokens, heads, head size] with contiguous channels")
    seqs, hs = seqused_k.shape[0], q.shape[2]
    if k_cache.dim() != 4 or k_cache.dtype not in (torch.uint8, torch.int8) or k_cache.stride(3) != 1:
        raise ValueError("key_weights: the key cache must be a (blocks, slots, heads, bytes) view of uint8 or int8 codes")
    nkv = k_cache.shape[2]
    widths = (hs,) if k_cache.dtype == torch.int8 else (hs // 2, hs // 2 + 4)  # (with the word's bytes behind the codes)
    if k_cache.shape[3] not in widths or k_scale_cache.shape != k_cache.shape[:3]:
        raise ValueError(f"key_weights: key codes {tuple(k_cache.shape)} and words {tuple(k_scale_cache.shape)} are not "
                         f"those of heads of {hs}")
    if out.dtype != torch.float32 or out.dim() != 3 or out.shape[:2] != (seqs, nkv) or out.stride(2) != 1:
        raise ValueError(f"key_weights: out must be fp32 [{seqs}, {nkv}, positions] with contiguous positions")
    if previous is not None and (previous.dtype != torch.float32 or previous.shape != out.shape or previous.stride(2) != 1):
        raise ValueError("key_weights: previous must be fp32, of out's shape, with contiguous positions")
    if max_seqlen_k is None:
        max_seqlen_k = out.shape[2]
    if max_seqlen_k > out.shape[2]:
        raise ValueError(f"key_weights: out has {out.shape[2]} positions, the longest context {max_seqlen_k}")
    os = out.stride()
    if 0 in os and _hip.repeats(out, os):
        raise ValueError("key_weights: rows of out share memory with each other")
    ps = (0, 0) if previous is None else previous.stride()
    if previous is not None and decay and (ps != os or previous.data_ptr() != out.data_ptr()):
        _check_previous(previous, out, ps, os, max_seqlen_k)
    _vector("seqused_k", seqused_k)
    _vector("cu_seqlens_q", cu_seqlens_q, seqs + 1)
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.shape[0] != seqs or block_table.stride(1) != 1:
        raise ValueError(f"key_weights: block_table must be int32 [{seqs}, blocks]")
    if query_signs is not None and (query_signs.dtype != torch.float32 or query_signs.shape != (hs,) or
                                    not query_signs.is_contiguous()):
        raise ValueError(f"key_weights: query_signs must be {hs} contiguous fp32 signs")
    _hip.no_derivatives("key_weights", q, k_scale_cache, out, previous, query_signs)
    index = q.get_device()
    if (index < 0 or not (index == k_cache.get_device() == k_scale_cache.get_device() == out.get_device() ==
                          cu_seqlens_q.get_device() == seqused_k.get_device() == block_table.get_device()) or
            (query_signs is not None and query_signs.get_device() != index) or
            (previous is not None and previous.get_device() != index)):
        _hip.same_device("key_weights", q, k_cache=k_cache, k_scale_cache=k_scale_cache, out=out, cu_seqlens_q=cu_seqlens_q,
                         seqused_k=seqused_k, block_table=block_table, query_signs=query_signs, previous=previous)
    if k_scale_cache.dtype not in _hip._WORD_DTYPES:
        raise ValueError(f"key_weights: scale words must be 4-byte elements, got {k_scale_cache.dtype}")
    cs, ws, qs = k_cache.stride(), k_scale_cache.stride(), q.stride()
    args = _hip.KeyWeightsArgs()
    _PACK.pack(args, k_cache.data_ptr(), cs[0], cs[1], cs[2], k_scale_cache.data_ptr(), ws[0], ws[1], ws[2],
               _hip.CODES_INT8 if k_cache.dtype == torch.int8 else _hip.CODES_INT4, k_cache.shape[0], k_cache.shape[1], nkv,
               hs, q.data_ptr(), qs[0], qs[1], cu_seqlens_q.data_ptr(), seqused_k.data_ptr(), block_table.data_ptr(),
               block_table.stride(0), block_table.shape[1], seqs, q.shape[0], q.shape[1],
               int(min(max_seqlen_q, q.shape[0])), int(max_seqlen_k), float(softmax_scale), float(decay),
               0 if query_signs is None else query_signs.data_ptr(), 0 if previous is None else previous.data_ptr(), ps[0],
               ps[1], out.data_ptr(), os[0], os[1], 0, 0)
    lib = _hip.lib()
    with _hip.on_device_of(q):
        need = lib.qp_key_weights_workspace_size(args)
        if need > 0:
            space = torch.empty(need, dtype=torch.uint8, device=q.device)
            args.workspace = space.data_ptr()
            args.workspace_bytes = need
        _hip.check(lib.qp_key_weights(args, _hip.stream_of(q)), "key_weights")
    return out
