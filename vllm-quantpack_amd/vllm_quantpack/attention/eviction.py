"""Eviction from the int4 / k8v4 paged cache by accumulated attention weight (`qp_evict`).

A long context's cache is cut down to a budget per sequence: every KV head keeps its own keys of largest weight, with the
first and the last positions. The kept cells move, packed as they are, to new blocks in the order of their positions, so
that the ordinary attention and store go on over the new block table and length, and the old blocks can be freed (other
sequences that share them are not touched). Keys carry their position with them: rotary embeddings are applied before the
store, and the engine goes on counting positions by itself.
"""
from __future__ import annotations

import torch

from .. import _hip

_PACK = _hip.Packer(_hip.EvictArgs)


def _table(name, t, seqs):
    if t.dtype != torch.int32 or t.dim() != 2 or t.shape[0] != seqs or t.stride(1) != 1:
        raise ValueError(f"evict_keys: {name} must be int32 [{seqs}, blocks]")


def _rows(name, t, dtype, seqs, nkv, length):
    shape = t.shape
    if (t.dtype != dtype or len(shape) != 3 or shape[0] != seqs or shape[1] != nkv or shape[2] < length or
            t.stride(2) != 1):
        raise ValueError(f"evict_keys: {name} must be {dtype} [{seqs}, {nkv}, {length} or more], contiguous in the last "
                         f"dimension, got {t.dtype} {tuple(t.shape)}")


def _check_places(weights, written, name, length, budget):
    """Places and weights are written while the weights are read, each by a workgroup of its own. (The two tensors' extents
    meet.)"""
    if _hip.share_memory(weights[..., :max(length, 0)], written[..., :max(budget, 0)]):
        raise ValueError(f"evict_keys: weights are read while {name} are written: give other tensors")


def evict_keys(k_cache, v_cache, k_scale_cache, v_scale_cache, weights, *, seqused_k, block_table, new_block_table, budget,
               max_seqlen_k=None, sinks=0, recent=0, kept=None, new_weights=None, new_seqused_k=None):
    """Keep min(seqused_k[i], budget) keys of every sequence i and KV head: the first `sinks`, the last `recent` and, of the
    others, those of largest weight (of equal ones the lower positions; NaN as the smallest). weights fp32 [sequences, NKV,
    L] (`key_weights`), max_seqlen_k <= L (L when None).

    The kept cells go to slots 0, 1, .. of new_block_table[i] (int32 [sequences, blocks], room for the budget, of blocks
    that no sequence of the call still uses), in the order of their positions. Returns (new_seqused_k int32 [sequences],
    kept int32 [sequences, NKV, budget] with the old positions, new_weights fp32 [sequences, NKV, budget] with their
    weights), made when None, with -1 and 0 past a sequence's count; given ones are left as they are there. Given
    ones share no memory with seqused_k and weights.

    No host synchronisation; the workspace comes from torch's caching allocator."""
    if k_cache.dim() != 4 or v_cache.dim() != 4 or k_cache.stride(3) != 1 or v_cache.stride(3) != 1:
        raise ValueError("evict_keys: the cache views must be (blocks, slots, heads, bytes) with contiguous bytes")
    k_shape, v_shape = k_cache.shape, v_cache.shape
    places, seqs, nkv = k_shape[:3], seqused_k.shape[0], k_shape[2]
    hs = v_shape[3] // 8 * 16  # (an int4 half's view may have its word's 4 bytes behind the codes)
    if (v_shape[:3] != places or k_scale_cache.shape != places or v_scale_cache.shape != places or
            (k_shape[3] if k_cache.dtype == torch.int8 else k_shape[3] // 8 * 16) != hs):
        raise ValueError("evict_keys: the four cache views do not belong together")
    if seqused_k.dtype != torch.int32 or seqused_k.dim() != 1 or not seqused_k.is_contiguous():
        raise ValueError("evict_keys: seqused_k must be a contiguous int32 vector")
    budget, sinks, recent = int(budget), int(sinks), int(recent)
    if max_seqlen_k is None:
        max_seqlen_k = weights.shape[-1]
    _rows("weights", weights, torch.float32, seqs, nkv, max_seqlen_k)
    _table("block_table", block_table, seqs)
    _table("new_block_table", new_block_table, seqs)
    dev = k_cache.device
    if kept is None:
        kept = torch.full((seqs, nkv, max(budget, 0)), -1, dtype=torch.int32, device=dev)
    if new_weights is None:
        new_weights = torch.zeros((seqs, nkv, max(budget, 0)), dtype=torch.float32, device=dev)
    if new_seqused_k is None:
        new_seqused_k = torch.empty(seqs, dtype=torch.int32, device=dev)
    _rows("kept", kept, torch.int32, seqs, nkv, budget)
    _rows("new_weights", new_weights, torch.float32, seqs, nkv, budget)
    if new_seqused_k.dtype != torch.int32 or new_seqused_k.shape != (seqs,) or not new_seqused_k.is_contiguous():
        raise ValueError(f"evict_keys: new_seqused_k must be {seqs} contiguous int32 entries")
    _hip.no_derivatives("evict_keys", weights, new_weights, k_scale_cache, v_scale_cache)
    table_at, new_table_at, used_at, new_used_at = (block_table.data_ptr(), new_block_table.data_ptr(), seqused_k.data_ptr(),
                                                    new_seqused_k.data_ptr())
    if seqs and block_table.numel() and new_table_at == table_at:
        raise ValueError("evict_keys: the kept cells move to other blocks: new_block_table must not be block_table")
    ws, ks, ns = weights.stride(), kept.stride(), new_weights.stride()
    if (0 in ks and _hip.repeats(kept, ks)) or (0 in ns and _hip.repeats(new_weights, ns)):
        raise ValueError("evict_keys: rows of kept or new_weights share memory with each other")
    weights_at, kept_at, new_weights_at = weights.data_ptr(), kept.data_ptr(), new_weights.data_ptr()
    if seqs:
        end = weights_at + 4 * ((seqs - 1) * ws[0] + (nkv - 1) * ws[1] + weights.shape[2])
        if kept_at < end and weights_at < kept_at + 4 * ((seqs - 1) * ks[0] + (nkv - 1) * ks[1] + kept.shape[2]):
            _check_places(weights, kept, "kept", max_seqlen_k, budget)
        if (new_weights_at < end and
                weights_at < new_weights_at + 4 * ((seqs - 1) * ns[0] + (nkv - 1) * ns[1] + new_weights.shape[2])):
            _check_places(weights, new_weights, "new_weights", max_seqlen_k, budget)
    if seqs and new_used_at < used_at + 4 * seqs and used_at < new_used_at + 4 * seqs:
        raise ValueError("evict_keys: seqused_k is read while the new one is written: give other tensors")
    index = k_cache.get_device()
    if index < 0 or not (index == v_cache.get_device() == k_scale_cache.get_device() == v_scale_cache.get_device() ==
                         weights.get_device() == seqused_k.get_device() == block_table.get_device() ==
                         new_block_table.get_device() == kept.get_device() == new_weights.get_device() ==
                         new_seqused_k.get_device()):
        _hip.same_device("evict_keys", k_cache, v_cache=v_cache, k_scale_cache=k_scale_cache, v_scale_cache=v_scale_cache,
                         weights=weights, seqused_k=seqused_k, block_table=block_table, new_block_table=new_block_table,
                         kept=kept, new_weights=new_weights, new_seqused_k=new_seqused_k)
    cache = _hip.paged_cache(k_cache, v_cache, k_scale_cache, v_scale_cache, hs)
    args = _hip.EvictArgs()
    _PACK.pack(args, weights_at, ws[0], ws[1], used_at, table_at, block_table.stride(0), new_table_at,
               new_block_table.stride(0), block_table.shape[1], new_block_table.shape[1], seqs, int(max_seqlen_k), budget,
               sinks, recent, kept_at, ks[0], ks[1], new_weights_at, ns[0], ns[1], new_used_at, 0, 0)
    lib = _hip.lib()
    with _hip.on_device_of(k_cache):
        need = lib.qp_evict_workspace_size(cache, args)
        space = torch.empty(max(need, 8), dtype=torch.uint8, device=dev)
        args.workspace = space.data_ptr()
        args.workspace_bytes = need
        _hip.check(lib.qp_evict(cache, args, _hip.stream_of(k_cache)), "evict_keys")
    return new_seqused_k, kept, new_weights
