"""Results written where an input lies, or beside one in the same buffer, where the operators allow it: the same bits as into
tensors of their own."""
import numpy as np
import pytest

from qp_testlib import i32, random_cache, torch_cache
from test_gpu_prompt import HEADS

pytestmark = pytest.mark.gpu


def _prompt_in_place(device, lens, hs, nq, nkv, num_splits, strided):
    import torch

    from vllm_quantpack.attention.prompt import prompt_attention
    g = torch.Generator(device=device).manual_seed(hs)
    T, K = sum(t for t, _ in lens), sum(n for _, n in lens)
    wide = torch.randn((T, 2 * nq if strided else nq, hs), generator=g, device=device).to(torch.bfloat16)
    q = wide[:, :nq]
    k, v = (torch.randn((K, nkv, hs), generator=g, device=device).to(torch.bfloat16) for _ in range(2))
    kw = dict(cu_seqlens_q=i32(np.cumsum([0] + [t for t, _ in lens]), device),
              cu_seqlens_k=i32(np.cumsum([0] + [n for _, n in lens]), device), max_seqlen_k=max(n for _, n in lens),
              num_splits=num_splits)
    want = prompt_attention(q, k, v, **kw)
    if strided:  # beside q, in the same rows
        assert torch.equal(prompt_attention(q, k, v, wide[:, nq:], **kw), want)
    assert prompt_attention(q, k, v, q, **kw) is q
    assert torch.equal(q, want)


@pytest.mark.parametrize("hs,nq,nkv", HEADS)
@pytest.mark.parametrize("num_splits", [0, 1, 3])
@pytest.mark.parametrize("strided", [False, True])
def test_prompt_in_the_queries_place(device, strided, num_splits, hs, nq, nkv):
    _prompt_in_place(device, [(70, 70), (1, 900), (33, 20), (130, 300)], hs, nq, nkv, num_splits, strided)


@pytest.mark.parametrize("hs", [64, 128])
def test_prompt_of_halved_keys_in_the_queries_place(device, hs):
    _prompt_in_place(device, [(700, 1300)], hs, 48, 24, 0, False)


@pytest.mark.parametrize("tokens", [1, 40])
def test_weights_beside_the_earlier_ones(device, tokens):
    import torch

    from vllm_quantpack.attention.key_weights import key_weights
    rng = np.random.default_rng(tokens)
    kv, _ = random_cache(rng, 40, 2, 16, 128)
    keep, (kc, _, ks, _) = torch_cache(kv, 128, "int4", device)
    q = torch.randn((2 * tokens, 8, 128), device=device).to(torch.bfloat16)
    kw = dict(cu_seqlens_q=i32([0, tokens, 2 * tokens], device), seqused_k=i32([300, 299], device), max_seqlen_q=tokens,
              block_table=i32(rng.permutation(40).reshape(2, 20), device), softmax_scale=0.05, decay=0.5, max_seqlen_k=300)
    buf = torch.rand((2, 2, 2, 300), device=device)
    want = key_weights(q, kc, ks, buf[:, 1].clone(), previous=buf[:, 0].clone(), **kw)
    key_weights(q, kc, ks, buf[:, 1], previous=buf[:, 0], **kw)
    assert torch.equal(buf[:, 1], want)
    key_weights(q, kc, ks, buf[:, 0], previous=buf[:, 0], **kw)
    assert torch.equal(buf[0, 0], want[0]) and torch.equal(buf[1, 0, :, :299], want[1, :, :299])


@pytest.mark.parametrize("n", [700, 9000])
def test_evicted_weights_beside_the_earlier_ones(device, n):
    import torch

    from vllm_quantpack.attention.eviction import evict_keys
    rng = np.random.default_rng(n)
    blocks = -(-n // 16)
    kv, _ = random_cache(rng, blocks + 20, 2, 16, 64)
    keep, views = torch_cache(kv, 64, "int4", device)
    buf = torch.rand((1, 2, n + 320), device=device)
    lens = i32([n, -1], device)
    kw = dict(seqused_k=lens[:1], block_table=i32([np.arange(blocks)], device), budget=320, max_seqlen_k=n, sinks=2, recent=9,
              new_block_table=i32([blocks + np.arange(20)], device))
    used, kept, weights = evict_keys(*views, buf[..., :n].clone(), **kw)
    cells = keep[blocks:].clone()
    got = evict_keys(*views, buf, new_weights=buf[..., n:], new_seqused_k=lens[1:], **kw)
    assert torch.equal(buf[..., n:], weights) and torch.equal(got[1], kept) and lens.tolist() == [n, 320]
    assert torch.equal(keep[blocks:], cells)
