"""key_weights where there is nothing to see, and where a query is no number."""
import numpy as np
import pytest

from qp_testlib import i32, random_cache, torch_cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens", [1, 40])
def test_weights_of_sequences_without_pages(device, tokens):
    """A block table of no columns holds no position: nothing is seen, and every entry is left as it was."""
    import torch

    from vllm_quantpack.attention.key_weights import key_weights
    kv, _ = random_cache(np.random.default_rng(1), 3, 2, 16, 64)
    keep, (kc, _, ks, _) = torch_cache(kv, 64, "int4", device)
    q = torch.randn((tokens, 4, 64), device=device).to(torch.bfloat16)
    table = i32([[0, 1, 2]], device)
    for none in (table[:, :0], torch.empty((1, 0), dtype=torch.int32, device=device)):
        out = torch.full((1, 2, 40), 7.0, device=device)
        key_weights(q, kc, ks, out, cu_seqlens_q=i32([0, tokens], device), seqused_k=i32([40], device), block_table=none,
                    max_seqlen_q=tokens, softmax_scale=0.1, previous=torch.ones_like(out))
        torch.cuda.synchronize()
        assert bool((out == 7.0).all())


@pytest.mark.parametrize("fmt,tokens", [("int4", 3), ("int8", 3), ("int4", 40), ("int8", 40)])
@pytest.mark.parametrize("bad", [0, 1, -1])
def test_weights_of_a_query_that_is_no_number(device, fmt, tokens, bad):
    """A query of NaN gives NaN to the keys that it sees, and nothing to the others: keys after it, and pages that do not exist."""
    import torch

    from vllm_quantpack.attention.key_weights import key_weights
    rng = np.random.default_rng(tokens)
    hs, n, row = 128, 300, bad % tokens
    kv, _ = random_cache(rng, 20, 2, 16, hs, fmt)
    keep, (kc, _, ks, _) = torch_cache(kv, hs, fmt, device)
    table = rng.permutation(20)[:19].astype(np.int32)
    table[3] = -1
    q = torch.randn((tokens, 4, hs), device=device).to(torch.bfloat16)
    kw = dict(cu_seqlens_q=i32([0, tokens], device), seqused_k=i32([n], device), block_table=i32([table], device),
              max_seqlen_q=tokens, softmax_scale=0.02)
    want = key_weights(q, kc, ks, torch.zeros((1, 2, n), device=device), **kw)
    q[row, 1] = float("nan")  # (a head of the first KV head)
    got = key_weights(q, kc, ks, torch.zeros((1, 2, n), device=device), **kw)
    torch.cuda.synchronize()
    sees = n - tokens + row + 1
    gone = torch.zeros(n, dtype=torch.bool, device=device)
    gone[48:64] = True
    assert bool((got[..., gone] == 0).all())
    assert bool(got[0, 0, :sees][~gone[:sees]].isnan().all())
    assert bool(got[0, 0, sees:].isfinite().all()) and torch.equal(got[0, 1], want[0, 1])
