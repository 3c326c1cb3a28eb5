"""key_weights where there is nothing to see."""
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
