"""The order that prompt_attention takes row blocks in, where the products of keys and heads are large."""
import pytest

from qp_testlib import i32

pytestmark = pytest.mark.gpu


def test_prompt_of_more_keys_than_the_longest_context_says(device):
    """2^22 + 97 keys under 512 query heads, 2^31 (key, head) pairs and more, where max_seqlen_k says 100 (it only lays out the
    work). Every key and value is the same, in numbers whose sums are exact."""
    import torch

    from vllm_quantpack.attention.prompt import prompt_attention
    hs, nq, lens = 64, 512, [(1, (1 << 22) + 97), (64, 64)]
    T, K = sum(t for t, _ in lens), sum(n for _, n in lens)
    q = torch.ones((T, nq, hs), dtype=torch.bfloat16, device=device)
    k = torch.zeros((1, 1, hs), dtype=torch.bfloat16, device=device).expand(K, 1, hs)
    row = torch.tensor([1.0, -1.0, 2.0, 0.5] * (hs // 4), dtype=torch.bfloat16, device=device)
    v = row.view(1, 1, hs).expand(K, 1, hs)
    out, lse = torch.full_like(q, 7.0), torch.zeros((T, nq), device=device)
    prompt_attention(q, k, v, out, cu_seqlens_q=i32([0, 1, 65], device), cu_seqlens_k=i32([0, lens[0][1], K], device),
                     max_seqlen_k=100, lse=lse, num_splits=1)
    torch.cuda.synchronize()
    assert bool((out == row).all())
    count = torch.tensor([lens[0][1]] + list(range(1, 65)), dtype=torch.float64)[:, None].log()
    assert bool(((lse.double().cpu() - count).abs() <= 6 * 2 ** -24 * count + 2 ** -20).all())
