"""Arguments of the operators of include/quantpack_ops.h that are looked at on the host, without a kernel running."""
import pytest
import torch

from test_ops_refusals import lib, weight_args  # noqa: F401  (the fixture)


def test_key_weights_of_sequences_without_pages(lib):  # noqa: F811
    """A block table of no columns holds no position: there is nothing to do, whether it has an address or not."""
    assert lib.qp_key_weights(weight_args(max_blocks=0), None) == 0
    assert lib.qp_key_weights(weight_args(max_blocks=0, block_table=None), None) == 0


# ------------------------------------------------------------------------------------------------- derivatives

def i32(x):
    return torch.tensor(x, dtype=torch.int32)


def _prompt(**change):
    from vllm_quantpack.attention.prompt import prompt_attention
    t = dict(q=torch.zeros((5, 8, 128), dtype=torch.bfloat16), k=torch.zeros((5, 2, 128), dtype=torch.bfloat16),
             v=torch.zeros((5, 2, 128), dtype=torch.bfloat16), out=torch.zeros((5, 8, 128), dtype=torch.bfloat16),
             lse=torch.zeros((5, 8)))
    t = {name: change.get(name, lambda x: x)(x) for name, x in t.items()}
    return prompt_attention(t["q"], t["k"], t["v"], t["out"], lse=t["lse"], cu_seqlens_q=i32([0, 5]))


def _weights(**change):
    from vllm_quantpack.attention.key_weights import key_weights
    t = dict(q=torch.zeros((1, 4, 64), dtype=torch.bfloat16), k_scale_cache=torch.zeros((3, 16, 2)), out=torch.zeros((1, 2, 40)),
             previous=torch.zeros((1, 2, 40)), query_signs=torch.ones(64))
    t = {name: change.get(name, lambda x: x)(x) for name, x in t.items()}
    return key_weights(t["q"], torch.zeros((3, 16, 2, 32), dtype=torch.uint8), t["k_scale_cache"], t["out"],
                       cu_seqlens_q=i32([0, 1]), seqused_k=i32([40]), block_table=i32([[0, 1, 2]]), max_seqlen_q=1,
                       softmax_scale=0.1, previous=t["previous"], query_signs=t["query_signs"])


def _evict(**change):
    from vllm_quantpack.attention.eviction import evict_keys
    t = dict(weights=torch.zeros((1, 2, 48)), new_weights=torch.zeros((1, 2, 32)), k_scale_cache=torch.zeros((6, 16, 2)),
             v_scale_cache=torch.zeros((6, 16, 2)))
    t = {name: change.get(name, lambda x: x)(x) for name, x in t.items()}
    kc = torch.zeros((6, 16, 2, 32), dtype=torch.uint8)
    return evict_keys(kc, kc, t["k_scale_cache"], t["v_scale_cache"], t["weights"], seqused_k=i32([48]),
                      block_table=i32([[0, 1, 2]]), new_block_table=i32([[3, 4]]), budget=32, new_weights=t["new_weights"])


CALLS = [(_prompt, n) for n in ("q", "k", "v", "out", "lse")] + \
        [(_weights, n) for n in ("q", "k_scale_cache", "out", "previous", "query_signs")] + \
        [(_evict, n) for n in ("weights", "new_weights", "k_scale_cache", "v_scale_cache")]


@pytest.mark.parametrize("call,name", CALLS)
def test_refuses_what_it_has_no_derivative_for(lib, call, name):  # noqa: F811
    """A result without the gradient or tangent that the argument carries would drop it without a word."""
    def grad(x):
        return x.clone().requires_grad_()

    with pytest.raises(NotImplementedError, match="backward"):
        call(**{name: grad})
    with torch.no_grad(), pytest.raises(ValueError, match="on a GPU"):  # (goes on to the next check)
        call(**{name: grad})
    with torch.autograd.forward_ad.dual_level():
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            call(**{name: lambda x: torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))})
        with pytest.raises(ValueError, match="on a GPU"):  # (no argument has a tangent)
            call()
