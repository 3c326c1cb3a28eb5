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


# ----------------------------------------------------------------------------------- results where inputs are read

def _places(call, ok, message, **change):
    with pytest.raises(ValueError, match="on a GPU" if ok else message):  # (past the check: the next one refuses the CPU)
        call(**{name: (lambda x, t=t: t) for name, t in change.items()})


def test_prompt_out_shares_no_memory_but_that_of_q(lib):  # noqa: F811
    qkv = torch.zeros((6, 20 * 128), dtype=torch.bfloat16)
    q, k, v, rest = (x.unflatten(1, (-1, 128)) for x in qkv.split([8 * 128, 2 * 128, 2 * 128, 8 * 128], dim=1))
    q5, k5, v5 = q[:5], k[:5], v[:5]
    for out in (q5, rest[:5], torch.zeros((5, 8, 128), dtype=torch.bfloat16), q5.as_strided(q5.shape, q5.stride())):
        _places(_prompt, True, "", q=q5, k=k5, v=v5, out=out)
    late = qkv.flatten()[128:].as_strided((5, 8, 128), (20 * 128, 128, 1))
    for name, out in (("q", q[1:6]), ("q", late), ("k", k[:5, :1].as_strided((5, 8, 128), (20 * 128, 128, 1))),
                      ("v", v[:5, 1:].as_strided((5, 8, 128), (20 * 128, 128, 1)))):
        _places(_prompt, False, f"shares memory with {name}", q=q5, k=k5, v=v5, out=out)
    heads = torch.zeros((5, 8, 128), dtype=torch.bfloat16)  # (as many KV heads as query heads: k is q is out)
    _places(_prompt, False, "shares memory with k", q=heads, k=heads, v=torch.zeros_like(heads), out=heads)
    _places(_prompt, False, "with each other", out=torch.zeros((1, 8, 128), dtype=torch.bfloat16).expand(5, 8, 128))
    _places(_prompt, False, "a place for every row", lse=torch.zeros((5, 1)).expand(5, 8))
    one = torch.zeros((1, 8, 128), dtype=torch.bfloat16)  # (of one token: its stride says nothing)
    from vllm_quantpack.attention.prompt import prompt_attention
    with pytest.raises(ValueError, match="on a GPU"):
        prompt_attention(one, one[:, :2].clone(), one[:, :2].clone(), one.as_strided(one.shape, (8, 128, 1)), cu_seqlens_q=i32([0, 1]))


def test_previous_weights_are_out_or_apart(lib):  # noqa: F811
    from vllm_quantpack.attention.key_weights import key_weights
    buf = torch.zeros((2, 2, 2, 100))
    kc, ks = torch.zeros((3, 16, 2, 32), dtype=torch.uint8), torch.zeros((3, 16, 2))

    def call(out, previous, decay=1.0, length=40):
        key_weights(torch.zeros((2, 4, 64), dtype=torch.bfloat16), kc, ks, out, cu_seqlens_q=i32([0, 1, 2]), seqused_k=i32([40, 40]),
                    block_table=i32([[0, 1, 2], [0, 1, 2]]), max_seqlen_q=1, softmax_scale=0.1, previous=previous, decay=decay,
                    max_seqlen_k=length)

    out = buf[:, 0, :, :40]
    for previous in (out, buf[:, 1, :, :40], buf[:, 0, :, 40:80], out.as_strided(out.shape, out.stride()), torch.zeros((2, 2, 40))):
        with pytest.raises(ValueError, match="on a GPU"):
            call(out, previous)
    for previous in (buf[:, 0, :, 1:41], buf[:, 0, :, 39:79], buf.view(4, 2, 100)[1:3, :, :40], out[:1].expand(2, 2, 40)):
        with pytest.raises(ValueError, match="previous shares"):
            call(out, previous)
        with pytest.raises(ValueError, match="on a GPU"):
            call(out, previous, decay=0.0)  # (not read)
    with pytest.raises(ValueError, match="on a GPU"):
        call(out, buf[:, 0, :, 39:79], length=39)  # (entries that the call neither reads nor writes)
    with pytest.raises(ValueError, match="with each other"):
        call(torch.zeros((2, 1, 40)).expand(2, 2, 40), None)


def test_evictions_write_apart_from_what_they_read(lib):  # noqa: F811
    from vllm_quantpack.attention.eviction import evict_keys
    kc, ks = torch.zeros((6, 16, 2, 32), dtype=torch.uint8), torch.zeros((6, 16, 2))
    buf, lens = torch.zeros((1, 2, 100)), i32([48, 48, 48])

    def call(**change):
        kw = dict(seqused_k=lens[:1], block_table=i32([[0, 1, 2]]), new_block_table=i32([[3, 4]]), budget=32, max_seqlen_k=48)
        evict_keys(kc, kc, ks, ks, buf, **{**kw, **change})

    for change in (dict(new_weights=buf[..., 48:80]), dict(new_weights=buf[..., 60:]), dict(new_seqused_k=lens[1:2]),
                   dict(kept=buf[..., 48:].view(torch.int32))):
        with pytest.raises(ValueError, match="on a GPU"):
            call(**change)
    for change in (dict(new_weights=buf[..., 47:]), dict(new_weights=buf[..., :32]), dict(new_weights=buf),
                   dict(kept=buf[..., 20:60].view(torch.int32)), dict(new_seqused_k=lens[:1])):
        with pytest.raises(ValueError, match="other tensors"):
            call(**change)
    two = torch.zeros((2, 2, 48))
    with pytest.raises(ValueError, match="other tensors"):  # (shifted by one)
        evict_keys(kc, kc, ks, ks, two, seqused_k=lens[:2], new_seqused_k=lens[1:], block_table=i32([[0, 1, 2]] * 2),
                   new_block_table=i32([[3], [4]]), budget=16)
    for change in (dict(kept=torch.zeros((1, 1, 32), dtype=torch.int32).expand(1, 2, 32)),
                   dict(new_weights=torch.zeros((1, 1, 32)).expand(1, 2, 32))):
        with pytest.raises(ValueError, match="with each other"):
            call(**change)
