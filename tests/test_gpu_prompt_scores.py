"""prompt_attention where a row's probabilities span more than its operand's type holds, and where its scores are very large.

Tolerances: those derived in test_gpu_prompt, but that fp16 probabilities may lose less: a row's reference is set 7 log2 units
below its largest score, so the largest probability is at least 2^7, and so is the row's sum. One below 2^-14 loses up to 2^-25
absolutely, n of them n 2^-25 / 2^7 = n 2^-32 of max |v|."""
import math

import pytest

from qp_testlib import i32
from test_gpu_prompt import HEADS, exact

pytestmark = pytest.mark.gpu


def _type(name):
    import torch
    return {"bf16": torch.bfloat16, "fp16": torch.float16}[name]


@pytest.mark.parametrize("hs,nq,nkv", HEADS)
@pytest.mark.parametrize("num_splits", [0, 1, 3])
@pytest.mark.parametrize("nearest,farthest", [(16.8, 17.2), (17.4, 18.2)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_many_small_weights_beside_a_large_one(device, dtype, nearest, farthest, num_splits, hs, nq, nkv):
    """65536 keys some 17 nats below the first one, whose value is 0: they alone make the output."""
    import torch

    from vllm_quantpack.attention.prompt import prompt_attention
    dtype, n = _type(dtype), 65536
    g = torch.Generator(device=device).manual_seed(hs)
    q = torch.zeros((1, nq, hs), dtype=dtype, device=device)
    q[..., 0] = 1.0
    k = torch.randn((n, nkv, hs), generator=g, device=device).to(dtype)
    k[..., 0] = (farthest - nearest) * torch.rand((n, nkv), generator=g, device=device).to(dtype)
    k[0, :, 0] = farthest
    v = (torch.rand((n, nkv, hs), generator=g, device=device) + 0.5).to(dtype)
    v[0] = 0.0
    lse = torch.zeros((1, nq), device=device)
    out = prompt_attention(q, k, v, cu_seqlens_q=i32([0, 1], device), cu_seqlens_k=i32([0, n], device), softmax_scale=1.0,
                           lse=lse, num_splits=num_splits)
    want, wlse, mean, big = exact(q, k, v, 1.0, True)
    u, s = torch.finfo(dtype).eps / 2, (hs + 4) * 2 ** -24 * big
    tol = u * want.abs() + ((1 + u) * u + 2 * s + (n + 64) * 2 ** -23) * mean
    if dtype == torch.float16:
        tol = tol + n * 2 ** -32 * float(v.abs().max())
    off = (out.double().cpu() - want).abs()
    assert bool((off <= tol).all()), f"off by {float((off / tol).max()):.1f} tolerances, {float((off / want).max()):.3f} of the output"
    assert bool(((lse.double().cpu() - wlse).abs() <= s + (n + 64) * 2 ** -23 + wlse.abs() * 2 ** -23).all())


@pytest.mark.parametrize("hs,nq,nkv", HEADS)
@pytest.mark.parametrize("num_splits", [0, 3])
@pytest.mark.parametrize("shift", [0, 576])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_scores_of_ten_million(device, dtype, shift, num_splits, hs, nq, nkv):
    """Scores that are whole numbers times 16384, up to 10^7 (and down to -10^7 with the shift): their sums are exact, every key
    but those of the largest score is at least 16384 nats away, and the row is the mean of those keys' values.

    Equal scores give equal probabilities, so the rows' are off by no more than their rounding, u each, the output's u, and
    2^-20 for the exponential, sums over few keys and the quotient. The log-sum-exp takes six roundings of 2^-24."""
    import torch

    from vllm_quantpack.attention.prompt import prompt_attention
    dtype, n, scale = _type(dtype), 300, 16384.0
    g = torch.Generator(device=device).manual_seed(hs)
    q = torch.zeros((n, nq, hs), device=device)
    k = torch.zeros((n, nkv, hs), device=device)
    q[..., :16] = torch.randint(-8, 9, (n, nq, 16), generator=g, device=device).float()
    k[..., :16] = torch.randint(-8, 9, (n, nkv, 16), generator=g, device=device).float()
    q[..., 16], k[..., 16] = 32.0, -shift / 32.0   # (every score less by the same)
    q, k = q.to(dtype), k.to(dtype)
    v = torch.randn((n, nkv, hs), generator=g, device=device).to(dtype)
    lse = torch.zeros((n, nq), device=device)
    out = prompt_attention(q, k, v, cu_seqlens_q=i32([0, n], device), softmax_scale=scale, lse=lse, num_splits=num_splits)
    u, group = torch.finfo(dtype).eps / 2, nq // nkv
    a = torch.einsum("thc,jhc->htj", q.double().cpu(), k.double().cpu().repeat_interleave(group, 1))
    a = a.masked_fill(torch.ones((n, n)).triu(1).bool(), -math.inf)
    p = (a == a.amax(-1, keepdim=True)).double()
    p = p / p.sum(-1, keepdim=True)
    vv = v.double().cpu().repeat_interleave(group, 1)
    want, mean = torch.einsum("htj,jhc->thc", p, vv), torch.einsum("htj,jhc->thc", p, vv.abs())
    off = (out.double().cpu() - want).abs()
    assert bool((off <= u * want.abs() + ((1 + u) * u + 2 ** -20) * mean).all())
    wlse = (scale * a.amax(-1) + (1 / p.amax(-1)).log()).t()
    assert float(wlse.abs().max()) > 4e6
    assert bool(((lse.double().cpu() - wlse).abs() <= 6 * 2 ** -24 * wlse.abs() + 2 ** -20).all())
