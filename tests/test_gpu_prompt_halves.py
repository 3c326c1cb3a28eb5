"""prompt_attention where two groups of waves halve the keys of each row block, against the definition in 64 bits. That is so
where there are as many workgroups as CUs and at most half as many more, contexts of 1024 keys or more, heads of 64 or 128 and
row blocks of 128; every test asserts that it is there. Tolerances: those derived in test_gpu_prompt."""
import math

import numpy as np
import pytest

from qp_testlib import i32

pytestmark = pytest.mark.gpu


def halves(lens, nq, nkv, hs, max_seqlen_k):
    """Whether the call's row blocks are halved: the library's rules for splits, row blocks and groups."""
    import torch
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    tokens, seqs, group = sum(t for t, _ in lens), len(lens), nq // nkv
    rows = tokens * group
    if hs == 128 and (rows <= 32 * seqs or (rows > 128 * seqs and max(-(-rows // 256), seqs) * nkv >= 2 * cus)):
        return False  # (blocks of 256 rows)
    share = {0: 1, 4: 2, 2: 4, 6: 4}.get(nkv % 8, 8)
    blocks = -(-(rows // 128 + seqs) // share) * share
    return max(-(-rows // 128), seqs) * nkv >= cus and 2 * blocks * nkv <= 3 * cus and max_seqlen_k >= 1024 and hs in (64, 128)


def exact(q, k, v, scale, causal):
    """(out, lse, mean |v|, largest scale sum |q_i k_i|) of one sequence: out and mean [tokens, heads, hs], lse [tokens, heads]."""
    import torch
    tokens, keys, group = q.shape[0], k.shape[0], q.shape[1] // k.shape[1]
    q, k, v = (x.double().cpu().transpose(0, 1) for x in (q, k, v))
    k, v = k.repeat_interleave(group, 0), v.repeat_interleave(group, 0)
    if not keys:
        return torch.zeros_like(q).transpose(0, 1), torch.full(q.shape[:2], -math.inf).t(), torch.zeros_like(q).transpose(0, 1), 0.0
    a = scale * torch.bmm(q, k.transpose(1, 2).contiguous())
    if causal:
        a.masked_fill_(torch.arange(keys)[None, :] > torch.arange(tokens)[:, None] + keys - tokens, -math.inf)
    lse = torch.logsumexp(a, -1)
    p = (a - lse.masked_fill(lse == -math.inf, 0.0)[..., None]).exp()
    big = float(scale * torch.bmm(q.abs(), k.abs().transpose(1, 2).contiguous()).max()) if tokens else 0.0
    return torch.bmm(p, v).transpose(0, 1), lse.t(), torch.bmm(p, v.abs()).transpose(0, 1), big


def run(device, lens, nq, nkv, hs, dtype, causal, seed):
    import torch

    from vllm_quantpack.attention.prompt import prompt_attention
    dtype = {"bf16": torch.bfloat16, "fp16": torch.float16}[dtype]
    longest = max(n for _, n in lens)
    assert halves(lens, nq, nkv, hs, longest)
    g = torch.Generator(device=device).manual_seed(seed)
    T, K = sum(t for t, _ in lens), sum(n for _, n in lens)
    q = (torch.randn((T, nq, hs), generator=g, device=device) * 2).to(dtype)
    k, v = (torch.randn((K, nkv, hs), generator=g, device=device).to(dtype) for _ in range(2))
    out, lse = torch.full_like(q, 7.0), torch.full((T, nq), 7.0, device=device)
    prompt_attention(q, k, v, out, cu_seqlens_q=i32(np.cumsum([0] + [t for t, _ in lens]), device),
                     cu_seqlens_k=i32(np.cumsum([0] + [n for _, n in lens]), device), max_seqlen_k=longest, causal=causal, lse=lse)
    u, tq, tk = torch.finfo(dtype).eps / 2, 0, 0
    for t, n in lens:
        want, wlse, mean, big = exact(q[tq:tq + t], k[tk:tk + n], v[tk:tk + n], hs ** -0.5, causal)
        s = (hs + 4) * 2 ** -24 * big
        tol = u * want.abs() + ((1 + u) * u + 2 * s + (n + 64) * 2 ** -23) * mean
        if dtype == torch.float16 and n:
            tol = tol + n * 2 ** -32 * float(v.abs().max())
        off = (out[tq:tq + t].double().cpu() - want).abs()
        assert bool((off <= tol + 1e-30).all()), (t, n, float((off / (tol + 1e-30)).max()))
        got, seen = lse[tq:tq + t].double().cpu(), wlse != -math.inf
        assert bool((got[~seen] == -math.inf).all())
        assert bool(((got[seen] - wlse[seen]).abs() <= s + (n + 64) * 2 ** -23 + wlse[seen].abs() * 2 ** -23).all()), (t, n)
        tq, tk = tq + t, tk + n


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("hs", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_sequences_of_all_lengths(device, causal, hs, dtype):
    """Contexts of one tile (whose second half is empty) and of none, halves that end in the middle of a tile, rows that see
    nothing, a sequence without queries; causal ones are taken longest first."""
    run(device, [(700, 1300), (1, 1100), (257, 257), (0, 40), (40, 64), (60, 65), (13, 10), (2, 0)], 32, 16, hs, dtype, causal, hs)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("hs", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("keys", [1024, 1300, 1345])
def test_one_sequence(device, keys, causal, hs, dtype):
    """One prompt after earlier keys: its blocks are taken in their order."""
    run(device, [(700, keys)], 48, 24, hs, dtype, causal, keys)


@pytest.mark.parametrize("hs", [64, 128])
def test_many_sequences(device, hs):
    """More sequences than are ordered by length, each with a row block of its own."""
    lens = [(20 + i, 30 + 70 * i) for i in range(12)] + [(3, 1200)]
    run(device, lens, 40, 20, hs, "bf16", True, hs)


@pytest.mark.parametrize("hs", [64, 128])
@pytest.mark.parametrize("at", [20, 640, 700, 1290])
def test_an_infinite_value(device, hs, at):
    """The rows that see it have it, the others and the other channels what the definition says without it."""
    import torch

    from vllm_quantpack.attention.prompt import prompt_attention
    T, K, nq, nkv = 700, 1300, 48, 24
    assert halves([(T, K)], nq, nkv, hs, K)
    g = torch.Generator(device=device).manual_seed(at)
    q = torch.randn((T, nq, hs), generator=g, device=device).to(torch.bfloat16)
    k, v = (torch.randn((K, nkv, hs), generator=g, device=device).to(torch.bfloat16) for _ in range(2))
    v[at, :, 3] = 0.0
    want, _, mean, big = exact(q, k, v, hs ** -0.5, True)
    v[at, :, 3] = -math.inf
    got = prompt_attention(q, k, v, cu_seqlens_q=i32([0, T], device), cu_seqlens_k=i32([0, K], device)).double().cpu()
    see = torch.arange(T) + K - T >= at
    assert bool((got[see][..., 3] == -math.inf).all())
    got[see, :, 3] = want[see, :, 3]
    u = torch.finfo(torch.bfloat16).eps / 2
    tol = u * want.abs() + ((1 + u) * u + 2 * (hs + 4) * 2 ** -24 * big + (K + 64) * 2 ** -23) * mean
    assert bool(((got - want).abs() <= tol).all())
