"""prompt_attention against the definition in 64 bits.

Tolerance of an output: it is rounded to the tensors' type, off by at most u |out| with u half a step of the type (2^-8 in
bf16, 2^-11 in fp16), and so is every probability that enters the second product. With A = sum p |v| / sum p the rounded
probabilities move the sum by at most u A, so |out - exact| <= u |exact| + (1 + u) u A. The fp32 part: scores are sums of hs
exact products, off by at most (hs + 4) 2^-24 B with B = the largest scale * sum |q_i k_i|, which moves every probability by that
share, in the sum and in its normaliser: 2 (hs + 4) 2^-24 B A; exponentials, sums over n keys (in any order) and the merge add
less than (n + 64) 2^-23 A. The log-sum-exp is off by (hs + 4) 2^-24 B + (n + 64) 2^-23 + |lse| 2^-23. fp16: a probability below
2^-14 of the type's range loses up to 2^-25 absolutely, and the largest one is at least 2^0: n 2^-25 A' more, A' = max |v|.
"""
import math

import pytest

pytestmark = pytest.mark.gpu


def exact(q, k, v, scale, causal):
    """(out, lse, A, B) of one sequence in 64 bits on the CPU: q [tokens, heads, hs], k and v [keys, kv heads, hs]."""
    import torch
    group = q.shape[1] // k.shape[1]
    q, k, v = (x.double().cpu().transpose(0, 1) for x in (q, k, v))
    tokens, keys = q.shape[1], k.shape[1]
    sight = torch.ones((tokens, keys), dtype=torch.bool)
    if causal:
        sight = torch.arange(keys)[None, :] <= torch.arange(tokens)[:, None] + keys - tokens
    out, lse = torch.zeros_like(q), torch.full(q.shape[:2], -math.inf, dtype=torch.float64)
    mean, big = torch.zeros_like(q), 0.0
    for h in range(q.shape[0]):
        kk, vv = k[h // group], v[h // group]
        for t in range(tokens):
            see = sight[t]
            if not bool(see.any()):
                continue
            a = scale * (kk[see] @ q[h, t])
            lse[h, t] = torch.logsumexp(a, 0)
            p = (a - lse[h, t]).exp()
            out[h, t] = (p[:, None] * vv[see]).sum(0)
            mean[h, t] = (p[:, None] * vv[see].abs()).sum(0)
            big = max(big, float(scale * (kk[see].abs() @ q[h, t].abs()).max()))
    return out.transpose(0, 1), lse.transpose(0, 1), mean.transpose(0, 1), big


def check(got, lse, q, k, v, scale, causal, dtype):
    import torch
    want, wlse, mean, big = exact(q, k, v, scale, causal)
    hs, n = q.shape[2], k.shape[0]
    u = torch.finfo(dtype).eps / 2
    s = (hs + 4) * 2 ** -24 * big
    tol = u * want.abs() + ((1 + u) * u + 2 * s + (n + 64) * 2 ** -23) * mean
    if dtype == torch.float16:
        tol = tol + n * 2 ** -25 * float(v.abs().max()) if n else tol
    diff = (got.double().cpu() - want).abs()
    assert bool((diff <= tol + 1e-30).all()), f"out off by {float((diff / (tol + 1e-30)).max()):.2f} tolerances"
    if lse is not None:
        got = lse.double().cpu()
        empty = wlse == -math.inf
        assert bool((got[empty] == -math.inf).all())
        ltol = s + (n + 64) * 2 ** -23 + wlse[~empty].abs() * 2 ** -23
        assert bool(((got[~empty] - wlse[~empty]).abs() <= ltol).all())


def cu(lens, device):
    import torch
    return torch.tensor([0] + list(lens), dtype=torch.int32).cumsum(0, dtype=torch.int32).to(device)


def run(device, lens, nq, nkv, hs, dtype, causal=True, seed=0, num_splits=0, spread=2.0, extra=0):
    """One call on a batch of (tokens, keys), every sequence checked; `extra` rows of q, k and v of no sequence."""
    import torch

    from vllm_quantpack.attention.prompt import prompt_attention
    g = torch.Generator(device=device).manual_seed(seed)
    T, K = sum(t for t, _ in lens) + extra, sum(n for _, n in lens) + extra
    q = (torch.randn((T, nq, hs), generator=g, device=device) * spread).to(dtype)
    k, v = (torch.randn((K, nkv, hs), generator=g, device=device).to(dtype) for _ in range(2))
    out, lse = torch.full_like(q, 7.0), torch.full((T, nq), 7.0, device=device)
    ret = prompt_attention(q, k, v, out, cu_seqlens_q=cu([t for t, _ in lens], device),
                           cu_seqlens_k=cu([n for _, n in lens], device), max_seqlen_k=max([n for _, n in lens] + [0]),
                           causal=causal, lse=lse, num_splits=num_splits)
    torch.cuda.synchronize()
    assert ret is out
    tq = tk = 0
    for t, n in lens:
        check(out[tq:tq + t], lse[tq:tq + t], q[tq:tq + t], k[tk:tk + n], v[tk:tk + n], hs ** -0.5, causal, dtype)
        tq, tk = tq + t, tk + n
    assert bool((out[tq:] == 7.0).all()) and bool((lse[tq:] == 7.0).all())


def _type(name):
    import torch
    return {"bf16": torch.bfloat16, "fp16": torch.float16}[name]


HEADS = [(64, 8, 2), (128, 8, 2), (256, 6, 1), (512, 4, 2)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("hs,nq,nkv", HEADS)
@pytest.mark.parametrize("tokens", [1, 2, 31, 64, 65, 130])
def test_one_prompt(device, tokens, hs, nq, nkv, dtype):
    run(device, [(tokens, tokens)], nq, nkv, hs, _type(dtype), seed=tokens)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("hs,nq,nkv", HEADS)
@pytest.mark.parametrize("causal", [True, False])
def test_packed_sequences(device, causal, hs, nq, nkv, dtype):
    """Lengths from one token on, a sequence without queries, one without keys, more queries than keys (whose first rows see
    nothing), and rows of no sequence."""
    run(device, [(5, 5), (0, 40), (70, 70), (1, 1), (33, 97), (9, 4), (3, 0), (64, 64)], nq, nkv, hs, _type(dtype),
        causal=causal, seed=hs, extra=3)


@pytest.mark.parametrize("nq,nkv", [(1, 1), (7, 7), (5, 1), (33, 1), (28, 4)])
def test_groups(device, nq, nkv):
    run(device, [(45, 45), (20, 83)], nq, nkv, 128, _type("bf16"), seed=nq)


@pytest.mark.parametrize("hs,nq,nkv", HEADS)
@pytest.mark.parametrize("splits", [0, 1, 3, 16, 128])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_few_rows_over_many_keys(device, dtype, splits, hs, nq, nkv):
    run(device, [(1, 1300), (2, 70), (1, 0), (4, 999)], nq, nkv, hs, _type(dtype), seed=splits, num_splits=splits)


@pytest.mark.parametrize("hs,nq,nkv", HEADS)
def test_large_scores(device, hs, nq, nkv):
    """Scores of several hundred, rising along the keys: the running maximum is raised again and again."""
    import torch

    from vllm_quantpack.attention.prompt import prompt_attention
    for dtype in (torch.bfloat16, torch.float16):
        n = 200
        g = torch.Generator(device=device).manual_seed(5)
        q = torch.randn((n, nq, hs), generator=g, device=device).to(dtype)
        ramp = torch.linspace(0.2, 8, n, device=device)[:, None, None]
        k = (torch.randn((n, nkv, hs), generator=g, device=device) * ramp).to(dtype)
        v = torch.randn((n, nkv, hs), generator=g, device=device).to(dtype)
        lse = torch.empty((n, nq), device=device)
        out = prompt_attention(q, k, v, cu_seqlens_q=cu([n], device), softmax_scale=1.0, lse=lse)
        check(out, lse, q, k, v, 1.0, True, dtype)


@pytest.mark.parametrize("hs,nq,nkv", HEADS)
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_values_out_of_sight(device, dtype, hs, nq, nkv):
    """NaN and infinities in keys and values that a row does not see: later keys of its sequence, and the next sequence's."""
    import torch

    from vllm_quantpack.attention.prompt import prompt_attention
    dtype = _type(dtype)
    g = torch.Generator(device=device).manual_seed(9)
    lens = [70, 41]
    q, k, v = (torch.randn((sum(lens), h, hs), generator=g, device=device).to(dtype) for h in (nq, nkv, nkv))
    clean = prompt_attention(q, k, v, cu_seqlens_q=cu(lens, device))
    for at in (69, 40, 71):
        for bad in (math.nan, math.inf, -math.inf):
            kb, vb = k.clone(), v.clone()
            kb[at, :, 1], vb[at, :, 3] = bad, bad
            out = prompt_attention(q, kb, vb, cu_seqlens_q=cu(lens, device))
            torch.cuda.synchronize()
            end = lens[0] if at < lens[0] else sum(lens)
            untouched = torch.ones(sum(lens), dtype=torch.bool)
            untouched[at:end] = False
            assert torch.equal(out[untouched], clean[untouched]), (at, bad)
            # the value alone is odd: the rows that see it have it in its channel, and only there
            out = prompt_attention(q, k, vb, cu_seqlens_q=cu(lens, device))
            assert torch.equal(out[untouched], clean[untouched])
            seen = out[at:end, :, 3].float()
            assert bool(seen.isnan().all() if math.isnan(bad) else (seen == bad).all()), (at, bad)
            rest = [c for c in range(hs) if c != 3]
            assert torch.equal(out[at:end][..., rest], clean[at:end][..., rest])


def test_strides(device):
    """q, k and v as views of one projection's output, and out and lse inside larger tensors."""
    import torch

    from vllm_quantpack.attention.prompt import prompt_attention
    nq, nkv, hs, n = 8, 2, 128, 90
    g = torch.Generator(device=device).manual_seed(3)
    qkv = torch.randn((n, (nq + 2 * nkv) * hs), generator=g, device=device).to(torch.bfloat16)
    q, k, v = (x.unflatten(1, (-1, hs)) for x in qkv.split([nq * hs, nkv * hs, nkv * hs], dim=1))
    wide = torch.full((n, 2 * nq, hs + 8), 5.0, dtype=torch.bfloat16, device=device)
    out = wide[:, ::2, 8:]
    lse = torch.zeros((nq, n), device=device).t()
    prompt_attention(q, k, v, out, cu_seqlens_q=cu([n], device), lse=lse)
    check(out, lse, q, k, v, hs ** -0.5, True, torch.bfloat16)
    assert bool((wide[:, 1::2] == 5.0).all()) and bool((wide[..., :8] == 5.0).all())
    # heads before tokens in memory
    kt, vt = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (k, v))
    assert torch.equal(prompt_attention(q, kt, vt, cu_seqlens_q=cu([n], device)), out)


def test_same_bits_and_graph(device):
    """The same bits at every call, and in replays of a captured one between eager calls (with splits: 2 calls share no
    workspace)."""
    import torch

    from vllm_quantpack.attention.prompt import prompt_attention
    g = torch.Generator(device=device).manual_seed(4)
    nq, nkv, hs = 8, 2, 128
    q = torch.randn((3, nq, hs), generator=g, device=device).to(torch.bfloat16)
    k, v = (torch.randn((3000, nkv, hs), generator=g, device=device).to(torch.bfloat16) for _ in range(2))
    cq, ck = cu([1, 2], device), cu([1000, 2000], device)
    out = torch.zeros_like(q)

    def call(q, out):
        return prompt_attention(q, k, v, out, cu_seqlens_q=cq, cu_seqlens_k=ck, max_seqlen_k=2000)

    want = call(q, torch.zeros_like(q)).clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(q, out)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        call(q, out)
    for i in range(4):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
        assert torch.equal(call(q, torch.zeros_like(q)), want)
        q.mul_(0.5)
        want = call(q, torch.zeros_like(q)).clone()
        torch.cuda.synchronize()


def test_another_stream(device):
    import torch

    from vllm_quantpack.attention.prompt import prompt_attention
    g = torch.Generator(device=device).manual_seed(6)
    q, k, v = (torch.randn((300, h, 64), generator=g, device=device).to(torch.float16) for h in (4, 2, 2))
    want = prompt_attention(q, k, v, cu_seqlens_q=cu([300], device))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = prompt_attention(q, k, v, cu_seqlens_q=cu([300], device))
    side.synchronize()
    assert torch.equal(got, want)
