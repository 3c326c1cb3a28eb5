"""Calls of prompt_attention, key_weights and evict_keys at the ends of what they allow: many sequences, several blocks of keys
per workgroup, offsets past 32 bits, streams that run at once, captured calls of every path. Tolerances are those derived at the
top of each operator's own tests; copies and repeated calls are compared bit by bit."""
import numpy as np
import pytest

from qp_testlib import i32, random_cache, torch_cache
from test_gpu_evict import expected
from test_gpu_evict import run as run_evict
from test_gpu_key_weights import run as run_weights
from test_gpu_prompt import check as check_prompt
from test_gpu_prompt import run as run_prompt

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------------------------- prompt_attention

@pytest.mark.parametrize("num_splits", [0, 1, 3])
@pytest.mark.parametrize("count", [62, 63, 64, 130])
def test_prompt_of_many_sequences(device, count, num_splits):
    """Around 63 sequences, which a workgroup looks at in one go, and more; some without queries or keys."""
    import torch
    rng = np.random.default_rng(count)
    lens = [(int(t), int(n)) for t, n in zip(rng.integers(0, 4, count), rng.integers(0, 70, count))]
    lens[0], lens[-1], lens[61] = (0, 5), (2, 40), (3, 0)
    run_prompt(device, lens, 4, 2, 64, torch.float16, num_splits=num_splits, seed=count, extra=3)


def test_prompt_groups_past_a_row_tile(device):
    """40 query heads per KV head: a token's rows lie in two row tiles."""
    import torch
    run_prompt(device, [(7, 100), (1, 3)], 80, 2, 128, torch.bfloat16, seed=5)
    run_prompt(device, [(3, 50)], 130, 1, 512, torch.bfloat16, seed=6)


@pytest.mark.parametrize("dtype,causal", [("bf16", True), ("fp16", False)])
def test_prompt_of_many_rows(device, dtype, causal):
    """Enough rows, of enough sequences, for the larger row blocks; blocks that are full, and some with a row in them."""
    import torch
    rng = np.random.default_rng(11)
    lens = [(int(t), int(t + n)) for t, n in zip(rng.integers(25, 50, 64), rng.integers(0, 90, 64))]
    lens[3], lens[9], lens[20], lens[63] = (300, 333), (64, 64), (129, 100), (1, 77)
    run_prompt(device, lens, 32, 8, 128, {"bf16": torch.bfloat16, "fp16": torch.float16}[dtype], causal=causal, seed=2)


@pytest.mark.parametrize("hs,nq,nkv", [(64, 16, 16), (128, 32, 16), (256, 16, 16), (512, 16, 8)])
def test_prompts_by_length(device, hs, nq, nkv):
    """Few sequences of many row blocks: earlier keys, none, fewer keys than queries, no queries, equal lengths. The longest
    context's bound only decides the order of the blocks, whatever it says."""
    import torch

    from vllm_quantpack.attention.prompt import prompt_attention
    lens = [(300, 300), (0, 70), (257, 900), (400, 130), (1, 512), (300, 300), (420, 421)]
    run_prompt(device, lens, nq, nkv, hs, torch.bfloat16, num_splits=1, seed=hs, extra=2)
    T, K = sum(t for t, _ in lens), sum(n for _, n in lens)
    g = torch.Generator(device=device).manual_seed(3)
    q = torch.randn((T, nq, hs), generator=g, device=device).to(torch.float16)
    k, v = (torch.randn((K, nkv, hs), generator=g, device=device).to(torch.float16) for _ in range(2))
    offsets = [i32(np.concatenate(([0], np.cumsum([x[i] for x in lens]))), device) for i in range(2)]

    def call(bound):
        return prompt_attention(q, k, v, cu_seqlens_q=offsets[0], cu_seqlens_k=offsets[1], max_seqlen_k=bound, num_splits=1)

    want = torch.cat([prompt_attention(q[a:b], k[c:d], v[c:d], cu_seqlens_q=i32([0, b - a], device),
                                       cu_seqlens_k=i32([0, d - c], device), num_splits=1)
                      for a, b, c, d in zip(offsets[0][:-1].tolist(), offsets[0][1:].tolist(), offsets[1][:-1].tolist(),
                                            offsets[1][1:].tolist()) if b > a])
    for bound in (0, 1, 64, 900, K):
        got = call(bound)
        assert bool(torch.isfinite(got.float()).all())
        # (a sequence for itself may have its rows in other blocks, whose running maxima differ: two results, each off by u of
        # itself and u of the mean |v|, u = 2^-11, and by far less for its fp32 part)
        assert torch.allclose(got.float(), want.float(), rtol=2 ** -10, atol=2 ** -10 * float(v.abs().max())), bound
        assert torch.equal(got, call(900)), bound


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("hs", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_prompt_of_halved_keys(device, causal, hs, dtype):
    """As many row blocks as CUs over long contexts, whose keys are halved between a workgroup's waves; contexts of one tile,
    and of none, among them."""
    import torch
    lens = [(300, 1300), (1, 1100), (257, 257), (0, 40), (40, 64), (60, 65), (130, 100), (2, 0)]
    run_prompt(device, lens, 48, 24, hs, {"bf16": torch.bfloat16, "fp16": torch.float16}[dtype], causal=causal, seed=hs)


@pytest.mark.parametrize("hs", [64, 128])
@pytest.mark.parametrize("at", [20, 600, 700, 1290])
def test_prompt_infinities_in_halved_keys(device, hs, at):
    """An infinite value reaches the rows that see its key and no others."""
    import torch

    from vllm_quantpack.attention.prompt import prompt_attention
    g = torch.Generator(device=device).manual_seed(at)
    T, K = 700, 1300
    q = torch.randn((T, 48, hs), generator=g, device=device).to(torch.bfloat16)
    k, v = (torch.randn((K, 24, hs), generator=g, device=device).to(torch.bfloat16) for _ in range(2))
    v[at, :, 3] = 0.0
    offsets = dict(cu_seqlens_q=i32([0, T], device), cu_seqlens_k=i32([0, K], device))
    want = prompt_attention(q, k, v, **offsets)
    v[at, :, 3] = float("inf")
    got = prompt_attention(q, k, v, **offsets)
    see = torch.arange(T, device=device) + K - T >= at
    assert bool((got[see][..., 3] == float("inf")).all())
    assert torch.equal(got[~see], want[~see])
    rest = [c for c in range(hs) if c != 3]
    assert torch.equal(got[..., rest], want[..., rest])


@pytest.mark.parametrize("hs,num_splits", [(128, 0), (512, 0), (64, 1)])
def test_prompt_offsets_past_32_bits(device, hs, num_splits):
    """Key and value rows 64 Ki elements apart: the last ones lie 2^32 elements from the first."""
    import torch

    from vllm_quantpack.attention.prompt import prompt_attention
    n, apart = 66000, 1 << 16
    g = torch.Generator(device=device).manual_seed(hs)
    far = torch.empty((n, apart), dtype=torch.bfloat16, device=device)
    q = torch.randn((2, 2, hs), generator=g, device=device).to(torch.bfloat16)
    k, v = far[:, :hs].unsqueeze(1), far[:, 1024:1024 + hs].unsqueeze(1)
    for x in (k, v):
        x.copy_(torch.randn((n, 1, hs), generator=g, device=device).to(torch.bfloat16))
    lse = torch.zeros((2, 2), device=device)
    offsets = i32([0, 2], device), i32([0, n], device)
    out = prompt_attention(q, k, v, cu_seqlens_q=offsets[0], cu_seqlens_k=offsets[1], lse=lse, num_splits=num_splits)
    torch.cuda.synchronize()
    check_prompt(out, lse, q, k.contiguous(), v.contiguous(), hs ** -0.5, True, torch.bfloat16)


def test_prompt_broadcast_inputs(device):
    """Keys and values of one head shared by all through a stride of 0, and one query row for all tokens."""
    import torch

    from vllm_quantpack.attention.prompt import prompt_attention
    g = torch.Generator(device=device).manual_seed(1)
    q = torch.randn((1, 8, 128), generator=g, device=device).to(torch.bfloat16).expand(70, 8, 128)
    k, v = (torch.randn((90, 1, 128), generator=g, device=device).to(torch.bfloat16).expand(90, 4, 128) for _ in range(2))
    offsets = dict(cu_seqlens_q=i32([0, 70], device), cu_seqlens_k=i32([0, 90], device))
    got = prompt_attention(q, k, v, **offsets)
    assert torch.equal(got, prompt_attention(q.contiguous(), k.contiguous(), v.contiguous(), **offsets))


# --------------------------------------------------------------------------------------------------- key_weights

@pytest.mark.parametrize("fmt,hs,nq,nkv,tokens,seqs,n", [
    ("int4", 64, 8, 4, 10, 16, 4200), ("int8", 64, 8, 4, 70, 16, 4200),      # 20 rows; 140 rows in three stages
    ("int4", 128, 8, 4, 12, 17, 4100), ("int8", 128, 8, 4, 34, 17, 4100),    # 24; 68 rows in two stages
    ("int4", 256, 8, 4, 14, 8, 4300), ("int8", 256, 4, 4, 33, 8, 4300),      # 28; 33
    ("int4", 512, 4, 4, 34, 8, 4300), ("int8", 512, 8, 4, 25, 8, 4300)])     # 34 rows and 50, two stages of 32
def test_weights_of_several_blocks(device, fmt, hs, nq, nkv, tokens, seqs, n):
    """Enough heads and keys for a workgroup to walk several blocks of keys; some contexts end in the middle of its walk."""
    lens = [(tokens, n - 37 * i) for i in range(seqs)]
    lens[1], lens[2], lens[3], lens[4] = (tokens, 1), (0, n // 2 + 1), (3, 129), (tokens, n // 2 + 130)
    run_weights(device, lens, fmt, hs, nq, nkv, decay=0.5, seed=hs + tokens)


def test_weights_of_eight_blocks(device):
    """Eight blocks per workgroup, and tokens that see only part of them."""
    lens = [(20, 4096 + 5 * i) for i in range(40)]
    lens[7], lens[8] = (20, 19), (20, 700)
    run_weights(device, lens, "int4", 64, 8, 8, seed=8)


@pytest.mark.parametrize("fmt", ["int4", "int8"])
@pytest.mark.parametrize("tokens", [1, 40])
def test_weights_offsets_past_32_bits(device, fmt, tokens):
    """The pages of a cache of more than 4 GiB, from its first to its last, against the same pages close together. Weights
    and queries with strides of their own."""
    import torch

    from vllm_quantpack.attention import k8v4_kv
    from vllm_quantpack.attention.key_weights import key_weights
    rng = np.random.default_rng(tokens)
    hs, nkv, bs, blocks, n = 512, 8, 16, 20, 315
    kv, _ = random_cache(rng, blocks, nkv, bs, hs, fmt)
    near, (kc, _, ks, _) = torch_cache(kv, hs, fmt, device)
    size = near[0].numel()
    many = (1 << 32) // size + 100
    far = torch.empty((many,) + tuple(near.shape[1:]), dtype=near.dtype, device=device)
    pages = np.concatenate(([0, many - 1], rng.permutation(np.arange(1, many - 1))[:blocks - 2])).astype(np.int32)
    far[torch.from_numpy(pages.astype(np.int64)).to(device)] = near
    fkc, _, fks, _ = (k8v4_kv.views if fmt == "int8" else k8v4_kv.int4_views)(far, hs)
    wide = torch.randn((tokens, 2 * nkv, 2 * hs), device=device).to(torch.bfloat16)
    q = wide[:, ::2, hs:]
    kw = dict(cu_seqlens_q=i32([0, tokens], device), seqused_k=i32([n], device), max_seqlen_q=tokens, max_seqlen_k=n,
              softmax_scale=0.02)
    want = key_weights(q.contiguous(), kc, ks, torch.zeros((1, nkv, n), device=device),
                       block_table=i32([np.arange(blocks)], device), **kw)
    room = torch.full((1, 2 * nkv, n + 9), 3.0, device=device)
    got = key_weights(q, fkc, fks, room[:, 1::2, 9:], block_table=i32([pages], device), **kw)
    assert torch.equal(got, want)
    assert bool((room[:, ::2] == 3.0).all()) and bool((room[..., :9] == 3.0).all())


def test_weights_of_a_loose_bound(device):
    """max_seqlen_q far above what there is: the same weights to rounding, whatever path it leads to."""
    import torch

    from vllm_quantpack.attention.key_weights import key_weights
    rng = np.random.default_rng(2)
    kv, _ = random_cache(rng, 30, 2, 16, 128)
    keep, (kc, _, ks, _) = torch_cache(kv, 128, "int4", device)
    q = torch.randn((2, 8, 128), device=device).to(torch.bfloat16)
    kw = dict(cu_seqlens_q=i32([0, 2], device), seqused_k=i32([470], device), block_table=i32([np.arange(30)], device),
              softmax_scale=0.05)
    outs = [key_weights(q, kc, ks, torch.zeros((1, 2, 470), device=device), max_seqlen_q=m, **kw) for m in (2, 500, 1 << 30)]
    # (exponentials and sums over n keys (n + 64) 2^-23 = 6e-5, scores 2 ln 2 (hs + 8) 2^-24 D = 5e-5 with D below 5)
    for x in outs[1:]:
        assert torch.allclose(x, outs[0], rtol=2e-4, atol=0)
    # at most max_seqlen_q of a sequence's tokens are counted, the first ones
    one = key_weights(q, kc, ks, torch.zeros((1, 2, 470), device=device), max_seqlen_q=1, **kw)
    assert torch.allclose(one.sum(-1), torch.full((1, 2), 4.0, device=device), rtol=2e-4)
    assert bool((one[..., 469] == 0).all()) and bool((outs[0][..., 469] > 0).all())


# ---------------------------------------------------------------------------------------------------- evict_keys

@pytest.mark.parametrize("kind", ["equal", "few values", "nan", "infinite", "close", "one bin"])
@pytest.mark.parametrize("budget", [1, 9000])
def test_evict_ties_in_long_contexts(device, kind, budget):
    """Contexts past 8192 positions, beside shorter ones and an empty one: their lists hold many or all of the weights."""
    rng = np.random.default_rng(7)
    shape = (4, 2, 20003)
    w = rng.standard_normal(shape).astype(np.float32)
    if kind == "equal":
        w[:] = 0.125
    elif kind == "few values":
        w = rng.integers(0, 3, shape).astype(np.float32)
    elif kind == "nan":
        w[rng.random(shape) < 0.7] = np.nan
    elif kind == "infinite":
        w[rng.random(shape) < 0.3] = np.inf
        w[rng.random(shape) < 0.3] = -np.inf
    elif kind == "close":
        w = (np.float32(1.0).view(np.uint32) + rng.integers(0, 900, shape).astype(np.uint32)).view(np.float32)
    elif kind == "one bin":  # of the upper 11 bits
        w = (1.0 + 0.1 * rng.random(shape)).astype(np.float32)
    run_evict(device, [20000, 8193, 0, 9001], budget, sinks=min(2, budget - 1), recent=0, hs=64, weights=w, seed=1)


@pytest.mark.parametrize("n", [8191, 8192, 8193, 16384, 16385, 140001])
def test_evict_around_the_parts(device, n):
    run_evict(device, [n, 100], min(n, 3000), sinks=3, recent=9, hs=64, seed=n)


def test_evict_everything_stays_in_a_long_context(device):
    rng = np.random.default_rng(3)
    w = rng.standard_normal((2, 2, 9003)).astype(np.float32)
    w[rng.random(w.shape) < 0.2] = np.nan
    run_evict(device, [9000, 8500], 9000, hs=64, weights=w)


def test_evict_offsets_past_32_bits_and_strides(device):
    """Old and new pages at both ends of a cache of more than 4 GiB; weights, places and tables with strides of their own."""
    import torch

    from vllm_quantpack.attention import k8v4_kv
    from vllm_quantpack.attention.eviction import evict_keys
    rng = np.random.default_rng(9)
    hs, nkv, bs, n, budget = 512, 8, 16, 315, 60
    kv, _ = random_cache(rng, 20, nkv, bs, hs, "int8")
    near, _ = torch_cache(kv, hs, "int8", device)
    many = (1 << 32) // near[0].numel() + 100
    far = torch.empty((many,) + tuple(near.shape[1:]), dtype=near.dtype, device=device)
    pages = np.concatenate(([0, many - 1], rng.permutation(np.arange(3, many - 3))[:18])).astype(np.int32)
    new = np.array([many - 2, 1, many - 3, 2], np.int32)
    at = torch.from_numpy(pages.astype(np.int64)).to(device)
    far[at] = near
    views = k8v4_kv.views(far, hs)
    wide = rng.random((1, 2 * nkv, n + 4)).astype(np.float32)
    weights = torch.from_numpy(wide).to(device)[:, 1::2, 4:]
    tables = torch.full((1, 60), -1, dtype=torch.int32, device=device)
    tables[0, :20], tables[0, 30:34] = torch.from_numpy(pages).to(device), torch.from_numpy(new).to(device)
    room = torch.full((1, 2 * nkv, budget + 7), -5, dtype=torch.int32, device=device)
    used, kept, nw = evict_keys(*views, weights, seqused_k=i32([n], device), block_table=tables[:, :20],
                                new_block_table=tables[:, 30:34], budget=budget, sinks=2, recent=5, kept=room[:, ::2, 7:])
    torch.cuda.synchronize()
    assert used.tolist() == [budget] and bool((room[:, 1::2] == -5).all()) and bool((room[..., :7] == -5).all())
    moved = far[torch.from_numpy(new.astype(np.int64)).to(device)].cpu().numpy()
    old = near.cpu().numpy()
    for g in range(nkv):
        pos = expected(wide[0, 1 + 2 * g, 4:], n, budget, 2, 5)
        assert np.array_equal(kept[0, g].cpu().numpy(), pos)
        assert np.array_equal(nw[0, g].cpu().numpy(), wide[0, 1 + 2 * g, 4:][pos])
        to = np.arange(budget)
        assert np.array_equal(moved[to // bs, g, to % bs], old[pos // bs, g, pos % bs])
    assert torch.equal(far[at], near)


# ------------------------------------------------------------------------------- calls at once, and captured ones

def _calls(device, seed):
    """A call of every path of the three operators, each as a function that returns fresh results."""
    import torch

    from vllm_quantpack.attention.eviction import evict_keys
    from vllm_quantpack.attention.key_weights import key_weights
    from vllm_quantpack.attention.prompt import prompt_attention
    rng = np.random.default_rng(seed)
    g = torch.Generator(device=device).manual_seed(seed)
    hs, nq, nkv, n = 128, 8, 2, 9000
    blocks = -(-n // 16)
    kv, _ = random_cache(rng, 2 * blocks + 80, nkv, 16, hs)
    keep, views = torch_cache(kv, hs, "int4", device)
    table = i32(rng.permutation(2 * blocks).reshape(2, blocks), device)
    new = i32(2 * blocks + np.arange(80).reshape(2, 40), device)
    used, short = i32([n, n - 777], device), i32([900, 17], device)
    q = torch.randn((80, nq, hs), generator=g, device=device).to(torch.bfloat16)
    k, v = (torch.randn((2 * n, nkv, hs), generator=g, device=device).to(torch.bfloat16) for _ in range(2))
    w = torch.rand((2, nkv, n), generator=g, device=device)
    ck = i32([0, n, 2 * n], device)

    def prompt(tokens):
        lse = torch.zeros((tokens, nq), device=device)
        out = prompt_attention(q[:tokens], k, v, cu_seqlens_q=i32_of(tokens), cu_seqlens_k=ck, max_seqlen_k=n, lse=lse)
        return out, lse

    offsets = {t: i32([0, t // 2, t], device) for t in (2, 80)}

    def i32_of(tokens):
        return offsets[tokens]

    def weigh(tokens):
        return (key_weights(q[:tokens], views[0], views[2], torch.zeros_like(w), cu_seqlens_q=i32_of(tokens), seqused_k=used,
                            block_table=table, max_seqlen_q=tokens // 2, softmax_scale=0.05, previous=w, decay=0.5),)

    def evict(lengths, most):
        keep[2 * blocks:].zero_()
        out = evict_keys(*views, w, seqused_k=lengths, block_table=table, new_block_table=new, budget=600, max_seqlen_k=most)
        return tuple(out) + (keep[2 * blocks:].add(0),)

    return [lambda: prompt(2), lambda: prompt(80), lambda: weigh(2), lambda: weigh(80), lambda: evict(used, n),
            lambda: evict(short, 900)]


def test_two_streams_at_once(device):
    """Two streams run all the calls on tensors of their own at the same time, in different orders."""
    import torch
    a, b = _calls(device, 1), _calls(device, 2)
    want = [[f() for f in a], [f() for f in b]]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(3):
        for i, f in enumerate(a):
            with torch.cuda.stream(streams[0]):
                got[0].append((i, f()))
            j = len(b) - 1 - i
            with torch.cuda.stream(streams[1]):
                got[1].append((j, b[j]()))
    torch.cuda.synchronize()
    for wants, results in zip(want, got):
        for i, res in results:
            for x, y in zip(wants[i], res):
                assert torch.equal(x, y), i


def test_captured_calls_of_every_path(device):
    """All the calls in one graph, replayed between eager calls, whose tensors take the place of what the capture freed."""
    import torch
    calls = _calls(device, 3)
    want = [f() for f in calls]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for f in calls:
            f()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):  # two graphs of one pool: neither's workspaces are the other's to keep
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0].pool() if graphs else None):
            outs.append([f() for f in calls])
        graphs.append(graph)
    for r in range(4):
        graph, out = graphs[r % 2], outs[r % 2]
        for res in out:
            for x in res:
                x.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for i, (a, b) in enumerate(zip(want, out)):
            for x, y in zip(a, b):
                assert torch.equal(x, y), (r, i)
        for a, f in zip(want, calls):
            for x, y in zip(a, f()):
                assert torch.equal(x, y)
        torch.cuda.synchronize()
