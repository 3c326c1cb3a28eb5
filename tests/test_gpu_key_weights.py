"""key_weights against the definition in 64 bits on the dequantised keys.

Tolerance: codes and queries enter the products exactly. A score in log2 units, S = c (sum q_i (code_i - 8) - sum(q) (zp - 8))
with c = scale s_k log2 e, is a sum of at most hs + 1 products in fp32, in any order, times c: off by at most
(hs + 8) 2^-24 D with D the largest |c| (sum |q_i (code_i - 8)| + 8 sum |q_i|) (int8: the first sum, over |code_i|). A
probability 2^(S - max) / sum is then off by the relative amount 2 ln 2 (hs + 8) 2^-24 D for the score and the normaliser,
and by less than (n + 64) 2^-23 for exponentials, sums and the join; a weight adds R rows' probabilities, (R + 4) 2^-24 more,
and the decayed earlier weight, off by 2^-23 of itself."""
import numpy as np
import pytest

from oracle import qp_oracle as O
from qp_testlib import bf16_tensor, i32, random_cache, torch_cache

pytestmark = pytest.mark.gpu


def exact(q, views, table, n, scale):
    """(weights [kv heads, n], D) of one sequence's query tokens q [tokens, heads, hs] (float64)."""
    K, _ = O.dequant_f64(views, table, n)
    tokens, nq, hs = q.shape
    nkv = K.shape[1]
    w, big = np.zeros((nkv, n)), 0.0
    pos = np.arange(n)
    codes, words = views.key[table[pos // views.key.shape[1]], pos % views.key.shape[1]], None
    words = views.key_word[table[pos // views.key.shape[1]], pos % views.key.shape[1]]
    if codes.dtype == np.int8:
        size, sk, extra = np.abs(codes.astype(np.float64)), words.view(np.float32).astype(np.float64), 0.0
    else:
        size = np.abs(np.stack((codes & 15, codes >> 4), -1).reshape(*codes.shape[:-1], hs).astype(np.float64) - 8)
        sk, extra = (words & np.uint32(0xFFFFFFF0)).view(np.float32).astype(np.float64), 8.0
    for h in range(nq):
        g = h // (nq // nkv)
        for t in range(tokens):
            see = n - tokens + t + 1
            if see <= 0:
                continue
            a = scale * (K[:see, g] @ q[t, h])
            p = np.exp(a - a.max())
            w[g, :see] += p / p.sum()
            aq = np.abs(q[t, h])
            big = max(big, float((scale * O.LOG2E * sk[:see, g] * (size[:see, g] @ aq + extra * aq.sum())).max()))
    return w, big


def run(device, lens, fmt, hs, nq, nkv, bs=16, layout="hnd", decay=None, seed=0, signs=False, spread=1.0, in_place=False,
        extra=0):
    """One call on a batch of (tokens, keys); entries past a sequence's keys and sequences' other rows stay as they were."""
    import torch

    from vllm_quantpack.attention import rht
    from vllm_quantpack.attention.key_weights import key_weights
    rng = np.random.default_rng(seed)
    counts = [-(-n // bs) for _, n in lens]
    kv, views = random_cache(rng, sum(counts) + 2, nkv, bs, hs, fmt, layout)
    keep, (kc, vc, ks, vs) = torch_cache(kv, hs, fmt, device)
    pool, at = rng.permutation(sum(counts) + 2), 0
    table = np.full((len(lens), max(counts + [1])), 2 ** 30, np.int32)  # (entries past a sequence are never followed)
    for i, c in enumerate(counts):
        table[i, :c] = pool[at:at + c]
        at += c
    T = sum(t for t, _ in lens) + extra
    bits = O.f32_to_bf16_bits(rng.standard_normal((T, nq, hs)).astype(np.float32) * spread)
    q = bf16_tensor(bits, device)
    qf = O.bf16_bits_to_f32(bits).astype(np.float64)
    scale = hs ** -0.5 * (1 / hs if signs else 1)
    if signs:  # (rows rotated on load have the bits of a separate rotation)
        qf = rht.single_rht(q).double().cpu().numpy()
    L = max(n for _, n in lens) + 5
    prev = rng.random((len(lens), nkv, L)).astype(np.float32) if decay is not None else None
    out = torch.full((len(lens), nkv, L), 7.0, device=device)
    pt = None if prev is None else torch.from_numpy(prev).to(device)
    if in_place:
        out = pt
    before = out.clone()
    cu = np.concatenate(([0], np.cumsum([t for t, _ in lens]))).astype(np.int32)
    got = key_weights(q, kc, ks, out, cu_seqlens_q=i32(cu, device), seqused_k=i32([n for _, n in lens], device),
                      block_table=i32(table, device), max_seqlen_q=max(t for t, _ in lens),
                      max_seqlen_k=max(n for _, n in lens), softmax_scale=scale,
                      query_signs=rht.signs(hs, device) if signs else None, previous=pt,
                      decay=1.0 if decay is None else decay)
    torch.cuda.synchronize()
    assert got is out
    res = out.cpu().numpy().astype(np.float64)
    for i, (t, n) in enumerate(lens):
        w, big = exact(qf[cu[i]:cu[i] + t], views, table[i], n, scale) if n else (np.zeros((nkv, 0)), 0.0)
        rows = t * (nq // nkv)
        tol = w * (2 * np.log(2) * (hs + 8) * 2 ** -24 * big + (n + 64) * 2 ** -23 + (rows + 4) * 2 ** -24)
        if decay is not None:
            w = w + decay * prev[i, :, :n].astype(np.float64)
            tol = tol + 2 ** -23 * w
        diff = np.abs(res[i, :, :n] - w)
        assert (diff <= tol + 1e-30).all(), (i, t, n, float((diff / (tol + 1e-30)).max()))
        assert (out[i, :, n:] == before[i, :, n:]).all()
    return out


CASES = [("int4", 64, 8, 2), ("int4", 128, 8, 2), ("int4", 256, 6, 1), ("int4", 512, 4, 2),
         ("int8", 64, 4, 1), ("int8", 128, 8, 2), ("int8", 256, 12, 2), ("int8", 512, 4, 2)]


@pytest.mark.parametrize("fmt,hs,nq,nkv", CASES)
@pytest.mark.parametrize("tokens,n", [(1, 1), (1, 33), (2, 300), (4, 1025), (40, 90)])
def test_one_sequence(device, tokens, n, fmt, hs, nq, nkv):
    run(device, [(tokens, n)], fmt, hs, nq, nkv, seed=n)


@pytest.mark.parametrize("fmt,hs,nq,nkv", CASES)
def test_batch(device, fmt, hs, nq, nkv):
    """Different lengths; a sequence without tokens, one without keys, one with more tokens than keys; rows of no sequence."""
    run(device, [(1, 700), (0, 50), (3, 3), (9, 4), (2, 0), (1, 1), (70, 640)], fmt, hs, nq, nkv, decay=0.9, seed=hs, extra=2)


@pytest.mark.parametrize("bs,layout", [(1, "hnd"), (5, "hnd"), (16, "nhd"), (48, "hnd"), (64, "nhd")])
@pytest.mark.parametrize("fmt", ["int4", "int8"])
def test_blocks_and_layouts(device, fmt, bs, layout):
    run(device, [(2, 131), (1, 64)], fmt, 128, 8, 2, bs=bs, layout=layout, seed=bs)


@pytest.mark.parametrize("decay", [0.0, 0.5, 1.0])
@pytest.mark.parametrize("in_place", [False, True])
def test_decay(device, decay, in_place):
    run(device, [(1, 200), (2, 77)], "int4", 128, 8, 2, decay=decay, in_place=in_place, seed=3)


def test_zero_decay_reads_no_earlier_weights(device):
    import torch

    from vllm_quantpack.attention.key_weights import key_weights
    rng = np.random.default_rng(1)
    kv, _ = random_cache(rng, 3, 2, 16, 64)
    keep, (kc, _, ks, _) = torch_cache(kv, 64, "int4", device)
    q = torch.randn((1, 4, 64), device=device).to(torch.bfloat16)
    kw = dict(cu_seqlens_q=i32([0, 1], device), seqused_k=i32([40], device), block_table=i32([[2, 0, 1]], device),
              max_seqlen_q=1, softmax_scale=0.1)
    out = torch.full((1, 2, 40), float("nan"), device=device)
    key_weights(q, kc, ks, out, previous=out, decay=0.0, **kw)
    assert torch.equal(out, key_weights(q, kc, ks, torch.zeros_like(out), **kw))
    assert bool(torch.allclose(out.sum(-1), torch.full((1, 2), 2.0, device=device), atol=1e-5))


@pytest.mark.parametrize("fmt,hs,nq,nkv", CASES)
def test_rotated_queries(device, fmt, hs, nq, nkv):
    run(device, [(1, 150), (3, 64)], fmt, hs, nq, nkv, signs=True, seed=8)


@pytest.mark.parametrize("fmt", ["int4", "int8"])
def test_large_scores(device, fmt):
    run(device, [(2, 500)], fmt, 128, 8, 2, spread=60.0, seed=2)


def test_many_rows(device):
    """More rows than one chunk of LDS holds, at every head size, and groups that do not divide a tile."""
    for hs, nq, nkv in ((64, 33, 1), (128, 14, 2), (256, 5, 1), (512, 6, 2)):
        run(device, [(67, 210), (50, 130)], "int4", hs, nq, nkv, seed=hs)


def test_pages_outside_the_cache(device):
    """Keys on a page that does not exist are not seen: the others share the weight, and those get none."""
    import torch

    from vllm_quantpack.attention.key_weights import key_weights
    rng = np.random.default_rng(4)
    kv, views = random_cache(rng, 4, 2, 16, 128)
    keep, (kc, _, ks, _) = torch_cache(kv, 128, "int4", device)
    q = torch.randn((1, 4, 128), device=device).to(torch.bfloat16)

    def call(table, n):
        out = torch.full((1, 2, 64), 7.0, device=device)
        return key_weights(q, kc, ks, out, cu_seqlens_q=i32([0, 1], device), seqused_k=i32([n], device),
                           block_table=i32([table], device), max_seqlen_q=1, softmax_scale=0.1)

    whole = call([1, 3], 32)
    for bad in (-1, 4, 2 ** 31 - 1, -2 ** 31):
        got = call([1, bad, 3], 48)
        assert bool((got[..., 16:32] == 0).all())
        both = torch.cat((got[..., :16], got[..., 32:48]), -1)
        assert bool(torch.allclose(both, whole[..., :32], rtol=1e-5))
        assert bool((got[..., 48:] == 7.0).all())
        assert bool((call([bad], 16)[..., :16] == 0).all())
    # a length beyond the block table's room, or the longest context, is cut there
    assert torch.equal(call([1, 3], 2 ** 31 - 1), whole)


def test_same_bits_and_graph(device):
    import torch

    from vllm_quantpack.attention.key_weights import key_weights
    rng = np.random.default_rng(5)
    kv, _ = random_cache(rng, 200, 2, 16, 128)
    keep, (kc, _, ks, _) = torch_cache(kv, 128, "int4", device)
    q = torch.randn((3, 8, 128), device=device).to(torch.bfloat16)
    table = i32(rng.permutation(200).reshape(2, 100), device)
    cu, used = i32([0, 1, 3], device), i32([1600, 900], device)
    prev = torch.rand((2, 2, 1600), device=device)

    def call(out):
        return key_weights(q, kc, ks, out, cu_seqlens_q=cu, seqused_k=used, block_table=table, max_seqlen_q=2,
                           softmax_scale=0.05, previous=prev, decay=0.9)

    out = torch.zeros_like(prev)
    want = call(torch.zeros_like(prev))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out)
    for i in range(4):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
        assert torch.equal(call(torch.zeros_like(prev)), want)
        q.mul_(0.7)
        want = call(torch.zeros_like(prev))
        torch.cuda.synchronize()
