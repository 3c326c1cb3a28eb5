"""evict_keys against a sort on the host. Everything it writes is copied or counted, so every comparison is exact."""
import numpy as np
import pytest

from qp_testlib import i32, random_cache, torch_cache

pytestmark = pytest.mark.gpu


def expected(w, n, budget, sinks, recent):
    """The kept positions of one sequence and head, ascending."""
    w = w[:n].astype(np.float64)
    rank = np.ones(n, int)
    rank[:sinks] = 0
    rank[max(0, n - recent):] = 0
    nan = np.isnan(w)
    order = sorted(range(n), key=lambda j: (rank[j], nan[j], 0 if nan[j] else -w[j], j))
    return np.sort(np.array(order[:min(n, budget)], int))


def run(device, lens, budget, sinks=0, recent=0, fmt="int4", hs=128, nkv=2, bs=16, layout="hnd", seed=0, weights=None,
        apart=False):
    """One call; the returned places, weights and lengths, and the whole cache, against the host's."""
    import torch

    from vllm_quantpack.attention.eviction import evict_keys
    rng = np.random.default_rng(seed)
    seqs, L = len(lens), max(lens) + 3
    counts, new = [-(-n // bs) for n in lens], [-(-min(n, budget) // bs) for n in lens]
    total = sum(counts) + sum(new) + 2
    kv, _ = random_cache(rng, total, nkv, bs, hs, fmt, layout)
    keep, views = torch_cache(kv, hs, fmt, device)
    if apart:  # codes and words in allocations of their own (an int4 view has its words' bytes behind the codes)
        views = tuple(x[..., :x.shape[3] // 8 * 8].contiguous() if x.dim() == 4 else x.contiguous() for x in views)
    pool, at = rng.permutation(total).astype(np.int32), 0
    table, new_table = np.zeros((seqs, max(counts + [1])), np.int32), np.zeros((seqs, max(new + [1])), np.int32)
    for t, cs in ((table, counts), (new_table, new)):
        for i, c in enumerate(cs):
            t[i, :c] = pool[at:at + c]
            at += c
    w = rng.lognormal(-3, 2, (seqs, nkv, L)).astype(np.float32) if weights is None else weights
    before = [x.cpu().numpy().copy() for x in views]
    kept = torch.full((seqs, nkv, budget + 1), -9, dtype=torch.int32, device=device)
    new_w = torch.full((seqs, nkv, budget + 2), -9.0, device=device)
    used, k2, w2 = evict_keys(*views, torch.from_numpy(w).to(device), seqused_k=i32(lens, device),
                              block_table=i32(table, device), new_block_table=i32(new_table, device), budget=budget,
                              max_seqlen_k=max(lens), sinks=sinks, recent=recent, kept=kept, new_weights=new_w)
    torch.cuda.synchronize()
    assert k2 is kept and w2 is new_w
    assert used.tolist() == [min(n, budget) for n in lens]
    kept, new_w = kept.cpu().numpy(), new_w.cpu().numpy()
    want = [x.copy() for x in before]
    for i, n in enumerate(lens):
        m = min(n, budget)
        for g in range(nkv):
            pos = expected(w[i, g], n, budget, sinks, recent)
            assert np.array_equal(kept[i, g, :m], pos), (i, g)
            assert np.array_equal(new_w[i, g, :m], w[i, g, pos], equal_nan=True)
            assert (kept[i, g, m:] == -9).all() and (new_w[i, g, m:] == -9).all()
            for a, b in zip(want, before):
                to = np.arange(m)
                a[new_table[i, to // bs], to % bs, g] = b[table[i, pos // bs], pos % bs, g]
    for a, x in zip(want, views):
        x = x.cpu().numpy()
        assert np.array_equal(np.ascontiguousarray(a).view(np.uint8), np.ascontiguousarray(x).view(np.uint8)), "cache bytes"
    return kept, new_w


@pytest.mark.parametrize("fmt", ["int4", "int8"])
@pytest.mark.parametrize("hs", [64, 128, 256, 512])
def test_formats(device, fmt, hs):
    run(device, [300, 17, 1500], 200, sinks=4, recent=16, fmt=fmt, hs=hs, seed=hs)


@pytest.mark.parametrize("bs,layout,apart", [(1, "hnd", False), (5, "hnd", False), (32, "nhd", False), (16, "hnd", True),
                                             (48, "nhd", True)])
@pytest.mark.parametrize("fmt", ["int4", "int8"])
def test_blocks_and_layouts(device, fmt, bs, layout, apart):
    run(device, [200, 333], 90, sinks=1, recent=7, fmt=fmt, bs=bs, layout=layout, apart=apart, seed=bs)


@pytest.mark.parametrize("lens,budget,sinks,recent", [
    ([1], 1, 0, 0), ([1], 1, 1, 0), ([1, 2, 3], 2, 0, 1), ([0, 5, 0], 3, 0, 0), ([64], 64, 0, 0), ([64], 63, 0, 0),
    ([64], 65, 0, 0), ([100], 40, 40, 0), ([100], 40, 0, 40), ([100], 40, 20, 20), ([30], 40, 20, 20), ([1024], 1, 0, 0),
    ([1025], 1024, 3, 3), ([5000, 4097, 4096], 2000, 4, 64), ([20000], 12345, 4, 128), ([70000], 500, 4, 32)])
def test_lengths(device, lens, budget, sinks, recent):
    run(device, lens, budget, sinks, recent, hs=64, seed=budget)


@pytest.mark.parametrize("kind", ["equal", "zeros", "few values", "negative", "both zeros", "infinite", "nan", "close"])
def test_ties_and_odd_weights(device, kind):
    rng = np.random.default_rng(7)
    shape = (2, 2, 3003)
    w = rng.standard_normal(shape).astype(np.float32)
    if kind == "equal":
        w[:] = 0.125
    elif kind == "zeros":
        w = np.where(rng.random(shape) < 0.9, 0, w).astype(np.float32)
    elif kind == "few values":
        w = rng.integers(0, 3, shape).astype(np.float32)
    elif kind == "negative":
        w = -np.abs(w)
    elif kind == "both zeros":
        w = np.where(rng.random(shape) < 0.5, np.float32(-0.0), np.float32(0.0))
    elif kind == "infinite":
        w[rng.random(shape) < 0.3] = np.inf
        w[rng.random(shape) < 0.3] = -np.inf
    elif kind == "nan":
        w = np.abs(w)
        w[rng.random(shape) < 0.6] = np.nan
    elif kind == "close":  # all in one bin of the first two histograms
        w = (np.float32(1.0).view(np.uint32) + rng.integers(0, 900, shape).astype(np.uint32)).view(np.float32)
    run(device, [3000, 2500], 1500, sinks=2, recent=5, hs=64, weights=w, seed=1)


def test_pages_outside_the_cache(device):
    """A cell whose old or new page does not exist is not moved; places and weights are there all the same."""
    import torch

    from vllm_quantpack.attention.eviction import evict_keys
    rng = np.random.default_rng(4)
    for fmt, apart in (("int4", False), ("int8", True)):
        kv, _ = random_cache(rng, 6, 2, 16, 64, fmt)
        keep, views = torch_cache(kv, 64, fmt, device)
        if apart:
            views = tuple(x[..., :x.shape[3] // 8 * 8].contiguous() if x.dim() == 4 else x.contiguous() for x in views)
        before = [x.clone() for x in views]
        w = torch.arange(48, dtype=torch.float32, device=device).expand(1, 2, 48).contiguous()
        for old, to in (([0, -1, 2], [4, 5]), ([0, 6, 2], [4, 5]), ([0, 1, 2], [4, -5]), ([0, 1, 2], [2 ** 31 - 1, 4])):
            used, kept, nw = evict_keys(*views, w, seqused_k=i32([48], device), block_table=i32([old], device),
                                        new_block_table=i32([to], device), budget=32)
            torch.cuda.synchronize()
            assert kept[0, 0].tolist() == list(range(16, 48)) and used.tolist() == [32]
            for x, b in zip(views, before):
                want = b.clone()
                for src, dst in zip(old[1:], to):
                    if 0 <= src < 6 and 0 <= dst < 6:
                        want[dst] = b[src]
                assert torch.equal(x, want)
            for x, b in zip(views, before):
                x.copy_(b)


def test_made_outputs_and_graph(device):
    import torch

    from vllm_quantpack.attention.eviction import evict_keys
    rng = np.random.default_rng(6)
    kv, _ = random_cache(rng, 40, 2, 16, 64)
    keep, views = torch_cache(kv, 64, "int4", device)
    w = torch.rand((2, 2, 250), device=device)
    kw = dict(seqused_k=i32([250, 20], device), block_table=i32(rng.permutation(32).reshape(2, 16), device),
              new_block_table=i32([[32, 33, 34, 35], [36, 37, 38, 39]], device), budget=60, sinks=1, recent=3)
    used, kept, nw = evict_keys(*views, w, **kw)
    assert bool((kept[1, :, 20:] == -1).all()) and bool((nw[1, :, 20:] == 0).all()) and used.tolist() == [60, 20]
    out = dict(kept=torch.empty_like(kept).fill_(-1), new_weights=torch.zeros_like(nw), new_seqused_k=torch.zeros_like(used))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        evict_keys(*views, w, **kw, **out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        evict_keys(*views, w, **kw, **out)
    for i in range(4):
        keep[32:] = 0
        graph.replay()
        torch.cuda.synchronize()
        got = keep[32:].clone()
        used, kept, nw = evict_keys(*views, w, **kw)
        torch.cuda.synchronize()
        assert torch.equal(got, keep[32:])
        assert torch.equal(out["kept"], kept) and torch.equal(out["new_weights"], nw) and torch.equal(out["new_seqused_k"], used)
        w.copy_(torch.rand_like(w))
