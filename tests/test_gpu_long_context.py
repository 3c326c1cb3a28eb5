"""A long request's life through the operators in turn: attention over the prompt's own keys and values, their store, the
weights from the prompt's last tokens, an eviction, and decode steps over the shorter cache, each against 64 bits."""
import numpy as np
import pytest

from oracle import qp_oracle as O
from qp_testlib import i32, to_f32, torch_cache
from test_gpu_prompt import check as check_prompt
from test_gpu_router import _call, _segm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt,hs,nq,nkv", [("int4", 64, 8, 2), ("int4", 128, 8, 2), ("int8", 256, 6, 1), ("int4", 512, 4, 2)])
def test_prompt_store_weigh_evict_decode(device, fmt, hs, nq, nkv):
    import torch

    from vllm_quantpack.attention import eviction, int4_kv, key_weights, prompt, rht
    bs, budget, sinks, recent, window = 16, 96, 4, 16, 8
    lens = [300, 77, 150]
    g = torch.Generator(device=device).manual_seed(hs)
    q, k, v = (torch.randn((sum(lens), h, hs), generator=g, device=device).to(torch.bfloat16) for h in (nq, nkv, nkv))
    cu = np.concatenate(([0], np.cumsum(lens))).astype(np.int32)

    # the prompts' attention, over what the model has just computed
    lse = torch.empty((sum(lens), nq), device=device)
    out = prompt.prompt_attention(q, k, v, cu_seqlens_q=i32(cu, device), lse=lse)
    for i, n in enumerate(lens):
        s = slice(cu[i], cu[i + 1])
        check_prompt(out[s], lse[s], q[s], k[s], v[s], hs ** -0.5, True, torch.bfloat16)

    # their store
    counts = [-(-n // bs) for n in lens]
    new = [-(-(budget + 8) // bs)] * len(lens)
    total = sum(counts) + sum(new)
    cell = O.int4_cell_bytes(hs) if fmt == "int4" else O.k8v4_cell_bytes(hs)
    cache, views = torch_cache(O.new_cache(total, nkv, bs, cell), hs, fmt, device)
    pool, at = np.random.default_rng(1).permutation(total).astype(np.int32), 0
    table, new_table = np.zeros((3, max(counts)), np.int32), np.zeros((3, new[0]), np.int32)
    for t, cs in ((table, counts), (new_table, new)):
        for i, c in enumerate(cs):
            t[i, :c] = pool[at:at + c]
            at += c
    kc, vc, ks, vs = views
    slots = np.concatenate([table[i, np.arange(n) // bs].astype(np.int64) * bs + np.arange(n) % bs for i, n in enumerate(lens)])
    int4_kv.reshape_and_cache_int4(k, v, kc, vc, torch.from_numpy(slots).to(device), k_scale_cache=ks, v_scale_cache=vs)

    # the weight of every key from the last tokens of its prompt
    last = np.concatenate([np.arange(cu[i + 1] - window, cu[i + 1]) for i in range(3)])
    qw = q[torch.from_numpy(last).to(device)]
    weights = torch.zeros((3, nkv, max(lens)), device=device)
    signs = rht.signs(hs, device)
    key_weights.key_weights(qw, kc, ks, weights, cu_seqlens_q=i32([0, window, 2 * window, 3 * window], device),
                            seqused_k=i32(lens, device), block_table=i32(table, device), max_seqlen_q=window,
                            softmax_scale=hs ** -0.5 / hs, query_signs=signs)
    torch.cuda.synchronize()

    def host():
        x = cache.cpu().numpy().view(np.uint8)
        return O.int4_views(x, hs) if fmt == "int4" else O.k8v4_views(x, hs)

    hv = host()
    qr = rht.single_rht(qw).double().cpu().numpy()
    for i, n in enumerate(lens):
        K, _ = O.dequant_f64(hv, table[i], n)
        w = np.zeros((nkv, n))
        for h in range(nq):
            for t in range(window):
                a = (K[:n - window + t + 1, h // (nq // nkv)] @ qr[i * window + t, h]) * hs ** -1.5
                p = np.exp(a - a.max())
                w[h // (nq // nkv), :len(p)] += p / p.sum()
        assert O.relerr(weights[i, :, :n].cpu().numpy(), w) < 2e-5  # (fp32 throughout, on the same rotated rows)
        assert (weights[i, :, n:] == 0).all()

    # the eviction: exactly what the weights say
    used, kept, _ = eviction.evict_keys(*views, weights, seqused_k=i32(lens, device), block_table=i32(table, device),
                                        new_block_table=i32(new_table, device), budget=budget, sinks=sinks, recent=recent)
    torch.cuda.synchronize()
    assert used.tolist() == [min(n, budget) for n in lens]
    wn, kn = weights.cpu().numpy(), kept.cpu().numpy()
    for i, n in enumerate(lens):
        for h in range(nkv):
            w = wn[i, h, :n].astype(np.float64)
            w[:sinks] = w[max(0, n - recent):] = np.inf
            want = np.sort(np.argsort(-w, kind="stable")[:min(n, budget)])
            assert np.array_equal(kn[i, h, :len(want)], want)

    # three decode steps over the new blocks: the kept keys and what is stored after them
    now = [min(n, budget) for n in lens]
    for step in range(3):
        kq, vq, qq = (torch.randn((3, h, hs), generator=g, device=device).to(torch.bfloat16) for h in (nkv, nkv, nq))
        slots = [int(new_table[i, now[i] // bs]) * bs + now[i] % bs for i in range(3)]
        int4_kv.reshape_and_cache_int4(kq, vq, kc, vc, torch.tensor(slots, device=device), k_scale_cache=ks, v_scale_cache=vs)
        now = [n + 1 for n in now]
        got = torch.empty_like(qq)
        _call(views, qq, got, i32([0, 1, 2, 3], device), i32(now, device), i32(new_table, device), 1, max(now),
              _segm(device, 3, 16, nq=nq, hs=hs), 16, hs=hs)
        torch.cuda.synchronize()
        after = host()
        qd = O.rht(to_f32(qq).astype(np.float64))
        for i in range(3):
            parts = [O.dequant_f64(hv, table[i], lens[i])]
            K, V = (np.zeros((now[i], nkv, hs)) for _ in range(2))
            m = min(lens[i], budget)
            for h in range(nkv):  # the kept keys from the cache as it was before, the stored ones from the new blocks
                K[:m, h], V[:m, h] = parts[0][0][kn[i, h, :m], h], parts[0][1][kn[i, h, :m], h]
            tail = O.dequant_f64(after, new_table[i], now[i])
            K[m:], V[m:] = tail[0][m:], tail[1][m:]
            want = O.rht(O.attention_f64(qd[i:i + 1], K, V, now[i], hs ** -1.5), inverse=True) / hs
            assert O.relerr(to_f32(got[i:i + 1]), want) < 5e-3  # as the attention's own tests
