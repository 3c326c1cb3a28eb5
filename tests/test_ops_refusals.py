"""What the operators of include/quantpack_ops.h refuse, on the host before anything runs, and their binding. No kernel runs
here."""
import ctypes
import os
import re
import shutil
import subprocess

import pytest
import torch

from conftest import REPO

HEADER = os.path.join(REPO, "include", "quantpack_ops.h")
STRUCTS = {"PromptArgs": "qp_prompt_args", "KeyWeightsArgs": "qp_key_weights_args", "EvictArgs": "qp_evict_args"}


@pytest.fixture(scope="module")
def lib():
    from vllm_quantpack import _hip
    if not os.path.exists(_hip.LIB_PATH):
        pytest.skip("library not built (python vllm-quantpack_amd/build.py)")
    return _hip.lib()


def test_binding_has_every_declared_entry_point(lib):
    from vllm_quantpack import _hip
    src = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    declared = set(re.findall(r"^\s*(?:const\s+)?\w+\s*\*?\s*(qp_\w+)\s*\(", src, flags=re.M))
    assert declared == set(_hip.OPS_SIGNATURES)
    for name in declared:
        assert hasattr(ctypes.CDLL(_hip.LIB_PATH), name), name


def test_ctypes_structs_have_the_header_layout(tmp_path):
    from vllm_quantpack import _hip
    if shutil.which("gcc") is None:
        pytest.skip("no gcc")
    lines = ['#include <stddef.h>', '#include <stdio.h>', '#include "quantpack_ops.h"', "int main(void) {"]
    want = []
    for py, c in STRUCTS.items():
        T = getattr(_hip, py)
        lines.append(f'  printf("{py} size %zu\\n", sizeof({c}));')
        want.append(f"{py} size {ctypes.sizeof(T)}")
        for name, _ in T._fields_:
            lines.append(f'  printf("{py} {name} %zu\\n", offsetof({c}, {name}));')
            want.append(f"{py} {name} {getattr(T, name).offset}")
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["  return 0;", "}"]) + "\n")
    subprocess.run(["gcc", "-I", os.path.join(REPO, "include"), str(src), "-o", str(exe)], check=True)
    assert subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split("\n")[:-1] == want


# ------------------------------------------------------------------------------------------------ qp_prompt

def prompt_args(**kw):
    from vllm_quantpack import _hip
    a = _hip.PromptArgs()
    a.query = a.key = a.value = a.out = a.cu_seqlens_q = a.cu_seqlens_k = 4096
    for f in ("query_stride", "key_stride", "value_stride", "out_stride"):
        setattr(a, f, _hip.I64x2(1024, 128))
    a.num_seqs, a.num_tokens, a.num_keys, a.num_q_heads, a.num_kv_heads, a.head_size = 1, 5, 5, 8, 2, 128
    a.max_seqlen_k, a.softmax_scale = 5, 0.1
    for name, value in kw.items():
        setattr(a, name, _hip.I64x2(*value) if isinstance(value, tuple) else value)
    return a


@pytest.mark.parametrize("bad,status,text", [
    (dict(query=None), -1, "null tensor"), (dict(key=None), -1, "null tensor"), (dict(cu_seqlens_k=None), -1, "null tensor"),
    (dict(head_size=96), -2, "head size"), (dict(dtype=1), -2, "bf16 or fp16"), (dict(num_q_heads=7), -1, "multiple"),
    (dict(num_kv_heads=0), -1, "multiple"), (dict(num_tokens=-1), -1, "sizes"), (dict(num_splits=129), -1, "splits"),
    (dict(softmax_scale=0.0), -1, "scale"), (dict(softmax_scale=float("nan")), -1, "scale"),
    (dict(softmax_scale=-1.0), -1, "scale"), (dict(query=4104), -1, "aligned"), (dict(key_stride=(1028, 128)), -1, "aligned"),
    (dict(out_stride=(1024, 132)), -1, "aligned"), (dict(value_stride=(-1024, 128)), -1, "negative"),
    (dict(key_stride=(1 << 23, 128)), -2, "apart"), (dict(num_splits=4), -1, "workspace"),
    (dict(num_splits=4, workspace=4100, workspace_bytes=1 << 30), -1, "aligned")])
def test_prompt_refusals(lib, bad, status, text):
    assert lib.qp_prompt(prompt_args(**bad), None) == status
    assert text in lib.qp_last_error().decode()


def test_prompt_refuses_null_arguments(lib):
    assert lib.qp_prompt(None, None) == -1
    assert lib.qp_prompt_workspace_size(None) == 0


def test_prompt_with_nothing_to_do(lib):
    assert lib.qp_prompt(prompt_args(num_tokens=0), None) == 0
    assert lib.qp_prompt(prompt_args(num_seqs=0), None) == 0


def test_prompt_workspace(lib):
    assert lib.qp_prompt_workspace_size(prompt_args(num_splits=4)) == 5 * 8 * 4 * 130 * 4
    assert lib.qp_prompt_workspace_size(prompt_args(num_splits=1)) == 0


def _tensors(tokens=5, nq=8, nkv=2, hs=128, dtype=torch.bfloat16):
    return (torch.zeros((tokens, nq, hs), dtype=dtype), torch.zeros((tokens, nkv, hs), dtype=dtype),
            torch.zeros((tokens, nkv, hs), dtype=dtype), torch.tensor([0, tokens], dtype=torch.int32))


def test_prompt_attention_refusals(lib):
    from vllm_quantpack.attention.prompt import prompt_attention
    q, k, v, cu = _tensors()
    with pytest.raises(ValueError, match="on a GPU"):
        prompt_attention(q, k, v, cu_seqlens_q=cu)
    with pytest.raises(NotImplementedError, match="bf16 or fp16"):
        prompt_attention(q.float(), k.float(), v.float(), cu_seqlens_q=cu)
    with pytest.raises(ValueError, match="must have q's type"):
        prompt_attention(q, k.half(), v, cu_seqlens_q=cu)
    with pytest.raises(ValueError, match="do not belong together"):
        prompt_attention(q, k, v[:3], cu_seqlens_q=cu)
    with pytest.raises(ValueError, match="do not belong together"):
        prompt_attention(q, k[..., :64], v[..., :64], cu_seqlens_q=cu)
    with pytest.raises(ValueError, match="do not belong together"):
        prompt_attention(q, k, v, torch.empty_like(q[:2]), cu_seqlens_q=cu)
    with pytest.raises(ValueError, match="contiguous"):
        prompt_attention(q, k.transpose(1, 2).contiguous().transpose(1, 2), v, cu_seqlens_q=cu)
    with pytest.raises(ValueError, match="int32"):
        prompt_attention(q, k, v, cu_seqlens_q=cu.long())
    with pytest.raises(ValueError, match="different batches"):
        prompt_attention(q, k, v, cu_seqlens_q=cu, cu_seqlens_k=torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="lse"):
        prompt_attention(q, k, v, cu_seqlens_q=cu, lse=torch.zeros((5, 7)))
    with pytest.raises(NotImplementedError, match="backward"):
        prompt_attention(q.requires_grad_(), k, v, cu_seqlens_q=cu)


# ------------------------------------------------------------------------------------------- qp_key_weights

def set_fields(a, kw):
    from vllm_quantpack import _hip
    for name, value in kw.items():
        obj, *rest = [a] + name.split("__")
        for r in rest[:-1]:
            obj = getattr(obj, r)
        types = {2: _hip.I64x2, 3: _hip.I64x3}
        setattr(obj, rest[-1], types[len(value)](*value) if isinstance(value, tuple) else value)
    return a


def half(hs, fmt=0):
    from vllm_quantpack import _hip
    cell = 264
    return _hip.CacheHalf(4096, _hip.I64x3(16 * cell, cell, 0), 4096 + hs // 2, _hip.I64x3(4 * cell, cell // 4, 0), fmt)


def weight_args(**kw):
    from vllm_quantpack import _hip
    a = _hip.KeyWeightsArgs()
    a.key = half(256)
    a.num_blocks, a.block_size, a.num_kv_heads, a.head_size = 8, 16, 1, 256
    a.query = a.cu_seqlens_q = a.seqused_k = a.block_table = a.out = 4096
    a.query_stride = _hip.I64x2(1024, 256)
    a.max_blocks, a.num_seqs, a.num_tokens, a.num_q_heads, a.max_query_len, a.max_seqlen_k = 4, 1, 1, 4, 1, 64
    a.softmax_scale, a.decay = 0.1, 1.0
    a.workspace, a.workspace_bytes = 4096, 1 << 20
    return set_fields(a, kw)


@pytest.mark.parametrize("bad,status,text", [
    (dict(out=None), -1, "null tensor"), (dict(query=None), -1, "null tensor"), (dict(key__codes=None), -1, "null tensor"),
    (dict(head_size=80), -2, "head size"), (dict(key__format=2), -1, "format"), (dict(num_kv_heads=3), -1, "multiple"),
    (dict(block_size=0), -1, "sizes"), (dict(num_tokens=-1), -1, "sizes"), (dict(num_seqs=65536), -2, "65535"),
    (dict(max_query_len=1 << 29), -2, "rows"), (dict(softmax_scale=0.0), -1, "scale"),
    (dict(key__code_stride=(66, 264, 0)), -1, "multiples of 4"), (dict(key__words=4098), -1, "4-byte"),
    (dict(query=4100), -1, "16-byte"), (dict(query_stride=(1020, 256)), -1, "16-byte"),
    (dict(workspace=None), -1, "workspace"), (dict(workspace_bytes=8), -1, "workspace"), (dict(workspace=4100), -1, "workspace")])
def test_key_weights_refusals(lib, bad, status, text):
    assert lib.qp_key_weights(weight_args(**bad), None) == status
    assert text in lib.qp_last_error().decode()


def test_key_weights_with_nothing_to_do(lib):
    assert lib.qp_key_weights(weight_args(num_seqs=0), None) == 0
    assert lib.qp_key_weights(weight_args(max_seqlen_k=0), None) == 0
    assert lib.qp_key_weights(None, None) == -1 and lib.qp_key_weights_workspace_size(None) == 0
    assert lib.qp_key_weights_workspace_size(weight_args()) > 0


def test_key_weights_python_refusals(lib):
    from vllm_quantpack.attention.key_weights import key_weights
    q, out = torch.zeros((1, 4, 64), dtype=torch.bfloat16), torch.zeros((1, 2, 40))
    kc, ks = torch.zeros((3, 16, 2, 32), dtype=torch.uint8), torch.zeros((3, 16, 2))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    kw = dict(cu_seqlens_q=i32([0, 1]), seqused_k=i32([40]), block_table=i32([[0, 1, 2]]), max_seqlen_q=1, softmax_scale=0.1)
    bad = [(ValueError, "on a GPU", (q, kc, ks, out), {}), (NotImplementedError, "bf16", (q.float(), kc, ks, out), {}),
           (ValueError, "contiguous channels", (q.transpose(0, 2), kc, ks, out), {}),
           (ValueError, "uint8 or int8", (q, kc.float(), ks, out), {}), (ValueError, "heads of", (q, kc[..., :16], ks, out), {}),
           (ValueError, "heads of", (q, kc, ks[:2], out), {}), (ValueError, "out must be", (q, kc, ks, out.double()), {}),
           (ValueError, "out must be", (q, kc, ks, out[:, :1]), {}),
           (ValueError, "longest context", (q, kc, ks, out), dict(max_seqlen_k=41)),
           (ValueError, "previous", (q, kc, ks, out), dict(previous=out[..., :30])),
           (ValueError, "seqused_k", (q, kc, ks, out), dict(seqused_k=torch.tensor([40]))),
           (ValueError, "cu_seqlens_q", (q, kc, ks, out), dict(cu_seqlens_q=i32([0, 1, 1]))),
           (ValueError, "block_table", (q, kc, ks, out), dict(block_table=i32([0, 1, 2]))),
           (ValueError, "query_signs", (q, kc, ks, out), dict(query_signs=torch.ones(32)))]
    for error, text, args, more in bad:
        with pytest.raises(error, match=text):
            key_weights(*args, **{**kw, **more})


# ------------------------------------------------------------------------------------------------- qp_evict

def evict_args(**kw):
    from vllm_quantpack import _hip
    c, a = _hip.PagedCache(), _hip.EvictArgs()
    c.key, c.value = half(256), half(256)
    c.num_blocks, c.block_size, c.num_kv_heads, c.head_size = 8, 16, 1, 256
    a.weights = a.seqused_k = a.block_table = a.new_block_table = a.kept = a.new_weights = a.new_seqused_k = 4096
    a.max_blocks, a.new_max_blocks, a.num_seqs, a.max_seqlen_k, a.budget, a.sinks, a.recent = 4, 2, 1, 64, 32, 1, 2
    a.workspace, a.workspace_bytes = 4096, 1 << 20
    set_fields(a, {k: v for k, v in kw.items() if not k.startswith("cache_")})
    set_fields(c, {k[6:]: v for k, v in kw.items() if k.startswith("cache_")})
    return c, a


@pytest.mark.parametrize("bad,status,text", [
    (dict(weights=None), -1, "null tensor"), (dict(kept=None), -1, "null tensor"), (dict(new_seqused_k=None), -1, "null tensor"),
    (dict(cache_value__codes=None), -1, "null cache"), (dict(cache_head_size=96), -2, "head size"),
    (dict(cache_value__format=1), -1, "values int4"), (dict(cache_block_size=0), -1, "cache sizes"),
    (dict(cache_num_blocks=1 << 28), -2, "slots"), (dict(num_seqs=-1), -1, "sizes"), (dict(num_seqs=1 << 16), -2, "65535"),
    (dict(budget=0, sinks=0, recent=0), -1, "budget"), (dict(sinks=31), -1, "budget"), (dict(sinks=-1), -1, "budget"),
    (dict(recent=2 ** 31 - 1, sinks=2 ** 31 - 1), -1, "budget"), (dict(budget=33), -1, "room"),
    (dict(new_max_blocks=1), -1, "room"), (dict(cache_key__code_stride=(66, 264, 0)), -1, "multiples of 4"),
    (dict(cache_value__words=4097), -1, "4-byte"), (dict(workspace=None), -1, "workspace"),
    (dict(workspace_bytes=4), -1, "workspace"), (dict(workspace=4100), -1, "workspace")])
def test_evict_refusals(lib, bad, status, text):
    assert lib.qp_evict(*evict_args(**bad), None) == status
    assert text in lib.qp_last_error().decode()


def test_evict_with_nothing_to_do(lib):
    assert lib.qp_evict(*evict_args(num_seqs=0), None) == 0
    assert lib.qp_evict(None, None, None) == -1 and lib.qp_evict_workspace_size(None, None) == 0


def test_evict_keys_refusals(lib):
    from vllm_quantpack.attention.eviction import evict_keys
    kc, ks = torch.zeros((6, 16, 2, 32), dtype=torch.uint8), torch.zeros((6, 16, 2))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    w, used = torch.zeros((1, 2, 48)), i32([48])
    kw = dict(seqused_k=used, block_table=i32([[0, 1, 2]]), new_block_table=i32([[3, 4]]), budget=32)
    bad = [(ValueError, "on a GPU", {}), (ValueError, "weights must be", dict(max_seqlen_k=49)),
           (ValueError, "block_table must be", dict(block_table=i32([[0], [1]]))),
           (ValueError, "new_block_table must be", dict(new_block_table=torch.zeros((1, 2)))),
           (ValueError, "kept must be", dict(kept=torch.zeros((1, 2, 31), dtype=torch.int32))),
           (ValueError, "new_weights must be", dict(new_weights=torch.zeros((1, 1, 32)))),
           (ValueError, "other tensors", dict(new_weights=w)), (ValueError, "other tensors", dict(new_seqused_k=used)),
           (ValueError, "int32 vector", dict(seqused_k=torch.tensor([48])))]
    for error, text, more in bad:
        with pytest.raises(error, match=text):
            evict_keys(kc, kc, ks, ks, w, **{**kw, **more})
    with pytest.raises(ValueError, match="belong together"):
        evict_keys(kc, kc[..., :16], ks, ks, w, **kw)
    with pytest.raises(ValueError, match="weights must be"):
        evict_keys(kc, kc, ks, ks, w.double(), **kw)


# ------------------------------------------------------------------------------------- sizes that a launch cannot take

def test_refuses_sizes_past_the_launch_limits(lib):
    big = dict(num_tokens=1 << 21, num_splits=2, workspace=4096, workspace_bytes=1 << 62)
    assert lib.qp_prompt(prompt_args(**big), None) == -2 and "rows for splits" in lib.qp_last_error().decode()
    assert lib.qp_prompt_workspace_size(prompt_args(**big)) == 0
    assert lib.qp_prompt(prompt_args(num_tokens=1 << 28), None) == -2 and "rows" in lib.qp_last_error().decode()
    assert lib.qp_key_weights(weight_args(max_query_len=1 << 23), None) == -2 and "rows" in lib.qp_last_error().decode()
    long = (1 << 30) + 1
    assert lib.qp_key_weights(weight_args(max_seqlen_k=long), None) == -2 and "positions" in lib.qp_last_error().decode()
    assert lib.qp_key_weights_workspace_size(weight_args(max_seqlen_k=long)) == 0
    assert lib.qp_evict(*evict_args(max_seqlen_k=long), None) == -2 and "positions" in lib.qp_last_error().decode()


def test_refuses_gradients_and_moves_in_place(lib):
    from vllm_quantpack.attention.eviction import evict_keys
    from vllm_quantpack.attention.key_weights import key_weights
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    q, kc, ks = torch.zeros((1, 4, 64), dtype=torch.bfloat16), torch.zeros((6, 16, 2, 32), dtype=torch.uint8), torch.zeros((6, 16, 2))
    table = i32([[0, 1, 2]])
    with pytest.raises(NotImplementedError, match="backward"):
        key_weights(q.requires_grad_(), kc, ks, torch.zeros((1, 2, 40)), cu_seqlens_q=i32([0, 1]), seqused_k=i32([40]),
                    block_table=table, max_seqlen_q=1, softmax_scale=0.1)
    with pytest.raises(ValueError, match="must not be block_table"):
        evict_keys(kc, kc, ks, ks, torch.zeros((1, 2, 48)), seqused_k=i32([48]), block_table=table, new_block_table=table,
                   budget=32)
