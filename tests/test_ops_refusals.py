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
STRUCTS = {"PromptArgs": "qp_prompt_args"}


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
