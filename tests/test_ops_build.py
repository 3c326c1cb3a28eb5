"""The build's checks of generated code reach the sources in csrc/ops, as those of csrc."""
import os
import re

import pytest

from test_boundary import _build_module

LOOPS = {"qp_prompt": 14, "qp_key_weights": 16}  # kernels that loop over MFMAs: instances by head, type, waves or pass


def _listing(build, name):
    path = os.path.join(build.OBJ, f"{name}.gfx.s")
    if not os.path.exists(path):
        pytest.skip("not built")
    return open(path).read()


def test_sources_with_mfmas():
    build = _build_module()
    ops = os.path.join(build.CSRC, "ops")
    found = [n[:-4] for n in sorted(os.listdir(ops)) if n.endswith(".hip") and build.has_mfma(open(os.path.join(ops, n)).read())]
    assert found == sorted(LOOPS)


def test_the_build_checks_every_source(monkeypatch):
    """build() compiles, checks and links all of csrc and csrc/ops (nothing is run here)."""
    build = _build_module()
    compiled, checked, linked = [], [], []

    class Done:
        returncode = 0

    monkeypatch.setattr(build, "_compile", lambda src, verbose: compiled.append(os.path.basename(src)) or False)
    monkeypatch.setattr(build, "_check_mfma", lambda src, verbose, scheduled: checked.append(os.path.basename(src)))
    monkeypatch.setattr(build.subprocess, "run", lambda cmd, **kw: linked.extend(cmd) or Done())
    monkeypatch.setattr(build.os, "replace", lambda a, b: None)
    build.build(jobs=1)
    want = sorted(n for d in ("", "ops") for n in os.listdir(os.path.join(build.CSRC, d)) if n.endswith(".hip"))
    assert sorted(compiled) == sorted(checked) == want and {"qp_prompt.hip", "qp_key_weights.hip", "qp_evict.hip"} <= set(want)
    assert sorted(os.path.basename(x) for x in linked if x.endswith(".o")) == [n[:-4] + ".o" for n in want]


@pytest.mark.parametrize("name", sorted(LOOPS))
def test_built_loops_hold_no_spill_code(name):
    build = _build_module()
    text = _listing(build, name)
    assert build.spills_in_mfma_loops(text) == [] and build.mfma_hazards(text) == []
    assert build.valu_writes_before_mfma(text) == []
    assert sum(1 for hot in build.mfma_loops(text).values() if hot) == LOOPS[name]


@pytest.mark.parametrize("name", sorted(LOOPS))
def test_vector_registers_that_spill(name):
    """The first pass of key_weights over int4 keys of 512 spills a few registers around its blocks of keys; no other kernel
    any."""
    text = _listing(_build_module(), name)
    spills = {fn: int(n) for fn, n in re.findall(r"\.name: +(_ZN\S+)\n(?:(?!\.name:).*\n)*? +\.vgpr_spill_count: +(\d+)", text)}
    assert len(spills) >= LOOPS[name]
    few = {fn: n for fn, n in spills.items() if n}
    assert few == {} or (all("key_weights_kernelILi512ELi0ELi1E" in fn for fn in few) and max(few.values()) <= 6), few
