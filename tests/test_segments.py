"""The rule by which a context's keys are cut into segments, compiled for the host from the kernels' own header."""
import os
import shutil
import subprocess

import pytest

from conftest import REPO
from test_boundary import _build_module

MAIN = r"""
#include <stdio.h>
#include "qp_common.h"
int main() {
  const int lens[] = {0, 1, 31, 32, 33, 255, 256, 257, 1300, 65536, 1 << 30}, counts[] = {1, 2, 3, 16, 128}, floors[] = {0, 32, 256};
  for (int n : lens)
    for (int s : counts)
      for (int f : floors) {
        const int seg = qp::segment_keys(n, s, f);
        printf("%d %d %d %d %d\n", n, s, f, seg, qp::segments_used(n, s, seg));
      }
}
"""


def test_segments_of_a_context(tmp_path):
    """Segments are whole 32-key chunks, no shorter than the floor; those in use hold all keys, and no keys are in use by none."""
    build = _build_module()
    if shutil.which(build.hipcc()) is None:
        pytest.skip("no hipcc")
    src, exe = tmp_path / "segments.hip", tmp_path / "segments"
    src.write_text(MAIN)
    subprocess.run([build.hipcc(), "--offload-host-only", "-O1", "-std=c++17", "-I", os.path.join(REPO, "include"), "-I", build.CSRC,
                    str(src), "-o", str(exe)], check=True)
    lines = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines()
    assert len(lines) == 11 * 5 * 3
    for line in lines:
        n, splits, floor, seg, used = map(int, line.split())
        assert seg % 32 == 0 and seg >= floor and seg * splits >= n
        assert seg <= max(floor, -(-n // splits) + 31)
        assert used == (-(-n // seg) if n else 0) and used <= splits
