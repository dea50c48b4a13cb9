"""Two HIP runtimes in one process: what does not see the GPU then says why (no
GPU needed: nothing sees one here)."""
from __future__ import annotations

import os
import subprocess
import sys

import pytest

torch = pytest.importorskip("torch")

from conftest import ROOT  # noqa: E402

OWN = os.path.join(os.path.dirname(torch.__file__), "lib", "libamdhip64.so")

PROGRAM = """
import sys
sys.path.insert(0, {path!r})
import {order}
import distlr_amd, torch, distlr_amd.losses
if torch.cuda.is_available():
    sys.exit(3)
for call in (lambda: distlr_amd.Engine(16), lambda: distlr_amd.Engine.create_group(16, 2),
             lambda: distlr_amd.losses.token_logprob(torch.zeros(2, 3), torch.zeros(2, dtype=torch.int64))):
    try:
        call()
    except distlr_amd.DLRError as e:
        print(e.code, "import torch before distlr_amd" in str(e), len(distlr_amd.hip_runtimes()))
"""


@pytest.mark.skipif(not os.path.exists(OWN), reason="torch brings no HIP runtime of its own")
@pytest.mark.parametrize("order,two", [("torch", False), ("distlr_amd", True), ("distlr_amd.losses", True)])
def test_the_cause_is_named(order, two):
    if torch.cuda.is_available():
        pytest.skip("every runtime sees the GPU at first here")
    prog = PROGRAM.format(path=os.path.join(ROOT, "dist-lr_amd"), order=order)
    out = subprocess.run([sys.executable, "-c", prog], check=True, capture_output=True, text=True).stdout.split("\n")
    n = 2 if two else 1
    assert out[:3] == [f"-4 {two} {n}", f"-4 {two} {n}", f"-1 {two} {n}"], out
