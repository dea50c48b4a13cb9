"""The gfx950 code of the softmax losses (CPU-only check): what no kernel of
dist-lr_amd/csrc may hold, in this file's dump (`make asm-losses`) and in the
engine's (`make asm`)."""
from __future__ import annotations

import functools
import os
import re
import subprocess

import pytest

from test_abi import ROOT, _kernel_bodies

pytestmark = pytest.mark.skipif(not os.path.exists("/opt/rocm/bin/hipcc"), reason="hipcc not available")


@functools.lru_cache(maxsize=None)
def dump(target, name):
    subprocess.run(["make", "-s", "-C", os.path.join(ROOT, "dist-lr_amd"), target], check=True)
    with open(os.path.join(ROOT, "dist-lr_amd", "build", name)) as f:
        return f.read()


def instructions(text):
    bodies = _kernel_bodies(text)
    assert len(bodies) > 20
    for name, body in bodies.items():
        for line in body:
            if line and not line.startswith((";", ".")):
                yield name[:80], line


def test_no_scalar_stores_or_atomics_in_the_losses():
    forbidden = pytest.importorskip("test_isa_scalar").FORBIDDEN  # the mnemonics, in a file that stays on the CPU
    bad = [at for at in instructions(dump("asm-losses", "dlr_losses.s")) if at[1].startswith(forbidden)]
    assert not bad, bad[:10]


@pytest.mark.parametrize("target,name", [("asm", "dlr_kernels.s"), ("asm-losses", "dlr_losses.s")])
def test_no_packed_32_bit_arithmetic(target, name):
    # some of its forms have given wrong results: the build turns it off
    bad = [at for at in instructions(dump(target, name)) if re.match(r"v_pk_(add|mul|fma)_f32\b", at[1])]
    assert not bad, bad[:10]


def test_the_losses_keep_their_vectors_in_registers():
    # no vector register is spilled; a kernel that nothing launches would not be tuned either
    text = dump("asm-losses", "dlr_losses.s")
    kernels = re.findall(r"^    \.name:\s+(\S+)", text, re.M)
    spills = [int(n) for n in re.findall(r"\.vgpr_spill_count:\s+(\d+)", text)]
    scratch = [int(n) for n in re.findall(r"\.private_segment_fixed_size:\s+(\d+)", text)]
    assert len(kernels) == len(spills) == len(scratch) > 20
    assert not any(spills) and not any(scratch), [k for k, n, s in zip(kernels, spills, scratch) if n or s]


def test_only_kernels_that_a_call_reaches():
    # rows in 16 bits are held by 512 threads at most (launch_policy_loss): 1,024 are for float32
    text = dump("asm-losses", "dlr_losses.s")
    held = re.findall(r"^    \.name:\s+(_ZN\S*k_policy_lossI\S+)", text, re.M)
    assert held and all("k_policy_lossIf" in k for k in held if "Li1024E" in k)
    for dtype, kinds in (("f", 6), ("DF16b", 5), ("DF16_", 5)):
        assert sum(("k_policy_lossI" + dtype + "L") in k for k in held) == kinds, held
