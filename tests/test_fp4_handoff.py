"""The 4-bit product by pairs of CTAs comes to its end whichever of its bounded waits gives up: tests/fp4_handoff_check.cpp tries every
order of events of the hand-off between its copying warps and its issuer, with the rule the kernel has (csrc/fp4_handoff.h). CPU only."""
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "comfyui-hy-nomas_b200", "csrc")


@pytest.mark.parametrize("steps,tile", [(1, 1), (3, 1), (13, 4), (12, 6), (11, 1), (16, 16)])
def test_every_order_ends(tmp_path, steps, tile):
    exe = os.path.join(tmp_path, "check")
    subprocess.check_call(["g++", "-O2", "-std=c++17", "-I" + CSRC, "-o", exe, os.path.join(HERE, "fp4_handoff_check.cpp")])
    r = subprocess.run([exe, str(steps), str(tile)], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0 and "stuck 0" in r.stdout, r.stdout + r.stderr
