"""The launches of the norms' ring kernels, for every width, type and form of
rows (mhc-proj_b200/csrc/ring_plan.h): a launch that needs more shared memory than
a kernel has by default, beside its static memory, has to ask for it.  The
plan is host C++ with no CUDA dependency; it is compiled here with g++."""
import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "mhc-proj_b200", "csrc")


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_every_width_has_a_launch_that_fits(tmp_path):
    exe = str(tmp_path / "ring_plan_check")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I", CSRC,
                    os.path.join(HERE, "ring_plan_check.cpp"), "-o", exe], check=True)
    out = subprocess.run([exe], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout.strip() == "ok", out.stdout + out.stderr
