"""Several backward passes over one graph of a loss that keeps its gradient from the
forward pass (tests/cpp/repeated_backward.cpp): each pass adds the same gradient."""
import os
import shutil
import subprocess

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("loss", ["distill", "cross_entropy"])
def test_every_pass_adds_the_same(cuda, tmp_path, loss):
    lib, exe = os.path.join(ROOT, "tinytrain_b200", "lib"), tmp_path / "repeated_backward"
    gxx = shutil.which("g++")
    assert gxx
    r = subprocess.run([gxx, "-std=c++20", "-O2", "-Wall", "-I" + os.path.join(ROOT, "include"),
                        os.path.join(ROOT, "tests", "cpp", "repeated_backward.cpp"), "-L" + lib,
                        "-ltinytrain", "-lttk", "-Wl,-rpath," + lib, "-o", str(exe)],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([str(exe), loss], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "ok" in r.stdout, r.stdout + r.stderr
