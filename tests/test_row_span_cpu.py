"""The bulk copies of rows that are no whole number of 16-byte words stay inside their
tensors (tests/cpp/row_span.cpp checks csrc/row_span.h on the host)."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_whole_words_stay_inside(tmp_path):
    gxx = shutil.which("g++")
    if not gxx:
        pytest.skip("no g++")
    exe = tmp_path / "row_span"
    r = subprocess.run([gxx, "-std=c++17", "-O1", "-Wall", "-Werror",
                        "-I" + os.path.join(ROOT, "tinytrain_b200", "csrc"),
                        os.path.join(ROOT, "tests", "cpp", "row_span.cpp"), "-o", str(exe)],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and "ok" in r.stdout, r.stdout
