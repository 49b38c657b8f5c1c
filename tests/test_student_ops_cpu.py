"""Refusals of the scaled embedding, residual norm and distillation entry
points: every bad argument is turned down with TTK_ERR_ARG and a message before
anything is launched, so the checks run on a machine without a GPU (the
pointers are never followed)."""
import pytest
import torch

PTR = 1 << 20  # a non-null, aligned address that no check follows
BIG = 1 << 40


def refused(name, *args):
    from tinytrain_b200 import _ttk
    with pytest.raises(_ttk.TtkError, match=r"\(1\): " + name[4:]):
        _ttk.call(name, *args)


def test_embedding_scaled_refusals():
    f, b = "ttk_embedding_scaled_fwd", "ttk_embedding_scaled_bwd"
    refused(f, 0, PTR, PTR, 4, 8, 16, 1.0, 0)
    refused(f, PTR, 0, PTR, 4, 8, 16, 1.0, 0)
    refused(f, PTR, PTR, 0, 4, 8, 16, 1.0, 0)
    refused(f, PTR, PTR, PTR, -1, 8, 16, 1.0, 0)
    refused(f, PTR, PTR, PTR, 4, 0, 16, 1.0, 0)
    refused(f, PTR, PTR, PTR, 4, 8, 0, 1.0, 0)
    refused(b, 0, PTR, PTR, 0, 4, 8, 16, 1.0, PTR, BIG, 0)
    refused(b, PTR, 0, PTR, 0, 4, 8, 16, 1.0, PTR, BIG, 0)
    refused(b, PTR, PTR, 0, 0, 4, 8, 16, 1.0, PTR, BIG, 0)
    refused(b, PTR, PTR, PTR, 0, 1 << 31, 8, 16, 1.0, PTR, BIG, 0)
    refused(b, PTR, PTR, PTR, 0, 4, 8, 1 << 31, 1.0, PTR, BIG, 0)
    refused(b, PTR, PTR, PTR, 0, 4, 8, 16, 1.0, 0, BIG, 0)
    refused(b, PTR, PTR, PTR, 0, 4, 8, 16, 1.0, PTR + 4, BIG, 0)
    from tinytrain_b200 import _ttk
    n = _ttk.call("ttk_embedding_scaled_bwd_workspace_size", 4, 8, 16)
    refused(b, PTR, PTR, PTR, 0, 4, 8, 16, 1.0, PTR, n - 1, 0)


def test_residual_norm_refusals():
    f, b = "ttk_residual_norm_fwd", "ttk_residual_norm_bwd"
    ok = [PTR, PTR, PTR, 0, 0, PTR, PTR, PTR, PTR, PTR, 0, 4, 64, 1.0, 1e-5, 0]
    for i, v in ((0, 0), (1, 0), (2, 0), (6, 0), (7, 0), (8, 0), (9, 0), (11, -1), (12, 0)):
        refused(f, *(v if j == i else a for j, a in enumerate(ok)))
    refused(f, *ok[:4], 1, *ok[5:])  # a gate's kind without a gate
    refused(f, *ok[:3], PTR, 5, *ok[5:])
    refused(f, *ok[:10], PTR, 4, 65, *ok[13:])  # planes of a width that is no multiple of 32
    refused(f, *ok[:10], PTR + 8, *ok[11:])
    refused(f, *ok[:5], 0, *ok[6:10], PTR, *ok[11:])  # planes without the second norm
    ok = [PTR] * 5 + [0, 0, PTR, PTR, PTR, PTR, PTR, PTR, PTR, 0, 0, 4, 64, 1.0, PTR, BIG, 0]
    for i, v in ((2, 0), (3, 0), (4, 0), (7, 0), (8, 0), (9, 0), (10, 0), (11, 0), (15, 16), (16, -1),
                 (17, 0), (19, 0), (19, PTR + 4), (20, 0)):
        refused(b, *(v if j == i else a for j, a in enumerate(ok)))
    refused(b, 0, 0, *ok[2:])
    refused(b, *ok[:6], 2, *ok[7:])


def test_distill_refusals():
    f = "ttk_distill_loss"
    ok = [PTR, 100, PTR, PTR, 0, 5, PTR, 0, 4, 100, 0.5, 2.0, 0.25, PTR, PTR, 100, PTR, BIG, 0]
    bad = [(0, 0), (1, 99), (2, 0), (3, 0), (4, 3), (4, -1), (5, -1), (5, 1025), (8, -1), (9, 0),
           (9, 1 << 31), (10, -0.1), (10, 1.1), (10, float("nan")), (11, 0.0), (11, -1.0),
           (11, float("inf")), (11, float("nan")), (13, 0), (15, 99), (16, 0), (16, PTR + 4), (17, 63)]
    for i, v in bad:
        refused(f, *(v if j == i else a for j, a in enumerate(ok)))
    refused(f, *ok[:14], PTR, 104, *ok[16:])  # in place with another stride


def test_front_end_refusals():
    """kernels.py turns down tensors it would misread: other types, shapes, strides, devices."""
    from tinytrain_b200 import kernels as K
    W, ids = torch.zeros(4, 8), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="W: expected a contiguous float32 CUDA"):
        K.embedding_scaled_fwd(W, ids)
    with pytest.raises(ValueError, match="x: expected"):
        K.residual_norm_fwd(W, W, W[0], W[0])
    with pytest.raises(ValueError, match="logits: expected"):
        K.distill_loss(W, torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 2))


def test_programs_compile(tmp_path):
    """The example and the device test program build against the headers and libraries."""
    import os
    import shutil
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    lib = os.path.join(root, "tinytrain_b200", "lib")
    gxx = shutil.which("g++")
    if not gxx:
        pytest.skip("no g++")
    for src in (("examples", "distill_student.cpp"), ("tests", "cpp", "student_ops.cpp")):
        r = subprocess.run([gxx, "-std=c++20", "-O1", "-Wall", "-Werror",
                            "-I" + os.path.join(root, "include"), os.path.join(root, *src),
                            "-L" + lib, "-ltinytrain", "-lttk", "-Wl,-rpath," + lib, "-o",
                            str(tmp_path / "prog")], capture_output=True, text=True)
        assert r.returncode == 0, r.stderr[-3000:]
