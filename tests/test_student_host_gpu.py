"""The C++ side of the student operators on the device: tests/cpp/student_ops.cpp
(the graph nodes against compositions of the other ops) and the example that
trains a student with them; and the operators inside a CUDA graph."""
import os
import shutil
import subprocess

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def build(src, out):
    lib = os.path.join(ROOT, "tinytrain_b200", "lib")
    gxx = shutil.which("g++")
    assert gxx
    r = subprocess.run([gxx, "-std=c++20", "-O2", "-Wall", "-I" + os.path.join(ROOT, "include"),
                        os.path.join(ROOT, *src), "-L" + lib, "-ltinytrain", "-lttk",
                        "-Wl,-rpath," + lib, "-o", str(out)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]


def test_nodes_against_compositions(cuda, tmp_path):
    exe = tmp_path / "student_ops"
    build(("tests", "cpp", "student_ops.cpp"), exe)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "ok" in r.stdout, r.stdout + r.stderr


def test_example_learns(cuda, tmp_path):
    exe = tmp_path / "distill_student"
    build(("examples", "distill_student.cpp"), exe)
    r = subprocess.run([str(exe), "30"], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    lines = [ln for ln in r.stdout.splitlines() if ln.startswith("step")]
    losses = [float(ln.split("loss")[1].split()[0]) for ln in lines]
    assert len(losses) >= 3 and losses[-1] < 0.7 * losses[0], r.stdout


def test_in_a_cuda_graph(cuda):
    """Recorded once and replayed on new contents of the same buffers: the bits of
    the calls made directly."""
    import torch

    from tinytrain_b200 import kernels as K
    g = torch.Generator(device=cuda).manual_seed(3)
    N, D, V, C, k = 700, 256, 900, 5000, 20

    def fill():
        return dict(ids=torch.randint(-1, V, (N,), device=cuda, generator=g),
                    W=torch.randn(V, D, device=cuda, generator=g),
                    x=torch.randn(N, D, device=cuda, generator=g),
                    b=torch.randn(N, D, device=cuda, generator=g),
                    w=torch.rand(D, device=cuda, generator=g) + 0.5,
                    logits=torch.randn(N, C, device=cuda, generator=g),
                    tid=torch.randint(0, C, (N, k), device=cuda, generator=g).int(),
                    top=torch.randn(N, k, device=cuda, generator=g),
                    t=torch.randint(0, C, (N,), device=cuda, generator=g))

    def run(s):
        e = K.embedding_scaled_fwd(s["W"], s["ids"], 2.0)
        h, y, r1, r2 = K.residual_norm_fwd(e, s["b"], s["w"], s["w"], gate=s["w"])
        d = K.residual_norm_bwd(s["x"], y, h, s["b"], s["w"], s["w"], r1, r2, gate=s["w"])
        dW = K.embedding_scaled_bwd(d[0], s["ids"], V, 2.0)
        loss, dl = K.distill_loss(s["logits"], s["tid"], s["top"], s["t"], alpha=0.5,
                                  temperature=2.0)
        return [e, h, y, *d, dW, loss, dl]

    s = fill()
    run(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(s)
    for _ in range(3):
        new = fill()
        for key, v in new.items():
            s[key].copy_(v)
        graph.replay()
        want = run(new)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
