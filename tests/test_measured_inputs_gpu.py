"""The inputs of the measured cases (perf/operators.py) are fixed by their seed: two
preparations of a case give the same bits, so that outputs made from one can be
compared with outputs made from the other."""
import os
import random
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "perf"))
import operators  # noqa: E402

DRAWN = [dict(operators.draw(random.Random(s)), name=f"drawn{s}") for s in range(12)]


def tensors(state):
    return {k: v for k, v in state.items() if torch.is_tensor(v)}


@pytest.mark.gpu
@pytest.mark.parametrize("case", operators.listed() + DRAWN, ids=lambda c: c["name"])
def test_same_seed_same_inputs(cuda, case):
    first = tensors(operators.prepare(case, 3))
    # the ids are made in microseconds: often, since what varies varies now and then
    for _ in range(30 if "ids" in first and case["op"].startswith("embed") else 3):
        again = tensors(operators.prepare(case, 3))
        assert first.keys() == again.keys()
        for name, t in first.items():
            assert torch.equal(t, again[name]), name
        del again
    other = tensors(operators.prepare(case, 4))
    assert any(not torch.equal(t, other[k]) for k, t in first.items())


@pytest.mark.parametrize("N,V,pad", [(1, 1000, False), (513, 1000, True), (32768, 32000, True)])
def test_token_frequencies(N, V, pad):
    """Ids in range, padding at the ends, and the first id as often as its share (five
    standard deviations)."""
    g = torch.Generator().manual_seed(7)
    ids = operators._tokens(N, V, pad, g)
    padded = torch.arange(N) % 512 >= 448 if pad else torch.zeros(N, dtype=torch.bool)
    assert ids.dtype == torch.int64 and ids.shape == (N,)
    assert ((ids == -1) == padded).all() and ids.max() < V and ids.min() >= -1
    n = int((~padded).sum())
    share = (1 / 2.7) / sum(1 / (r + 2.7) for r in range(V))
    assert abs(int((ids == 0).sum()) - n * share) <= 5 * (n * share * (1 - share)) ** 0.5 + 1


@pytest.mark.parametrize("N", [1, 448, 449, 512, 700, 32768])
def test_padding_is_no_work(N):
    """A gradient's bytes count the rows of dout that have a token."""
    D, V = 64, 1000
    live = sum(i % 512 < 448 for i in range(N))
    case = dict(op="embed_bwd", N=N, D=D, V=V, pad=True)
    assert operators.work(case)["bytes"] == 4 * live * D + 4 * V * D + 8 * N
    assert operators.work(dict(case, pad=False))["bytes"] == 4 * N * D + 4 * V * D + 8 * N
