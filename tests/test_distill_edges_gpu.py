"""Distillation loss at the ends of its types' ranges and in the forms that the dispatch
takes for many rows. Definition and bounds as in test_distill_gpu.py."""
import math

import pytest
import torch

import test_distill_gpu as base

pytestmark = pytest.mark.gpu
U = base.U
# (rows, classes) of every kernel form: a warp per row; 8, 4 and 2 warps a row, each CTA
# over several rows
FORMS = [(1300, 700), (1300, 3001), (200, 5000), (1500, 5000), (700, 12000), (700, 33001)]


@pytest.mark.parametrize("N,C", [(5, 700), (1300, 700), (400, 5000)])
@pytest.mark.parametrize("offset,T", [(1e5, 3.0), (-1e5, 0.7), (1e6, 1.5)])
def test_teacher_logits_far_from_zero(cuda, N, C, offset, T):
    """A constant added to all teacher logits of a row changes nothing: their differences
    are exact, and only they are divided by T."""
    from tinytrain_b200 import kernels as KN
    x, ids, top, t, _ = base.make(N, C, 40, cuda)
    top = (top * 8).round() / 8 + offset  # eighths: the sums are exact
    out = KN.distill_loss(x, ids, top, t, alpha=0.5, temperature=T)
    base.check(out, base.define(x, ids, top, t, 0.5, T), x, T)
    near = KN.distill_loss(x, ids, top - offset, t, alpha=0.5, temperature=T)
    assert torch.equal(near[0], out[0]) and torch.equal(near[1], out[1])
    assert base.status() == 0


@pytest.mark.parametrize("N,C", [(6, 700), (1302, 700), (402, 5000)])
@pytest.mark.parametrize("T", [0.5, 0.01])
def test_teacher_logits_at_the_types_ends(cuda, N, C, T):
    """Lists of the lowest value alone are uniform, entries at the lowest value beside
    others have probability 0, and the largest values share a list: z / T is no fp32
    number in any of them."""
    from tinytrain_b200 import kernels as KN
    x, ids, top, t, _ = base.make(N, C, 7, cuda, spread=0.3)
    low, high = torch.finfo(torch.float32).min, torch.finfo(torch.float32).max
    top[0::3] = low
    top[1::3, 3:] = low
    top[2::3, :2] = high
    out = KN.distill_loss(x, ids, top, t, alpha=0.5, temperature=T)
    base.check(out, base.define(x, ids, top, t, 0.5, T), x, T)
    assert torch.isfinite(out[0]).all() and torch.isfinite(out[1]).all()
    assert base.status() == 0


@pytest.mark.parametrize("N,C", [(6, 700), (1302, 700), (402, 5000)])
@pytest.mark.parametrize("T", [1.0, 2.0, 4.0])
def test_listed_classes_at_the_lowest_value(cuda, N, C, T):
    """A label or a listed class whose logit is the type's lowest value has a large
    finite loss, 3.4e38 for the label: a few roundings of the one term that counts."""
    from tinytrain_b200 import kernels as KN
    x, ids, top, t, _ = base.make(N, C, 5, cuda)
    low = torch.finfo(torch.float32).min
    t = (ids[:, 0].long() + 1) % C
    x[0, t[0]] = low
    loss, d = KN.distill_loss(x, ids, top, t, alpha=0.5, temperature=T, grad_scale=0.5)
    want = base.define(x, ids, top, t, 0.5, T, scale=0.5)[0]
    assert abs(float(loss[2]) / float(want[2]) - 1) <= 8 * U
    assert abs(float(loss[0]) / float(want[0]) - 1) <= 8 * U
    assert abs(float(loss[1]) / float(want[1]) - 1) <= 400 * U
    x, ids, top, t, _ = base.make(N, C, 5, cuda)
    x[0, ids[0, 1].long()] = low
    t[:] = -1
    loss, d = KN.distill_loss(x, ids, top, t, alpha=1.0, temperature=T, grad_scale=0.125 / T)
    want = base.define(x, ids, top, t, 1.0, T, scale=0.125 / T)[0]
    assert float(loss[2]) == 0
    # p of one entry, with the teacher's exponential and sum around it
    assert abs(float(loss[0]) / float(want[0]) - 1) <= 60 * U
    assert torch.isfinite(d).all()
    assert base.status() == 0
