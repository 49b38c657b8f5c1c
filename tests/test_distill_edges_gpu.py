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


@pytest.mark.parametrize("N,C", FORMS)
@pytest.mark.parametrize("alpha,T", [(1.0, 1.0), (0.5, 1.0), (0.5, 2.0)])
@pytest.mark.parametrize("K", [5, 33, 200])
def test_forms(cuda, N, C, alpha, T, K):
    """Loss and gradient, loss alone, the gradient in place, and without labels, in every
    kernel form with a CTA or a warp over several rows."""
    from tinytrain_b200 import kernels as KN
    x, ids, top, t, _ = base.make(N, C, K, cuda)
    for labels in (t, None):
        want = base.define(x, ids, top, labels, alpha, T)
        out = KN.distill_loss(x, ids, top, labels, alpha=alpha, temperature=T)
        base.check(out, want, x, T)
        only, _ = KN.distill_loss(x, ids, top, labels, alpha=alpha, temperature=T, want_grad=False)
        base.check((only, None), want, x, T)
        work = x.clone()
        loss, d = KN.distill_loss(work, ids, top, labels, alpha=alpha, temperature=T, dlogits=work)
        assert torch.equal(d, out[1]) and torch.equal(loss, out[0])
    assert base.status() == 0


@pytest.mark.parametrize("N,C", FORMS)
def test_longest_lists(cuda, N, C):
    """Lists of 1000 of the classes (700 of 700): the largest tables in shared memory."""
    from tinytrain_b200 import kernels as KN
    K = min(C, 1000)
    x, ids, top, t, _ = base.make(N, C, K, cuda)
    want = base.define(x, ids, top, t, 0.5, 2.0)
    base.check(KN.distill_loss(x, ids, top, t, alpha=0.5, temperature=2.0), want, x, 2.0)
    only, _ = KN.distill_loss(x, ids, top, t, alpha=0.5, temperature=2.0, want_grad=False)
    base.check((only, None), want, x, 2.0)
    # without labels one temperature is left
    base.check(KN.distill_loss(x, ids, top, alpha=0.5, temperature=2.0),
               base.define(x, ids, top, None, 0.5, 2.0), x, 2.0)
    assert base.status() == 0


@pytest.mark.parametrize("N,C", FORMS)
@pytest.mark.parametrize("K", [8, 40, 300])
@pytest.mark.parametrize("T", [1.0, 2.0])
def test_repeated_classes(cuda, N, C, K, T):
    """Some rows list classes more than once, the rows around them do not: the lists take
    turns in two buffers."""
    from tinytrain_b200 import kernels as KN
    x, ids, top, t, g = base.make(N, C, K, cuda)
    some = torch.rand(N, device=cuda, generator=g) < 0.4
    few = torch.randint(0, max(2, K // 3), (N, K), device=cuda, generator=g).int()
    ids = torch.where(some[:, None], few, ids).contiguous()
    t = torch.where(some, t % max(2, K // 3), t)
    want = base.define(x, ids, top, t, 0.5, T)
    out = KN.distill_loss(x, ids, top, t, alpha=0.5, temperature=T)
    base.check(out, want, x, T)
    assert torch.equal(KN.distill_loss(x, ids, top, t, alpha=0.5, temperature=T)[1], out[1])
    assert base.status() == 0


@pytest.mark.parametrize("N,C", FORMS)
@pytest.mark.parametrize("pad,shift", [(24, 0), (1, 0), (0, 1), (3, 2)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_strides_and_teacher_types(cuda, N, C, pad, shift, dtype):
    """Rows of wider buffers that start on any 4-byte boundary, the gradient beside them, in
    rows of another alignment and in place; teachers of every type."""
    from tinytrain_b200 import kernels as KN
    x, ids, top, t, _ = base.make(N, C, 9, cuda, dtype)
    buf = torch.full((N * (C + pad) + shift,), 77.0, device=cuda)
    view = buf[shift:].view(N, C + pad)[:, :C]
    view.copy_(x)
    wide = torch.full((N, C + 5), -3.0, device=cuda)
    for T in (1.0, 2.0):
        want = base.define(x, ids, top, t, 0.5, T)
        base.check(KN.distill_loss(view, ids, top, t, alpha=0.5, temperature=T), want, x, T)
        out = KN.distill_loss(view, ids, top, t, alpha=0.5, temperature=T, dlogits=wide[:, :C])
        base.check(out, want, x, T)
        assert (wide[:, C:] == -3.0).all()
    out = KN.distill_loss(view, ids, top, t, alpha=0.5, temperature=T, dlogits=view)
    base.check(out, want, x, T)
    if pad:
        assert (buf[shift:].view(N, C + pad)[:, C:] == 77.0).all()
    assert base.status() == 0


@pytest.mark.parametrize("N,C", FORMS)
@pytest.mark.parametrize("T", [1.0, 2.0])
def test_masks_and_not_numbers(cuda, N, C, T):
    """Rows with -inf classes, ragged lists, missing labels and weights of zero; then NaN in
    one row's logits and -inf in the whole of another: only those rows' gradients are NaN."""
    from tinytrain_b200 import kernels as KN
    K = 24
    x, ids, top, t, g = base.make(N, C, K, cuda)
    x[:, : C // 3] = -math.inf
    allowed = torch.where(torch.isinf(x), -1e4, x)
    top, ids = allowed.topk(K, 1)
    t = ids[:, 3].contiguous()
    n = torch.randint(0, K + 1, (N, 1), device=cuda, generator=g)
    ids = torch.where(torch.arange(K, device=cuda) < n, ids, -1).int().contiguous()
    t[torch.rand(N, device=cuda, generator=g) < 0.2] = -1
    w = (torch.rand(N, device=cuda, generator=g) > 0.3).float() * 1.5
    w[[1, 2, 3]] = 1.0
    t[[1, 2]] = C - 1
    clean = torch.where((w == 0)[:, None], 0.0, x)
    x[w == 0] = math.nan
    # -inf - -inf on the rows that count: the definition's terms of probability 0
    want = base.define(torch.where(torch.isinf(clean), -1e30, clean), ids, top, t, 0.6, T, w)
    out = KN.distill_loss(x, ids, top, t, alpha=0.6, temperature=T, row_weight=w)
    base.check(out, want, torch.where(torch.isinf(clean), 0.0, clean), T)
    assert (out[1][w == 0] == 0).all()
    x[1, C - 2] = math.nan
    x[2] = -math.inf
    loss, d = KN.distill_loss(x, ids, top, t, alpha=0.6, temperature=T, row_weight=w)
    assert torch.isnan(loss[0]) and torch.isnan(d[1]).all() and torch.isnan(d[2]).all()
    rest = torch.ones(N, dtype=torch.bool, device=cuda)
    rest[[1, 2]] = False
    assert torch.equal(d[rest], out[1][rest])
    assert base.status() == 0
