"""Distillation loss on a teacher's top logits and its gradient, against the
definition in 64 bits.

Tolerance, with u = 2^-24: exp is the hardware's 2^x (4 u) of an argument
|x - m| / T with 3 roundings, so a term of a softmax is within
(4 + 3 |x - m| / T) u; the sums behind it add at most (C / 256 + 40) u. A
gradient element is within that many u of alpha T (q_T + P) + (1 - alpha)(q_1 +
onehot), times the row's weight; a loss within that many u of the terms'
magnitudes sum_k p_k (|log p_k| + |log q_T| + 1) and |log q_1| + 1.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def status():
    from tinytrain_b200 import _ttk
    return _ttk.device_status()


def make(N, C, K, dev, dtype=torch.float32, seed=0, spread=3.0):
    g = torch.Generator(device=dev).manual_seed(31 * N + C + K + seed)
    x = torch.randn(N, C, device=dev, generator=g) * spread
    teacher = x + torch.randn(N, C, device=dev, generator=g)
    top, ids = teacher.topk(K, 1)
    t = torch.randint(0, C, (N,), device=dev, generator=g)
    return x, ids.int().contiguous(), top.to(dtype).contiguous(), t, g


def define(x, ids, top, t, alpha, T, w=None, scale=None):
    """(loss [3], gradient, their magnitudes) in 64 bits; ids -1 and t None / -1 as documented."""
    x, z = x.double(), top.double() / T
    N, C = x.shape
    scale = 1.0 / N if scale is None else scale
    w = torch.ones(N, device=x.device, dtype=torch.float64) if w is None else w.double()
    w = w * scale
    z = torch.where(ids >= 0, z, -math.inf)
    has = (z > -math.inf).any(1)
    p = torch.where(has[:, None], torch.softmax(z, 1), 0.0)
    P = torch.zeros_like(x).scatter_add_(1, ids.clamp(min=0).long(), p)
    lq, l1 = torch.log_softmax(x / T, 1), torch.log_softmax(x, 1)
    lqk = lq.gather(1, ids.clamp(min=0).long())
    on = p > 0
    lp = torch.where(on, torch.log(p), 0.0)
    kd = torch.where(on, p * (lp - lqk), 0.0).sum(1)
    kdm = torch.where(on, p * (lp.abs() + lqk.abs() + 1), 0.0).sum(1)
    onehot = torch.zeros_like(x)
    lab = torch.zeros(N, dtype=torch.bool, device=x.device) if t is None else t >= 0
    if t is not None:
        onehot[lab, t[lab]] = 1.0
    ce = torch.where(onehot > 0, -l1, 0.0).sum(1)
    off = (w == 0) | (~has & ~lab)
    zero = lambda v: torch.where(off if v.dim() == 1 else off[:, None], 0.0, v)  # noqa: E731
    kd, kdm, ce = zero(kd), zero(kdm), zero(ce)
    hasd, labd = has.double()[:, None], lab.double()[:, None]
    grad = w[:, None] * (alpha * T * (hasd * lq.exp() - P) + (1 - alpha) * (labd * l1.exp() - onehot))
    gmag = w.abs()[:, None] * (alpha * T * (hasd * lq.exp() + P) + (1 - alpha) * (labd * l1.exp() + onehot))
    KD, CE = (w * kd).sum(), (w * ce).sum()
    KDm, CEm = (w.abs() * kdm).sum(), (w.abs() * (ce.abs() + lab.double())).sum()
    mix = lambda a, b: torch.stack([(alpha * T * T * a if alpha else 0 * b)  # noqa: E731
                                    + ((1 - alpha) * b if alpha < 1 else 0 * a), a, b])
    return mix(KD, CE), zero(grad), mix(KDm, CEm), zero(gmag)


def check(out, want, x, T):
    (loss, d), (rl, rd, ml, md) = out, want
    C = x.shape[1]
    xd = x.double()
    fin = torch.where(torch.isinf(xd), 0.0, xd)
    far = (fin.max(1, keepdim=True).values - fin).abs()
    c = 4 + 3 * far / min(T, 1.0) + C / 256 + 40
    err = (loss.double() - rl).abs()
    assert (err <= (float(c.max())) * U * ml).all(), (err / (U * ml), float(c.max()))
    if d is not None:
        bad = ~((d.double() - rd).abs() <= c * U * md + 1e-37)
        assert not bad.any(), float(((d.double() - rd).abs() / (U * md + 1e-37)).max())


@pytest.mark.parametrize("N,C,K", [(1, 1, 1), (1, 2, 2), (3, 5, 3), (2, 31, 7), (5, 32, 32),
                                   (17, 1000, 16), (4, 1023, 100), (3, 4096, 1024), (7, 8193, 64),
                                   (300, 2048, 20), (33, 32000, 64), (5, 32001, 8), (2, 49999, 50),
                                   (3, 65536, 33), (2, 131072, 16), (1, 262147, 5), (2, 600000, 9)])
@pytest.mark.parametrize("alpha,T", [(1.0, 1.0), (0.5, 2.0), (0.0, 1.0), (0.3, 0.5), (1.0, 4.0)])
def test_loss_and_gradient(cuda, N, C, K, alpha, T):
    from tinytrain_b200 import kernels as KN
    x, ids, top, t, _ = make(N, C, K, cuda)
    want = define(x, ids, top, t, alpha, T)
    keep = x.clone()
    out = KN.distill_loss(x, ids, top, t, alpha=alpha, temperature=T)
    check(out, want, x, T)
    assert torch.equal(x, keep)
    # loss alone
    only, none = KN.distill_loss(x, ids, top, t, alpha=alpha, temperature=T, want_grad=False)
    assert none is None
    check((only, None), want, x, T)
    # the gradient over the logits, and equal bits of equal calls
    loss2, d2 = KN.distill_loss(keep, ids, top, t, alpha=alpha, temperature=T, dlogits=keep)
    assert d2.data_ptr() == keep.data_ptr()
    assert torch.equal(d2, out[1]) and torch.equal(loss2, out[0])
    # without labels
    out = KN.distill_loss(x, ids, top, alpha=alpha, temperature=T)
    check(out, define(x, ids, top, None, alpha, T), x, T)
    assert float(out[0][2]) == 0.0
    assert status() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_teacher_types(cuda, dtype):
    from tinytrain_b200 import kernels as KN
    x, ids, top, t, _ = make(40, 5000, 30, cuda, dtype)
    check(KN.distill_loss(x, ids, top, t, alpha=0.7, temperature=1.5),
          define(x, ids, top, t, 0.7, 1.5), x, 1.5)


@pytest.mark.parametrize("C", [700, 3001, 32000, 70001])
def test_ragged_lists_labels_and_masked_rows(cuda, C):
    """Short and empty lists, entries of -inf, rows without a label, rows with
    neither, masked rows full of NaN, negative and uneven weights, another scale."""
    from tinytrain_b200 import kernels as KN
    N, K = 61, 24
    x, ids, top, t, g = make(N, C, K, cuda)
    n = torch.randint(0, K + 1, (N, 1), device=cuda, generator=g)
    n[3] = 0
    n[4] = 0
    gap = torch.rand(N, K, device=cuda, generator=g) < 0.2  # absent entries anywhere
    ids = torch.where((torch.arange(K, device=cuda) < n) & ~gap, ids, -1).contiguous()
    top = torch.where(ids >= 0, top, math.nan).contiguous()  # not to be read
    top[7] = torch.where(ids[7] >= 0, -math.inf, top[7])
    t[::5] = -1
    t[4] = -1  # row 4: neither list nor label
    x[4] = math.nan
    w = torch.rand(N, device=cuda, generator=g) * 2 - 0.5
    w[::7] = 0
    x[::7] = math.nan
    out = KN.distill_loss(x, ids, top, t, alpha=0.6, temperature=2.0, row_weight=w, grad_scale=0.25)
    off = (w == 0) | (torch.arange(N, device=cuda) == 4)
    clean = torch.where(off[:, None], 0.0, x)
    want = define(clean, ids, torch.where(ids >= 0, top, 0.0), t, 0.6, 2.0, w, 0.25)
    check(out, want, clean, 2.0)
    assert (out[1][off] == 0).all()
    assert status() == 0


def test_every_row_masked(cuda):
    from tinytrain_b200 import kernels as KN
    x, ids, top, t, _ = make(9, 100, 4, cuda)
    loss, d = KN.distill_loss(x * math.nan, ids, top, t, row_weight=torch.zeros(9, device=cuda))
    assert (loss == 0).all() and (d == 0).all()
    loss, d = KN.distill_loss(x * math.nan, torch.full_like(ids, -1), top, torch.full_like(t, -1))
    assert (loss == 0).all() and (d == 0).all()


@pytest.mark.parametrize("C", [300, 32000])
def test_masked_classes(cuda, C):
    """Student logits of -inf and of the type's lowest value: probability 0. A
    teacher entry on a class of -inf makes the loss infinite, the gradient finite."""
    from tinytrain_b200 import kernels as KN
    x, ids, top, t, g = make(8, C, 6, cuda)
    x[:, : C // 3] = -math.inf
    x[1, C // 3:C // 2] = torch.finfo(torch.float32).min
    allowed = torch.where(torch.isinf(x) | (x < -1e30), -1e4, x)
    top, ids = allowed.topk(6, 1)
    ids, t = ids.int().contiguous(), ids[:, 2].contiguous()
    want = define(x, ids, top, t, 0.5, 2.0)
    loss, d = KN.distill_loss(x, ids, top, t, alpha=0.5, temperature=2.0)
    assert torch.isfinite(loss).all() and torch.isfinite(d).all()
    assert (d[:, : C // 3] == 0).all()
    near = torch.where(x < -1e30, 0.0, x)
    check((loss, d), want, near, 2.0)
    ids[2, 0] = 1  # a masked class
    loss, d = KN.distill_loss(x, ids, top, t, alpha=0.5, temperature=2.0)
    assert torch.isinf(loss[:2]).all() and (loss[:2] > 0).all() and torch.isfinite(loss[2])
    _, rd, _, md = define(x, ids, top, t, 0.5, 2.0)
    assert ((d.double() - rd).abs() <= 300 * U * md + 1e-37).all()
    # a row without any class
    x[3] = -math.inf
    loss, d = KN.distill_loss(x, ids, top, t, alpha=0.5, temperature=2.0)
    assert torch.isnan(loss[0]) and torch.isnan(d[3]).all() and torch.isfinite(d[4]).all()
    assert status() == 0


def test_nan_reaches_the_loss(cuda):
    from tinytrain_b200 import kernels as KN
    x, ids, top, t, _ = make(3, 2000, 5, cuda)
    bad = x.clone()
    bad[1, 77] = math.nan
    loss, d = KN.distill_loss(bad, ids, top, t, alpha=0.5)
    assert torch.isnan(loss[0]) and torch.isnan(d[1]).all() and torch.isfinite(d[[0, 2]]).all()
    bad = top.clone()
    bad[1, 2] = math.nan
    loss, d = KN.distill_loss(x, ids, bad, t, alpha=0.5)
    assert torch.isnan(loss[0]) and torch.isnan(d[1, ids[1].long()]).all()
    assert torch.isfinite(d[[0, 2]]).all()


def test_repeated_classes_add_up(cuda):
    """A class listed several times has the sum of its entries' probabilities,
    and the label's class may be listed: one place of the gradient, in a fixed order."""
    from tinytrain_b200 import kernels as KN
    N, C, K = 20, 5000, 200
    x, ids, top, t, g = make(N, C, K, cuda)
    ids = torch.randint(0, 40, (N, K), device=cuda, generator=g).int()
    t = torch.randint(0, 40, (N,), device=cuda, generator=g)
    want = define(x, ids, top, t, 0.5, 2.0)
    out = KN.distill_loss(x, ids, top, t, alpha=0.5, temperature=2.0)
    check(out, want, x, 2.0)
    for _ in range(3):
        assert torch.equal(KN.distill_loss(x, ids, top, t, alpha=0.5, temperature=2.0)[1], out[1])


@pytest.mark.parametrize("C,pad,shift", [(1000, 24, 0), (999, 1, 0), (1001, 0, 1), (4096, 3, 2),
                                         (32000, 64, 0), (32000, 0, 3), (31999, 4, 1)])
def test_row_strides_and_alignment(cuda, C, pad, shift):
    """Rows of wider buffers, starting on any 4-byte boundary; columns past C stay."""
    from tinytrain_b200 import kernels as KN
    N, K = 12, 9
    x, ids, top, t, g = make(N, C, K, cuda)
    buf = torch.full((N * (C + pad) + shift,), 77.0, device=cuda)
    view = buf[shift:].view(N, C + pad)[:, :C]
    view.copy_(x)
    want = KN.distill_loss(x, ids, top, t, alpha=0.5, temperature=2.0)
    ref = define(x, ids, top, t, 0.5, 2.0)
    out = KN.distill_loss(view, ids, top, t, alpha=0.5, temperature=2.0)
    check(out, ref, x, 2.0)
    wide = torch.full((N, C + 5), -3.0, device=cuda)
    loss, d = KN.distill_loss(view, ids, top, t, alpha=0.5, temperature=2.0, dlogits=wide[:, :C])
    check((loss, d), ref, x, 2.0)
    assert (wide[:, C:] == -3.0).all()
    loss, d = KN.distill_loss(view, ids, top, t, alpha=0.5, temperature=2.0, dlogits=view)
    check((loss, d), ref, x, 2.0)
    if pad:
        assert (buf[shift:].view(N, C + pad)[:, C:] == 77.0).all()
    assert torch.equal(want[0], KN.distill_loss(x, ids, top, t, alpha=0.5, temperature=2.0)[0])
    assert status() == 0


def test_ids_out_of_range_are_reported(cuda):
    from tinytrain_b200 import kernels as KN
    x, ids, top, t, _ = make(6, 300, 5, cuda)
    bad, tb = ids.clone(), t.clone()
    bad[1, 2] = 300
    bad[2, 0] = -7
    out = KN.distill_loss(x, bad, top, t, alpha=0.5)
    assert status() == 2
    keep = torch.where((bad >= 0) & (bad < 300), bad, -1)
    check(out, define(x, keep, top, t, 0.5, 1.0), x, 1.0)
    tb[3] = 300
    out = KN.distill_loss(x, ids, top, tb, alpha=0.5)
    assert status() == 2
    tb[3] = -1
    check(out, define(x, ids, top, tb, 0.5, 1.0), x, 1.0)


def test_gradient_against_differences(cuda):
    """Central differences of the kernel's loss along a random direction v. The
    loss is a mean of rows of size about 1; with step s the truncation is below
    s^2 |L'''| / 6 <= s^2 and the rounding below 100 u |L| / s: for s = 2^-7
    under 1e-4 and 1e-3."""
    from tinytrain_b200 import kernels as KN
    x, ids, top, t, g = make(16, 700, 12, cuda, spread=1.0)
    v = torch.randn(x.shape, device=cuda, generator=g)
    for alpha, T in ((1.0, 1.0), (0.5, 2.0), (0.0, 1.0)):
        s = 2.0 ** -7
        L = [float(KN.distill_loss(x + k * s * v, ids, top, t, alpha=alpha, temperature=T,
                                   want_grad=False)[0][0].double()) for k in (-1, 1)]
        _, d = KN.distill_loss(x, ids, top, t, alpha=alpha, temperature=T)
        ana = float((d.double() * v.double()).sum())
        assert abs((L[1] - L[0]) / (2 * s) - ana) <= 2e-3, (alpha, T, L, ana)


def test_no_rows(cuda):
    from tinytrain_b200 import kernels as KN
    x = torch.empty(0, 50, device=cuda)
    ids = torch.empty(0, 4, dtype=torch.int32, device=cuda)
    loss, d = KN.distill_loss(x, ids, torch.empty(0, 4, device=cuda))
    assert (loss == 0).all() and d.shape == (0, 50)
    # and no teacher entries: the loss of the labels alone
    x, _, _, t, _ = make(5, 50, 4, cuda)
    ids = torch.empty(5, 0, dtype=torch.int32, device=cuda)
    top = torch.empty(5, 0, device=cuda)
    out = KN.distill_loss(x, ids, top, t, alpha=0.0)
    l1 = torch.log_softmax(x.double(), 1)
    ce = -l1.gather(1, t[:, None]).mean()
    assert abs(float(out[0][0]) - float(ce)) <= 60 * U * (float(ce) + 1)
    assert status() == 0


@pytest.mark.parametrize("C", [40, 5000, 32000, 40000])
def test_rows_at_the_lowest_value(cuda, C):
    """Rows whose logits are all the type's lowest value are uniform, as softmax
    has them; a part of a row at that value next to ordinary logits has
    probability 0."""
    from tinytrain_b200 import kernels as KN
    low = torch.finfo(torch.float32).min
    x = torch.full((3, C), low, device=cuda)
    x[1, C - 3:] = torch.tensor([1.0, 2.0, 3.0], device=cuda)
    x[2, :] = -math.inf
    x[2, C // 2] = low
    ids = torch.full((3, 1), C - 1, dtype=torch.int32, device=cuda)
    ids[2] = C // 2
    t = ids[:, 0].long()
    for T in (1.0, 2.0):
        loss, d = KN.distill_loss(x, ids, torch.zeros(3, 1, device=cuda), t, alpha=0.5,
                                  temperature=T, grad_scale=1.0)
        q = torch.zeros(2, 3, C, dtype=torch.float64, device=cuda)  # at T, at 1
        for i, k in enumerate((1 / T, 1.0)):
            q[i, 0] = 1.0 / C
            q[i, 1, C - 3:] = torch.softmax(k * torch.tensor([1.0, 2.0, 3.0], dtype=torch.float64), 0)
            q[i, 2, C // 2] = 1.0
        hit = torch.zeros(3, C, dtype=torch.float64, device=cuda).scatter_(1, t[:, None], 1.0)
        want = 0.5 * T * (q[0] - hit) + 0.5 * (q[1] - hit)
        mag = 0.5 * T * (q[0] + hit) + 0.5 * (q[1] + hit)
        c = 60 + C / 256
        assert ((d.double() - want).abs() <= c * U * mag).all()
        kd, ce = (-(torch.log(v[torch.arange(3, device=cuda), t])).sum() for v in q)
        ref = torch.stack([0.5 * T * T * kd + 0.5 * ce, kd, ce])
        assert ((loss.double() - ref).abs() <= c * U * (ref + 3)).all()
    assert status() == 0


@pytest.mark.parametrize("C", [1000, 3200, 3500, 6000, 10000, 15001, 20000, 40000, 60001])
@pytest.mark.parametrize("K", [33, 200, 256, 500, 1000])
def test_long_lists(cuda, C, K):
    """Long lists leave less room for the row: rows that do not fit beside them."""
    from tinytrain_b200 import kernels as KN
    x, ids, top, t, _ = make(9, C, K, cuda)
    want = define(x, ids, top, t, 0.5, 2.0)
    check(KN.distill_loss(x, ids, top, t, alpha=0.5, temperature=2.0), want, x, 2.0)
    check(KN.distill_loss(x, ids, top, t, alpha=0.5, temperature=2.0, want_grad=False), want, x, 2.0)


@pytest.mark.parametrize("N,C,K", [(700, 5000, 40), (1300, 700, 12), (2500, 3584, 7), (1200, 3585, 300),
                                   (900, 12000, 64), (700, 33001, 16), (3000, 17, 5), (1184, 4, 2)])
def test_many_rows(cuda, N, C, K):
    """More rows than run at once, with labels, lists and masks of all kinds between them."""
    from tinytrain_b200 import kernels as KN
    x, ids, top, t, g = make(N, C, K, cuda)
    n = torch.randint(0, K + 1, (N, 1), device=cuda, generator=g)
    ids = torch.where(torch.arange(K, device=cuda) < n, ids, -1).contiguous()
    t[torch.rand(N, device=cuda, generator=g) < 0.2] = -1
    w = (torch.rand(N, device=cuda, generator=g) > 0.3).float() * 1.5
    want = define(x, ids, top, t, 0.7, 2.0, w)
    out = KN.distill_loss(x, ids, top, t, alpha=0.7, temperature=2.0, row_weight=w)
    check(out, want, x, 2.0)
    again = KN.distill_loss(x, ids, top, t, alpha=0.7, temperature=2.0, row_weight=w, dlogits=x)
    assert torch.equal(again[0], out[0]) and torch.equal(again[1], out[1])
    assert status() == 0


@pytest.mark.parametrize("stride", [1, 64, 128])
@pytest.mark.parametrize("K", [33, 64, 300])
@pytest.mark.parametrize("twice", [False, True])
def test_lists_of_regular_classes(cuda, K, stride, twice):
    """Classes at a constant stride, whose hashes fall together, all different or
    with one of them listed a second time at the end."""
    from tinytrain_b200 import kernels as KN
    N, C = 5, 128 * 300
    x, ids, top, t, _ = make(N, C, K, cuda)
    ids = (torch.arange(K, device=cuda) * stride).int().repeat(N, 1)
    if twice:
        ids[:, K - 1] = ids[:, 1]
    out = KN.distill_loss(x, ids, top, t, alpha=0.5, temperature=2.0)
    check(out, define(x, ids, top, t, 0.5, 2.0), x, 2.0)
