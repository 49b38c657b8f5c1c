"""Residual norm (norm after a block, gate, residual scale, residual add, norm
before the next block), forward and backward, against the formulas in 64 bits.

Tolerance: every output is a short chain of fp32 operations on sums over a row
(or, for the weights' gradients, over the rows as well). With u = 2^-24, a sum
taken in chains of n additions is within n u of the sum of the terms'
magnitudes. So each formula is also evaluated in 64 bits with every term made
positive, and each element has to be within c u of that: c = D / 32 + 40 for the
chains of a row (32 lanes at least share a row) and the operations around them,
plus the number of rows for sums over rows.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
GATES = ["none", "scalar", "column", "row", "full"]
SIZES = [(1, 1), (1, 256), (3, 20), (5, 33), (2, 128), (37, 64), (64, 257), (129, 768), (300, 1111),
         (1000, 256), (50, 2048), (9, 2050), (17, 4096), (33, 4100), (5, 8192), (3, 12000),
         (2500, 96)]


def status():
    from tinytrain_b200 import _ttk
    return _ttk.device_status()


def make(R, D, kind, dev, seed=0):
    g = torch.Generator(device=dev).manual_seed(1000 * R + D + seed)
    rn = lambda *s: torch.randn(s, device=dev, generator=g)  # noqa: E731
    shape = dict(none=None, scalar=(1,), column=(D,), row=(R, 1), full=(R, D))[kind]
    gate = None if shape is None else torch.rand(shape, device=dev, generator=g) * 2 - 0.5
    return dict(x=2 * rn(R, D), b=rn(R, D) * 0.3, w1=1 + 0.3 * rn(D), w2=1 + 0.3 * rn(D), gate=gate,
                dh=rn(R, D), dy=rn(R, D))


def forward64(s, alpha, eps):
    """h, y and their magnitudes (every term positive)."""
    x, b, w1, w2 = (s[k].double() for k in ("x", "b", "w1", "w2"))
    g = 1.0 if s["gate"] is None else s["gate"].double()
    r1 = (b.square().mean(1, keepdim=True) + eps) ** -0.5
    u = g * (b * r1 * w1)
    h, hm = alpha * x + u, (alpha * x).abs() + u.abs()
    r2 = (h.square().mean(1, keepdim=True) + eps) ** -0.5
    r2m = r2 * (1 + (hm * h.abs()).mean(1, keepdim=True) * r2 ** 2)  # |d r2| for |dh| = hm
    return h, hm, h * r2 * w2, hm * r2 * w2.abs() + h.abs() * r2m * w2.abs(), r1, r2


def backward64(s, h, r1, r2, alpha, dh, dy, positive=False):
    """(dx, db, dw_post, dw_next, dgate per element); `positive`: the magnitudes."""
    pos = (lambda t: t.abs()) if positive else (lambda t: t)
    sgn = 1.0 if positive else -1.0
    b, w1, w2, h = (pos(t.double()) for t in (s["b"], s["w1"], s["w2"], h))
    g = 1.0 if s["gate"] is None else pos(s["gate"].double())
    r1, r2 = r1.double()[:, None], r2.double()[:, None]
    D = b.shape[1]
    dh = torch.zeros_like(b) if dh is None else pos(dh.double())
    dy = torch.zeros_like(b) if dy is None else pos(dy.double())
    e = dy * w2
    H = dh + r2 * e + sgn * h * r2 ** 3 / D * (e * h).sum(1, keepdim=True)
    f = H * g * w1
    db = r1 * f + sgn * b * r1 ** 3 / D * (f * b).sum(1, keepdim=True)
    return alpha * H, db, (H * g * b * r1).sum(0), (dy * h * r2).sum(0), H * b * r1 * w1


def to_gate(full, gate):
    if gate.dim() == 1:
        return full.sum().reshape(1) if gate.numel() == 1 else full.sum(0)
    return full.sum_to_size(gate.shape)


def within(got, ref, mag, c, what):
    err = (got.double() - ref).abs()
    bad = ~(err <= c * U * mag + 1e-37)
    assert not bad.any(), (what, float((err / (U * mag + 1e-37)).max()), c)


@pytest.mark.parametrize("R,D", SIZES)
@pytest.mark.parametrize("kind", GATES)
def test_forward(cuda, R, D, kind):
    from tinytrain_b200 import kernels as K
    s = make(R, D, kind, cuda)
    alpha, eps = 0.75, 1e-5
    h, y, r1, r2 = K.residual_norm_fwd(s["x"], s["b"], s["w1"], s["w2"], gate=s["gate"],
                                       residual_scale=alpha, eps=eps)
    h64, hm, y64, ym, r1_64, r2_64 = forward64(s, alpha, eps)
    c = D / 32 + 40
    within(h, h64, hm, c, "h")
    within(y, y64, ym, c, "y")
    within(r1, r1_64[:, 0], r1_64[:, 0], c, "rstd_post")
    # r2 moves with h: |d r2| <= r2^3 mean(|h| |dh|)
    within(r2, r2_64[:, 0], r2_64[:, 0] * (1 + (hm * h64.abs()).mean(1) * r2_64[:, 0] ** 2), c,
           "rstd_next")
    # without the second norm
    h2, none, r1b, none2 = K.residual_norm_fwd(s["x"], s["b"], s["w1"], gate=s["gate"],
                                               residual_scale=alpha, eps=eps)
    assert none is None and none2 is None
    assert torch.equal(h2, h) and torch.equal(r1b, r1)
    assert status() == 0


@pytest.mark.parametrize("R,D", SIZES)
@pytest.mark.parametrize("kind", GATES)
@pytest.mark.parametrize("into", ["both", "dh", "dy"])
def test_backward(cuda, R, D, kind, into):
    from tinytrain_b200 import kernels as K
    s = make(R, D, kind, cuda)
    alpha, eps = 0.75, 1e-5
    h, _, r1, r2 = K.residual_norm_fwd(s["x"], s["b"], s["w1"], s["w2"], gate=s["gate"],
                                       residual_scale=alpha, eps=eps)
    dh = s["dh"] if into != "dy" else None
    dy = s["dy"] if into != "dh" else None
    args = (dh, dy, h, s["b"], s["w1"], s["w2"], r1, r2)
    got = K.residual_norm_bwd(*args, gate=s["gate"], residual_scale=alpha)
    ref = list(backward64(s, h, r1, r2, alpha, dh, dy))
    mag = list(backward64(s, h, r1, r2, alpha, dh, dy, positive=True))
    if kind == "none":
        assert got[4] is None
    else:
        ref[4], mag[4] = to_gate(ref[4], s["gate"]), to_gate(mag[4], s["gate"])
    c = D / 32 + 40
    names = ["dx", "db", "dw_post", "dw_next", "dgate"]
    over_rows = [False, False, True, True, kind in ("scalar", "column")]
    for i in range(4 if kind == "none" else 5):
        if i == 3 and dy is None:
            assert got[3] is None
            continue
        within(got[i].reshape(ref[i].shape), ref[i], mag[i],
               c + (R if over_rows[i] else 0) + (D if i == 4 and kind == "scalar" else 0), names[i])
    # equal calls, equal bits
    again = K.residual_norm_bwd(*args, gate=s["gate"], residual_scale=alpha)
    for p, q in zip(got, again):
        assert (p is None and q is None) or torch.equal(p, q)
    # the same added to what is there
    have = [torch.randn_like(t) if t is not None else None for t in got]
    acc = K.residual_norm_bwd(*args, gate=s["gate"], residual_scale=alpha,
                              **{n: None if t is None else t.clone() for n, t in zip(names, have)})
    for p, q, t, n in zip(acc, got, have, names):
        if p is not None:
            within(p, q.double() + t.double(), q.double().abs() + t.double().abs(), 2, n + " added")
    assert status() == 0


@pytest.mark.parametrize("R,D", [(64, 256), (1000, 2048), (37, 96), (5, 8192), (3, 32)])
def test_planes_bit_for_bit(cuda, R, D):
    from tinytrain_b200 import kernels as K
    s = make(R, D, "column", cuda)
    _, y, _, _, planes = K.residual_norm_fwd(s["x"], s["b"], s["w1"], s["w2"], gate=s["gate"],
                                             planes=True)
    h2, y2, _, _ = K.residual_norm_fwd(s["x"], s["b"], s["w1"], s["w2"], gate=s["gate"])
    assert torch.equal(y, y2)
    assert torch.equal(planes, K.gemm_split(y))
    assert status() == 0


@pytest.mark.parametrize("kind", GATES)
def test_gradient_against_differences(cuda, kind):
    """The directional derivative of L = <h, A> + <y, B> along a random direction
    of every input, by central differences of the kernel's own forward (L summed
    in 64 bits). With step s the truncation is about s^2 of L's size and the
    rounding 40 u / s of the terms' magnitudes: s = 2^-6 makes them 2.4e-4 and
    1.5e-4 of L's magnitude, in the norm below."""
    from tinytrain_b200 import kernels as K
    R, D, alpha, eps = 6, 160, 0.5, 1e-5
    s = make(R, D, kind, cuda)
    g = torch.Generator(device=cuda).manual_seed(9)
    A, B = (torch.randn(R, D, device=cuda, generator=g) for _ in range(2))
    dirs = {k: torch.randn(s[k].shape, device=cuda, generator=g) * s[k].abs().mean()
            for k in ("x", "b", "w1", "w2", "gate") if s[k] is not None}

    def L(step):
        t = {k: s[k] if s[k] is None or k not in dirs else s[k] + step * dirs[k]
             for k in ("x", "b", "w1", "w2", "gate")}
        h, y, _, _ = K.residual_norm_fwd(t["x"], t["b"], t["w1"], t["w2"], gate=t["gate"],
                                         residual_scale=alpha, eps=eps)
        return (h.double() * A.double()).sum() + (y.double() * B.double()).sum()

    step = 2.0 ** -6
    num = (L(step) - L(-step)) / (2 * step)
    h, y, r1, r2 = K.residual_norm_fwd(s["x"], s["b"], s["w1"], s["w2"], gate=s["gate"],
                                       residual_scale=alpha, eps=eps)
    dx, db, dw1, dw2, dg = K.residual_norm_bwd(A, B, h, s["b"], s["w1"], s["w2"], r1, r2,
                                               gate=s["gate"], residual_scale=alpha)
    ana = sum((d.double() * dirs[k].double()).sum() for d, k in
              ((dx, "x"), (db, "b"), (dw1, "w1"), (dw2, "w2"), (dg, "gate")) if k in dirs)
    size = ((h.double() * A.double()).square().sum() + (y.double() * B.double()).square().sum()).sqrt()
    assert (num - ana).abs() <= 2e-3 * size, (float(num), float(ana), float(size))


def test_zero_block_output(cuda):
    """b = 0 leaves h = alpha x; the gradient of b is then r1 f, r1 = eps^-1/2."""
    from tinytrain_b200 import kernels as K
    R, D, eps = 4, 128, 1e-5
    s = make(R, D, "none", cuda)
    b = torch.zeros_like(s["b"])
    h, y, r1, r2 = K.residual_norm_fwd(s["x"], b, s["w1"], s["w2"], residual_scale=0.5, eps=eps)
    assert torch.equal(h, 0.5 * s["x"])
    assert ((r1.double() - eps ** -0.5).abs() <= 4 * U * eps ** -0.5).all()
    dx, db, dw1, _, _ = K.residual_norm_bwd(s["dh"], None, None, b, s["w1"], None, r1, None,
                                            residual_scale=0.5)
    assert torch.equal(dx, 0.5 * s["dh"])
    assert (dw1 == 0).all()
    ref = r1.double()[:, None] * s["dh"].double() * s["w1"].double()
    within(db, ref, ref.abs(), 4, "db")


def test_no_rows(cuda):
    from tinytrain_b200 import kernels as K
    D = 96
    e = torch.empty(0, D, device=cuda)
    w = torch.ones(D, device=cuda)
    h, y, r1, r2 = K.residual_norm_fwd(e, e, w, w)
    assert h.shape == y.shape == (0, D)
    dx, db, dw1, dw2, dg = K.residual_norm_bwd(e, e, h, e, w, w, r1, r2, gate=w.clone())
    assert (dw1 == 0).all() and (dw2 == 0).all() and (dg == 0).all()
    have = torch.randn(D, device=cuda)
    _, _, dw1, _, _ = K.residual_norm_bwd(e, e, h, e, w, w, r1, r2, dw_post=have.clone())
    assert torch.equal(dw1, have)
    assert status() == 0


@pytest.mark.parametrize("D", [128, 131, 2048])
@pytest.mark.parametrize("kind", ["none", "column", "full"])
def test_unaligned_tensors(cuda, D, kind):
    """Tensors that start off a 16-byte boundary take another path, within the same bounds."""
    from tinytrain_b200 import kernels as K
    R, alpha, eps = 37, 0.5, 1e-5
    s = make(R, D, kind, cuda)

    def off(t):
        return None if t is None else torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape)

    u = {k: off(v) for k, v in s.items()}
    h, y, r1, r2 = K.residual_norm_fwd(u["x"], u["b"], u["w1"], u["w2"], gate=u["gate"],
                                       residual_scale=alpha, eps=eps)
    h64, hm, y64, ym, _, _ = forward64(s, alpha, eps)
    c = D / 32 + 40
    within(h, h64, hm, c, "h")
    within(y, y64, ym, c, "y")
    got = K.residual_norm_bwd(u["dh"], u["dy"], off(h), u["b"], u["w1"], u["w2"], r1, r2,
                              gate=u["gate"], residual_scale=alpha)
    ref = list(backward64(s, h, r1, r2, alpha, s["dh"], s["dy"]))
    mag = list(backward64(s, h, r1, r2, alpha, s["dh"], s["dy"], positive=True))
    for i, name in enumerate(("dx", "db", "dw_post", "dw_next")):
        within(got[i], ref[i], mag[i], c + (R if i > 1 else 0), name)
    if kind != "none":
        within(got[4], to_gate(ref[4], s["gate"]), to_gate(mag[4], s["gate"]), c + R, "dgate")
    assert status() == 0


@pytest.mark.parametrize("R,D", [(5000, 66), (3001, 1111), (2003, 999), (1500, 2049), (700, 4095),
                                 (600, 8191), (40000, 32)])
def test_many_rows_of_odd_widths(cuda, R, D):
    """More rows than the machine holds at once: every slot runs over several rows."""
    from tinytrain_b200 import kernels as K
    alpha, eps = 0.75, 1e-5
    for kind in ("column", "full"):
        s = make(R, D, kind, cuda)
        h, y, r1, r2 = K.residual_norm_fwd(s["x"], s["b"], s["w1"], s["w2"], gate=s["gate"],
                                           residual_scale=alpha, eps=eps)
        h64, hm, y64, ym, _, _ = forward64(s, alpha, eps)
        c = D / 32 + 40
        within(h, h64, hm, c, "h")
        within(y, y64, ym, c, "y")
        got = K.residual_norm_bwd(s["dh"], s["dy"], h, s["b"], s["w1"], s["w2"], r1, r2,
                                  gate=s["gate"], residual_scale=alpha)
        ref = list(backward64(s, h, r1, r2, alpha, s["dh"], s["dy"]))
        mag = list(backward64(s, h, r1, r2, alpha, s["dh"], s["dy"], positive=True))
        for i, name in enumerate(("dx", "db", "dw_post", "dw_next")):
            within(got[i], ref[i], mag[i], c + (R if i > 1 else 0), name)
        within(got[4], to_gate(ref[4], s["gate"]), to_gate(mag[4], s["gate"]),
               c + (R if kind == "column" else 0), "dgate")
    assert status() == 0
