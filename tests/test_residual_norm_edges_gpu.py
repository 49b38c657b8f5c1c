"""Residual norm at its edges: rows narrower than a 16-byte word, whose last words
lie across the tensors' ends. Bounds as in test_residual_norm_gpu.py."""
import pytest
import torch

import test_residual_norm_gpu as base

pytestmark = pytest.mark.gpu


def compare(R, D, kind, s, alpha, eps):
    from tinytrain_b200 import kernels as K
    h, y, r1, r2 = K.residual_norm_fwd(s["x"], s["b"], s["w1"], s["w2"], gate=s["gate"],
                                       residual_scale=alpha, eps=eps)
    h64, hm, y64, ym, _, _ = base.forward64(s, alpha, eps)
    c = D / 32 + 40
    base.within(h, h64, hm, c, "h")
    base.within(y, y64, ym, c, "y")
    got = K.residual_norm_bwd(s["dh"], s["dy"], h, s["b"], s["w1"], s["w2"], r1, r2,
                              gate=s["gate"], residual_scale=alpha)
    ref = list(base.backward64(s, h, r1, r2, alpha, s["dh"], s["dy"]))
    mag = list(base.backward64(s, h, r1, r2, alpha, s["dh"], s["dy"], positive=True))
    if s["gate"] is not None:
        ref[4], mag[4] = base.to_gate(ref[4], s["gate"]), base.to_gate(mag[4], s["gate"])
    for i, name in enumerate(("dx", "db", "dw_post", "dw_next", "dgate")):
        if got[i] is not None:
            rows = R + D if i == 4 and kind == "scalar" else R if i in (2, 3, 4) else 0
            base.within(got[i].reshape(ref[i].shape), ref[i], mag[i], c + rows, name)
    assert base.status() == 0


@pytest.mark.parametrize("R", [1, 2, 3, 4, 5, 6, 7, 1001, 5003])
@pytest.mark.parametrize("D", [1, 2, 3, 5])
@pytest.mark.parametrize("kind", base.GATES)
def test_narrow_rows(cuda, R, D, kind):
    compare(R, D, kind, base.make(R, D, kind, cuda), 0.75, 1e-5)


@pytest.mark.parametrize("kind", base.GATES)
def test_no_rows(cuda, kind):
    """Without rows nothing is read: the sums are zero, or what they are added to stays."""
    from tinytrain_b200 import kernels as K
    D = 40
    s = base.make(0, D, kind, cuda)
    e, r = s["x"], torch.empty(0, device=cuda)
    args = (e, e, e, e, s["w1"], s["w2"], r, r)
    _, _, dw1, dw2, dg = K.residual_norm_bwd(*args, gate=s["gate"])
    assert (dw1 == 0).all() and (dw2 == 0).all() and (dg is None or (dg == 0).all())
    have = torch.randn(D, device=cuda)
    keep = None if s["gate"] is None else torch.randn_like(s["gate"])
    got = K.residual_norm_bwd(*args, gate=s["gate"], dw_post=have.clone(), dw_next=have.clone(),
                              dgate=None if keep is None else keep.clone())
    assert torch.equal(got[2], have) and torch.equal(got[3], have)
    assert keep is None or torch.equal(got[4], keep)
    assert base.status() == 0


@pytest.mark.parametrize("size,eps", [(1e14, 1e-5), (1e-14, 0.0), (1e-14, 1e-30)])
@pytest.mark.parametrize("R,D", [(7, 128), (5, 1111), (3, 8192), (4, 12000)])
@pytest.mark.parametrize("kind", ["none", "column", "full"])
def test_sizes_far_from_one(cuda, R, D, kind, size, eps):
    """Rows of 1e14 or 1e-14: the third power of a row's 1 / rms is no fp32 number, but
    every output is one."""
    s = base.make(R, D, kind, cuda)
    s["x"], s["b"] = s["x"] * size, s["b"] * size
    if size < 1:  # the residual and the gated norm of b of one size
        s["w1"] = s["w1"] * size
    compare(R, D, kind, s, 0.75, eps)


def test_sums_over_many_rows(cuda):
    """The weights' and the gate's gradients over 32768 rows are not one chain of
    additions. An addition in fp32 is off by about 0.4 u of its result, u = 2^-24, so a
    chain of n random terms by 0.4 u sqrt(n / 2) of its sum: 16 rows, 7 such sums, 9
    blocks and 32 of those give 2.3 u together, with the terms' own rounding 2.6 u; one
    chain of 110 rows in place of the first two would give 3.6 u and more."""
    from tinytrain_b200 import kernels as K
    R, D, alpha, eps = 32768, 2048, 0.75, 1e-5
    s = base.make(R, D, "column", cuda)
    h, _, r1, r2 = K.residual_norm_fwd(s["x"], s["b"], s["w1"], s["w2"], gate=s["gate"],
                                       residual_scale=alpha, eps=eps)
    got = K.residual_norm_bwd(s["dh"], s["dy"], h, s["b"], s["w1"], s["w2"], r1, r2,
                              gate=s["gate"], residual_scale=alpha)
    ref = list(base.backward64(s, h, r1, r2, alpha, s["dh"], s["dy"]))
    ref[4] = base.to_gate(ref[4], s["gate"])
    for i in (2, 3, 4):
        err = (got[i].double() - ref[i]).norm() / ref[i].norm()
        assert err <= 3 * base.U, (i, float(err / base.U))


def test_gradients_of_nothing(cuda):
    """A gate's gradient without a gate is refused; w_next's without dy stays as it is."""
    from tinytrain_b200 import kernels as K
    R, D = 5, 64
    s = base.make(R, D, "none", cuda)
    r1 = torch.ones(R, device=cuda)
    have = torch.randn(D, device=cuda)
    with pytest.raises(ValueError, match="dgate: there is no gate"):
        K.residual_norm_bwd(s["dh"], None, None, s["b"], s["w1"], None, r1, None, dgate=have)
    got = K.residual_norm_bwd(s["dh"], None, None, s["b"], s["w1"], None, r1, None,
                              dw_next=have.clone())
    assert torch.equal(got[3], have)


@pytest.mark.parametrize("R,D", [(100000, 32), (90000, 66), (80000, 304), (30000, 1111), (20000, 2048),
                                 (6000, 8190), (5500, 8192)])
@pytest.mark.parametrize("kind", ["column", "row", "full"])
def test_slots_of_many_rows(cuda, R, D, kind):
    """Slots of more than 32 rows, whose sums go through shared memory, in every form of the
    kernel: several slots a block or one, whole words or not, two or four words a thread."""
    compare(R, D, kind, base.make(R, D, kind, cuda), 0.75, 1e-5)
