"""Scaled embedding lookup and its gradient by sorted tokens.

The lookup is one multiplication per element and is compared bit for bit. A
gradient element is a sum of n products: any order of n additions in fp32
differs from the exact sum by at most about (n + 1) u sum|terms|, u = 2^-24,
plus the multiplication by the scale; that bound is checked element by element
against sums in 64 bits.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def status():
    from tinytrain_b200 import _ttk
    return _ttk.device_status()


def tokens(kind, N, V, g, dev):
    if kind == "uniform":
        return torch.randint(0, V, (N,), device=dev, generator=g)
    if kind == "one":  # every position the same token
        return torch.full((N,), min(3, V - 1), device=dev, dtype=torch.int64)
    if kind == "text":  # frequencies of text, ends padded
        ids = torch.multinomial(1.0 / (torch.arange(V, device=dev, dtype=torch.float32) + 2.7), N,
                                replacement=True, generator=g)
        ids[torch.arange(N, device=dev) % 16 >= 13] = -1
        return ids
    if kind == "ends":  # the first and the last row of the table
        return torch.where(torch.rand(N, device=dev, generator=g) < 0.5, 0, V - 1)
    assert kind == "padding"
    return torch.full((N,), -1, device=dev, dtype=torch.int64)


SIZES = [(1, 1, 1), (1, 256, 32000), (7, 20, 5), (33, 64, 1), (100, 768, 255), (255, 257, 256),
         (1000, 1111, 257), (2048, 256, 32000), (4097, 132, 65535), (5000, 96, 65536),
         (300, 2048, 100003), (3000, 4100, 700), (20001, 64, 1000)]


@pytest.mark.parametrize("N,D,V", SIZES)
@pytest.mark.parametrize("kind", ["uniform", "one", "text", "ends", "padding"])
def test_lookup_and_gradient(cuda, N, D, V, kind):
    from tinytrain_b200 import kernels as K
    g = torch.Generator(device=cuda).manual_seed(N + 7 * D + V)
    ids = tokens(kind, N, V, g, cuda)
    W = torch.randn(V, D, device=cuda, generator=g)
    scale = math.sqrt(D)
    live = (ids >= 0)[:, None]
    out = K.embedding_scaled_fwd(W, ids, scale)
    s32 = torch.tensor(scale, dtype=torch.float32, device=cuda)
    assert torch.equal(out, torch.where(live, W[ids.clamp(min=0)] * s32, 0.0))

    dout = torch.randn(N, D, device=cuda, generator=g)
    rows = torch.where(live, dout.double() * s32.double(), 0.0)
    at = ids.clamp(min=0)
    ref = torch.zeros(V, D, device=cuda, dtype=torch.float64).index_add_(0, at, rows)
    mag = torch.zeros(V, D, device=cuda, dtype=torch.float64).index_add_(0, at, rows.abs())
    n = torch.bincount(at[ids >= 0], minlength=V).double()[:, None]
    dW = K.embedding_scaled_bwd(dout, ids, V, scale)
    assert ((dW.double() - ref).abs() <= (n + 2) * U * mag).all()
    assert (dW[(n == 0).squeeze(1)] == 0).all()
    # the same call gives the same bits
    assert torch.equal(dW, K.embedding_scaled_bwd(dout, ids, V, scale))

    base = torch.randn(V, D, device=cuda, generator=g)
    acc = K.embedding_scaled_bwd(dout, ids, V, scale, dW=base.clone(), accumulate=True)
    tol = (n + 2) * U * mag + U * (ref + base.double()).abs()
    assert ((acc.double() - (ref + base.double())).abs() <= tol).all()
    assert torch.equal(acc[(n == 0).squeeze(1)], base[(n == 0).squeeze(1)])
    assert status() == 0


def test_unaligned_tensors(cuda):
    """Rows that start off a 16-byte boundary take another path, with the same results."""
    from tinytrain_b200 import _ttk
    from tinytrain_b200 import kernels as K
    N, D, V = 513, 128, 700
    g = torch.Generator(device=cuda).manual_seed(5)
    ids = torch.randint(0, V, (N,), device=cuda, generator=g)

    def off(rows):
        return torch.randn(rows * D + 1, device=cuda, generator=g)[1:].view(rows, D)

    W, dout = off(V), off(N)
    out, dW = off(N), off(V)
    s = torch.cuda.current_stream().cuda_stream
    _ttk.call("ttk_embedding_scaled_fwd", W.data_ptr(), ids.data_ptr(), out.data_ptr(), N, D, V,
              0.5, s)
    assert torch.equal(out, K.embedding_scaled_fwd(W.clone(), ids, 0.5))
    ws = K.workspace(_ttk.call("ttk_embedding_scaled_bwd_workspace_size", N, D, V))
    _ttk.call("ttk_embedding_scaled_bwd", dout.data_ptr(), ids.data_ptr(), dW.data_ptr(), 0, N, D,
              V, 0.5, ws.data_ptr(), ws.numel(), s)
    ref = torch.zeros(V, D, device=cuda, dtype=torch.float64).index_add_(0, ids, 0.5 * dout.double())
    mag = torch.zeros(V, D, device=cuda, dtype=torch.float64).index_add_(
        0, ids, 0.5 * dout.double().abs())
    n = torch.bincount(ids, minlength=V).double()[:, None]
    assert ((dW.double() - ref).abs() <= (n + 2) * U * mag).all()
    assert status() == 0


def test_no_tokens(cuda):
    from tinytrain_b200 import kernels as K
    V, D = 37, 12
    ids = torch.empty(0, dtype=torch.int64, device=cuda)
    none = torch.empty(0, D, device=cuda)
    W = torch.randn(V, D, device=cuda)
    assert K.embedding_scaled_fwd(W, ids, 2.0).shape == (0, D)
    dW = torch.full((V, D), 5.0, device=cuda)
    assert torch.equal(K.embedding_scaled_bwd(none, ids, V, 2.0, dW=dW.clone(), accumulate=True), dW)
    assert (K.embedding_scaled_bwd(none, ids, V, 2.0, dW=dW) == 0).all()
    assert status() == 0


def test_ids_out_of_range_are_reported(cuda):
    from tinytrain_b200 import kernels as K
    V, D = 50, 64
    W = torch.randn(V, D, device=cuda)
    ids = torch.tensor([3, V, 4, -2, 3, -1, 1 << 40], device=cuda)
    good = torch.tensor([True, False, True, False, True, False, False], device=cuda)
    out = K.embedding_scaled_fwd(W, ids, 1.0)
    assert status() == 2
    assert torch.equal(out, torch.where(good[:, None], W[ids.clamp(0, V - 1)], 0.0))
    dout = torch.randn(7, D, device=cuda)
    dW = K.embedding_scaled_bwd(dout, ids, V)
    assert status() == 2
    ref = torch.zeros(V, D, device=cuda)
    ref[3] = dout[0] + dout[4]
    ref[4] = dout[2]
    assert torch.equal(dW, ref)
    # padding alone is no error
    K.embedding_scaled_bwd(dout, torch.full_like(ids, -1), V)
    assert status() == 0


def test_gradient_against_differences(cuda):
    """<dW, E> against the change of <out, G> along E: the lookup is linear, so
    the difference quotient is exact up to rounding: 2^-24 of each product and
    of each sum of its parts, in 64 bits after that."""
    from tinytrain_b200 import kernels as K
    g = torch.Generator(device=cuda).manual_seed(1)
    N, D, V = 200, 48, 60
    ids = tokens("text", N, V, g, cuda)
    W, E = torch.randn(V, D, device=cuda, generator=g), torch.randn(V, D, device=cuda, generator=g)
    G = torch.randn(N, D, device=cuda, generator=g)
    lo, hi = (K.embedding_scaled_fwd((W + s * E), ids, 3.0).double() for s in (-1.0, 1.0))
    num = ((hi - lo) * G.double()).sum() / 2
    dW = K.embedding_scaled_bwd(G, ids, V, 3.0).double()
    ana = (dW * E.double()).sum()
    mag = ((hi.abs() + lo.abs()) * G.double().abs()).sum() / 2 + N * (dW.abs() * E.double().abs()).sum()
    assert (num - ana).abs() <= 4 * U * mag


def test_other_stream(cuda):
    """The calls run on the current stream, ordered with the work around them."""
    from tinytrain_b200 import kernels as K
    g = torch.Generator(device=cuda).manual_seed(2)
    N, D, V = 4096, 512, 2000
    ids = torch.randint(0, V, (N,), device=cuda, generator=g)
    dout = torch.randn(N, D, device=cuda, generator=g)
    want = K.embedding_scaled_bwd(2 * dout, ids, V, 1.5)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = K.embedding_scaled_bwd(dout + dout, ids, V, 1.5) + 0.0
    torch.cuda.current_stream().wait_stream(st)
    assert torch.equal(got, want)


@pytest.mark.parametrize("N,D,V", [(10, 4, 100), (3, 1, 4000), (60, 8, 900), (4096, 4, 1000),
                                   (4097, 3, 2000), (5000, 1, 33), (70000, 2, 3000)])
def test_small_tables(cuda, N, D, V):
    """Tables of a few KB (one block zeroes them all) with tokens past the first 32."""
    from tinytrain_b200 import kernels as K
    g = torch.Generator(device=cuda).manual_seed(N)
    for kind in ("uniform", "ends", "text"):
        ids = tokens(kind, N, V, g, cuda)
        dout = torch.randn(N, D, device=cuda, generator=g)
        at, rows = ids.clamp(min=0), torch.where((ids >= 0)[:, None], dout.double(), 0.0)
        ref = torch.zeros(V, D, device=cuda, dtype=torch.float64).index_add_(0, at, rows)
        mag = torch.zeros(V, D, device=cuda, dtype=torch.float64).index_add_(0, at, rows.abs())
        n = torch.bincount(at[ids >= 0], minlength=V).double()[:, None]
        dW = torch.full((V, D), 9.0, device=cuda)  # written, not added to
        K.embedding_scaled_bwd(dout, ids, V, 1.0, dW=dW)
        assert ((dW.double() - ref).abs() <= (n + 2) * U * mag).all()
        assert (dW[(n == 0).squeeze(1)] == 0).all()
    assert status() == 0
