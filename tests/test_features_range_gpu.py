"""Feature-map operators at the ends of their types' ranges and of their sizes: rows far from zero,
variances beyond float32, float16 factors beyond float16, long reductions, many input dimensions.
Bounds as in test_features_gpu, counted from the arithmetic."""
import math

import pytest

import test_features_gpu as base
from test_features_gpu import DT, E23, E24, act_ref, check, half_step, norm_depth, randn, sum_error

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ft(gpb_lib):
    from mojogp_b200 import features
    yield features
    features.check_device(0)


# ------------------------------------------------------------------ layer norm
# Rows of at most a vector per thread, of several, unaligned, and too wide for registers.
@pytest.mark.parametrize("rows,cols", [(50, 16), (1000, 64), (40, 1000), (40, 999), (700, 2048), (5, 4096),
                                       (3, 16384), (3, 20001)])
@pytest.mark.parametrize("dtype,mean", [("fp32", 1e4), ("fp32", -3e5), ("bf16", 512.0), ("fp16", 1000.0)])
def test_layer_norm_backward_far_from_zero(ft, rows, cols, dtype, mean):
    """xhat = (x - mean) rstd is a subtraction and a product, each off by 2^-24 of its own result: the
    rows' distance from zero does not show, whatever their alignment."""
    t = DT[dtype]
    x, dy = randn(31, rows, cols, dtype=t, shift=mean), randn(32, rows, cols, dtype=t)
    w = randn(33, cols, scale=0.3, shift=1.0)
    X, D, W = x.double(), dy.double(), w.double()
    mu = X.mean(1)
    rs = 1 / torch.sqrt(((X - mu[:, None]) ** 2).mean(1) + 1e-5)
    m, r = mu.float(), rs.float()
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(w)
    ws = torch.empty(ft.layer_norm_workspace(rows, cols), dtype=torch.uint8, device="cuda")
    ft.layer_norm_backward(dx, dy, x, m, r, w, dweight=dw, dbias=db, workspace=ws)
    R = r.double()[:, None]
    xh = (X - m.double()[:, None]) * R
    e_x = 2.1 * E24 * xh.abs()
    g = norm_depth(cols) * E24
    G = D * W
    mg, mgx = G.mean(1, keepdim=True), (G * xh).mean(1, keepdim=True)
    ref = R * (G - mg - xh * mgx)
    e_mg = g * G.abs().mean(1, keepdim=True) * 1.01
    e_mgx = (g * (G * xh).abs().mean(1, keepdim=True) + (G.abs() * e_x).mean(1, keepdim=True)) * 1.01
    bound = R * (6 * E24 * (G.abs() + mg.abs() + (xh * mgx).abs()) + e_mg + xh.abs() * e_mgx
                 + e_x * mgx.abs()) * 1.01
    check(dx, ref, bound + half_step(t) * (ref.abs() + bound))
    k = (rows + 20) * E24
    ref, mag = (D * xh).sum(0), (D * xh).abs().sum(0)
    bound = k * mag + (D.abs() * e_x).sum(0)
    check(dw, ref, bound + E24 * (ref.abs() + bound))


# One vector per thread of few and many rows, several vectors, unaligned rows of few and many, wide rows.
@pytest.mark.parametrize("rows,cols", [(3, 16), (5000, 64), (40, 1000), (40, 999), (700, 999), (700, 4096),
                                       (3, 20001)])
def test_layer_norm_of_an_infinite_variance(ft, rows, cols):
    """A variance beyond float32 is infinite in the formula's float32: rstd = 0 and out = bias."""
    x = randn(34, rows, cols, scale=1e20)
    x[1] = randn(35, cols)
    w, b = randn(36, cols), randn(37, cols)
    y, rstd = torch.empty_like(x), torch.empty(rows, device="cuda")
    ft.layer_norm(y, x, w, b, rstd=rstd)
    far = torch.arange(rows, device="cuda") != 1
    assert (rstd[far] == 0).all() and torch.equal(y[far], b.expand(rows, cols)[far])
    one = torch.empty((1, cols), device="cuda")
    ft.layer_norm(one, x[1:2], w, b)
    torch.testing.assert_close(y[1:2], one, rtol=1e-5, atol=1e-5)
