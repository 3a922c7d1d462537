"""Feature-map operators at the ends of their types' ranges and of their sizes: rows far from zero,
variances beyond float32, float16 factors beyond float16, long reductions, many input dimensions.
Bounds as in test_features_gpu, counted from the arithmetic."""
import math

import pytest

import test_features_gpu as base
from test_features_gpu import DT, E23, E24, act_ref, check, half_step, norm_depth, randn, sum_error

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def give_memory_back():
    yield
    if torch.cuda.memory_reserved() > 8 << 30:
        torch.cuda.empty_cache()


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


# ------------------------------------------------------------------- gated unit
def gated_grads_in_range(ft, rows, inner, outer, act, x_scale, w_scale, up_bias, dy_scale, want):
    """float16 gradients `want` of factors dout up act' and dout act that float16 itself does not hold.
    They are kept as float16 parts of their values times one power of two: off by half a step of the
    type (U), or by half the smallest step: 2^-25 where the largest factor is 2^-4 to 2^15, 2^-37
    of the largest otherwise."""
    t, u = torch.float16, half_step(torch.float16)
    x = randn(41, rows, inner, dtype=t, scale=x_scale)
    wg, wu = (randn(s, outer, inner, dtype=t, scale=w_scale) for s in (42, 43))
    bg = randn(44, outer, dtype=t, scale=0.3)
    bu = randn(45, outer, dtype=t, scale=0.2 * up_bias, shift=up_bias)
    dy = randn(46, rows, outer, dtype=t, scale=dy_scale)
    out = {"dx": torch.zeros_like(x), "dw_gate": torch.zeros_like(wg), "dw_up": torch.zeros_like(wu),
           "db_gate": torch.zeros_like(bg), "db_up": torch.zeros_like(bu)}
    out = {k: out[k] for k in want}
    ws = torch.full((ft.gated_unit_workspace(rows, inner, outer, t, backward=True),), 0xFF,
                    dtype=torch.uint8, device="cuda")
    ft.gated_unit_backward(dy, x, wg, wu, bg, bu, activation=act, workspace=ws, **out)
    X, G, U, D = x.double(), wg.double(), wu.double(), dy.double()
    gate, up = X @ G.T + bg.double(), X @ U.T + bu.double()
    e = sum_error(inner, False)
    eg = e * (X.abs() @ G.abs().T) + E23 * gate.abs()
    eu = e * (X.abs() @ U.abs().T) + E23 * up.abs()
    val, slope = act_ref(act, gate)
    ev = 1.13 * eg + 2.0 ** -22 * (4 + gate * gate) * val.abs()
    es = eg + 2.0 ** -21 * (1 + gate.abs())
    dg, du = D * up * slope, D * val
    largest = max(dg.abs().max().item(), du.abs().max().item())
    tiny = max(2.0 ** -37 * largest, 2.0 ** -25 if largest > 0.06 else 0.0)
    edg = D.abs() * (slope.abs() * eu + up.abs() * es + es * eu) + 2.0 ** -22 * dg.abs()
    edg = edg + u * (dg.abs() + edg) + tiny
    edu = D.abs() * ev + E23 * du.abs()
    edu = edu + u * (du.abs() + edu) + tiny
    if "dx" in out:
        ref = dg @ G + du @ U
        e = sum_error(2 * outer, False)
        bound = edg @ G.abs() + edu @ U.abs()
        bound = bound + e * ((dg.abs() + edg) @ G.abs() + (du.abs() + edu) @ U.abs())
        check(out["dx"], ref, bound + u * (ref.abs() + bound))
    e = sum_error(rows, False)
    for name, d, ed in (("gate", dg, edg), ("up", du, edu)):
        if "dw_" + name in out:
            ref = d.T @ X
            bound = ed.T @ X.abs() + e * ((d.abs() + ed).T @ X.abs())
            check(out["dw_" + name], ref, bound + u * (ref.abs() + bound))
        if "db_" + name in out:
            ref = d.sum(0)
            bound = ed.sum(0) + (rows + 20) * E24 * (d.abs() + ed).sum(0)
            check(out["db_" + name], ref, bound + u * (ref.abs() + bound))
    return dg, du, largest, out


# On both sides of the CUDA-core path's bound, with split and unsplit projections, unaligned rows, both
# weights in one tile, and on CTA pairs with one part per factor.
RANGE_SHAPES = [(2, 520, 520), (3, 520, 520), (9, 64, 48), (100, 64, 48), (33, 71, 65), (140, 2100, 130),
                (300, 96, 300), (2660, 1800, 1000)]


@pytest.mark.parametrize("act", ["silu", "sigmoid"])
@pytest.mark.parametrize("rows,inner,outer", RANGE_SHAPES)
def test_gated_unit_float16_factors_beyond_the_type(ft, rows, inner, outer, act):
    """up of some 300 under a gradient of some 200: factors up to 10^6, gradients within float16."""
    s = 0.02 / math.sqrt(max(1, max(inner, outer, rows) / 100))
    dg, _, largest, _ = gated_grads_in_range(ft, rows, inner, outer, act, s, s, 300.0,
                                             200.0 if act == "silu" else 400.0,
                                             ["dx", "dw_gate", "dw_up"])
    assert largest > 65504


@pytest.mark.parametrize("rows,inner,outer", RANGE_SHAPES)
def test_gated_unit_float16_factors_below_the_type(ft, rows, inner, outer):
    """A gradient of a few of float16's smallest steps, 2^-24, against large weights (dx) and large inputs
    (the weight gradients)."""
    w = 2.0 ** 10
    for names, xs, wscale in ((["dx"], 2.0 ** -10 / math.sqrt(inner), w),
                              (["dw_gate", "dw_up"], w, 2.0 ** -10 / math.sqrt(inner))):
        _, _, largest, _ = gated_grads_in_range(ft, rows, inner, outer, "silu", xs, wscale, 0.5,
                                                2.0 ** -22, names)
        assert largest < 2.0 ** -15


def test_gated_unit_float16_factors_repeat_and_in_a_graph(ft):
    """A captured call follows its inputs: the factors' scale is found anew at each replay."""
    rows, inner, outer, t = 200, 64, 96, torch.float16
    x, dy = randn(1, rows, inner, dtype=t, scale=0.02), randn(2, rows, outer, dtype=t)
    wg, wu = randn(3, outer, inner, dtype=t, scale=0.02), randn(4, outer, inner, dtype=t, scale=0.02)
    bg, bu = randn(5, outer, dtype=t), randn(6, outer, dtype=t, shift=300.0)
    ws = torch.empty(ft.gated_unit_workspace(rows, inner, outer, t, backward=True), dtype=torch.uint8,
                     device="cuda")

    def call(out, stream=None):
        ft.gated_unit_backward(dy, x, wg, wu, bg, bu, dx=out[0], dw_gate=out[1], dw_up=out[2],
                               workspace=ws, stream=stream)

    new = lambda: [torch.zeros_like(x), torch.zeros_like(wg), torch.zeros_like(wu)]
    got = new()
    call(got)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(got, torch.cuda.current_stream().cuda_stream)
    for scale in (200.0, 2.0 ** -20, 0.0, 1.0, 200.0):
        dy.copy_(randn(2, rows, outer, scale=scale))
        want = new()
        call(want)
        graph.replay()
        torch.cuda.synchronize()
        for g, v in zip(got, want):
            assert torch.isfinite(v).all() and torch.equal(g, v), scale
            assert (v != 0).any() == (scale != 0)


@pytest.mark.parametrize("rows,inner,outer", [(100, 64, 48), (140, 2100, 130), (2660, 1800, 1000)])
def test_gated_unit_float16_non_finite_factors_stay_their_own(ft, rows, inner, outer):
    """A row with an infinite or NaN gradient leaves the other rows' dx as it is, scaled or not."""
    t = torch.float16
    x, dy = randn(1, rows, inner, dtype=t, scale=0.02), randn(2, rows, outer, dtype=t, scale=200.0)
    wg, wu = (randn(s, outer, inner, dtype=t, scale=0.2 / math.sqrt(inner)) for s in (3, 4))
    bg, bu = randn(5, outer, dtype=t), randn(6, outer, dtype=t, shift=300.0)
    ws = torch.empty(ft.gated_unit_workspace(rows, inner, outer, t, backward=True), dtype=torch.uint8,
                     device="cuda")
    want, got = torch.zeros_like(x), torch.zeros_like(x)
    ft.gated_unit_backward(dy, x, wg, wu, bg, bu, dx=want, workspace=ws)
    dy[3, 5], dy[rows - 2, 7] = float("inf"), float("nan")
    ft.gated_unit_backward(dy, x, wg, wu, bg, bu, dx=got, workspace=ws)
    rest = torch.ones(rows, dtype=torch.bool, device="cuda")
    rest[3] = rest[rows - 2] = False
    assert torch.isfinite(want).all() and torch.equal(got[rest], want[rest])
    assert not torch.isfinite(got[3]).any() and not torch.isfinite(got[rows - 2]).any()


# Reductions of one sign, in sizes whose tiles alone fill the SMs. The tensor core truncates each term at 2^-25
# of the accumulator, which holds half of its final value on average: a range of 2^14 terms is at most
# 2^-12 short of its sum of magnitudes. The joins add 2^-24 a range, the activation 2^-21.
SHORT = 2.0 ** -12 + 2.0 ** -16 + 2.0 ** -21


def positive(seed, *shape):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.rand(shape, generator=g, device="cuda", dtype=torch.float16) * 2.0 ** -6


def test_gated_unit_long_reduction(ft):
    t = torch.float16
    rows, inner, outer = 1280, 1 << 20, 1000
    x, wu = positive(3, rows, inner), positive(4, outer, inner)
    wg = torch.zeros_like(wu)  # sigmoid(0) = 1/2
    ws = torch.empty(ft.gated_unit_workspace(rows, inner, outer, t), dtype=torch.uint8, device="cuda")
    out = torch.empty((rows, outer), dtype=t, device="cuda")
    ft.gated_unit(out, x, wg, wu, activation="sigmoid", workspace=ws)
    i, j = torch.arange(0, rows, 161, device="cuda"), torch.arange(0, outer, 99, device="cuda")
    ref = 0.5 * torch.stack([(x[a].double()[None] * wu[j].double()).sum(1) for a in i])
    check(out[i][:, j], ref, SHORT * ref + half_step(t) * (1 + SHORT) * ref)


def test_gated_unit_long_reduction_of_the_weight_gradients(ft):
    t = torch.float16
    rows, inner, outer = 1 << 18, 2432, 1000
    x, dy, wu = positive(5, rows, inner), positive(6, rows, outer), positive(7, outer, inner)
    wg, dwu = torch.zeros_like(wu), torch.zeros_like(wu)
    ws = torch.empty(ft.gated_unit_workspace(rows, inner, outer, t, backward=True), dtype=torch.uint8,
                     device="cuda")
    ft.gated_unit_backward(dy, x, wg, wu, dw_up=dwu, activation="sigmoid", workspace=ws)
    i, j = torch.arange(0, inner, 97, device="cuda"), torch.arange(0, outer, 61, device="cuda")
    ref = (dy[:, j].double() / 2).T @ x[:, i].double()
    # dup = dout / 2 is exact in float16 but for its smallest steps, whatever the factors' scale.
    bound = SHORT * ref + 2.0 ** -25 * x[:, i].double().sum(0)
    check(dwu[j][:, i], ref, bound + half_step(t) * (ref + bound))


def test_gated_unit_long_reduction_of_the_input_gradient(ft):
    t = torch.float16
    rows, inner, outer = 2432, 1000, 1 << 18
    x, dy, wu = positive(8, rows, inner), positive(9, rows, outer), positive(10, outer, inner)
    wg, dx = torch.zeros_like(wu), torch.zeros_like(x)
    ws = torch.empty(ft.gated_unit_workspace(rows, inner, outer, t, backward=True), dtype=torch.uint8,
                     device="cuda")
    ft.gated_unit_backward(dy, x, wg, wu, dx=dx, activation="sigmoid", workspace=ws)
    i, j = torch.arange(0, inner, 97, device="cuda"), torch.arange(0, rows, 61, device="cuda")
    ref = (dy[j].double() / 2) @ wu[:, i].double()
    bound = SHORT * ref + 2.0 ** -25 * wu[:, i].double().sum(0)
    check(dx[j][:, i], ref, bound + half_step(t) * (ref + bound))
