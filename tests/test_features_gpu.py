"""Feature-map operators on the GPU against their formulas in 64 bits.

Tolerances are bounds, element by element, counted from the arithmetic: an
output's rounding is half a step of its type (U), an fp32 sum of k terms is off
by at most k 2^-24 of the sum of magnitudes (2^-23 on the tensor cores, which
truncate), and first-order error propagation through the formulas does the
rest. dgate and dup are rounded once to the operands' type (float32 inputs:
2^-24)."""
import ctypes as C
import math

import numpy as np
import pytest

from mojogp_b200 import _lib

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

E24, E23 = 2.0 ** -24, 2.0 ** -23
DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def half_step(t):
    return torch.finfo(t).eps / 2


@pytest.fixture(scope="module")
def ft(gpb_lib):
    from mojogp_b200 import features
    yield features
    features.check_device(0)


def randn(seed, *shape, dtype=torch.float32, scale=1.0, shift=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale + shift).to(dtype)


def strided(t, pad, offset=0):
    """The same values in a block with a longer row stride (and an offset start)."""
    rows, cols = t.shape
    big = torch.full((rows * (cols + pad) + offset + 16,), 7.0, dtype=t.dtype, device="cuda")
    v = big[offset:offset + rows * (cols + pad)].view(rows, cols + pad)[:, :cols]
    v.copy_(t)
    return v


def check(got, ref, bound, floor=2.0 ** -24):
    got = got.double()
    assert torch.isfinite(got).all()
    excess = ((got - ref).abs() - bound - floor).max().item()
    assert excess <= 0, f"largest error beyond the bound: {excess:.3e}"


# ------------------------------------------------------------------ layer norm
def norm_depth(cols):
    return min(cols, 70 + math.ceil(cols / 1024)) + 4


NORM_SHAPES = [(1, 1), (1, 4096), (3, 2), (7, 5), (33, 16), (5, 33), (130, 64), (9, 100), (17, 255),
               (4, 256), (3, 1000), (65, 1024), (2, 1025), (5, 4095), (3, 8192), (2, 16384), (2, 9001),
               (1, 40000), (1000, 8)]


@pytest.mark.parametrize("dtype,wdtype", [("fp32", "fp32"), ("fp16", "fp16"), ("fp16", "fp32"),
                                          ("bf16", "bf16"), ("bf16", "fp32")])
@pytest.mark.parametrize("rows,cols", NORM_SHAPES)
def test_layer_norm(ft, rows, cols, dtype, wdtype):
    t, wt = DT[dtype], DT[wdtype]
    x = randn(1, rows, cols, dtype=t, scale=1.5, shift=0.5)
    w, b = randn(2, cols, dtype=wt, scale=0.3, shift=1.0), randn(3, cols, dtype=wt)
    dy = randn(4, rows, cols, dtype=t)
    y, mean, rstd = torch.empty_like(x), torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    ft.layer_norm(y, x, w, b, eps=1e-5, mean=mean, rstd=rstd)
    X, W, B, D = x.double(), w.double(), b.double(), dy.double()
    mu = X.mean(1, keepdim=True)
    var = ((X - mu) ** 2).mean(1, keepdim=True)
    rs = 1 / torch.sqrt(var + 1e-5)
    g = norm_depth(cols) * E24
    e_d = g * X.abs().mean(1, keepdim=True) + E24 * (X.abs() + mu.abs())
    sd = torch.sqrt(var)
    e_var = 2 * sd * e_d.amax(1, keepdim=True) + e_d.amax(1, keepdim=True) ** 2 + g * var
    e_rs = 0.5 * e_var / (var + 1e-5) * 1.01 + 6 * E24
    xh = (X - mu) * rs
    ref = xh * W + B
    bound = W.abs() * (rs * e_d + xh.abs() * e_rs) * 1.01 + 6 * E24 * ((xh * W).abs() + B.abs())
    check(y, ref, bound + half_step(t) * (ref.abs() + bound))
    check(mean, mu[:, 0], g * X.abs().mean(1))
    check(rstd, rs[:, 0], rs[:, 0] * e_rs[:, 0])

    # Backward, from the statistics the forward pass wrote.
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
    ws = torch.empty(ft.layer_norm_workspace(rows, cols), dtype=torch.uint8, device="cuda")
    ft.layer_norm_backward(dx, dy, x, mean, rstd, w, dweight=dw, dbias=db, workspace=ws)
    M, R = mean.double()[:, None], rstd.double()[:, None]
    xh = (X - M) * R
    e_x = 3 * E24 * (X.abs() + M.abs()) * R
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
    check(dw, ref, bound + half_step(wt) * (ref.abs() + bound))
    ref, bound = D.sum(0), k * D.abs().sum(0)
    check(db, ref, bound + half_step(wt) * (ref.abs() + bound))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("pad,offset", [(8, 0), (3, 0), (0, 1), (5, 3)])
def test_layer_norm_strides_and_in_place(ft, dtype, pad, offset):
    t = DT[dtype]
    for rows, cols in [(37, 64), (6, 2000)]:
        x, dy = randn(5, rows, cols, dtype=t), randn(6, rows, cols, dtype=t)
        w, b = randn(7, cols), randn(8, cols)
        y = torch.empty_like(x)
        mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
        ft.layer_norm(y, x, w, b, mean=mean, rstd=rstd)
        xs = strided(x, pad, offset)
        # The kernels for aligned and unaligned rows sum in different orders: equal up to a rounding.
        tol = dict(rtol=2 * half_step(t) + 1e-5, atol=2 * half_step(t) + 1e-5)
        ys = strided(torch.zeros_like(x), pad, offset)
        ft.layer_norm(ys, xs, w, b)
        torch.testing.assert_close(ys, y, **tol)
        full = torch.as_strided(ys, (rows - 1, pad), (cols + pad, 1), ys.storage_offset() + cols)
        assert (full == 7).all()  # between the rows nothing is written
        ws = torch.empty(ft.layer_norm_workspace(rows, cols), dtype=torch.uint8, device="cuda")
        dx, dw = torch.empty_like(x), torch.empty_like(w)
        ft.layer_norm_backward(dx, dy, x, mean, rstd, w, dweight=dw, workspace=ws)
        dys, dw2 = strided(dy, pad, offset), torch.empty_like(w)
        ft.layer_norm_backward(dys, dys, xs, mean, rstd, w, dweight=dw2, workspace=ws)  # in place
        torch.testing.assert_close(dys, dx, **tol)
        torch.testing.assert_close(dw2, dw, rtol=1e-4, atol=1e-4)
        ft.layer_norm(xs, xs, w, b)  # in place
        torch.testing.assert_close(xs, y, **tol)


def test_layer_norm_options_and_repeats(ft):
    x, dy = randn(9, 300, 96), randn(10, 300, 96)
    one, zero = torch.ones(96, device="cuda"), torch.zeros(96, device="cuda")
    y, y1 = torch.empty_like(x), torch.empty_like(x)
    mean, rstd = torch.empty(300, device="cuda"), torch.empty(300, device="cuda")
    ft.layer_norm(y, x, mean=mean, rstd=rstd)
    ft.layer_norm(y1, x, one, zero)
    assert torch.equal(y, y1)
    dx, dx1 = torch.empty_like(x), torch.empty_like(x)
    ws = torch.empty(ft.layer_norm_workspace(300, 96), dtype=torch.uint8, device="cuda")
    dw, db = torch.empty(96, device="cuda"), torch.empty(96, device="cuda")
    ft.layer_norm_backward(dx, dy, x, mean, rstd)
    ft.layer_norm_backward(dx1, dy, x, mean, rstd, one, dweight=dw, dbias=db, workspace=ws)
    assert torch.equal(dx, dx1)
    dw1, db1 = torch.empty_like(dw), torch.empty_like(db)
    ft.layer_norm_backward(None, dy, x, mean, rstd, one, dweight=dw1, workspace=ws)
    ft.layer_norm_backward(None, dy, x, mean, rstd, one, dbias=db1, workspace=ws)
    assert torch.equal(dw, dw1) and torch.equal(db, db1)
    # No rows: nothing to norm, zero weight gradients.
    e = torch.empty((0, 96), device="cuda")
    ft.layer_norm(e, e.clone(), one, zero)
    ft.layer_norm_backward(e, e, e, e[:, 0], e[:, 0], one, dweight=dw, dbias=db, workspace=ws)
    assert (dw == 0).all() and (db == 0).all()
    ft.layer_norm_backward(e, e, e, e[:, 0], e[:, 0], one)  # and nothing else to do
    # A constant row has variance 0: rstd = 1 / sqrt(eps), y = bias.
    c = torch.full((2, 96), 3.25, device="cuda")
    ft.layer_norm(y[:2], c, one, zero, eps=1e-4, rstd=rstd[:2])
    assert (y[:2] == 0).all()
    torch.testing.assert_close(rstd[:2], torch.full((2,), 100.0, device="cuda"))


# ------------------------------------------------------------------- gated unit
def act_ref(name, z):
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if name == "gelu":
        cdf = torch.special.ndtr(z)
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "sigmoid":
        s = torch.sigmoid(z)
        return s, s * (1 - s)
    v = torch.tanh(z)
    return v, 1 - v * v


def sum_error(k, f32):
    """Relative to the sum of magnitudes: k truncating additions; float32 inputs promote every 256
    terms and drop plane products below 2^-23."""
    return (min(k, 256) + k / 256 + 10) * E23 if f32 else (k + 10) * E23


def gated_case(ft, rows, inner, outer, dtype, act, bias, transform=lambda t: t, seed=0):
    t = DT[dtype]
    f32 = dtype == "fp32"
    u = half_step(t)
    x = transform(randn(seed + 11, rows, inner, dtype=t))
    wg = transform(randn(seed + 12, outer, inner, dtype=t, scale=inner ** -0.5))
    wu = transform(randn(seed + 13, outer, inner, dtype=t, scale=inner ** -0.5))
    bg = randn(seed + 14, outer, dtype=t, scale=0.3) if bias else None
    bu = randn(seed + 15, outer, dtype=t, scale=0.3) if bias else None
    dy = transform(randn(seed + 16, rows, outer, dtype=t))
    ws = torch.empty(max(16, ft.gated_unit_workspace(rows, inner, outer, t)), dtype=torch.uint8,
                     device="cuda")
    out = transform(torch.zeros((rows, outer), dtype=t, device="cuda"))
    ft.gated_unit(out, x, wg, wu, bg, bu, activation=act, workspace=ws)
    X, G, U, D = x.double(), wg.double(), wu.double(), dy.double()
    gate, up = X @ G.T, X @ U.T
    e = sum_error(inner, f32)
    eg, eu = e * (X.abs() @ G.abs().T), e * (X.abs() @ U.abs().T)
    if bias:
        gate, up = gate + bg.double(), up + bu.double()
    eg, eu = eg + E23 * gate.abs(), eu + E23 * up.abs()
    val, slope = act_ref(act, gate)
    ev = 1.13 * eg + 2.0 ** -22 * (4 + gate * gate) * val.abs()
    es = eg + 2.0 ** -21 * (1 + gate.abs())
    ref = val * up
    bound = (up.abs() * ev + val.abs() * eu + ev * eu) + E23 * ref.abs()
    check(out, ref, bound + u * (ref.abs() + bound))

    need = ft.gated_unit_workspace(rows, inner, outer, t, backward=True)
    ws = torch.full((max(16, need),), 0xFF, dtype=torch.uint8, device="cuda")  # NaN patterns
    dx = transform(torch.zeros((rows, inner), dtype=t, device="cuda"))
    dwg = transform(torch.zeros((outer, inner), dtype=t, device="cuda"))
    dwu = transform(torch.zeros((outer, inner), dtype=t, device="cuda"))
    dbg, dbu = torch.zeros(outer, dtype=t, device="cuda"), torch.zeros(outer, dtype=t, device="cuda")
    ft.gated_unit_backward(dy, x, wg, wu, bg, bu, dx=dx, dw_gate=dwg, dw_up=dwu, db_gate=dbg,
                           db_up=dbu, activation=act, workspace=ws)
    dg, du = D * up * slope, D * val
    op = E24 if f32 else u
    tiny = 2.0 ** -25 if dtype == "fp16" else 0.0
    edg = D.abs() * (slope.abs() * eu + up.abs() * es + es * eu) + 2.0 ** -22 * dg.abs()
    edg = edg + op * (dg.abs() + edg) + tiny
    edu = D.abs() * ev + E23 * du.abs()
    edu = edu + op * (du.abs() + edu) + tiny
    ref = dg @ G + du @ U
    e = sum_error(2 * outer, f32)
    bound = edg @ G.abs() + edu @ U.abs()
    bound = bound + e * ((dg.abs() + edg) @ G.abs() + (du.abs() + edu) @ U.abs())
    check(dx, ref, bound + u * (ref.abs() + bound))
    e = sum_error(rows, f32)
    for got, d, ed, gb in ((dwg, dg, edg, dbg), (dwu, du, edu, dbu)):
        ref = d.T @ X
        bound = ed.T @ X.abs() + e * ((d.abs() + ed).T @ X.abs())
        check(got, ref, bound + u * (ref.abs() + bound))
        ref = d.sum(0)
        bound = ed.sum(0) + (rows + 20) * E24 * (d.abs() + ed).sum(0)
        check(gb, ref, bound + u * (ref.abs() + bound))
    return out, dx, dwg, dwu, dbg, dbu


GATED_SHAPES = [(1, 1, 1), (1, 64, 48), (2, 7, 3), (3, 100, 130), (8, 256, 2500), (9, 8, 1), (9, 1, 9),
                (16, 64, 64), (33, 72, 65), (64, 17, 33), (100, 136, 64), (127, 64, 129),
                (128, 64, 128), (129, 65, 130), (130, 200, 96), (257, 513, 31), (300, 96, 300),
                (1000, 24, 16), (700, 320, 257), (2100, 40, 8)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,inner,outer", GATED_SHAPES)
def test_gated_unit(ft, rows, inner, outer, dtype):
    act = ["silu", "gelu", "sigmoid", "tanh"][(rows + inner + outer) % 4]
    gated_case(ft, rows, inner, outer, dtype, act, bias=(rows + outer) % 2 == 0)


# Sizes whose products all run on CTA pairs (16-bit), with an odd number of row tiles and ragged edges.
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,inner,outer", [(2660, 1800, 1000), (9500, 264, 1200), (2561, 1928, 1024)])
def test_gated_unit_large(ft, rows, inner, outer, dtype):
    gated_case(ft, rows, inner, outer, dtype, "gelu", True)


# Few tiles: a long reduction is split (projections from 2048 columns, dx from 512 outputs) and the ranges
# end unevenly; a few rows on either side of the CUDA-core path's bound, rows that a 16-byte vector cannot
# read among them.
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,inner,outer", [
    (2, 520, 520), (3, 520, 520), (3, 517, 523), (5, 517, 523), (8, 520, 520), (9, 520, 520),
    (3, 2100, 130), (11, 2048, 7), (16, 4104, 72), (40, 5000, 33), (100, 2050, 40), (130, 3100, 200),
    (290, 2048, 64), (20, 40, 1030), (129, 8, 2100), (260, 264, 800)])
def test_gated_unit_few_tiles(ft, rows, inner, outer, dtype):
    act = ["silu", "gelu", "sigmoid", "tanh"][(rows + inner + outer) % 4]
    gated_case(ft, rows, inner, outer, dtype, act, bias=(rows + outer) % 3 > 0)


def test_gated_unit_split_repeats(ft):
    """Split reductions join in a fixed order: results repeat bit for bit."""
    full = gated_case(ft, 50, 4096, 96, "bf16", "silu", True)
    again = gated_case(ft, 50, 4096, 96, "bf16", "silu", True)
    for a, b in zip(full, again):
        assert torch.equal(a, b)


def test_gated_unit_split_outputs_alone_and_in_a_graph(ft):
    rows, inner, outer, t = 50, 4096, 530, torch.bfloat16
    full = gated_case(ft, rows, inner, outer, "bf16", "silu", True)
    x, dy = randn(11, rows, inner, dtype=t), randn(16, rows, outer, dtype=t)
    wg = randn(12, outer, inner, dtype=t, scale=inner ** -0.5)
    wu = randn(13, outer, inner, dtype=t, scale=inner ** -0.5)
    bg, bu = randn(14, outer, dtype=t, scale=0.3), randn(15, outer, dtype=t, scale=0.3)
    ws = torch.empty(ft.gated_unit_workspace(rows, inner, outer, t, backward=True), dtype=torch.uint8,
                     device="cuda")
    names = ["dx", "dw_gate", "dw_up", "db_gate", "db_up"]
    for name, want in zip(names, full[1:]):
        got = torch.empty_like(want)
        ft.gated_unit_backward(dy, x, wg, wu, bg, bu, workspace=ws, **{name: got})
        assert torch.equal(got, want), name
    got = [torch.zeros_like(v) for v in full]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        stream = torch.cuda.current_stream().cuda_stream
        ft.gated_unit(got[0], x, wg, wu, bg, bu, workspace=ws, stream=stream)
        ft.gated_unit_backward(dy, x, wg, wu, bg, bu, workspace=ws, stream=stream,
                               **dict(zip(names, got[1:])))
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    for g, w in zip(got, full):
        assert torch.equal(g, w)


def test_gated_unit_split_padding_stays_out_of_the_sums(ft):
    """The rows of a split product's last tile past the caller's add nothing to any gradient, whatever a
    bias holds."""
    rows, inner, outer, t = 33, 2048, 70, torch.bfloat16
    x, dy = randn(1, rows, inner, dtype=t), randn(2, rows, outer, dtype=t)
    wg, wu = randn(3, outer, inner, dtype=t, scale=0.02), randn(4, outer, inner, dtype=t, scale=0.02)
    bg, bu = torch.zeros(outer, dtype=t, device="cuda"), torch.zeros(outer, dtype=t, device="cuda")
    bu[5] = float("inf")
    ws = torch.full((ft.gated_unit_workspace(rows, inner, outer, t, backward=True),), 0xFF,
                    dtype=torch.uint8, device="cuda")
    dbg, dbu = torch.zeros_like(bg), torch.zeros_like(bg)
    ft.gated_unit_backward(dy, x, wg, wu, bg, bu, db_gate=dbg, db_up=dbu, workspace=ws)
    gate = x.double() @ wg.double().T
    val, _ = act_ref("silu", gate)
    want = (dy.double() * val).sum(0)
    eg = sum_error(inner, False) * (x.double().abs() @ wg.double().abs().T)
    ev = 1.13 * eg + 2.0 ** -22 * (4 + gate * gate) * val.abs()
    term = dy.double().abs() * ev
    bound = term.sum(0) + (rows + 20) * E24 * ((dy.double() * val).abs() + term).sum(0)
    check(dbu, want, bound + half_step(t) * (want.abs() + bound))
    keep = torch.arange(outer, device="cuda") != 5
    assert torch.isfinite(dbg[keep]).all() and not torch.isfinite(dbg[5])


@pytest.mark.parametrize("rows", [3, 140])
@pytest.mark.parametrize("pad,offset", [(8, 0), (3, 0), (0, 1), (5, 3)])
def test_gated_unit_split_strides(ft, rows, pad, offset):
    gated_case(ft, rows, 2304, 144, "bf16", "gelu", True, transform=lambda v: strided(v, pad, offset))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("act", ["silu", "gelu", "sigmoid", "tanh"])
@pytest.mark.parametrize("rows", [5, 150])
def test_gated_unit_activations(ft, rows, act, dtype):
    gated_case(ft, rows, 48, 72, dtype, act, bias=True)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("rows", [4, 140])
@pytest.mark.parametrize("pad,offset", [(8, 0), (3, 0), (0, 1), (5, 3)])
def test_gated_unit_strides(ft, rows, pad, offset, dtype):
    gated_case(ft, rows, 72, 136, dtype, "silu", True, transform=lambda v: strided(v, pad, offset))


def test_gated_unit_partial_outputs_and_repeats(ft):
    for rows in (3, 400):
        full = gated_case(ft, rows, 80, 100, "bf16", "gelu", True)
        again = gated_case(ft, rows, 80, 100, "bf16", "gelu", True)
        for a, b in zip(full, again):
            assert torch.equal(a, b)
        t = torch.bfloat16
        x = randn(11, rows, 80, dtype=t)
        wg, wu = randn(12, 100, 80, dtype=t, scale=80 ** -0.5), randn(13, 100, 80, dtype=t, scale=80 ** -0.5)
        bg, bu = randn(14, 100, dtype=t, scale=0.3), randn(15, 100, dtype=t, scale=0.3)
        dy = randn(16, rows, 100, dtype=t)
        ws = torch.empty(ft.gated_unit_workspace(rows, 80, 100, t, backward=True), dtype=torch.uint8,
                         device="cuda")
        names = ["dx", "dw_gate", "dw_up", "db_gate", "db_up"]
        for name, want in zip(names, full[1:]):
            got = torch.empty_like(want)
            ft.gated_unit_backward(dy, x, wg, wu, bg, bu, activation="gelu", workspace=ws,
                                   **{name: got})
            assert torch.equal(got, want), name


def test_gated_unit_no_rows(ft):
    t = torch.float16
    e = torch.empty((0, 24), dtype=t, device="cuda")
    o = torch.empty((0, 40), dtype=t, device="cuda")
    w = randn(1, 40, 24, dtype=t)
    w2 = randn(2, 40, 24, dtype=t)
    ft.gated_unit(o, e, w, w2)
    dw, dw2 = torch.ones_like(w), torch.ones_like(w)
    db, db2 = torch.ones(40, dtype=t, device="cuda"), torch.ones(40, dtype=t, device="cuda")
    ft.gated_unit_backward(o, e, w, w2, dw_gate=dw, dw_up=dw2, db_gate=db, db_up=db2)
    for v in (dw, dw2, db, db2):
        assert (v == 0).all()
    ft.gated_unit_backward(o, e, w, w2, dx=e)


def test_gated_unit_padding_stays_out_of_the_sums(ft):
    """A bias that is not finite makes the outputs of its own column what the formula says; the rows
    that pad the last tile add nothing to the bias gradients."""
    for t in (torch.bfloat16, torch.float32):
        x, wg, wu = randn(1, 70, 32, dtype=t), randn(2, 40, 32, dtype=t), randn(3, 40, 32, dtype=t)
        bg, bu = torch.zeros(40, dtype=t, device="cuda"), torch.zeros(40, dtype=t, device="cuda")
        bg[7] = float("inf")  # sigmoid 1, slope 0
        dy = randn(4, 70, 40, dtype=t)
        ws = torch.empty(ft.gated_unit_workspace(70, 32, 40, t, backward=True), dtype=torch.uint8,
                         device="cuda")
        out = torch.empty_like(dy)
        ft.gated_unit(out, x, wg, wu, bg, bu, activation="sigmoid", workspace=ws)
        dbg, dbu = torch.empty_like(bg), torch.empty_like(bu)
        ft.gated_unit_backward(dy, x, wg, wu, bg, bu, db_gate=dbg, db_up=dbu, activation="sigmoid",
                               workspace=ws)
        assert torch.isfinite(out).all() and torch.isfinite(dbu).all() and dbg[7] == 0


def test_non_finite_rows_stay_their_own(ft):
    """A row with NaN or infinity leaves every other row's results as they were."""
    for t in (torch.bfloat16, torch.float32):
        x, wg, wu = randn(1, 300, 64, dtype=t), randn(2, 48, 64, dtype=t), randn(3, 48, 64, dtype=t)
        ws = torch.empty(ft.gated_unit_workspace(300, 64, 48, t), dtype=torch.uint8, device="cuda")
        a, b = (torch.empty((300, 48), dtype=t, device="cuda") for _ in range(2))
        ft.gated_unit(a, x, wg, wu, workspace=ws)
        na, nb = torch.empty_like(x), torch.empty_like(x)
        ft.layer_norm(na, x)
        x[17, 3], x[130, 63] = float("nan"), float("inf")
        ft.gated_unit(b, x, wg, wu, workspace=ws)
        ft.layer_norm(nb, x)
        rest = torch.ones(300, dtype=torch.bool, device="cuda")
        rest[17] = rest[130] = False
        assert torch.equal(a[rest], b[rest]) and torch.equal(na[rest], nb[rest])
        assert not torch.isfinite(b[17]).any() and not torch.isfinite(nb[17]).any()


def test_gated_unit_gradient_against_differences(ft):
    """Central differences of the fp64 formula confirm the formula's own gradient, and the kernel's
    float32 gradient follows it to the differences' error (h^2 terms ~1e-6, and 2^-24 / h)."""
    rows, inner, outer = 20, 12, 10
    x, wg, wu = (randn(s, *sh, scale=0.5) for s, sh in ((1, (rows, inner)), (2, (outer, inner)),
                                                        (3, (outer, inner))))
    dy = randn(4, rows, outer)

    def loss(a, g, u):
        return (act_ref("silu", a @ g.T)[0] * (a @ u.T) * dy.double()).sum()

    ws = torch.empty(ft.gated_unit_workspace(rows, inner, outer, torch.float32, backward=True),
                     dtype=torch.uint8, device="cuda")
    dx, dwg, dwu = torch.empty_like(x), torch.empty_like(wg), torch.empty_like(wu)
    ft.gated_unit_backward(dy, x, wg, wu, dx=dx, dw_gate=dwg, dw_up=dwu, workspace=ws)
    h = 1e-4
    args = [x.double(), wg.double(), wu.double()]
    for which, got in enumerate((dx, dwg, dwu)):
        for i, j in [(0, 0), (3, 7), (9, 11), (5, 2)]:
            hi, lo = [v.clone() for v in args], [v.clone() for v in args]
            hi[which][i, j] += h
            lo[which][i, j] -= h
            diff = (loss(*hi) - loss(*lo)) / (2 * h)
            assert abs(diff - got[i, j].double()) < 2e-5 * (1 + abs(diff))


# -------------------------------------------------------------------- dropout
def philox_keep(count, p, seed, offset):
    """Philox4x32-10 in NumPy uint64 (block e // 4, word e % 4)."""
    lo = np.uint64(0xFFFFFFFF)
    s32 = np.uint64(32)
    blk = np.arange((count + 3) // 4, dtype=np.uint64)
    c = [blk & lo, blk >> s32, np.full_like(blk, offset & 0xFFFFFFFF), np.full_like(blk, offset >> 32)]
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(10):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> s32) ^ c[1] ^ np.uint64(k0), p1 & lo, (p0 >> s32) ^ c[3] ^ np.uint64(k1), p0 & lo]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    words = np.stack(c, 1).reshape(-1)[:count]
    return words, words >= np.uint64(math.floor(p * 2 ** 32))


def test_philox_known_answers():
    """Published test vectors of Philox4x32-10 (counter and key all zeros, all ones)."""
    w, _ = philox_keep(4, 0.0, 0, 0)
    assert [int(v) for v in w] == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 5), (1, 4096), (70, 64), (13, 17), (33, 4), (5, 1003)])
@pytest.mark.parametrize("residual", [False, True])
def test_dropout(ft, rows, cols, dtype, residual):
    t = DT[dtype]
    p, seed, offset = 0.3, 0x1234_5678_9ABC_DEF0, 0xFEDC_BA98_7654_3210
    x = randn(21, rows, cols, dtype=t)
    res = randn(22, rows, cols, dtype=t) if residual else None
    _, keep = philox_keep(rows * cols, p, seed, offset)
    keep = torch.from_numpy(keep.reshape(rows, cols)).cuda()
    if rows * cols > 4000:
        assert abs(keep.double().mean().item() - 0.7) < 5 * math.sqrt(0.21 / (rows * cols))
    kept = torch.where(keep, x.double() / (1 - p), 0.0)
    ref = kept + res.double() if residual else kept
    bound = 3 * E24 * (kept.abs() + ref.abs())
    bound = bound + half_step(t) * (ref.abs() + bound)
    for pad, off in [(0, 0), (8, 0), (3, 0), (0, 1)]:
        xs = strided(x, pad, off)
        rs = strided(res, pad, off) if residual else None
        out = strided(torch.zeros_like(x), pad, off)
        ft.dropout(out, xs, p, seed, offset=offset, residual=rs)
        check(out, ref, bound)
        if not residual:
            assert torch.equal(out != 0, keep & (x != 0))
            dx = torch.empty_like(x)
            ft.dropout_backward(dx, xs, p, seed, offset=offset)  # the same mask
            assert torch.equal(dx, out)
        ft.dropout(xs, xs, p, seed, offset=offset, residual=rs)  # in place
        assert torch.equal(xs, out)


def test_dropout_edges(ft):
    x = randn(23, 40, 24)
    x[3, 5], x[7, 1] = float("nan"), float("inf")
    y = torch.empty_like(x)
    ft.dropout(y, x, 0.0, 5)
    assert torch.equal(torch.nan_to_num(y), torch.nan_to_num(x))  # p = 0 keeps everything
    _, keep = philox_keep(x.numel(), 0.5, 2 ** 64 - 1, 0)
    keep = torch.from_numpy(keep.reshape(x.shape)).cuda()
    ft.dropout(y, x, 0.5, 2 ** 64 - 1)
    assert (y[~keep] == 0).all()  # dropped elements are 0 whatever they held
    e = torch.empty((0, 24), device="cuda")
    ft.dropout(e, e, 0.5, 1)
    # Element indices beyond 2^32 / 4 blocks reach the counter's second word through the offset form:
    # one row of a very long strided block keeps its own indices.
    ft.dropout(y, x, 1.0 - 2.0 ** -40, 9)
    assert (torch.nan_to_num(y) == 0).sum() >= x.numel() - 1


# -------------------------------------------------------------- input gradient
def kernel_cases():
    from mojogp_b200 import kernel as k
    return {
        "rbf": k.RBF(), "rbf_ard": k.RBF(ard=True), "m12": k.Matern12(), "m12_ard": k.Matern12(ard=True),
        "m32": k.Matern32(ard=True), "m52": k.Matern52(), "rq": k.RQ(), "rq_ard": k.RQ(ard=True),
        "scaled": 2.0 * k.Matern52(ard=True), "dims": k.RBF(active_dims=[1]),
        "sum": k.RBF() + k.Linear(), "prod": k.Periodic() * k.Matern32(ard=True),
        "poly": k.Polynomial() + k.Matern12(), "nested": 0.5 * (k.RBF() * k.RQ()) + k.Periodic(ard=True),
    }


def bilinear64(spec, params, X, a, b):
    from oracle import kernels as ok
    K = ok.kernel_matrix(spec, params, X)
    return sum(a[c] @ K @ b[c] for c in range(a.shape[0]))


@pytest.mark.parametrize("name", sorted(kernel_cases()))
@pytest.mark.parametrize("n,d,t", [(1, 2, 1), (37, 3, 2), (300, 2, 5), (129, 5, 16), (90, 2, 19)])
def test_input_gradient_against_differences(gpb_lib, name, n, d, t):
    """Central differences of the float64 oracle's bilinear form: their error is h^2 and
    2^-53 / h of the form's magnitude, below 1e-6 of the gradient's scale at h = 1e-5; the kernel's
    float32 sums add at most (n / 8 + 60) 2^-23 of the sum of magnitudes."""
    from mojogp_b200.kernel import make_ard_kernel
    from mojogp_b200.provider import DeviceBuffer, Provider
    rng = np.random.default_rng(n * 31 + d)
    k = kernel_cases()[name].resolve_ard(d)
    X = rng.uniform(-1, 1, (n, d)).astype(np.float32)
    params = k.get_initial_params().astype(np.float32)
    params = np.where(params == np.round(params), params, params * rng.uniform(0.8, 1.2, params.shape))
    params = params.astype(np.float32)
    a, b = rng.standard_normal((t, n)).astype(np.float32), rng.standard_normal((t, n)).astype(np.float32)
    prov = Provider(X, k, params, 0.1)
    out = DeviceBuffer((n, d))
    prov.input_gradient(out, DeviceBuffer.from_host(a), DeviceBuffer.from_host(b), t)
    prov.synchronize()
    got = out.download()
    X64, a64, b64 = X.astype(np.float64), a.astype(np.float64), b.astype(np.float64)
    spec = k.to_spec(d)
    h = 1e-5
    mag = (np.abs(a64).T @ np.abs(b64) + np.abs(b64).T @ np.abs(a64)).sum(1)
    for i in sorted({0, n // 2, n - 1}):
        for q in range(d):
            hi, lo = X64.copy(), X64.copy()
            hi[i, q] += h
            lo[i, q] -= h
            diff = (bilinear64(spec, params, hi, a64, b64) - bilinear64(spec, params, lo, a64, b64)) / (2 * h)
            assert abs(got[i, q] - diff) < 4e-5 * (mag[i] + 1), (i, q, got[i, q], diff)


@pytest.mark.parametrize("leaf", ["rbf", "m12", "m32", "m52", "rq"])
@pytest.mark.parametrize("n,d,t,ard", [(1, 1, 1, False), (2, 1, 4, False), (500, 1, 11, False),
                                       (777, 8, 16, True), (600, 17, 3, True), (300, 33, 16, True),
                                       (300, 64, 7, False), (257, 12, 20, True)])
def test_input_gradient_formula(gpb_lib, leaf, n, d, t, ard):
    from mojogp_b200 import kernel as km
    from mojogp_b200.provider import Provider
    cls = {"rbf": km.RBF, "m12": km.Matern12, "m32": km.Matern32, "m52": km.Matern52, "rq": km.RQ}[leaf]
    k = (cls(ard=True) if ard else cls()).resolve_ard(d)
    rng = np.random.default_rng(5)
    nl = d if ard else 1
    ls = rng.uniform(0.5, 2.0, nl).astype(np.float32)
    tail = [0.8, 1.3] if leaf == "rq" else [1.3]
    params = np.concatenate([ls, tail]).astype(np.float32)
    x = torch.rand((n, d), generator=torch.Generator().manual_seed(1)) * 2 - 1
    if n > 2:
        x[1] = x[0]  # a repeated point contributes nothing, and no NaN
    a, b = randn(2, t, n), randn(3, t, n)
    prov = Provider(x.numpy(), k, params, 0.1)
    out = torch.empty((n, d), device="cuda")
    prov.input_gradient(out, a, b, t, stream=torch.cuda.current_stream().cuda_stream)
    X, A, B = x.double().cuda(), a.double(), b.double()
    L = torch.from_numpy(ls).double().cuda()
    diff = (X[:, None] - X[None]) / L
    s = (diff ** 2).sum(2)
    r = torch.sqrt(s.clamp(min=1e-20))
    os_ = float(params[-1])
    if leaf == "rbf":
        psi = torch.exp(-s / 2)
    elif leaf == "m12":
        psi = torch.exp(torch.clamp(-r, min=-20) if ard else -r) / r
    elif leaf == "m32":
        psi = 3 * torch.exp(torch.clamp(-math.sqrt(3) * r, min=-20))
    elif leaf == "m52":
        psi = 5 / 3 * (1 + math.sqrt(5) * r) * torch.exp(torch.clamp(-math.sqrt(5) * r, min=-20))
    else:
        al = float(params[-2])
        psi = (1 + s / (2 * al)) ** (-al - 1)
    w = (A.T @ B + B.T @ A) * psi * os_
    ref = -(w[:, :, None] * diff).sum(1) / L
    mag = ((A.abs().T @ B.abs() + B.abs().T @ A.abs()) * psi * os_ * (1 + s + r))[:, :, None]
    bound = (mag * diff.abs()).sum(1) / L * (n / 8 + 4 * t + d + 60) * E23
    check(out, ref, bound)
    again = torch.empty_like(out)
    prov.input_gradient(again, a, b, t, stream=torch.cuda.current_stream().cuda_stream)
    assert torch.equal(out, again)


# -------------------------------------------------- streams, graphs, two calls
def test_operators_on_another_stream_and_in_a_graph(ft):
    t = torch.bfloat16
    rows, inner, outer = 200, 64, 96
    x, w, b = randn(1, rows, inner, dtype=t), randn(2, inner), randn(3, inner)
    wg, wu = randn(4, outer, inner, dtype=t, scale=0.1), randn(5, outer, inner, dtype=t, scale=0.1)

    def layer(stream, bufs):
        norm, mid, out, dmid, dnorm, dx, dwg, dwu, mean, rstd, ws, ws2, dw = bufs
        ft.layer_norm(norm, x, w, b, mean=mean, rstd=rstd, stream=stream)
        ft.gated_unit(mid, norm, wg, wu, workspace=ws, stream=stream)
        ft.dropout(out, mid, 0.1, 7, stream=stream)
        ft.dropout_backward(dmid, out, 0.1, 7, stream=stream)
        ft.gated_unit_backward(dmid, norm, wg, wu, dx=dnorm, dw_gate=dwg, dw_up=dwu, workspace=ws,
                               stream=stream)
        ft.layer_norm_backward(dx, dnorm, x, mean, rstd, w, dweight=dw, workspace=ws2, stream=stream)

    def buffers():
        e = lambda *s, dtype=t: torch.zeros(s, dtype=dtype, device="cuda")
        ws = max(ft.gated_unit_workspace(rows, inner, outer, t, backward=True),
                 ft.gated_unit_workspace(rows, inner, outer, t))
        return (e(rows, inner), e(rows, outer), e(rows, outer), e(rows, outer), e(rows, inner),
                e(rows, inner), e(outer, inner), e(outer, inner), e(rows, dtype=torch.float32),
                e(rows, dtype=torch.float32), e(ws, dtype=torch.uint8),
                e(ft.layer_norm_workspace(rows, inner), dtype=torch.uint8),
                e(inner, dtype=torch.float32))

    want = buffers()
    layer(None, want)
    torch.cuda.synchronize()
    outs = [0, 1, 2, 3, 4, 5, 6, 7, 12]
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    b1, b2 = buffers(), buffers()
    torch.cuda.synchronize()
    for _ in range(5):  # two calls at once, each with its own workspace
        layer(one.cuda_stream, b1)
        layer(two.cuda_stream, b2)
    torch.cuda.synchronize()
    for got in (b1, b2):
        for i in outs:
            assert torch.equal(got[i], want[i]), i
    b3 = buffers()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        layer(torch.cuda.current_stream().cuda_stream, b3)
    for i in outs:
        b3[i].zero_()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    for i in outs:
        assert torch.equal(b3[i], want[i]), i


def test_device_buffers(ft):
    """The operators on provider.DeviceBuffer arrays, without tensors."""
    from mojogp_b200.provider import DeviceBuffer
    rng = np.random.default_rng(0)
    x = rng.standard_normal((50, 20)).astype(np.float32)
    xd, out = DeviceBuffer.from_host(x), DeviceBuffer((50, 20))
    ft.layer_norm(out, xd, eps=1e-5)
    ref = (x - x.mean(1, keepdims=True)) / np.sqrt(x.var(1, keepdims=True) + 1e-5)
    np.testing.assert_allclose(out.download(), ref, rtol=1e-4, atol=1e-5)
    h = DeviceBuffer.from_host(x.astype(np.float16))
    o = DeviceBuffer((50, 20), dtype=np.float16)
    ft.dropout(o, h, 0.0, 1)
    assert np.array_equal(o.download(), x.astype(np.float16))
