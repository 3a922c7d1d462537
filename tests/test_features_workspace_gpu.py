"""Where arguments may lie: the gated unit's workspace at every alignment that it may have, with guards on
both sides, and blocks that are column ranges of one matrix."""
import pytest

from test_features_gpu import DT, randn

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ft(gpb_lib):
    from mojogp_b200 import features
    yield features
    features.check_device(0)


# CUDA-core rows, split projections and dx, split weight gradients, plain tiles, CTA pairs.
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,inner,outer", [(2, 520, 520), (20, 4104, 72), (100, 136, 64), (3000, 40, 33),
                                              (300, 517, 300), (2660, 1800, 1000)])
def test_gated_unit_workspace_alignment(ft, rows, inner, outer, dtype):
    t = DT[dtype]
    x, dy = randn(1, rows, inner, dtype=t), randn(2, rows, outer, dtype=t)
    wg, wu = (randn(s, outer, inner, dtype=t, scale=inner ** -0.5) for s in (3, 4))
    bg, bu = randn(5, outer, dtype=t), randn(6, outer, dtype=t)
    forward = ft.gated_unit_workspace(rows, inner, outer, t)
    backward = ft.gated_unit_workspace(rows, inner, outer, t, backward=True)
    block = torch.empty(max(forward, backward) + 512, dtype=torch.uint8, device="cuda")
    want = None
    for off in (0, 16, 32, 48, 240):
        got = [torch.zeros_like(v) for v in (dy, x, wg, wu, bg, bu)]
        for need, call in ((forward, lambda ws: ft.gated_unit(got[0], x, wg, wu, bg, bu, workspace=ws)),
                           (backward, lambda ws: ft.gated_unit_backward(
                               dy, x, wg, wu, bg, bu, dx=got[1], dw_gate=got[2], dw_up=got[3],
                               db_gate=got[4], db_up=got[5], workspace=ws))):
            block.fill_(0xA5)
            call(block[off:off + need] if need else None)
            assert (block[:off] == 0xA5).all() and (block[off + need:] == 0xA5).all()
        if want is None:
            want = got
        for g, w in zip(got, want):
            assert torch.isfinite(g).all() and torch.equal(g, w), off


# Column widths whose rows are 16-byte aligned (64, 256) or not (33, 777), in few and many rows.
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("rows,cols", [(40, 64), (700, 256), (40, 33), (900, 777)])
def test_column_ranges_of_one_matrix(ft, rows, cols, dtype):
    """Inputs and outputs side by side in one matrix: the same results as in matrices of their own."""
    t = DT[dtype]

    def apart(*shapes):
        return [torch.full(s, 7.0, dtype=t, device="cuda") for s in shapes]

    def beside(*shapes):
        big = torch.full((shapes[0][0], sum(s[1] for s in shapes)), 7.0, dtype=t, device="cuda")
        return list(big.split([s[1] for s in shapes], 1))

    n, tall = (rows, cols), (48, cols)
    w, b = randn(1, cols), randn(2, cols)
    X, D, G, U = (randn(s, *k, dtype=t) for s, k in ((3, n), (4, n), (5, tall), (6, tall)))
    D2 = randn(7, rows, 48, dtype=t)
    results = []
    for layout in (apart, beside):
        x, norm, dy, dx, drop = layout(n, n, n, n, n)
        dwg, dwu, wg, wu = layout(tall, tall, tall, tall)
        x2, out, dout, dx2 = layout(n, (rows, 48), (rows, 48), n)
        for v, k in ((x, X), (dy, D), (wg, G / 8), (wu, U / 8), (x2, X), (dout, D2)):
            v.copy_(k)
        mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
        ws = torch.empty(max(ft.gated_unit_workspace(rows, cols, 48, t, backward=True),
                             ft.gated_unit_workspace(rows, cols, 48, t), 16), dtype=torch.uint8, device="cuda")
        ws2 = torch.empty(ft.layer_norm_workspace(rows, cols), dtype=torch.uint8, device="cuda")
        dw = torch.empty_like(w)
        ft.layer_norm(norm, x, w, b, mean=mean, rstd=rstd)
        ft.layer_norm_backward(dx, dy, x, mean, rstd, w, dweight=dw, workspace=ws2)
        ft.dropout(drop, dy, 0.3, 11, residual=norm)
        ft.gated_unit(out, x2, wg, wu, workspace=ws)
        ft.gated_unit_backward(dout, x2, wg, wu, dx=dx2, dw_gate=dwg, dw_up=dwu, workspace=ws)
        assert torch.equal(x, X) and torch.equal(dy, D) and torch.equal(x2, X) and torch.equal(dout, D2)
        results.append([norm, dx, dw, drop, out, dx2, dwg, dwu])
    # Other alignments sum in another order: equal up to a rounding of the type (test_features_gpu).
    step = torch.finfo(t).eps
    for a, c in zip(*results):
        torch.testing.assert_close(a, c, rtol=step + 1e-5, atol=(step + 1e-5) * max(1.0, a.abs().max().item() / 8))
