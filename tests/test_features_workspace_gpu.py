"""The gated unit's workspace at every alignment that it may have, with guards on both sides."""
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
