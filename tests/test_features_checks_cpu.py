"""Argument checks and size queries of the feature-map operators, without a GPU."""
import pytest

from mojogp_b200 import _lib
from test_features_cpu import MB, FakeArray, arr, refuse


@pytest.fixture()
def ft(gpb_lib):
    from mojogp_b200 import features
    return features


def no_device(fn, *a, **kw):
    """The call passes its checks: it ends where it looks for its device (64, which no machine here has)."""
    with pytest.raises(_lib.GPBError) as e:
        fn(*a, **kw)
    assert not isinstance(e.value, ValueError) and "device 64" in str(e.value)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("rows,inner,outer", [(1, 64, 48), (4, 600, 500), (16, 4104, 72), (100, 64, 64),
                                              (300, 517, 33), (3000, 1024, 2048)])
@pytest.mark.parametrize("backward", [False, True])
def test_gated_workspace_base_is_rounded_up(gpb_lib, rows, inner, outer, dtype, backward):
    """The kernels store 32-byte sectors into the workspace, whose base need only be 16-byte aligned: the
    parts, 256-byte multiples from the rounded base, still end inside the size asked for."""
    from mojogp_b200 import features as ft
    need = ft.gated_unit_workspace(rows, inner, outer, dtype, backward=backward)
    if need == 0:
        assert not backward and rows <= 8  # the CUDA cores' forward pass has none
        return
    parts = need // 256 * 256
    for base in (1 << 20, (1 << 20) + 16, (1 << 20) + 32, (1 << 20) + 48):
        rounded = -(-base // 32) * 32
        assert rounded + parts <= base + need


def test_gated_workspace_of_any_allowed_alignment_is_taken(ft):
    n = dict(device=64)
    x, w, u, y = arr((64, 8), **n), arr((6, 8), 2, **n), arr((6, 8), 3, **n), arr((64, 6), 4, **n)
    need = ft.gated_unit_workspace(64, 8, 6, "float32", backward=True)
    for off in (0, 16, 32):
        ws = FakeArray((need,), dtype="uint8", ptr=512 * MB + off, **n)
        no_device(ft.gated_unit, y, x, w, u, workspace=ws)
        no_device(ft.gated_unit_backward, y, x, w, u, dx=arr((64, 8), 5, **n), workspace=ws)
    for off in (4, 8, 24):
        ws = FakeArray((need,), dtype="uint8", ptr=512 * MB + off, **n)
        refuse("aligned", ft.gated_unit_backward, y, x, w, u, dx=arr((64, 8), 5, **n), workspace=ws)
    short = FakeArray((need - 1,), dtype="uint8", ptr=512 * MB, **n)
    refuse("workspace", ft.gated_unit_backward, y, x, w, u, dx=arr((64, 8), 5, **n), workspace=short)


def test_layer_norm_backward_keeps_dx_off_its_other_inputs(ft):
    """Rows of dx are written while other rows still read weight, mean and rstd."""
    x, d, dx = arr((4, 8)), arr((4, 8), 2), arr((4, 8), 3)
    w, m, r = arr((8,), 4), arr((4,), 5), arr((4,), 6)
    inside = lambda n: FakeArray((n,), ptr=dx.data_ptr() + 64)
    refuse("dx overlaps weight", ft.layer_norm_backward, dx, d, x, m, r, inside(8))
    refuse("dx overlaps weight", ft.layer_norm_backward, dx, d, x, inside(4), r, w)
    refuse("dx overlaps weight", ft.layer_norm_backward, dx, d, x, m, inside(4))


def columns(ptr, first, count, rows=4, ld=24, **kw):
    """Columns [first, first + count) of a float32 matrix with `ld` columns."""
    return FakeArray((rows, count), ptr=ptr + 4 * first, strides=(ld, 1), device=64, **kw)


def test_column_ranges_of_one_matrix_do_not_overlap(ft):
    big, other, n = 64 * MB, 128 * MB, dict(device=64)
    m, r, v = (FakeArray((k,), ptr=i * 64 * MB, **n) for k, i in ((4, 3), (4, 4), (8, 5)))
    ws = FakeArray((1 << 20,), dtype="uint8", ptr=512 * MB, **n)
    a, b, c = (columns(big, f, 8) for f in (0, 8, 16))
    for x, y in ((a, b), (b, a), (a, c), (c, b)):
        no_device(ft.layer_norm, y, x)
        no_device(ft.dropout, y, x, 0.5, 1)
        no_device(ft.dropout, y, x, 0.5, 1, residual=y)
        no_device(ft.cast, y, x)
        no_device(ft.layer_norm_backward, y, x, columns(other, 0, 8), m, r, dweight=v, workspace=ws)
    w, u = (FakeArray((8, 8), ptr=i * 64 * MB, **n) for i in (6, 7))
    no_device(ft.gated_unit, b, a, w, u)
    no_device(ft.gated_unit_backward, b, a, w, u, dx=c, workspace=ws)
    no_device(ft.gated_unit_backward, b, a, w, u, dw_gate=columns(other, 0, 8, 8),
              dw_up=columns(other, 8, 8, 8), workspace=ws)
    # One column shared, from either side; rows that wrap around; other strides.
    for first in (1, 7, 23):
        y = columns(big, 16 + first, 8) if first == 1 else columns(big, first, 8)
        refuse("overlap", ft.layer_norm, y, columns(big, 0, 8) if first != 1 else c)
        refuse("overlap", ft.gated_unit, y, columns(big, 0, 8) if first != 1 else c, w, u)
    refuse("overlap", ft.layer_norm, columns(big, 8, 8, ld=32), a)
    refuse("overlap", ft.dropout, b, columns(other, 0, 8), 0.5, 1, residual=columns(big, 9, 8))
    refuse("two outputs", ft.gated_unit_backward, b, a, w, u, dw_gate=columns(other, 0, 8, 8),
           dw_up=columns(other, 4, 8, 8), workspace=ws)
    # A single row between two others' columns.
    no_device(ft.layer_norm, columns(big, 24 + 8, 8, rows=1), columns(big, 24 + 16, 8, rows=1))
    refuse("overlap", ft.layer_norm, columns(big, 24 + 8, 8, rows=1), columns(big, 24 + 12, 8, rows=1))
