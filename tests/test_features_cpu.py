"""Refusals of the feature-map operators: every argument error is raised before any device work, so
they are tested without a GPU, on arrays that only look like device arrays."""
import ctypes as C

import numpy as np
import pytest

from mojogp_b200 import _lib


class FakeDevice:
    def __init__(self, index=0, kind="cuda"):
        self.index, self.type = index, kind

    def __repr__(self):
        return f"{self.type}:{self.index}"


class FakeArray:
    """Shape, strides, type, device and address of a device array; nothing behind it."""

    def __init__(self, shape, dtype="float32", ptr=1 << 20, strides=None, device=0, kind="cuda"):
        self.shape = tuple(shape)
        self.dtype = np.dtype(dtype) if dtype != "bfloat16" else "torch.bfloat16"
        self._ptr = ptr
        self._strides = strides
        self.device = FakeDevice(device, kind)

    def data_ptr(self):
        return self._ptr

    def stride(self):
        if self._strides is not None:
            return self._strides
        out, step = [], 1
        for s in reversed(self.shape):
            out.append(step)
            step *= s
        return tuple(reversed(out))

    def is_contiguous(self):
        return self._strides is None

    def numel(self):
        return int(np.prod(self.shape, dtype=np.int64))

    def element_size(self):
        return 2 if self.dtype == "torch.bfloat16" else self.dtype.itemsize


MB = 1 << 20


def arr(shape, i=1, **kw):
    return FakeArray(shape, ptr=i * 64 * MB, **kw)


@pytest.fixture()
def ft(gpb_lib):
    from mojogp_b200 import features
    return features


def refuse(match, fn, *a, **kw):
    with pytest.raises(ValueError, match=match):
        fn(*a, **kw)


def test_layer_norm_refusals(ft):
    x, y, v = arr((4, 8)), arr((4, 8), 2), arr((8,), 3)
    refuse("2-D", ft.layer_norm, y, arr((4, 8, 2)))
    refuse("shape", ft.layer_norm, arr((4, 9), 2), x)
    refuse("element type", ft.layer_norm, arr((4, 8), 2, dtype="float16"), x)
    refuse("element type", ft.layer_norm, y, arr((4, 8), dtype="float64"))
    refuse("CUDA device", ft.layer_norm, y, arr((4, 8), kind="cpu"))
    refuse("on device 1", ft.layer_norm, arr((4, 8), 2, device=1), x)
    refuse("unit column stride", ft.layer_norm, y, arr((4, 8), strides=(1, 4)))
    refuse("leading dimension", ft.layer_norm, y, arr((4, 8), strides=(0, 1)))  # broadcast rows
    refuse("entries", ft.layer_norm, y, x, arr((9,), 3))
    refuse("float32 or of x", ft.layer_norm, y, x, arr((8,), 3, dtype="float16"))
    refuse("different element type", ft.layer_norm, arr((4, 8), 2, dtype="float16"),
           arr((4, 8), dtype="float16"), v, arr((8,), 4, dtype="float16"))
    refuse("different element type", ft.layer_norm, y, x, mean=arr((4,), 4, dtype="float16"))
    refuse("eps", ft.layer_norm, y, x, eps=-1.0)
    refuse("eps", ft.layer_norm, y, x, eps=float("nan"))
    refuse("aligned", ft.layer_norm, y, FakeArray((4, 8), ptr=MB + 2))
    refuse("overlaps", ft.layer_norm, FakeArray((4, 8), ptr=MB + 32), FakeArray((4, 8), ptr=MB))
    refuse("device array", ft.layer_norm, y, np.zeros((4, 8), np.float32))
    refuse("columns", ft.layer_norm, arr((4, 0), 2), arr((4, 0)))
    refuse("mean or rstd overlaps", ft.layer_norm, y, x, mean=FakeArray((4,), ptr=y.data_ptr()))
    refuse("overlap", ft.layer_norm, y, x, mean=arr((4,), 9), rstd=arr((4,), 9))
    refuse("weight or bias", ft.layer_norm, y, x, FakeArray((8,), ptr=y.data_ptr()))
    m, r = arr((4,), 5), arr((4,), 6)
    d, dx = arr((4, 8), 7), arr((4, 8), 8)
    refuse("no output", ft.layer_norm_backward, None, d, x, m, r)
    refuse("workspace", ft.layer_norm_backward, dx, d, x, m, r, v, dweight=arr((8,), 9))
    refuse("workspace", ft.layer_norm_backward, dx, d, x, m, r, v, dweight=arr((8,), 9),
           workspace=arr((16,), 10, dtype="uint8"))
    ws = arr((1 << 20,), 10, dtype="uint8")
    refuse("two outputs", ft.layer_norm_backward, dx, d, x, m, r, v, dweight=arr((8,), 9),
           dbias=arr((8,), 9), workspace=ws)
    refuse("overlaps an input", ft.layer_norm_backward, dx, d, x, m, r, v, dweight=v, workspace=ws)
    refuse("overlaps", ft.layer_norm_backward, FakeArray((4, 8), ptr=MB + 32),
           FakeArray((4, 8), ptr=MB), x, m, r)


def test_gated_unit_refusals(ft):
    x, w, u, y = arr((4, 8)), arr((6, 8), 2), arr((6, 8), 3), arr((4, 6), 4)
    refuse("activation", ft.gated_unit, y, x, w, u, activation="step")
    refuse("activation", ft.gated_unit, y, x, w, u, activation=3)
    refuse("shape", ft.gated_unit, y, x, arr((6, 9), 2), u)
    refuse("shape", ft.gated_unit, y, x, w, arr((5, 8), 3))
    refuse("shape", ft.gated_unit, arr((4, 7), 4), x, w, u)
    refuse("element type", ft.gated_unit, y, x, arr((6, 8), 2, dtype="float16"), u)
    refuse("one row stride", ft.gated_unit, y, x, w, arr((6, 8), 3, strides=(16, 1)))
    refuse("entries", ft.gated_unit, y, x, w, u, arr((7,), 5))
    refuse("overlaps", ft.gated_unit, FakeArray((4, 6), ptr=x.data_ptr() + 16), x, w, u)
    refuse("inner", ft.gated_unit, arr((4, 6), 4), arr((4, 0)), arr((6, 0), 2), arr((6, 0), 3))
    big = arr((64, 8))
    refuse("workspace", ft.gated_unit, arr((64, 6), 4), big, w, u)
    refuse("workspace", ft.gated_unit, arr((64, 6), 4), big, w, u,
           workspace=arr((16,), 5, dtype="uint8"))
    need = ft.gated_unit_workspace(64, 8, 6, "float32")
    refuse("aligned", ft.gated_unit, arr((64, 6), 4), big, w, u,
           workspace=FakeArray((need + 8,), dtype="uint8", ptr=8 + 512 * MB))
    refuse("workspace overlaps", ft.gated_unit, arr((64, 6), 4), big, w, u,
           workspace=FakeArray((need,), dtype="uint8", ptr=big.data_ptr()))
    dy = arr((4, 6), 6)
    ws = arr((1 << 20,), 7, dtype="uint8")
    refuse("no output", ft.gated_unit_backward, dy, x, w, u, workspace=ws)
    refuse("workspace", ft.gated_unit_backward, dy, x, w, u, dx=arr((4, 8), 8))
    refuse("shape", ft.gated_unit_backward, dy, x, w, u, dx=arr((4, 9), 8), workspace=ws)
    refuse("overlap", ft.gated_unit_backward, dy, x, w, u, dx=x, workspace=ws)
    refuse("two outputs", ft.gated_unit_backward, dy, x, w, u, dw_gate=arr((6, 8), 9),
           dw_up=arr((6, 8), 9), workspace=ws)
    refuse("one row stride", ft.gated_unit_backward, dy, x, w, u, dw_gate=arr((6, 8), 9),
           dw_up=arr((6, 8), 10, strides=(9, 1)), workspace=ws)


def test_dropout_refusals(ft):
    x, y = arr((4, 8)), arr((4, 8), 2)
    for p in (-0.1, 1.0, 2.0, float("nan")):
        refuse("probability", ft.dropout, y, x, p, 1)
    refuse("seed", ft.dropout, y, x, 0.5, -1)
    refuse("offset", ft.dropout, y, x, 0.5, 1, offset=1 << 64)
    refuse("shape", ft.dropout, arr((4, 7), 2), x, 0.5, 1)
    refuse("residual", ft.dropout, y, x, 0.5, 1, residual=arr((5, 8), 3))
    refuse("overlaps", ft.dropout, FakeArray((4, 8), ptr=x.data_ptr() + 4), x, 0.5, 1)
    refuse("overlaps residual", ft.dropout, y, x, 0.5, 1,
           residual=FakeArray((4, 8), ptr=y.data_ptr() + 4))


def test_c_entry_refusals(gpb_lib):
    """The C entries' own checks of what the Python layer cannot pass."""
    p = C.c_void_p(1 << 20)
    q = C.c_void_p(1 << 24)
    bad = _lib.ERR_INVALID
    assert gpb_lib.gpb_layer_norm(0, None, 9, 9, 1, 8, p, 8, q, 8, None, None, 1e-5, None, None) == bad
    assert gpb_lib.gpb_layer_norm(0, None, 0, 0, 1, 8, None, 8, q, 8, None, None, 1e-5, None, None) == bad
    assert gpb_lib.gpb_layer_norm(0, None, 0, 1, 1, 8, p, 8, q, 8, None, None, 1e-5, None, None) == bad
    assert gpb_lib.gpb_layer_norm(0, None, 0, 0, -1, 8, p, 8, q, 8, None, None, 1e-5, None, None) == bad
    assert gpb_lib.gpb_layer_norm_workspace(1, 0, None) == bad
    assert gpb_lib.gpb_dropout(0, None, 7, 1, 1, p, 1, q, 1, None, 0, 0.5, 1, 0) == bad
    assert gpb_lib.gpb_dropout(0, None, 0, 1 << 30, 1 << 30, p, 1 << 30, q, 1 << 30, None, 0, 0.5, 1,
                               0) == bad
    assert gpb_lib.gpb_gated_unit(0, None, 0, 7, 1, 8, 8, p, 8, q, 8, p, q, 8, None, None, None, 0) == bad
    n = C.c_int64()
    assert gpb_lib.gpb_gated_unit_workspace(0, 1 << 40, 8, 8, 0, C.byref(n)) == bad
    assert gpb_lib.gpb_gated_unit_workspace(0, 8, 1 << 30, 8, 0, C.byref(n)) == bad
    assert gpb_lib.gpb_input_gradient(None, p, q, q, 1, None) == bad
    assert gpb_lib.gpb_feature_status(0, None) == bad


def test_workspace_sizes_follow_the_sizes_alone(gpb_lib):
    from mojogp_b200 import features as ft
    assert ft.layer_norm_workspace(0, 8) > 0
    assert ft.layer_norm_workspace(100, 64) == ft.layer_norm_workspace(100, 64)
    assert ft.gated_unit_workspace(1, 64, 64, "bfloat16") == 0
    assert ft.gated_unit_workspace(100, 64, 64, "bfloat16", backward=True) >= 2 * 100 * 64 * 2
    # float32 weights are three 16-bit planes; x has room for an aligned copy
    assert ft.gated_unit_workspace(100, 64, 64, "float32") >= 3 * 2 * 2 * 64 * 64 + 4 * 100 * 64


def test_feature_map_refusals_and_shapes():
    from mojogp_b200 import FeatureMap, RBF, SingleOutputGP
    for kw, match in [(dict(widths=[]), "widths"), (dict(widths=[0]), "widths"),
                      (dict(widths=[65]), "at most 64"), (dict(widths=[4], activation="x"), "activation"),
                      (dict(widths=[4], dropout=1.0), "dropout"), (dict(widths=[4], dtype="f64"), "dtype"),
                      (dict(widths=[4], seed=-1), "seed")]:
        refuse(match, FeatureMap, **kw)
    fm = FeatureMap([100, 8])
    refuse("at least one", fm.build, 0)
    fm.build(30)
    assert [p.shape for p in fm.parameters] == [(30,), (30,), (100, 30), (100, 30), (100,), (100,),
                                               (100,), (100,), (8, 100), (8, 100), (8,), (8,)]
    refuse("built for 30", fm.build, 31)
    same = FeatureMap.from_config(fm.config(), fm.parameters)
    assert all(np.array_equal(a, b) for a, b in zip(same.parameters, fm.parameters))
    refuse("do not match", FeatureMap.from_config, fm.config(), fm.parameters[:-1])
    with pytest.raises(TypeError, match="FeatureMap"):
        SingleOutputGP(RBF(), feature_map="wide")
    X, y = np.zeros((4, 30), np.float32), np.zeros(4, np.float32)
    refuse("needs a feature_map", SingleOutputGP(RBF()).fit, X, y, feature_learning_rate=0.1)
    refuse("feature_learning_rate", SingleOutputGP(RBF(), feature_map=fm).fit, X, y,
           feature_learning_rate=0.0)
    with pytest.raises(NotImplementedError, match="one GPU"):
        SingleOutputGP(RBF(), feature_map=fm).fit(X, y, comm=object())
    refuse("built for 30", SingleOutputGP(RBF(), feature_map=fm).fit, X[:, :20], y)
    refuse("2D", fm.upload, np.zeros(30, np.float32))


def test_bfloat16_rounding():
    from mojogp_b200.feature_map import _to_bfloat16_bits
    a = np.array([1.0, 1.00390625, 1.01171875, -3.4e38, np.inf, np.nan], np.float32)
    bits = _to_bfloat16_bits(a)
    assert list(bits[:3]) == [0x3F80, 0x3F80, 0x3F82]  # ties to even
    assert bits[3] == 0xFF80 and bits[4] == 0x7F80 and (bits[5] & 0x7FFF) > 0x7F80


def test_cast_and_provider_refusals(ft):
    refuse("shape", ft.cast, arr((4, 7), 2, dtype="float16"), arr((4, 8)))
    refuse("not one of", ft.cast, arr((4, 8), 2, dtype="int32"), arr((4, 8)))
    refuse("on device 1", ft.cast, arr((4, 8), 2, dtype="float16", device=1), arr((4, 8)))
    p, q = C.c_void_p(1 << 20), C.c_void_p(1 << 24)
    lib = _lib.lib()
    assert lib.gpb_cast(0, None, 5, 0, 1, 1, p, 1, q, 1) == _lib.ERR_INVALID
    assert lib.gpb_set_inputs(None, p, None) == _lib.ERR_INVALID
    z = C.c_double()
    assert lib.gpb_bbmm_inputs(None, p, 1, 1, 1, 1, 0.1, 0, 0, C.byref(z), C.byref(z), C.byref(z),
                               None, p) == _lib.ERR_INVALID
