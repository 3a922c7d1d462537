"""Operators of a learned feature map over the C ABI (layer norm, gated unit, dropout).

A GP takes at most 64 input dimensions; a feature map brings wider inputs
under it. The functions here are its operators, forward and backward, each
writing into arrays the caller passes (outputs first, as the provider's
operations do). An array is a provider.DeviceBuffer, or any device array
object with `data_ptr()`, `shape`, `stride()`, `dtype` and `device` (a CUDA
tensor, say): float32, float16 or bfloat16, two-dimensional [rows, columns]
with unit column stride and any row stride, or one-dimensional for weights,
biases and statistics.

Calls are asynchronous on `stream` (an integer CUDA stream handle; None or 0
is the legacy default stream), allocate nothing, and can be captured into a
CUDA graph; where one takes a workspace, it is any array of at least the bytes
the matching *_workspace function returns, not shared by calls that may run at
the same time. Argument errors raise ValueError before any device work.
"""
from __future__ import annotations

import ctypes as C
import functools

import numpy as np

from . import _lib

_DTYPES = {"float32": 0, "float16": 1, "bfloat16": 2}
_CODES: dict = {}
ACTIVATIONS = {"silu": 0, "gelu": 1, "sigmoid": 2, "tanh": 3}


def _dtype_code(dtype) -> int:
    """GPB_DTYPE_* of a NumPy or tensor element type, or of its name."""
    code = _CODES.get(dtype)
    if code is None:
        name = getattr(dtype, "name", None) or str(dtype).rsplit(".", 1)[-1]
        if name not in _DTYPES:
            raise ValueError(f"element type {name} is not one of {sorted(_DTYPES)}")
        code = _CODES[dtype] = _DTYPES[name]
    return code


class _View:
    """Pointer, sizes, leading dimension, element type and device of an array."""

    __slots__ = ("ptr", "shape", "ld", "code", "device")

    def __init__(self, a, name: str, ndim: int):
        self.shape = shape = a.shape
        if len(shape) != ndim:
            raise ValueError(f"{name} must be {ndim}-D, got shape {shape}")
        try:
            self.ptr = a.data_ptr()
        except AttributeError:
            if not (hasattr(a, "ptr") and hasattr(a, "nbytes")):
                raise ValueError(f"{name} must be a device array, got {type(a).__name__}") from None
            self.ptr, self.device, self.ld = a.ptr, a.device, shape[-1]
            self.code = _element_code(a)
            if self.ptr is None:
                raise ValueError(f"{name} was freed") from None
            return
        self.device = index = a.device.index
        if index is None or a.device.type != "cuda":
            raise ValueError(f"{name} must be on a CUDA device, got {a.device}")
        strides = a.stride()
        if strides[-1] != 1 and shape[-1] > 1:
            raise ValueError(f"{name} must have unit column stride, got strides {strides}")
        self.ld = strides[0] if ndim == 2 and shape[0] > 1 else shape[-1]
        dtype = a.dtype
        self.code = _CODES[dtype] if dtype in _CODES else _dtype_code(dtype)


def _element_code(a) -> int:
    return _dtype_code(getattr(a, "element_type", None) or a.dtype)


def _vector(a, name: str, size: int, like: "_View", code: int) -> int | None:
    """Pointer of a [size] vector of element type `code`, or None."""
    if a is None:
        return None
    v = _View(a, name, 1)
    if v.shape[0] != size:
        raise ValueError(f"{name} must have {size} entries, got {v.shape[0]}")
    if v.code != code:
        raise ValueError(f"{name} has a different element type")
    if v.device != like.device:
        raise ValueError(f"{name} is on device {v.device}, expected {like.device}")
    return v.ptr


def _matrix(a, name: str, shape: tuple, like: "_View") -> "_View":
    v = _View(a, name, 2)
    if v.shape != shape:
        raise ValueError(f"{name} must have shape {shape}, got {v.shape}")
    if v.code != like.code:
        raise ValueError(f"{name} has a different element type")
    if v.device != like.device:
        raise ValueError(f"{name} is on device {v.device}, expected {like.device}")
    return v


def _workspace(a, like: "_View") -> tuple:
    """(pointer, bytes) of a scratch array; the call itself checks the size."""
    if a is None:
        return None, 0
    data_ptr = getattr(a, "data_ptr", None)
    if data_ptr is not None:
        if a.device.type != "cuda":
            raise ValueError(f"workspace must be on a CUDA device, got {a.device}")
        if not a.is_contiguous():
            raise ValueError("workspace must be contiguous")
        ptr, size, device = data_ptr(), a.numel() * a.element_size(), a.device.index
    else:
        ptr, size, device = a.ptr, a.nbytes, a.device
    if device != like.device:
        raise ValueError(f"workspace is on device {device}, expected {like.device}")
    return ptr, size


def check_device(device: int = 0) -> None:
    """Wait for `device` and raise if a bounded wait inside an operator's kernel
    gave up since the last check (its outputs are then not valid)."""
    word = C.c_int32()
    _lib.call("gpb_feature_status", int(device), C.byref(word))
    if word.value:
        raise _lib.GPBError(_lib.ERR_DEVICE, f"device error word {word.value} "
                            "(bounded wait gave up in a feature-map kernel)")


# ------------------------------------------------------------- layer norm
def layer_norm(out, x, weight=None, bias=None, *, eps: float = 1e-5, mean=None, rstd=None,
               stream=None) -> None:
    """out = (x - mean) rstd weight + bias over each row of x [rows, columns].

    weight and bias [columns] are float32 or of x's type; `mean` and `rstd`
    [rows], float32, are written where given (the backward pass needs them).
    out may be x itself."""
    xv = _View(x, "x", 2)
    rows, cols = xv.shape
    ov = _matrix(out, "out", xv.shape, xv)
    pcode = xv.code
    for a in (weight, bias):
        if a is not None:
            pcode = _element_code(a)
            break
    if pcode not in (0, xv.code):
        raise ValueError("weight and bias must be float32 or of x's type")
    _lib.call("gpb_layer_norm", xv.device, stream, xv.code, pcode, rows, cols, ov.ptr, ov.ld,
              xv.ptr, xv.ld, _vector(weight, "weight", cols, xv, pcode),
              _vector(bias, "bias", cols, xv, pcode), eps,
              _vector(mean, "mean", rows, xv, 0), _vector(rstd, "rstd", rows, xv, 0))


@functools.lru_cache(maxsize=256)
def layer_norm_workspace(rows: int, cols: int) -> int:
    """Workspace bytes of layer_norm_backward with weight or bias gradients."""
    n = C.c_int64()
    _lib.call("gpb_layer_norm_workspace", rows, cols, C.byref(n))
    return n.value


def layer_norm_backward(dx, dout, x, mean, rstd, weight=None, *, dweight=None, dbias=None,
                        workspace=None, stream=None) -> None:
    """Gradients of layer_norm from dout, x and the forward pass's statistics.

    dx (None, dout or x themselves allowed), dweight and dbias are written
    where given; dweight and dbias are of weight's type (float32 or x's type
    when there is no weight) and need a workspace."""
    xv = _View(x, "x", 2)
    rows, cols = xv.shape
    dv = _matrix(dout, "dout", xv.shape, xv)
    ov = _matrix(dx, "dx", xv.shape, xv) if dx is not None else None
    pcode = xv.code
    for a in (weight, dweight, dbias):
        if a is not None:
            pcode = _element_code(a)
            break
    if pcode not in (0, xv.code):
        raise ValueError("weight and its gradient must be float32 or of x's type")
    wptr, wbytes = _workspace(workspace, xv)
    _lib.call("gpb_layer_norm_backward", xv.device, stream, xv.code, pcode, rows, cols,
              ov.ptr if ov else None, ov.ld if ov else 0, dv.ptr, dv.ld, xv.ptr, xv.ld,
              _vector(mean, "mean", rows, xv, 0), _vector(rstd, "rstd", rows, xv, 0),
              _vector(weight, "weight", cols, xv, pcode),
              _vector(dweight, "dweight", cols, xv, pcode),
              _vector(dbias, "dbias", cols, xv, pcode), wptr, wbytes)


# ------------------------------------------------------------- gated unit
def _activation(name: str) -> int:
    try:
        return ACTIVATIONS[name]
    except (KeyError, TypeError):
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, got {name!r}") from None


@functools.lru_cache(maxsize=256)
def gated_unit_workspace(rows: int, inner: int, outer: int, dtype, backward: bool = False) -> int:
    """Workspace bytes of gated_unit (or of its backward pass) for x [rows,
    inner] and weights [outer, inner] of element type `dtype`."""
    n = C.c_int64()
    _lib.call("gpb_gated_unit_workspace", _dtype_code(dtype), rows, inner, outer, int(backward),
              C.byref(n))
    return n.value


def _gated_inputs(x, w_gate, w_up, b_gate, b_up):
    xv = _View(x, "x", 2)
    g = _View(w_gate, "w_gate", 2)
    outer = g.shape[0]
    g = _matrix(w_gate, "w_gate", (outer, xv.shape[1]), xv)
    u = _matrix(w_up, "w_up", (outer, xv.shape[1]), xv)
    if g.ld != u.ld:
        raise ValueError(f"w_gate and w_up must have one row stride, got {g.ld} and {u.ld}")
    return (xv, g, u, _vector(b_gate, "b_gate", outer, xv, xv.code),
            _vector(b_up, "b_up", outer, xv, xv.code))


def gated_unit(out, x, w_gate, w_up, b_gate=None, b_up=None, *, activation: str = "silu",
               workspace=None, stream=None) -> None:
    """out = act(x w_gate' + b_gate) * (x w_up' + b_up).

    x [rows, inner], w_gate and w_up [outer, inner], biases [outer] or None,
    out [rows, outer], all of one element type. `activation` is "silu",
    "gelu" (exact), "sigmoid" or "tanh"."""
    act = _activation(activation)
    xv, g, u, bg, bu = _gated_inputs(x, w_gate, w_up, b_gate, b_up)
    rows, inner = xv.shape
    outer = g.shape[0]
    ov = _matrix(out, "out", (rows, outer), xv)
    wptr, wbytes = _workspace(workspace, xv)
    _lib.call("gpb_gated_unit", xv.device, stream, xv.code, act, rows, inner, outer, ov.ptr, ov.ld,
              xv.ptr, xv.ld, g.ptr, u.ptr, g.ld, bg, bu, wptr, wbytes)


def gated_unit_backward(dout, x, w_gate, w_up, b_gate=None, b_up=None, *, dx=None, dw_gate=None,
                        dw_up=None, db_gate=None, db_up=None, activation: str = "silu",
                        workspace=None, stream=None) -> None:
    """Gradients of gated_unit from dout [rows, outer] and the forward inputs
    (the projections are recomputed): dx, dw_gate, dw_up, db_gate and db_up are
    written where given, in x's element type."""
    act = _activation(activation)
    xv, g, u, bg, bu = _gated_inputs(x, w_gate, w_up, b_gate, b_up)
    rows, inner = xv.shape
    outer = g.shape[0]
    dv = _matrix(dout, "dout", (rows, outer), xv)
    xo = _matrix(dx, "dx", xv.shape, xv) if dx is not None else None
    go = _matrix(dw_gate, "dw_gate", g.shape, xv) if dw_gate is not None else None
    uo = _matrix(dw_up, "dw_up", g.shape, xv) if dw_up is not None else None
    if go and uo and go.ld != uo.ld:
        raise ValueError(f"dw_gate and dw_up must have one row stride, got {go.ld} and {uo.ld}")
    wo = go or uo
    wptr, wbytes = _workspace(workspace, xv)
    _lib.call("gpb_gated_unit_backward", xv.device, stream, xv.code, act, rows, inner, outer,
              dv.ptr, dv.ld, xv.ptr, xv.ld, g.ptr, u.ptr, g.ld, bg, bu,
              xo.ptr if xo else None, xo.ld if xo else 0, go.ptr if go else None,
              uo.ptr if uo else None, wo.ld if wo else 0,
              _vector(db_gate, "db_gate", outer, xv, xv.code),
              _vector(db_up, "db_up", outer, xv, xv.code), wptr, wbytes)


# ---------------------------------------------------------------- dropout
def dropout(out, x, p: float, seed: int, *, offset: int = 0, residual=None, stream=None) -> None:
    """out = keep ? x / (1 - p) : 0, plus `residual` where given.

    The mask is a function of (seed, offset) and the element's index row *
    columns + column alone (Philox4x32-10), so dropout_backward with the same
    two numbers regenerates it. out may be x or residual themselves."""
    xv = _View(x, "x", 2)
    ov = _matrix(out, "out", xv.shape, xv)
    rv = _matrix(residual, "residual", xv.shape, xv) if residual is not None else None
    for name, v in (("seed", seed), ("offset", offset)):
        if not 0 <= v < 1 << 64:
            raise ValueError(f"{name} must be in [0, 2^64), got {v}")
    _lib.call("gpb_dropout", xv.device, stream, xv.code, xv.shape[0], xv.shape[1], ov.ptr, ov.ld,
              xv.ptr, xv.ld, rv.ptr if rv else None, rv.ld if rv else 0, p, seed, offset)


def dropout_backward(dx, dout, p: float, seed: int, *, offset: int = 0, stream=None) -> None:
    """dx = keep ? dout / (1 - p) : 0 with the mask of dropout(p, seed, offset);
    the residual's gradient is dout itself. dx may be dout."""
    dropout(dx, dout, p, seed, offset=offset, stream=stream)


def cast(out, x, *, stream=None) -> None:
    """out = x in out's element type, rounded to nearest ([rows, columns])."""
    xv = _View(x, "x", 2)
    ov = _View(out, "out", 2)
    if ov.shape != xv.shape:
        raise ValueError(f"out must have shape {xv.shape}, got {ov.shape}")
    if ov.device != xv.device:
        raise ValueError(f"out is on device {ov.device}, expected {xv.device}")
    _lib.call("gpb_cast", xv.device, stream, ov.code, xv.code, *xv.shape, ov.ptr, ov.ld, xv.ptr,
              xv.ld)
