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
CUDA graph (after a first call on the device outside of any capture); where one
takes a workspace, it is any 16-byte aligned array of at least the bytes the
matching *_workspace function returns, not shared by calls that may run at the
same time. Argument errors raise ValueError before any device work.
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


def _element_code(a) -> int:
    return _dtype_code(getattr(a, "element_type", None) or a.dtype)


def _where(a, name: str) -> tuple:
    """(pointer, device, strides) of a device array; a DeviceBuffer is contiguous."""
    try:
        ptr = a.data_ptr()
    except AttributeError:
        if not (hasattr(a, "ptr") and hasattr(a, "nbytes")):
            raise ValueError(f"{name} must be a device array, got {type(a).__name__}") from None
        if a.ptr is None:
            raise ValueError(f"{name} was freed") from None
        return a.ptr, a.device, None
    device = a.device.index
    if device is None or a.device.type != "cuda":
        raise ValueError(f"{name} must be on a CUDA device, got {a.device}")
    return ptr, device, a.stride()


def _matrix(a, name: str, rows: int = -1, cols: int = -1, code: int = -1, device: int = -1) -> tuple:
    """(pointer, rows, columns, leading dimension, type, device) of a matrix; sizes, type and
    device that are given (not -1) have to agree."""
    ptr, dev, strides = _where(a, name)
    shape = a.shape
    if len(shape) != 2:
        raise ValueError(f"{name} must be 2-D, got shape {tuple(shape)}")
    r, c = shape
    if rows >= 0 and (r != rows or c != cols):
        raise ValueError(f"{name} must have shape ({rows}, {cols}), got {tuple(shape)}")
    ld = c
    if strides is not None:
        if strides[1] != 1 and c > 1:
            raise ValueError(f"{name} must have unit column stride, got strides {strides}")
        if r > 1:
            ld = strides[0]
        dtype = a.dtype
        kind = _CODES[dtype] if dtype in _CODES else _dtype_code(dtype)
    else:
        kind = _element_code(a)
    if code >= 0:
        if kind != code:
            raise ValueError(f"{name} has a different element type")
        if dev != device:
            raise ValueError(f"{name} is on device {dev}, expected {device}")
    return ptr, r, c, ld, kind, dev


def _vector(a, name: str, size: int, code: int, device: int) -> int | None:
    """Pointer of a [size] vector of element type `code` on `device`, or None."""
    if a is None:
        return None
    ptr, dev, strides = _where(a, name)
    shape = a.shape
    if len(shape) != 1:
        raise ValueError(f"{name} must be 1-D, got shape {tuple(shape)}")
    if shape[0] != size:
        raise ValueError(f"{name} must have {size} entries, got {shape[0]}")
    if strides is not None:
        if strides[0] != 1 and size > 1:
            raise ValueError(f"{name} must have unit stride, got {strides}")
        dtype = a.dtype
        kind = _CODES[dtype] if dtype in _CODES else _dtype_code(dtype)
    else:
        kind = _element_code(a)
    if kind != code:
        raise ValueError(f"{name} has a different element type")
    if dev != device:
        raise ValueError(f"{name} is on device {dev}, expected {device}")
    return ptr


def _workspace(a, device: int) -> tuple:
    """(pointer, bytes) of a scratch array; the call itself checks the size."""
    if a is None:
        return None, 0
    ptr, dev, strides = _where(a, "workspace")
    if strides is None:
        size = a.nbytes
    elif a.is_contiguous():
        size = a.numel() * a.element_size()
    else:
        raise ValueError("workspace must be contiguous")
    if dev != device:
        raise ValueError(f"workspace is on device {dev}, expected {device}")
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
    xp, rows, cols, x_ld, code, dev = _matrix(x, "x")
    op, _, _, out_ld, _, _ = _matrix(out, "out", rows, cols, code, dev)
    pcode = code
    for a in (weight, bias):
        if a is not None:
            pcode = _element_code(a)
            break
    if pcode not in (0, code):
        raise ValueError("weight and bias must be float32 or of x's type")
    _lib.call("gpb_layer_norm", dev, stream, code, pcode, rows, cols, op, out_ld, xp, x_ld,
              _vector(weight, "weight", cols, pcode, dev), _vector(bias, "bias", cols, pcode, dev),
              eps, _vector(mean, "mean", rows, 0, dev), _vector(rstd, "rstd", rows, 0, dev))


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
    xp, rows, cols, x_ld, code, dev = _matrix(x, "x")
    dp, _, _, dout_ld, _, _ = _matrix(dout, "dout", rows, cols, code, dev)
    op, out_ld = None, 0
    if dx is not None:
        op, _, _, out_ld, _, _ = _matrix(dx, "dx", rows, cols, code, dev)
    pcode = code
    for a in (weight, dweight, dbias):
        if a is not None:
            pcode = _element_code(a)
            break
    if pcode not in (0, code):
        raise ValueError("weight and its gradient must be float32 or of x's type")
    wptr, wbytes = _workspace(workspace, dev)
    _lib.call("gpb_layer_norm_backward", dev, stream, code, pcode, rows, cols, op, out_ld, dp,
              dout_ld, xp, x_ld, _vector(mean, "mean", rows, 0, dev),
              _vector(rstd, "rstd", rows, 0, dev), _vector(weight, "weight", cols, pcode, dev),
              _vector(dweight, "dweight", cols, pcode, dev),
              _vector(dbias, "dbias", cols, pcode, dev), wptr, wbytes)


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
    """x, w_gate and w_up as matrices and the biases' pointers, checked against one another."""
    xm = _matrix(x, "x")
    inner, code, dev = xm[2], xm[4], xm[5]
    if len(w_gate.shape) != 2:
        raise ValueError(f"w_gate must be 2-D, got shape {tuple(w_gate.shape)}")
    outer = w_gate.shape[0]
    g = _matrix(w_gate, "w_gate", outer, inner, code, dev)
    u = _matrix(w_up, "w_up", outer, inner, code, dev)
    if g[3] != u[3]:
        raise ValueError(f"w_gate and w_up must have one row stride, got {g[3]} and {u[3]}")
    return (xm, g, u, _vector(b_gate, "b_gate", outer, code, dev),
            _vector(b_up, "b_up", outer, code, dev))


def gated_unit(out, x, w_gate, w_up, b_gate=None, b_up=None, *, activation: str = "silu",
               workspace=None, stream=None) -> None:
    """out = act(x w_gate' + b_gate) * (x w_up' + b_up).

    x [rows, inner], w_gate and w_up [outer, inner], biases [outer] or None,
    out [rows, outer], all of one element type. `activation` is "silu",
    "gelu" (exact), "sigmoid" or "tanh"."""
    act = _activation(activation)
    (xp, rows, inner, x_ld, code, dev), g, u, bg, bu = _gated_inputs(x, w_gate, w_up, b_gate, b_up)
    outer = g[1]
    op, _, _, out_ld, _, _ = _matrix(out, "out", rows, outer, code, dev)
    wptr, wbytes = _workspace(workspace, dev)
    _lib.call("gpb_gated_unit", dev, stream, code, act, rows, inner, outer, op, out_ld, xp, x_ld,
              g[0], u[0], g[3], bg, bu, wptr, wbytes)


def gated_unit_backward(dout, x, w_gate, w_up, b_gate=None, b_up=None, *, dx=None, dw_gate=None,
                        dw_up=None, db_gate=None, db_up=None, activation: str = "silu",
                        workspace=None, stream=None) -> None:
    """Gradients of gated_unit from dout [rows, outer] and the forward inputs
    (the projections are recomputed): dx, dw_gate, dw_up, db_gate and db_up are
    written where given, in x's element type. With 16-bit types the gradients'
    factors dout up act' and dout act are rounded to two parts of the type where
    rows * inner * outer is at most 2^31, to one above; in float16 times a power
    of two of the call, so that they may pass its range."""
    act = _activation(activation)
    (xp, rows, inner, x_ld, code, dev), g, u, bg, bu = _gated_inputs(x, w_gate, w_up, b_gate, b_up)
    outer = g[1]
    dp, _, _, dout_ld, _, _ = _matrix(dout, "dout", rows, outer, code, dev)
    dxp, dx_ld, dgp, dup, dw_ld = None, 0, None, None, 0
    if dx is not None:
        dxp, _, _, dx_ld, _, _ = _matrix(dx, "dx", rows, inner, code, dev)
    if dw_gate is not None:
        dgp, _, _, dw_ld, _, _ = _matrix(dw_gate, "dw_gate", outer, inner, code, dev)
    if dw_up is not None:
        dup, _, _, ld, _, _ = _matrix(dw_up, "dw_up", outer, inner, code, dev)
        if dgp is not None and ld != dw_ld:
            raise ValueError(f"dw_gate and dw_up must have one row stride, got {dw_ld} and {ld}")
        dw_ld = ld
    wptr, wbytes = _workspace(workspace, dev)
    _lib.call("gpb_gated_unit_backward", dev, stream, code, act, rows, inner, outer, dp, dout_ld, xp,
              x_ld, g[0], u[0], g[3], bg, bu, dxp, dx_ld, dgp, dup, dw_ld,
              _vector(db_gate, "db_gate", outer, code, dev),
              _vector(db_up, "db_up", outer, code, dev), wptr, wbytes)


# ---------------------------------------------------------------- dropout
def dropout(out, x, p: float, seed: int, *, offset: int = 0, residual=None, stream=None) -> None:
    """out = keep ? x / (1 - p) : 0, plus `residual` where given.

    The mask is a function of (seed, offset) and the element's index row *
    columns + column alone (Philox4x32-10), so dropout_backward with the same
    two numbers regenerates it. out may be x or residual themselves."""
    xp, rows, cols, x_ld, code, dev = _matrix(x, "x")
    op, _, _, out_ld, _, _ = _matrix(out, "out", rows, cols, code, dev)
    rp, r_ld = None, 0
    if residual is not None:
        rp, _, _, r_ld, _, _ = _matrix(residual, "residual", rows, cols, code, dev)
    for name, v in (("seed", seed), ("offset", offset)):
        if not 0 <= v < 1 << 64:
            raise ValueError(f"{name} must be in [0, 2^64), got {v}")
    _lib.call("gpb_dropout", dev, stream, code, rows, cols, op, out_ld, xp, x_ld, rp, r_ld, p, seed,
              offset)


def dropout_backward(dx, dout, p: float, seed: int, *, offset: int = 0, stream=None) -> None:
    """dx = keep ? dout / (1 - p) : 0 with the mask of dropout(p, seed, offset);
    the residual's gradient is dout itself. dx may be dout."""
    dropout(dx, dout, p, seed, offset=offset, stream=stream)


def cast(out, x, *, stream=None) -> None:
    """out = x in out's element type, rounded to nearest ([rows, columns])."""
    xp, rows, cols, x_ld, code, dev = _matrix(x, "x")
    op, r, c, out_ld, ocode, odev = _matrix(out, "out")
    if (r, c) != (rows, cols):
        raise ValueError(f"out must have shape ({rows}, {cols}), got ({r}, {c})")
    if odev != dev:
        raise ValueError(f"out is on device {odev}, expected {dev}")
    _lib.call("gpb_cast", dev, stream, ocode, code, rows, cols, op, out_ld, xp, x_ld)
