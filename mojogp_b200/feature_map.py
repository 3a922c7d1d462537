"""FeatureMap: a learned map from wide inputs to a GP's input dimensions.

A stack of layers, each a layer norm over the layer's inputs, a gated unit
act(x Wg' + bg) * (x Wu' + bu) and, while training, dropout; a layer whose
width does not change adds its input. The last layer has no dropout. The
operators are mojogp_b200.features; weights live on the host in float32 (the
master copy an optimiser moves) and on the device in the map's element type.
SingleOutputGP(kernel, feature_map=FeatureMap([64, 16])) trains it with the
kernel by the marginal likelihood.
"""
from __future__ import annotations

from typing import Optional, Sequence

import numpy as np

from . import features
from .provider import DeviceBuffer

MAX_OUTPUTS = 64  # input dimensions a provider takes (GPB_MAX_DIM)
_EPS = 1e-5
_KEEP = 1 << 26  # bytes of activations that a prediction leaves for the next one (a new buffer costs some 0.1 ms)


def _to_bfloat16_bits(a: np.ndarray) -> np.ndarray:
    """float32 to bfloat16 bit patterns, rounded to nearest even."""
    u = np.ascontiguousarray(a, np.float32).view(np.uint32)
    r = ((u + np.uint32(0x7FFF) + ((u >> np.uint32(16)) & np.uint32(1))) >> np.uint32(16))
    quiet = (u >> np.uint32(16)) | np.uint32(0x40)
    return np.where(np.isnan(a), quiet, r).astype(np.uint16)


class _Array(DeviceBuffer):
    """A device buffer of one of the operators' element types (NumPy has no bfloat16)."""

    def __init__(self, shape, device: int, element_type: str):
        super().__init__(shape, device, np.uint16 if element_type == "bfloat16" else element_type)
        self.element_type = element_type

    def put(self, a: np.ndarray) -> "_Array":
        a = np.asarray(a, np.float32)
        self.upload(_to_bfloat16_bits(a) if self.element_type == "bfloat16"
                    else a.astype(self.dtype))
        return self

    def get(self) -> np.ndarray:
        a = self.download()
        if self.element_type == "bfloat16":
            return (a.astype(np.uint32) << np.uint32(16)).view(np.float32)
        return a.astype(np.float32)


class FeatureMap:
    """widths: output columns of each layer; the last is the GP's input
    dimension (at most 64). dtype: "float32" (default), "float16" or
    "bfloat16", the operators' element type. dropout: probability after every
    layer but the last, while training."""

    def __init__(self, widths: Sequence[int], *, activation: str = "silu", norm: bool = True,
                 dropout: float = 0.0, dtype: str = "float32", seed: int = 0):
        widths = [int(w) for w in widths]
        if not widths or min(widths) < 1:
            raise ValueError(f"widths must be positive, got {widths}")
        if widths[-1] > MAX_OUTPUTS:
            raise ValueError(f"the last width is the GP's input dimension (at most {MAX_OUTPUTS}), "
                             f"got {widths[-1]}")
        if activation not in features.ACTIVATIONS:
            raise ValueError(f"activation must be one of {sorted(features.ACTIVATIONS)}, "
                             f"got {activation!r}")
        if not 0.0 <= dropout < 1.0:
            raise ValueError(f"dropout must be in [0, 1), got {dropout}")
        if dtype not in ("float32", "float16", "bfloat16"):
            raise ValueError(f"dtype must be float32, float16 or bfloat16, got {dtype!r}")
        if not 0 <= int(seed) < 1 << 63:
            raise ValueError(f"seed must be in [0, 2^63), got {seed}")
        self.widths, self.activation, self.norm = widths, activation, bool(norm)
        self.dropout, self.dtype, self.seed = float(dropout), dtype, int(seed)
        self.input_dim: Optional[int] = None
        self.parameters: list = []  # host float32 arrays, per layer: norm w, b; Wg, Wu, bg, bu
        self._device_params: Optional[list] = None
        self._run: Optional[dict] = None
        self._device = 0
        self._stale = True  # the device copies are older than `parameters`
        self.version = 0  # counts the weights' changes

    # ------------------------------------------------------------- weights
    @property
    def output_dim(self) -> int:
        return self.widths[-1]

    @property
    def _per_layer(self) -> int:
        return 6 if self.norm else 4

    def build(self, input_dim: int) -> "FeatureMap":
        """Draw the weights for `input_dim` columns (once)."""
        input_dim = int(input_dim)
        if self.input_dim is not None:
            if input_dim != self.input_dim:
                raise ValueError(f"feature map was built for {self.input_dim} columns, got {input_dim}")
            return self
        if input_dim < 1:
            raise ValueError("feature map needs at least one input column")
        rng = np.random.default_rng(self.seed)
        inner = input_dim
        for outer in self.widths:
            if self.norm:
                self.parameters += [np.ones(inner, np.float32), np.zeros(inner, np.float32)]
            for _ in range(2):
                self.parameters.append((rng.standard_normal((outer, inner)) / np.sqrt(inner))
                                       .astype(np.float32))
            # The gate starts open (bias 1), the values unshifted.
            self.parameters += [np.ones(outer, np.float32), np.zeros(outer, np.float32)]
            inner = outer
        self.input_dim = input_dim
        return self

    def snapshot(self) -> list:
        return [p.copy() for p in self.parameters]

    def restore(self, saved: Sequence[np.ndarray]) -> None:
        for p, s in zip(self.parameters, saved, strict=True):
            p[...] = s
        self.parameters_changed()

    def parameters_changed(self) -> None:
        """The host weights moved: the device copies follow at the next forward,
        which `backward` needs first (it recomputes from the weights)."""
        self._stale = True
        self.version += 1
        if self._run is not None:
            self._run["ready"] = False

    def _params(self, device: int) -> list:
        if self._device_params is None or self._device != device:
            self._device_params = [
                _Array(p.shape, device, "float32" if self.norm and i % self._per_layer < 2
                       else self.dtype) for i, p in enumerate(self.parameters)]
            self._device = device
            self._run = None
            self._stale = True
        if self._stale:
            for d, p in zip(self._device_params, self.parameters):
                d.put(p)
            self._stale = False
        return self._device_params

    # ------------------------------------------------------------- running
    def upload(self, X: np.ndarray, device: int = 0) -> DeviceBuffer:
        """X [n, input_dim] on the device in the map's element type."""
        X = np.asarray(X, np.float32)
        if X.ndim != 2:
            raise ValueError(f"X must be 2D, got shape {X.shape}")
        self.build(X.shape[1])
        return _Array(X.shape, device, self.dtype).put(X)

    def _workspace_bytes(self, n: int, training: bool) -> int:
        need, inner = 16, self.input_dim
        for outer in self.widths:
            need = max(need, features.gated_unit_workspace(n, inner, outer, self.dtype))
            if training:
                need = max(need, features.gated_unit_workspace(n, inner, outer, self.dtype, backward=True),
                           features.layer_norm_workspace(n, inner) if self.norm else 0)
            inner = outer
        return need

    def _buffers(self, n: int, device: int, training: bool) -> dict:
        """Activations, gradients and the workspace for n rows, kept between calls of one size; the
        backward pass's share of the workspace only where it is trained."""
        run = self._run
        if run is None or run["n"] != n or run["device"] != device:
            self._run = None
            run = {"n": n, "device": device, "layers": [], "grads": None, "ready": False,
                   "workspace": None}
            inner = self.input_dim
            for outer in self.widths:
                lay = {"out": _Array((n, outer), device, self.dtype)}
                if self.norm:
                    lay["norm"] = _Array((n, inner), device, self.dtype)
                    lay["mean"], lay["rstd"] = (_Array((n,), device, "float32") for _ in range(2))
                run["layers"].append(lay)
                inner = outer
            if self.dtype != "float32":
                run["features"] = DeviceBuffer((n, self.output_dim), device)
            self._run = run
        need = self._workspace_bytes(n, training)
        if run["workspace"] is None or run["workspace"].nbytes < need:
            run["workspace"] = None
            run["workspace"] = DeviceBuffer((need,), device, np.uint8)
        return run

    def release(self) -> None:
        """Free the device activations (they are made again when needed)."""
        self._run = None

    def _dropout_seed(self, step: int, layer: int) -> tuple:
        return self.seed, step * len(self.widths) + layer

    def forward(self, x: DeviceBuffer, *, training: bool = False, step: int = 0) -> DeviceBuffer:
        """Features [n, output_dim], float32, of the rows of x (from `upload`);
        the buffer is the map's own and holds until the next call. Asynchronous
        on the default stream: `features.check_device` after it (as `backward`
        and `transform` do) raises if a kernel's bounded wait gave up. With
        `training`, dropout is drawn from (seed, step) and the activations are
        kept for `backward`."""
        if self.input_dim is None or tuple(x.shape[1:]) != (self.input_dim,):
            raise ValueError(f"x must be [n, {self.input_dim}], got {tuple(x.shape)}")
        n, device = x.shape[0], x.device
        params = self._params(device)
        run = self._buffers(n, device, training)
        run["ready"] = False
        ws, last = run["workspace"], len(self.widths) - 1
        cur = x
        for i, lay in enumerate(run["layers"]):
            p = params[i * self._per_layer:(i + 1) * self._per_layer]
            lay["in"] = cur
            unit_in = cur
            if self.norm:
                features.layer_norm(lay["norm"], cur, p[0], p[1], eps=_EPS, mean=lay["mean"],
                                    rstd=lay["rstd"])
                unit_in = lay["norm"]
            wg, wu, bg, bu = p[-4:]
            out = lay["out"]
            features.gated_unit(out, unit_in, wg, wu, bg, bu, activation=self.activation,
                                workspace=ws)
            lay["p"] = self.dropout if training and i < last else 0.0
            lay["joined"] = cur.shape[1] == out.shape[1]
            lay["key"] = self._dropout_seed(step, i)
            if lay["p"] > 0.0 or lay["joined"]:
                features.dropout(out, out, lay["p"], lay["key"][0], offset=lay["key"][1],
                                 residual=cur if lay["joined"] else None)
            cur = out
        run["ready"] = training
        if self.dtype == "float32":
            return cur
        features.cast(run["features"], cur)
        return run["features"]

    def backward(self, grad: DeviceBuffer) -> list:
        """Gradients of every entry of `parameters` (host, float32) from the
        gradient [n, output_dim] (float32) of the last training forward's features."""
        run = self._run
        if run is None or not run["ready"]:
            raise RuntimeError("backward needs a forward(training=True) before it")
        n, device = run["n"], run["device"]
        if tuple(grad.shape) != (n, self.output_dim):
            raise ValueError(f"grad must be [{n}, {self.output_dim}], got {tuple(grad.shape)}")
        params, ws = self._params(device), run["workspace"]
        if run["grads"] is None:
            run["grads"] = [_Array(p.shape, device, p.element_type) for p in params]
            for i, (lay, outer) in enumerate(zip(run["layers"], self.widths)):
                inner = lay["in"].shape[1]
                if i + 1 < len(self.widths) or self.dtype != "float32":
                    lay["dout"] = _Array((n, outer), device, self.dtype)
                lay["dmid"] = _Array((n, outer), device, self.dtype)
                lay["dunit"] = _Array((n, inner), device, self.dtype)
        out = run["grads"]
        layers = run["layers"]
        # float16 gradients are scaled by a power of two: the per-sample NLL's are of order 1/n, below
        # float16's normal range (6e-5), while a weight's gradient sums n of them and must stay
        # below 65504. The largest input gradient goes to 2^13 / n, at most 1.
        scale = 1.0
        if self.dtype == "float16":
            host = grad.download()
            top = float(np.max(np.abs(host)))
            if 0.0 < top < np.inf:
                scale = 2.0 ** np.floor(min(0.0, 13.0 - np.log2(n)) - np.log2(top))
                grad = DeviceBuffer.from_host(host * np.float32(scale), device)
        if self.dtype == "float32":
            layers[-1]["dout"] = grad
        else:
            features.cast(layers[-1]["dout"], grad)
        for i in reversed(range(len(layers))):
            lay = layers[i]
            p = params[i * self._per_layer:(i + 1) * self._per_layer]
            g = out[i * self._per_layer:(i + 1) * self._per_layer]
            dmid = lay["dout"]
            if lay["p"] > 0.0:
                dmid = lay["dmid"]
                features.dropout_backward(dmid, lay["dout"], lay["p"], lay["key"][0],
                                          offset=lay["key"][1])
            wg, wu, bg, bu = p[-4:]
            need_dx = self.norm or i > 0
            features.gated_unit_backward(
                dmid, lay["norm"] if self.norm else lay["in"], wg, wu, bg, bu,
                dx=lay["dunit"] if need_dx else None, dw_gate=g[-4], dw_up=g[-3], db_gate=g[-2],
                db_up=g[-1], activation=self.activation, workspace=ws)
            if self.norm:
                features.layer_norm_backward(
                    lay["dunit"] if i > 0 else None, lay["dunit"], lay["in"], lay["mean"],
                    lay["rstd"], p[0], dweight=g[0], dbias=g[1], workspace=ws)
            if i > 0:
                below = layers[i - 1]["dout"]
                # The layer's input also reaches its output directly where the widths agree.
                features.dropout(below, lay["dunit"], 0.0, 0,
                                 residual=lay["dout"] if lay["joined"] else None)
        grads = [g.get() / np.float32(scale) for g in out]
        features.check_device(device)
        return grads

    def transform(self, X: np.ndarray, device: int = 0, block: int = 65536) -> np.ndarray:
        """Features of host rows (no dropout), `block` rows at a time."""
        X = np.asarray(X, np.float32)
        if X.ndim != 2 or self.input_dim is None or X.shape[1] != self.input_dim:
            raise ValueError(f"X must be [n, {self.input_dim}], got {X.shape}")
        out = np.empty((X.shape[0], self.output_dim), np.float32)
        for b in range(0, X.shape[0], block):
            out[b:b + block] = self.forward(self.upload(X[b:b + block], device)).download()
            features.check_device(device)
        held = self._run["layers"] if self._run is not None else []
        if sum(b.nbytes for lay in held for b in lay.values() if isinstance(b, DeviceBuffer)) > _KEEP:
            self.release()
        return out

    # -------------------------------------------------------------- persist
    def config(self) -> dict:
        return {"widths": self.widths, "activation": self.activation, "norm": self.norm,
                "dropout": self.dropout, "dtype": self.dtype, "seed": self.seed,
                "input_dim": self.input_dim}

    @classmethod
    def from_config(cls, config: dict, parameters: Sequence[np.ndarray]) -> "FeatureMap":
        kw = dict(config)
        input_dim = kw.pop("input_dim")
        fm = cls(kw.pop("widths"), **kw).build(input_dim)
        if len(parameters) != len(fm.parameters) or any(
                np.shape(a) != b.shape for a, b in zip(parameters, fm.parameters)):
            raise ValueError("saved feature-map weights do not match its widths")
        fm.restore([np.asarray(a, np.float32) for a in parameters])
        return fm
