"""The operators of a learned feature map under a Gaussian process, as measured work.

A GP takes at most 64 input dimensions, so wide inputs (embeddings, sensor
vectors) are first mapped down by a small network that is trained with the
kernel's parameters. Its operators are a layer norm, a gated projection unit
(both projections, the activation and the product in one), dropout from a
counter-based generator, and the gradient of the kernel's bilinear form with
respect to the inputs, which is what the network's backward pass starts from.

`run` computes one pass: in elementary torch operations where `own` is false,
through mojogp_b200 where it is true. Cases are plain dicts; sizes are rows
(training points) by columns (features).
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
_ACTIVATIONS = ("silu", "gelu", "sigmoid", "tanh")
_LEAVES = ("rbf", "matern12", "matern32", "matern52")
_EPS = 1e-5


# ------------------------------------------------------------------- cases
def listed():
    return [
        # One prediction point through a wide norm: the smallest call.
        dict(name="norm-1x4096-bf16", op="norm", rows=1, cols=4096, dtype="bf16", wdtype="bf16",
             stats=False),
        # The benchmark's million rows of 16 features, with the statistics kept for training.
        dict(name="norm-1Mx16-fp32", op="norm", rows=1_000_000, cols=16, dtype="fp32",
             wdtype="fp32", stats=True),
        # Training on wide embeddings: every gradient of the norm.
        dict(name="norm-grad-16384x4096-bf16", op="norm_grad", rows=16384, cols=4096,
             dtype="bf16", wdtype="fp32"),
        # Odd row count, width that is no multiple of a warp's vector.
        dict(name="norm-grad-5003x1000-fp16", op="norm_grad", rows=5003, cols=1000, dtype="fp16",
             wdtype="fp16"),
        # One prediction point through a wide unit: bound by reading the weights.
        dict(name="gated-1x2048x8192-bf16", op="gated", rows=1, inner=2048, outer=8192,
             dtype="bf16", act="silu", bias=False),
        # A training batch through a wide unit: bound by the tensor cores.
        dict(name="gated-8192x2048x8192-bf16", op="gated", rows=8192, inner=2048, outer=8192,
             dtype="bf16", act="silu", bias=False),
        # Its backward pass, at half the widths.
        dict(name="gated-grad-8192x1024x4096-bf16", op="gated_grad", rows=8192, inner=1024,
             outer=4096, dtype="bf16", act="gelu", bias=True),
        # 50,000 training points of 768 features down to 64 inputs, single precision.
        dict(name="gated-grad-50000x768x64-fp32", op="gated_grad", rows=50000, inner=768,
             outer=64, dtype="fp32", act="sigmoid", bias=True),
        # The feature map of a 2,000-point fit: launch latency.
        dict(name="dropout-2000x64-fp32", op="dropout", rows=2000, cols=64, dtype="fp32",
             p=0.1, residual=False),
        # Dropout joined to the residual sum of a wide unit.
        dict(name="dropout-16384x4096-bf16-residual", op="dropout", rows=16384, cols=4096,
             dtype="bf16", p=0.2, residual=True),
        # The 1-D fit of 2,000 points, 10 probes.
        dict(name="input-grad-rbf-2000x1", op="input_grad", rows=2000, dim=1, cols=11,
             leaf="rbf", ard=False),
        # 20,000 points in 8 dimensions, the target and 15 probes.
        dict(name="input-grad-matern52-20000x8", op="input_grad", rows=20000, dim=8, cols=16,
             leaf="matern52", ard=True),
    ]


def _log_int(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi], odd values among them."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "norm_grad", "gated", "gated", "gated_grad", "gated_grad",
                     "dropout", "dropout_grad", "input_grad"])
    dtype = rng.choice(["bf16", "fp16", "fp32"])
    if op in ("norm", "norm_grad"):
        cols = _log_int(rng, 1, 16384)
        rows = _log_int(rng, 1, min(1_000_000, 67_000_000 // cols))
        case = dict(op=op, rows=rows, cols=cols, dtype=dtype, wdtype=rng.choice([dtype, "fp32"]))
        if op == "norm":
            case["stats"] = rng.random() < 0.5
        return case
    if op in ("gated", "gated_grad"):
        inner, outer = _log_int(rng, 1, 8192), _log_int(rng, 1, 8192)
        budget = 137_000_000_000 // (3 if op == "gated_grad" else 1)
        rows = _log_int(rng, 1, max(1, min(100_000, budget // (inner * outer),
                                           400_000_000 // max(inner, outer))))
        return dict(op=op, rows=rows, inner=inner, outer=outer, dtype=dtype,
                    act=rng.choice(_ACTIVATIONS), bias=rng.random() < 0.5)
    if op in ("dropout", "dropout_grad"):
        cols = _log_int(rng, 1, 16384)
        rows = _log_int(rng, 1, min(1_000_000, 67_000_000 // cols))
        case = dict(op=op, rows=rows, cols=cols, dtype=dtype, p=round(rng.uniform(0.0, 0.9), 3))
        if op == "dropout":
            case["residual"] = rng.random() < 0.5
        return case
    return dict(op=op, rows=_log_int(rng, 1, 20000), dim=_log_int(rng, 1, 32),
                cols=rng.randint(1, 16), leaf=rng.choice(_LEAVES), ard=rng.random() < 0.5)


def work(case):
    """Bytes and operations a pass cannot do without: each input read once, each output written
    once, the multiply-adds of the formulas."""
    op = case["op"]
    if op in ("norm", "norm_grad"):
        e, w = _BYTES[case["dtype"]], _BYTES[case["wdtype"]]
        r, c = case["rows"], case["cols"]
        if op == "norm":
            return {"bytes": 2 * r * c * e + 2 * c * w + (8 * r if case["stats"] else 0),
                    "flops": 8 * r * c}
        return {"bytes": 3 * r * c * e + 8 * r + 3 * c * w, "flops": 14 * r * c}
    if op in ("gated", "gated_grad"):
        e = _BYTES[case["dtype"]]
        m, k, n = case["rows"], case["inner"], case["outer"]
        b = 2 * n if case["bias"] else 0
        if op == "gated":
            return {"bytes": e * (m * k + 2 * n * k + b + m * n), "flops": 4 * m * n * k}
        return {"bytes": e * (2 * m * k + 4 * n * k + 2 * b + m * n), "flops": 12 * m * n * k}
    if op in ("dropout", "dropout_grad"):
        e, r, c = _BYTES[case["dtype"]], case["rows"], case["cols"]
        return {"bytes": e * r * c * (3 if case.get("residual") else 2), "flops": 2 * r * c}
    n, d, t = case["rows"], case["dim"], case["cols"]
    return {"bytes": 4 * (2 * n * d + 2 * n * t), "flops": n * n * (5 * d + 4 * t + 8)}


# ----------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, shape, dtype, scale=1.0, shift=0.0):
    x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)
    return (x * scale + shift).to(dtype)


def _inputs(case, seed):
    g = _generator(seed)
    op = case["op"]
    s = dict(case)
    if op in ("norm", "norm_grad"):
        t, wt = _TYPES[case["dtype"]], _TYPES[case["wdtype"]]
        r, c = case["rows"], case["cols"]
        s["x"] = _normal(g, (r, c), t, 1.5, 0.5)
        s["weight"] = _normal(g, (c,), wt, 0.2, 1.0)
        s["bias"] = _normal(g, (c,), wt, 0.2)
        if op == "norm_grad":
            s["dout"] = _normal(g, (r, c), t)
            x = s["x"].double()
            mean = x.mean(dim=1)
            s["mean"] = mean.float()
            s["rstd"] = (((x - mean[:, None]) ** 2).mean(dim=1) + _EPS).rsqrt().float()
    elif op in ("gated", "gated_grad"):
        t = _TYPES[case["dtype"]]
        m, k, n = case["rows"], case["inner"], case["outer"]
        s["x"] = _normal(g, (m, k), t)
        s["w_gate"] = _normal(g, (n, k), t, k ** -0.5)
        s["w_up"] = _normal(g, (n, k), t, k ** -0.5)
        s["b_gate"] = _normal(g, (n,), t, 0.1) if case["bias"] else None
        s["b_up"] = _normal(g, (n,), t, 0.1) if case["bias"] else None
        if op == "gated_grad":
            s["dout"] = _normal(g, (m, n), t)
    elif op in ("dropout", "dropout_grad"):
        t = _TYPES[case["dtype"]]
        shape = (case["rows"], case["cols"])
        s["x"] = _normal(g, shape, t)
        s["residual_in"] = _normal(g, shape, t) if case.get("residual") else None
        s["seed"] = (int(seed) * 0x9E3779B97F4A7C15 + 12345) & 0xFFFFFFFFFFFFFFFF
        s["offset"] = (int(seed) * 0xD1342543DE82EF95 + 7) & 0xFFFFFFFFFFFFFFFF
    else:
        n, d, t = case["rows"], case["dim"], case["cols"]
        s["x"] = torch.rand((n, d), generator=g, device="cuda") * 2 - 1
        s["a"] = _normal(g, (t, n), torch.float32)
        s["b"] = _normal(g, (t, n), torch.float32)
        nl = d if case["ard"] else 1
        s["scales"] = torch.rand(nl, generator=g, device="cuda") * 1.5 + 0.5
        s["outputscale"] = 1.3
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own and case["op"] == "input_grad":
        from mojogp_b200 import kernel as kernels
        from mojogp_b200.provider import Provider
        leaf = {"rbf": kernels.RBF, "matern12": kernels.Matern12, "matern32": kernels.Matern32,
                "matern52": kernels.Matern52}[case["leaf"]]
        k = kernels.make_ard_kernel(leaf(ard=True), case["dim"]) if case["ard"] else leaf()
        params = np.append(s["scales"].cpu().numpy(), np.float32(s["outputscale"]))
        s["provider"] = Provider(s["x"].cpu().numpy(), k.resolve_ard(case["dim"]), params, 0.1)
    return s


# --------------------------------------------------------------- plain form
def _plain_norm(s):
    x = s["x"].float()
    mean = x.mean(dim=1)
    centred = x - mean[:, None]
    rstd = 1.0 / torch.sqrt((centred * centred).mean(dim=1) + _EPS)
    y = centred * rstd[:, None] * s["weight"].float() + s["bias"].float()
    y = y.to(s["x"].dtype)
    return (y, mean, rstd) if s["stats"] else (y,)


def _plain_norm_grad(s):
    x, dy, rstd = s["x"].float(), s["dout"].float(), s["rstd"][:, None]
    xhat = (x - s["mean"][:, None]) * rstd
    g = dy * s["weight"].float()
    dx = rstd * (g - g.mean(dim=1, keepdim=True) - xhat * (g * xhat).mean(dim=1, keepdim=True))
    wt = s["weight"].dtype
    return dx.to(s["x"].dtype), (dy * xhat).sum(dim=0).to(wt), dy.sum(dim=0).to(wt)


def _plain_activation(name, z):
    """The activation and its derivative."""
    if name == "tanh":
        value = 1.0 - 2.0 / (torch.exp(2.0 * z) + 1.0)
        return value, 1.0 - value * value
    if name == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    sig = 1.0 / (1.0 + torch.exp(-z))
    if name == "sigmoid":
        return sig, sig * (1.0 - sig)
    return z * sig, sig * (1.0 + z * (1.0 - sig))


def _plain_projections(s):
    x = s["x"].float()
    gate = x @ s["w_gate"].float().T
    up = x @ s["w_up"].float().T
    if s["b_gate"] is not None:
        gate = gate + s["b_gate"].float()
        up = up + s["b_up"].float()
    return x, gate, up


def _plain_gated(s):
    _, gate, up = _plain_projections(s)
    return ((_plain_activation(s["act"], gate)[0] * up).to(s["x"].dtype),)


def _plain_gated_grad(s):
    t = s["x"].dtype
    x, gate, up = _plain_projections(s)
    act, slope = _plain_activation(s["act"], gate)
    dy = s["dout"].float()
    dgate, dup = dy * up * slope, dy * act
    dx = dgate @ s["w_gate"].float() + dup @ s["w_up"].float()
    out = [dx.to(t), (dgate.T @ x).to(t), (dup.T @ x).to(t)]
    if s["b_gate"] is not None:
        out += [dgate.sum(dim=0).to(t), dup.sum(dim=0).to(t)]
    return tuple(out)


def _plain_words(count, seed, offset):
    """One 32-bit word per element from Philox4x32-10 (Salmon et al., 2011): the block counter is
    (element // 4, offset), the key is the seed, element e takes word e % 4 of its block."""
    mask = 0xFFFFFFFF
    blocks = torch.arange((count + 3) // 4, device="cuda", dtype=torch.int64)
    c0, c1 = blocks & mask, blocks >> 32
    c2, c3 = torch.full_like(blocks, offset & mask), torch.full_like(blocks, offset >> 32)
    k0, k1 = seed & mask, seed >> 32
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = (((p1 >> 32) & mask) ^ c1 ^ k0, p1 & mask,
                          ((p0 >> 32) & mask) ^ c3 ^ k1, p0 & mask)
        k0, k1 = (k0 + 0x9E3779B9) & mask, (k1 + 0xBB67AE85) & mask
    return torch.stack((c0, c1, c2, c3), dim=1).reshape(-1)[:count]


def _plain_dropout(s):
    x = s["x"]
    keep = _plain_words(x.numel(), s["seed"], s["offset"]) >= int(s["p"] * 4294967296.0)
    y = torch.where(keep.reshape(x.shape), x.float() * (1.0 / (1.0 - s["p"])),
                    torch.zeros((), device="cuda"))
    if s["residual_in"] is not None:
        y = y + s["residual_in"].float()
    return (y.to(x.dtype),)


def _pull(leaf, sq, outputscale):
    """psi with dk/dx_i = -psi (x_i - x_j) / l^2, from the scaled squared distance; the kernels
    bound the exponent of the Matern-3/2 and -5/2 leaves (and of an ARD Matern-1/2) at -20."""
    if leaf == "rbf":
        return outputscale * torch.exp(-0.5 * sq)
    r = torch.sqrt(torch.clamp(sq, min=1e-20))
    if leaf in ("matern12", "matern12-ard"):
        e = torch.exp(torch.clamp(-r, min=-20.0) if leaf == "matern12-ard" else -r)
        return outputscale * e / r
    if leaf == "matern32":
        return 3.0 * outputscale * torch.exp(torch.clamp(-math.sqrt(3.0) * r, min=-20.0))
    r5 = math.sqrt(5.0) * r
    return (5.0 / 3.0) * outputscale * (1.0 + r5) * torch.exp(torch.clamp(-r5, min=-20.0))


def _plain_input_grad(s):
    x, a, b = s["x"], s["a"], s["b"]
    n, d = x.shape
    leaf = "matern12-ard" if s["leaf"] == "matern12" and s["ard"] else s["leaf"]
    out = torch.empty_like(x)
    step = max(1, min(n, 400_000_000 // (n * d)))
    for i in range(0, n, step):
        j = min(n, i + step)
        diff = (x[i:j, None, :] - x[None, :, :]) / s["scales"]
        pull = _pull(leaf, (diff * diff).sum(dim=2), s["outputscale"])
        weight = (a[:, i:j].T @ b + b[:, i:j].T @ a) * pull
        out[i:j] = -(weight[:, :, None] * diff).sum(dim=1) / s["scales"]
    return (out,)


_PLAIN = {"norm": _plain_norm, "norm_grad": _plain_norm_grad, "gated": _plain_gated,
          "gated_grad": _plain_gated_grad, "dropout": _plain_dropout,
          "dropout_grad": _plain_dropout, "input_grad": _plain_input_grad}


# ------------------------------------------------------------- the framework
def _own(s):
    from mojogp_b200 import features
    op = s["op"]
    stream = torch.cuda.current_stream().cuda_stream
    x = s["x"]
    if op == "norm":
        y = torch.empty_like(x)
        mean = torch.empty(x.shape[0], device="cuda") if s["stats"] else None
        rstd = torch.empty(x.shape[0], device="cuda") if s["stats"] else None
        features.layer_norm(y, x, s["weight"], s["bias"], eps=_EPS, mean=mean, rstd=rstd,
                            stream=stream)
        return (y, mean, rstd) if s["stats"] else (y,)
    if op == "norm_grad":
        dx = torch.empty_like(x)
        dw, db = torch.empty_like(s["weight"]), torch.empty_like(s["weight"])
        ws = torch.empty(features.layer_norm_workspace(*x.shape), dtype=torch.uint8, device="cuda")
        features.layer_norm_backward(dx, s["dout"], x, s["mean"], s["rstd"], s["weight"],
                                     dweight=dw, dbias=db, workspace=ws, stream=stream)
        return dx, dw, db
    if op in ("gated", "gated_grad"):
        m, k = x.shape
        n = s["w_gate"].shape[0]
        need = features.gated_unit_workspace(m, k, n, x.dtype, backward=op == "gated_grad")
        ws = torch.empty(need, dtype=torch.uint8, device="cuda")
        weights = (s["w_gate"], s["w_up"], s["b_gate"], s["b_up"])
        if op == "gated":
            y = torch.empty((m, n), dtype=x.dtype, device="cuda")
            features.gated_unit(y, x, *weights, activation=s["act"], workspace=ws, stream=stream)
            return (y,)
        dx = torch.empty_like(x)
        dwg, dwu = torch.empty_like(s["w_gate"]), torch.empty_like(s["w_up"])
        dbg = dbu = None
        if s["b_gate"] is not None:
            dbg, dbu = torch.empty_like(s["b_gate"]), torch.empty_like(s["b_up"])
        features.gated_unit_backward(s["dout"], x, *weights, dx=dx, dw_gate=dwg, dw_up=dwu,
                                     db_gate=dbg, db_up=dbu, activation=s["act"], workspace=ws,
                                     stream=stream)
        return (dx, dwg, dwu) if dbg is None else (dx, dwg, dwu, dbg, dbu)
    if op == "dropout":
        y = torch.empty_like(x)
        features.dropout(y, x, s["p"], s["seed"], offset=s["offset"], residual=s["residual_in"],
                         stream=stream)
        return (y,)
    if op == "dropout_grad":
        dx = torch.empty_like(x)
        features.dropout_backward(dx, x, s["p"], s["seed"], offset=s["offset"], stream=stream)
        return (dx,)
    out = torch.empty_like(x)
    s["provider"].input_gradient(out, s["a"], s["b"], s["cols"], stream=stream)
    return (out,)


def run(state):
    return _own(state) if own else _PLAIN[state["op"]](state)


# -------------------------------------------------------------------- exact
def _exact_keep(count, p, seed, offset):
    """The generator again, in 64-bit unsigned NumPy on the host, block range by block range."""
    u32 = np.uint64(32)
    low = np.uint64(0xFFFFFFFF)
    border = np.uint64(int(p * 4294967296.0))
    keep = np.empty(((count + 3) // 4, 4), dtype=bool)
    for begin in range(0, keep.shape[0], 1 << 15):
        end = min(keep.shape[0], begin + (1 << 15))
        block = np.arange(begin, end, dtype=np.uint64)
        w = [block & low, block >> u32,
             np.full(end - begin, offset & 0xFFFFFFFF, np.uint64),
             np.full(end - begin, offset >> 32, np.uint64)]
        key = [seed & 0xFFFFFFFF, seed >> 32]
        for _ in range(10):
            first = w[0] * np.uint64(0xD2511F53)
            third = w[2] * np.uint64(0xCD9E8D57)
            w = [(third >> u32) ^ w[1] ^ np.uint64(key[0]), third & low,
                 (first >> u32) ^ w[3] ^ np.uint64(key[1]), first & low]
            key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
        for lane in range(4):
            keep[begin:end, lane] = w[lane] >= border
    return keep.reshape(-1)[:count]


def exact(case, seed):
    op = case["op"]
    s = _inputs(case, seed)
    x = s["x"].double()
    if op == "norm":
        var, mean = torch.var_mean(x, dim=1, correction=0)
        rstd = (var + _EPS).pow(-0.5)
        y = torch.addcmul(s["bias"].double(), (x - mean.unsqueeze(1)) * rstd.unsqueeze(1),
                          s["weight"].double())
        return (y, mean, rstd) if case["stats"] else (y,)
    if op == "norm_grad":
        # With the statistics as given: the projection of g on the complement of (1, xhat).
        scale = s["rstd"].double().unsqueeze(1)
        unit = (x - s["mean"].double().unsqueeze(1)) * scale
        dy = s["dout"].double()
        g = dy * s["weight"].double()
        c = x.shape[1]
        along = torch.einsum("rc,rc->r", g, unit).unsqueeze(1) / c
        dx = (g - g.sum(dim=1, keepdim=True) / c - unit * along) * scale
        return dx, torch.einsum("rc,rc->c", dy, unit), dy.sum(dim=0)
    if op in ("gated", "gated_grad"):
        wg, wu = s["w_gate"].double(), s["w_up"].double()
        gate, up = torch.einsum("mk,nk->mn", x, wg), torch.einsum("mk,nk->mn", x, wu)
        if s["b_gate"] is not None:
            gate += s["b_gate"].double()
            up += s["b_up"].double()
        act = case["act"]
        if act == "tanh":
            value, slope = gate.tanh(), gate.cosh().pow(-2)
        elif act == "gelu":
            normal = torch.special.ndtr(gate)
            value = gate * normal
            slope = normal + gate * torch.exp(gate.square() / -2) / math.sqrt(2 * math.pi)
        else:
            sig = torch.sigmoid(gate)
            value = sig if act == "sigmoid" else gate * sig
            slope = sig * torch.sigmoid(-gate)
            if act == "silu":
                slope = sig + gate * slope
        if op == "gated":
            return (value * up,)
        dy = s["dout"].double()
        left, right = dy * up * slope, dy * value
        out = (torch.einsum("mn,nk->mk", left, wg) + torch.einsum("mn,nk->mk", right, wu),
               torch.einsum("mn,mk->nk", left, x), torch.einsum("mn,mk->nk", right, x))
        return out if s["b_gate"] is None else out + (left.sum(dim=0), right.sum(dim=0))
    if op in ("dropout", "dropout_grad"):
        keep = torch.from_numpy(_exact_keep(x.numel(), case["p"], s["seed"], s["offset"]))
        y = torch.zeros_like(x)
        keep = keep.to(x.device).reshape(x.shape)
        y[keep] = x[keep] / (1.0 - case["p"])
        return (y + s["residual_in"].double(),) if case.get("residual") else (y,)
    # out_i = d/dx_i of sum_ij a_i k(x_i, x_j) b_j, summed over the columns.
    a, b, ls = s["a"].double(), s["b"].double(), s["scales"].double()
    n, d = x.shape
    os_ = s["outputscale"]
    scaled = (x / ls).contiguous()
    out = torch.empty_like(x)
    for i in range(0, n, 1000):
        rows = scaled[i:i + 1000]
        sq = torch.zeros((rows.shape[0], n), dtype=torch.float64, device="cuda")
        for q in range(d):
            sq += (rows[:, q:q + 1] - scaled[:, q]).square()
        dist = sq.clamp(min=1e-20).sqrt()
        if case["leaf"] == "rbf":
            psi = os_ * torch.exp(sq / -2)
        elif case["leaf"] == "matern12":
            psi = os_ / dist * torch.exp(torch.maximum(-dist, torch.full_like(dist, -20.0))
                                         if case["ard"] else -dist)
        elif case["leaf"] == "matern32":
            psi = 3 * os_ * torch.exp((-(3 ** 0.5) * dist).clamp(min=-20))
        else:
            psi = 5 * os_ / 3 * (1 + 5 ** 0.5 * dist) * torch.exp((-(5 ** 0.5) * dist).clamp(min=-20))
        m = psi * (torch.einsum("ti,tj->ij", a[:, i:i + 1000], b)
                   + torch.einsum("ti,tj->ij", b[:, i:i + 1000], a))
        # sum_j m_ij (x_j - x_i): pairs first, so that near points do not cancel.
        for q in range(d):
            out[i:i + 1000, q] = (m * (scaled[:, q] - rows[:, q:q + 1])).sum(dim=1) / ls[q if case["ard"] else 0]
    return (out,)
