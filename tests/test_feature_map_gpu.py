"""The feature map as it is used: its layers run together, forward and backward, against a 64-bit
restatement; the NLL's gradient by the kernel's inputs; and a GP trained over a map."""
import math

import numpy as np
import pytest

from mojogp_b200 import engine
from mojogp_b200.feature_map import FeatureMap, _Array, _to_bfloat16_bits
from mojogp_b200.kernel import RBF, Matern32, Matern52, Periodic, make_ard_kernel
from mojogp_b200.provider import DeviceBuffer, Provider
from oracle import bbmm as ob
from oracle import kernels as ok

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def keep_mask(shape, p, seed, offset):
    from test_features_gpu import philox_keep
    _, keep = philox_keep(int(np.prod(shape)), p, seed, offset)
    return torch.from_numpy(keep.reshape(shape))


def restated(fm, params, x, step=None):
    """The map's formulas in torch float64 on the host; step = training step (dropout) or None."""
    act = {"silu": lambda z: z * torch.sigmoid(z), "gelu": lambda z: z * torch.special.ndtr(z),
           "sigmoid": torch.sigmoid, "tanh": torch.tanh}[fm.activation]
    it = iter(params)
    last = len(fm.widths) - 1
    for i in range(len(fm.widths)):
        h = x
        if fm.norm:
            w, b = next(it), next(it)
            c = x - x.mean(1, keepdim=True)
            h = c / torch.sqrt((c * c).mean(1, keepdim=True) + 1e-5) * w + b
        wg, wu, bg, bu = next(it), next(it), next(it), next(it)
        y = act(h @ wg.T + bg) * (h @ wu.T + bu)
        if step is not None and i < last and fm.dropout > 0:
            keep = keep_mask(tuple(y.shape), fm.dropout, fm.seed, step * len(fm.widths) + i)
            y = torch.where(keep, y / (1 - fm.dropout), torch.zeros((), dtype=y.dtype))
        x = x + y if x.shape[1] == y.shape[1] else y
    return x


MAPS = [dict(widths=[5]), dict(widths=[16, 16, 4], dropout=0.25), dict(widths=[24, 24, 24], activation="gelu"),
        dict(widths=[40, 8], norm=False, activation="tanh", dropout=0.1),
        dict(widths=[64, 64], activation="sigmoid")]


# Each operator's result is off by at most 2^-17 of its sum of magnitudes in float32 (64 terms), by
# half a step of the type (2^-11, 2^-8) in 16 bits; a pass runs up to 5 operators a layer over 3
# layers, there and back, and the norms pass an error on with a factor below 4.
@pytest.mark.parametrize("dtype,tol", [("float32", 2.0 ** -17 * 30 * 4), ("float16", 2.0 ** -11 * 30 * 4),
                                       ("bfloat16", 2.0 ** -8 * 30 * 2)])
@pytest.mark.parametrize("kw", MAPS)
@pytest.mark.parametrize("n", [1, 7, 333])
def test_map_forward_and_backward(gpb_lib, kw, n, dtype, tol):
    fm = FeatureMap(dtype=dtype, seed=3, **kw)
    rng = np.random.default_rng(4)
    X = rng.standard_normal((n, 24)).astype(np.float32)
    data = fm.upload(X)
    for p in fm.parameters:  # off the initial 0 / 1 of norms and biases
        p += (0.1 * rng.standard_normal(p.shape)).astype(np.float32)
    fm.parameters_changed()
    grad = rng.standard_normal((n, fm.output_dim)).astype(np.float32)
    out = fm.forward(data, training=True, step=6)
    got = out.download()
    grads = fm.backward(DeviceBuffer.from_host(grad))
    params = [torch.tensor(p, dtype=torch.float64, requires_grad=True) for p in fm.parameters]
    ref = restated(fm, params, torch.from_numpy(X).double(), step=6)
    (ref * torch.from_numpy(grad).double()).sum().backward()
    ref = ref.detach().numpy()
    assert np.linalg.norm(got - ref) <= tol * np.linalg.norm(ref)
    scale = max(float(p.grad.norm()) for p in params)
    for i, (g, p) in enumerate(zip(grads, params)):
        assert g.dtype == np.float32 and g.shape == tuple(p.shape)
        assert np.linalg.norm(g - p.grad.numpy()) <= tol * scale, i
    # Without training there is no dropout, and the same rows give the same features.
    plain = restated(fm, params, torch.from_numpy(X).double()).detach().numpy()
    got = fm.transform(X, block=100)
    assert np.linalg.norm(got - plain) <= tol * np.linalg.norm(plain)
    with pytest.raises(RuntimeError):
        fm.backward(DeviceBuffer.from_host(grad))


def test_map_gradient_against_differences(gpb_lib):
    """Central differences of the 64-bit restatement (error h^2 ~ 1e-8) against the device gradient
    (float32, bound above)."""
    fm = FeatureMap([16, 16, 4], dropout=0.25, seed=1)
    rng = np.random.default_rng(0)
    X = rng.standard_normal((50, 12)).astype(np.float32)
    data = fm.upload(X)
    grad = rng.standard_normal((50, 4)).astype(np.float32)
    fm.forward(data, training=True, step=2)
    grads = fm.backward(DeviceBuffer.from_host(grad))
    scale = max(np.linalg.norm(g) for g in grads)

    def loss(params):
        with torch.no_grad():
            return float((restated(fm, params, torch.from_numpy(X).double(), step=2)
                          * torch.from_numpy(grad)).sum())

    base = [torch.tensor(p, dtype=torch.float64) for p in fm.parameters]
    for i in range(len(base)):
        flat = rng.integers(0, base[i].numel())
        hi, lo = [p.clone() for p in base], [p.clone() for p in base]
        hi[i].view(-1)[flat] += 1e-4
        lo[i].view(-1)[flat] -= 1e-4
        diff = (loss(hi) - loss(lo)) / 2e-4
        assert abs(diff - grads[i].reshape(-1)[flat]) < 2.0 ** -17 * 120 * scale + 1e-6, i


def test_bfloat16_round_trip(gpb_lib):
    a = np.array([[1.0, -2.5, 3.14159, 1e-30, 65504.0, np.inf, -np.inf, np.nan, 1.00390625]], np.float32)
    t = torch.from_numpy(a).to(torch.bfloat16)
    got = _Array(a.shape, 0, "bfloat16").put(a).get()
    assert np.array_equal(got, t.float().numpy(), equal_nan=True)
    assert np.array_equal(_to_bfloat16_bits(a)[0, :7], t.view(torch.int16).numpy().astype(np.uint16)[0, :7])


@pytest.mark.parametrize("kind", ["rbf", "m52_ard", "product"])
def test_nll_gradient_by_inputs(gpb_lib, kind):
    """dNLL/dX = d/dX of (-1/2 a'Ka + 1/(2P) sum u_c'Kz_c) / n at fixed a = K^-1 y, u_c = K^-1 z_c,
    from a 64-bit solve with the engine's probes. The CG runs to float32 accuracy (condition number
    ~1e3: solves within 1e-4, as the engine's own NLL tests), so does the gradient."""
    rng = np.random.default_rng(1)
    n, d, P, noise = 300, 3, 6, 0.25
    X = rng.uniform(-1, 1, (n, d)).astype(np.float32)
    y = np.sin(3 * X[:, 0]).astype(np.float32)
    k, p = {"rbf": (RBF(), [0.7, 1.1]), "m52_ard": (make_ard_kernel(Matern52(ard=True), d), [0.6, 0.9, 1.2, 1.0]),
            "product": (Periodic() * Matern32(), [1.1, 1.7, 1.0, 0.8, 0.9])}[kind]
    p = np.array(p, np.float32)
    prov = Provider(X, k, p, noise)
    grad = DeviceBuffer((n, d))
    res = engine.bbmm_inputs(prov, y, grad, num_probes=P, max_cg_iter=250, max_tridiag_iter=30,
                             cg_tol=0.0, iteration=5)
    plain = engine.bbmm(prov, y, num_probes=P, max_cg_iter=250, max_tridiag_iter=30, cg_tol=0.0,
                        iteration=5)
    assert res["nll"] == plain["nll"] and np.array_equal(res["grads"], plain["grads"])
    spec = k.to_spec(d)
    K = ok.kernel_matrix(spec, p, X.astype(np.float64)) + noise * np.eye(n)
    z = ob.hash_gaussian(np.arange(P * n, dtype=np.uint64), 5 * 104729 + 42).reshape(P, n).astype(np.float64)
    alpha, u = np.linalg.solve(K, y.astype(np.float64)), np.linalg.solve(K, z.T).T
    assert abs(res["mean_grad"] + alpha.sum() / n) < 1e-4 * np.abs(alpha).sum() / n

    def form(Xh):
        M = ok.kernel_matrix(spec, p, Xh)
        return (-0.5 * alpha @ M @ alpha + 0.5 / P * sum(u[c] @ M @ z[c] for c in range(P))) / n

    got = grad.download()
    X64 = X.astype(np.float64)
    ref = np.zeros((12, d))
    rows = rng.choice(n, 12, replace=False)
    for r, i in enumerate(rows):
        for q in range(d):
            hi, lo = X64.copy(), X64.copy()
            hi[i, q] += 1e-5
            lo[i, q] -= 1e-5
            ref[r, q] = (form(hi) - form(lo)) / 2e-5
    assert np.linalg.norm(got[rows] - ref) < 1e-3 * np.linalg.norm(ref)


def test_set_inputs_matches_a_new_provider(gpb_lib):
    rng = np.random.default_rng(2)
    A, B = (rng.standard_normal((500, 4)).astype(np.float32) for _ in range(2))
    k, p = RBF(), np.array([0.8, 1.0], np.float32)
    v = rng.standard_normal((500, 16)).astype(np.float32)
    prov = Provider(A, k, p, 0.1)
    prov.matvec_host(v)
    prov.set_inputs(DeviceBuffer.from_host(B))
    fresh = Provider(B, k, p, 0.1)
    assert np.array_equal(prov.matvec_host(v), fresh.matvec_host(v))
    with pytest.raises(ValueError):
        prov.set_inputs(DeviceBuffer((500, 3)))
    with pytest.raises(ValueError):
        prov.set_inputs(DeviceBuffer((500, 4), dtype=np.float16))


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_gp_over_a_feature_map(gpb_lib, tmp_path, dtype):
    """200 input columns, beyond the 64 a kernel takes; fit, predict, save and load."""
    from mojogp_b200 import SingleOutputGP
    rng = np.random.default_rng(3)
    X = rng.standard_normal((400, 200)).astype(np.float32)
    y = np.tanh(X[:, 0] + 0.5 * X[:, 1]).astype(np.float32)
    fm = FeatureMap([32, 4], dropout=0.1, dtype=dtype)
    gp = SingleOutputGP(RBF(), feature_map=fm)
    tr = gp.fit(X[:300], y[:300], max_iterations=8, learning_rate=0.02, method="matrix_free")
    assert tr.iterations == 8 and np.all(np.isfinite(tr.nll_history))
    assert any(np.any(a != b) for a, b in zip(fm.parameters, FeatureMap([32, 4]).build(200).parameters))
    mean, std = gp.predict(X[300:], return_std=True)
    assert mean.shape == (100,) and np.all(np.isfinite(mean)) and np.all(std > 0)
    # The GP over the map is the plain GP over the map's outputs with the same parameters.
    feats = fm.transform(X)
    K = ok.kernel_matrix(gp.kernel.to_spec(4), tr.params, feats[:300].astype(np.float64))
    Ks = ok.kernel_matrix(gp.kernel.to_spec(4), tr.params, feats[300:].astype(np.float64),
                          feats[:300].astype(np.float64))
    mu = Ks @ np.linalg.solve(K + tr.noise * np.eye(300), y[:300] - tr.mean) + tr.mean
    assert np.sqrt(np.mean((mean - mu) ** 2)) < 2e-2  # the alpha solve stops at 1e-3
    _, var = gp.predict(X[300:310], return_var=True, variance_method="exact")
    assert np.all(var > 0)
    gp.save(str(tmp_path / "m"))
    again = SingleOutputGP.load(str(tmp_path / "m"))
    assert again.feature_map.dtype == dtype
    mean2, _ = again.predict(X[300:], return_std=True)
    np.testing.assert_allclose(mean2, mean, rtol=0, atol=2e-3)


def test_gp_over_a_feature_map_options(gpb_lib):
    from mojogp_b200 import fit_gp
    rng = np.random.default_rng(5)
    X = rng.standard_normal((150, 10)).astype(np.float32)
    y = X[:, 0].astype(np.float32)
    gp = fit_gp(X, y, Matern52(ard=True), feature_map=FeatureMap([6]), max_iterations=6,
                lr_schedule="cosine", feature_learning_rate=0.005, enable_early_stopping=True,
                early_stop_patience=2, early_stop_tol=1e9)
    assert gp.training_result.converged and gp.training_result.iterations == 3
    gp.fit(X, y, max_iterations=2, observation_noise=np.full(150, 0.05, np.float32), learn_noise=False)
    assert gp.noise == 0.0
    assert gp.score(X, y) <= 1.0
