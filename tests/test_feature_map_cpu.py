"""FeatureMap and its training loop on the host: the library's calls are stood in for by host memory and by
operators that compute nothing, so that what the Python layer does around them shows without a GPU."""
import ctypes as C
import gc

import numpy as np
import pytest

from mojogp_b200 import _lib, engine, features
from mojogp_b200.feature_map import FeatureMap
from mojogp_b200.kernel import RBF
from mojogp_b200.provider import DeviceBuffer, Provider


class HostCalls:
    """Stands in for _lib.call: allocations and copies in host memory, size queries by the library itself,
    operators and provider calls by nothing. `word` is what the device's error word holds."""

    def __init__(self, real):
        self.real, self.word, self.names, self.memory = real, 0, [], {}

    def __call__(self, name, *args):
        self.names.append(name)
        if name.endswith("_workspace"):
            return self.real(name, *args)
        if name == "gpb_device_alloc":
            block = np.zeros(args[1], np.uint8)
            self.memory[block.ctypes.data] = block
            args[2]._obj.value = block.ctypes.data
        elif name in ("gpb_memcpy_h2d", "gpb_memcpy_d2h"):
            C.memmove(args[1], args[2], args[3])
        elif name == "gpb_feature_status":
            args[1]._obj.value, self.word = self.word, 0
        elif name == "gpb_provider_create":
            args[-1]._obj.value = 1
        elif name == "gpb_get_noise":
            args[1]._obj.value = 0.1


@pytest.fixture()
def host(gpb_lib, monkeypatch):
    calls = HostCalls(_lib.call)
    monkeypatch.setattr(_lib, "call", calls)

    def no_lib():
        raise RuntimeError("the library is stood in for")

    monkeypatch.setattr(_lib, "lib", no_lib)
    yield calls
    gc.collect()  # buffers and providers go while they are stood in for


def gave_up(fn, *a, **kw):
    with pytest.raises(_lib.GPBError, match="gave up") as e:
        fn(*a, **kw)
    assert e.value.status == _lib.ERR_DEVICE


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_a_wait_that_gave_up_raises(host, dtype):
    fm = FeatureMap([6, 3], dropout=0.2, dtype=dtype).build(5)
    X = np.ones((7, 5), np.float32)
    assert fm.transform(X).shape == (7, 3)
    host.word = 1
    gave_up(fm.transform, X)
    grad = DeviceBuffer.from_host(np.ones((7, 3), np.float32))
    fm.forward(fm.upload(X), training=True)
    assert len(fm.backward(grad)) == len(fm.parameters)
    fm.forward(fm.upload(X), training=True)
    host.word = 1
    gave_up(fm.backward, grad)


def fit(fm, provider, X, iterations, **kw):
    return engine.train_features(provider, fm, X, np.zeros(X.shape[0], np.float32),
                                 max_iterations=iterations, num_probes=2, **kw)


@pytest.mark.parametrize("at", [0, 1, 2, 3, 4])
def test_training_ends_where_a_wait_gave_up(host, monkeypatch, at):
    """Whichever check of the loop sees the word, the weights it would have moved stay as they were."""
    fm = FeatureMap([4, 2]).build(5)
    X = np.ones((6, 5), np.float32)
    prov = Provider(np.zeros((6, 2), np.float32), RBF(), np.ones(2, np.float32), 0.1)
    checks = []
    real = features.check_device

    def check(device=0):
        checks.append(fm.snapshot())
        host.word = int(len(checks) == at + 1)
        real(device)

    monkeypatch.setattr(features, "check_device", check)
    with pytest.raises(_lib.GPBError):
        fit(fm, prov, X, 2)
    assert len(checks) == at + 1
    if at < 4:  # two checks a step, before the step's own update
        assert all(np.array_equal(a, b) for a, b in zip(fm.parameters, checks[-1]))
    prov.handle = None


# ------------------------------------------------------------- the training loop's rules
def script(seed, count, nan_at, params, shapes):
    """What `count` steps find: NLLs (NaN at nan_at), gradients, some beyond the clip or not finite."""
    rng = np.random.default_rng(seed)
    steps = []
    for i in range(count):
        g = rng.standard_normal(params + 1) * 3
        g[i % (params + 1)] *= 100  # clipped before the softplus factor
        if i == 1:
            g[0] = np.nan
        if i == 4:
            g[1] = np.inf
        maps = [rng.standard_normal(s) * (200 if i % 3 == 0 else 1) for s in shapes]
        steps.append(dict(nll=float("nan") if i in nan_at else 5.0 - i + (3.0 if i == 2 else 0.0), grads=g,
                          mean_grad=[0.7, -250.0, float("nan")][i % 3], cg_iters=1, maps=maps))
    return steps


def restated(steps, raw, mean, weights, lr, flr, cosine, init_mean):
    """The rules of the library's own loop (gpb_train) with the map's weights beside: the state that each
    step starts from, and the best one."""
    clip = lambda g: 0.0 if g != g or abs(g) > 1e30 else max(-100.0, min(100.0, g))
    vec = np.concatenate([raw, [mean]] + [w.ravel() for w in weights]).astype(np.float64)
    k = len(raw)
    m, v, t = np.zeros_like(vec), np.zeros_like(vec), 0
    best, seen, half, states = (1e30, vec.copy(), m.copy(), v.copy(), 0), [], 1.0, []
    for i, s in enumerate(steps):
        states.append(vec.copy())
        if np.isnan(s["nll"]):
            half *= 0.5
            _, vec, m, v, t = best
            vec, m, v = vec.copy(), m.copy(), v.copy()
            continue
        if s["nll"] < best[0]:
            best = (s["nll"], vec.copy(), m.copy(), v.copy(), t)
        g = np.concatenate([s["grads"], [s["mean_grad"]]] + [a.ravel() for a in s["maps"]])
        g = np.array([clip(float(x)) for x in g])
        g[:k] *= 1 / (1 + np.exp(-vec[:k]))
        t += 1
        m, v = 0.9 * m + 0.1 * g, 0.999 * v + 0.001 * g * g
        rate = np.full(vec.shape, lr)
        rate[k + 1:] = flr
        low = 1 / 20
        rate *= low + 0.5 * (1 - low) * (1 + np.cos(np.pi * i / len(steps))) if cosine else half
        vec = vec - rate * (m / (1 - 0.9 ** t)) / (np.sqrt(v / (1 - 0.999 ** t)) + 1e-8)
        vec[:k] = np.clip(vec[:k], -20, 20)
        if not abs(vec[k]) <= 1000:
            vec[k] = init_mean
    return states, best


@pytest.mark.parametrize("cosine", [False, True])
@pytest.mark.parametrize("nan_at", [(), (0,), (3,), (3, 4, 7)])
@pytest.mark.parametrize("lr", [0.05, 400.0])  # the second one drives the mean away
def test_training_moves_as_the_library_does(host, monkeypatch, nan_at, cosine, lr):
    fm = FeatureMap([3, 2], seed=2).build(4)
    X = np.random.default_rng(0).standard_normal((6, 4)).astype(np.float32)
    prov = Provider(np.zeros((6, 2), np.float32), RBF(), np.array([0.8, 1.3], np.float32), 0.1)
    start = fm.snapshot()
    steps = script(3, 9, nan_at, prov.num_params, [p.shape for p in start])
    states, at = [], iter(steps)
    now = {}

    def step(provider, y, x_grad, **kw):
        now.update(next(at))
        states.append(np.concatenate([np.append(provider.params, provider._noise), [-float(y[0])]]
                                     + [p.ravel() for p in fm.parameters]).astype(np.float64))
        return {k: now[k] for k in ("nll", "grads", "mean_grad", "cg_iters")}

    monkeypatch.setattr(engine, "bbmm_inputs", step)
    monkeypatch.setattr(fm, "backward", lambda grad: now["maps"])
    out = fit(fm, prov, X, len(steps), learning_rate=lr, feature_learning_rate=0.01, use_cosine_lr=cosine,
              init_mean=0.5)
    softplus = lambda r: np.logaddexp(0.0, r)
    raw = np.log(np.expm1(np.array([0.8, 1.3, 0.1], np.float32).astype(np.float64)))
    want, best = restated(steps, raw, 0.5, start, lr, 0.01, cosine, 0.5)
    for i, (got, ref) in enumerate(zip(states, want, strict=True)):
        # float32 weights and parameters: a rounding per step of each
        ref = np.concatenate([softplus(ref[:3]), ref[3:]])
        np.testing.assert_allclose(got, ref, rtol=20 * 2.0 ** -24, atol=20 * 2.0 ** -24 * (1 + 0.05 * lr),
                                   err_msg=str(i))
    assert out["final_nll"] == best[0] and out["iterations"] == len(steps)
    np.testing.assert_allclose(out["params"], softplus(best[1][:2]), rtol=2e-6)
    np.testing.assert_allclose(np.concatenate([p.ravel() for p in fm.parameters]), best[1][4:], rtol=2e-6,
                               atol=2e-6)
    assert abs(out["mean"] - best[1][3]) < 1e-4
    assert len(out["iter_times_ms"]) == len(steps)
    prov.handle = None


def test_training_skips_a_nan_in_the_early_stop_count(host, monkeypatch):
    fm = FeatureMap([2]).build(4)
    X = np.ones((6, 4), np.float32)
    prov = Provider(np.zeros((6, 2), np.float32), RBF(), np.ones(2, np.float32), 0.1)
    nlls = iter([3.0, float("nan"), float("nan"), 4.0, float("nan"), 5.0, 6.0])
    zero = dict(grads=np.zeros(3), mean_grad=0.0, cg_iters=1)
    monkeypatch.setattr(engine, "bbmm_inputs", lambda *a, **kw: dict(zero, nll=next(nlls)))
    monkeypatch.setattr(fm, "backward", lambda grad: [np.zeros(p.shape) for p in fm.parameters])
    out = fit(fm, prov, X, 7, enable_early_stopping=True, early_stop_patience=2)
    assert out["converged"] and out["iterations"] == 6
    prov.handle = None


# ------------------------------------------------------------- whose weights a result has
def test_a_model_refuses_another_fits_weights(host, monkeypatch, tmp_path):
    """Two models over one map: the first one's training inputs came from weights that the second one's fit
    moved, so its answers would mix both."""
    from mojogp_b200 import SingleOutputGP
    monkeypatch.setattr(engine, "bbmm_inputs", lambda provider, *a, **kw: dict(
        nll=1.0, grads=np.ones(provider.num_params + 1), mean_grad=0.1, cg_iters=1))
    fm = FeatureMap([4, 2])
    rng = np.random.default_rng(0)
    X, y = rng.standard_normal((8, 5)).astype(np.float32), np.ones(8, np.float32)
    one, two = SingleOutputGP(RBF(), feature_map=fm), SingleOutputGP(RBF(), feature_map=fm)
    one.fit(X, y, max_iterations=2, method="matrix_free")
    one._check_map()
    one.save(str(tmp_path / "one"))
    two.fit(X, y, max_iterations=2, method="matrix_free")
    two._check_map()
    for call in (lambda: one.predict(X), lambda: one.predict(X, return_std=True),
                 lambda: one.score(X, y), lambda: one.save(str(tmp_path / "again"))):
        with pytest.raises(RuntimeError, match="weights changed"):
            call()
    fm.restore(fm.snapshot())
    with pytest.raises(RuntimeError, match="weights changed"):
        two.predict(X)
    loaded = SingleOutputGP.load(str(tmp_path / "one"))
    loaded._check_map()
    one._provider.handle = None
    one.fit(X, y, max_iterations=1, method="matrix_free")
    one._check_map()
    for gp in (one, two, loaded):
        gp._provider.handle = None


def test_backward_needs_the_weights_of_its_forward(host):
    fm = FeatureMap([3, 2]).build(4)
    grad = DeviceBuffer.from_host(np.ones((5, 2), np.float32))
    fm.forward(fm.upload(np.ones((5, 4), np.float32)), training=True)
    fm.backward(grad)
    fm.parameters[2] += 1.0
    fm.parameters_changed()
    with pytest.raises(RuntimeError, match="forward"):
        fm.backward(grad)


# ------------------------------------------------------------- device memory
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_predictions_take_no_training_memory(host, dtype):
    fm = FeatureMap([256, 8], dtype=dtype).build(20)
    backward = max(features.gated_unit_workspace(3000, k, n, dtype, backward=True)
                   for k, n in ((20, 256), (256, 8)))
    forward = max(features.gated_unit_workspace(3000, k, n, dtype) for k, n in ((20, 256), (256, 8)))
    assert forward < backward
    host.memory.clear()
    fm.transform(np.zeros((3000, 20), np.float32))
    assert fm._run["workspace"].nbytes == forward
    kept = fm._run["layers"][0]["out"].ptr
    fm.transform(np.zeros((3000, 20), np.float32))
    assert fm._run["layers"][0]["out"].ptr == kept  # a small prediction's buffers serve the next one
    grad = DeviceBuffer.from_host(np.zeros((3000, 8), np.float32))
    fm.forward(fm.upload(np.zeros((3000, 20), np.float32)), training=True)
    assert fm._run["workspace"].nbytes >= backward and fm._run["layers"][0]["out"].ptr == kept
    fm.backward(grad)
    wide = FeatureMap([512, 8], dtype=dtype).build(300)
    wide.transform(np.zeros((40000, 300), np.float32))
    assert wide._run is None  # some 100 MB go back
