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
