"""Forms that the operators' other tests do not reach: element indices past the generator's first counter
word, and the input gradient of a preconditioned step."""
import math

import numpy as np
import pytest

from mojogp_b200 import engine
from mojogp_b200.kernel import RBF, Matern32, Matern52
from mojogp_b200.provider import DeviceBuffer, Provider

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def give_memory_back():
    yield
    if torch.cuda.memory_reserved() > 8 << 30:
        torch.cuda.empty_cache()


def philox_words(first_block, blocks, seed, offset):
    """Philox4x32-10 in NumPy uint64, from any block."""
    lo, s32 = np.uint64(0xFFFFFFFF), np.uint64(32)
    blk = np.arange(first_block, first_block + blocks, dtype=np.uint64)
    c = [blk & lo, blk >> s32, np.full_like(blk, offset & 0xFFFFFFFF), np.full_like(blk, offset >> 32)]
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(10):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> s32) ^ c[1] ^ np.uint64(k0), p1 & lo, (p0 >> s32) ^ c[3] ^ np.uint64(k1), p0 & lo]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return np.stack(c, 1).reshape(-1)


@pytest.mark.parametrize("cols", [1 << 14, (1 << 14) - 3])
def test_dropout_of_more_than_2_32_blocks(gpb_lib, cols):
    """2^34 elements and more: the last rows' blocks reach the counter's second word, and their offsets
    pass 32 bits."""
    from mojogp_b200 import features as ft
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB of device memory")
    rows = (1 << 34) // cols + 3
    x = torch.empty((rows, cols), dtype=torch.bfloat16, device="cuda")
    x[-8:] = 1.0
    p, seed, offset = 0.25, 0x0123_4567_89AB_CDEF, 77
    ft.dropout(x, x, p, seed, offset=offset)
    first = (rows - 8) * cols
    assert first < 1 << 34 < first + 7 * cols
    words = philox_words(first // 4, 2 * cols + 2, seed, offset)[first % 4:][:8 * cols]
    keep = torch.from_numpy(words >= np.uint64(math.floor(p * 2 ** 32))).cuda().view(8, cols)
    want = torch.where(keep, torch.tensor(1 / (1 - p), device="cuda").to(torch.bfloat16), 0.0)
    assert torch.equal(x[-8:], want.to(torch.bfloat16))


@pytest.mark.parametrize("rank", [0, 5, 60])
@pytest.mark.parametrize("name", ["rbf", "m32", "m52"])
@pytest.mark.parametrize("P", [3, 18])
def test_input_gradient_of_a_preconditioned_step(gpb_lib, name, rank, P):
    """k depends on x / l, so for one lengthscale sum_i x_i' dNLL/dx_i = -l dNLL/dl, probes and
    preconditioner included: both sides are forms of the same solves. Each is a float32 sum of n^2
    terms over P + 1 columns, off by at most (n / 8 + 4 P + 60) 2^-23 of its magnitudes, which the
    gradient's own terms bound here: some 1e-3 of sum |x_i' dNLL/dx_i| with the probes' cancellation."""
    rng = np.random.default_rng(P + rank)
    n, d = 400, 2
    X = rng.uniform(-1, 1, (n, d)).astype(np.float32)
    y = np.sin(3 * X[:, 0] - X[:, 1]).astype(np.float32)
    k = {"rbf": RBF(), "m32": Matern32(), "m52": Matern52()}[name]
    params = np.array([0.6, 1.2], np.float32)
    prov = Provider(X, k, params, 0.2)
    grad = DeviceBuffer((n, d))
    kw = dict(num_probes=P, max_cg_iter=300, cg_tol=0.0, precond_rank=rank, iteration=3)
    res = engine.bbmm_inputs(prov, y, grad, **kw)
    plain = engine.bbmm(prov, y, **kw)
    assert res["nll"] == plain["nll"] and np.array_equal(res["grads"], plain["grads"])
    g = grad.download().astype(np.float64)
    pulls = (X * g).sum(1)
    assert np.abs(pulls).sum() > 0
    assert abs(pulls.sum() + params[0] * res["grads"][0]) < 1e-3 * np.abs(pulls).sum()
