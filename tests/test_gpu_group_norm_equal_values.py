"""Group norm of values that are all alike and no sum of powers of two: roundings of a long sum of them all go the same way."""
import numpy as np
import pytest

import norm_dense_muon as R
from dopt_amd import ops

pytestmark = pytest.mark.gpu
F32 = np.float32


# every form of the norm: rows, held groups, parts, runs of pixels, and the rest (rows of two values, more than 1024 channels of one value, more
# than 8192 channels last)
@pytest.mark.parametrize("n,c,h,w,groups,last", [
    (3, 96, 1, 1, 3, False), (2, 64, 32, 32, 2, False), (2, 64, 32, 32, 2, True), (1, 16, 300, 301, 1, False), (1, 12, 300, 301, 1, True), (1, 3000, 1, 1, 1, False),
    (2, 4000, 1, 2, 1, False), (1, 300000, 1, 3, 1, False), (1, 8448, 64, 64, 1, True), (1, 9000, 63, 65, 1, True)], ids=str)
def test_equal_values(n, c, h, w, groups, last):
    r = np.random.default_rng(c)
    value, eps = F32(0.1), 1e-5
    x = np.full((n, h, w, c) if last else (n, c, h, w), value)
    scale, bias = (1 + 0.2 * r.standard_normal(c)).astype(F32), (0.2 * r.standard_normal(c)).astype(F32)
    got = ops.group_norm(ops.tensor(x), ops.tensor(scale), ops.tensor(bias), groups, eps, "none", last).numpy()
    y, mean, rstd = got[:x.size].reshape(x.shape), got[x.size:x.size + n * groups], got[x.size + n * groups:]
    # a tree of short chains: some 40 additions in a row at most, which are off by half a step of the sum each, in any direction
    off = 40 * R.E * float(value)
    assert np.abs(mean - value).max() <= off
    exact = 1 / np.sqrt(np.float64(eps))   # (of off^2 beside eps nothing is left)
    assert np.abs(rstd - exact).max() <= 8 * R.E * exact
    per = (1, 1, 1, c) if last else (1, c, 1, 1)
    want, bound = bias.reshape(per).astype(np.float64), off * exact * np.abs(scale.reshape(per)) * 1.01 + 4 * R.E * np.abs(bias.reshape(per))
    assert (np.abs(y - want) <= bound).all(), np.abs(y - want).max()


# ... and of many samples, whose sums are added behind the gradient
@pytest.mark.parametrize("n,c,h,w,groups,last", [
    (1 << 20, 8, 1, 1, 2, False), ((1 << 20) + 9, 8, 1, 2, 1, True), ((1 << 20) + 5, 4, 2, 2, 1, False), ((1 << 20) + 5, 4, 1, 2, 1, False), ((1 << 20) + 5, 4, 1, 3, 1, True),
    (2, 64, 32, 32, 2, False), (2, 64, 32, 32, 2, True), (1, 16, 300, 301, 1, False), (1, 12, 300, 301, 1, True), (2, 4000, 1, 2, 1, False),
    (1, 300000, 1, 3, 1, False), (1, 8448, 64, 64, 1, True)], ids=str)
def test_equal_gradients(n, c, h, w, groups, last):
    """The bias' gradient is a sum of them."""
    r = np.random.default_rng(n + c)
    dy = np.full((n, h, w, c) if last else (n, c, h, w), F32(0.1))
    x = r.standard_normal(dy.shape, F32)
    one, stats = np.ones(c, F32), np.concatenate([np.zeros(n * groups, F32), np.ones(n * groups, F32)])
    got = ops.group_norm_grad(ops.tensor(dy), ops.tensor(x), ops.tensor(one), ops.tensor(np.zeros(c, F32)), ops.tensor(stats), groups, "none", last).numpy()
    dbias = got[x.size + c:].astype(np.float64)
    want = float(F32(0.1)) * n * h * w
    # chains of at most 256, 64 and 64 additions, one after the other, each off by half a step of its own sum
    assert np.abs(dbias / want - 1).max() <= 384 * R.E, np.abs(dbias / want - 1).max()


@pytest.mark.parametrize("c", [1028, 1027])
def test_equal_gradients_of_a_long_sample(c):
    """A thread's own sums: 16384 pixels of one channels-last sample."""
    n, inner = 1, 1 << 20
    x = ops.tensor(np.full((n, inner, c), F32(0.1)))
    one = ops.tensor(np.ones(c, F32))
    out = ops.group_norm_grad(x, x, one, ops.tensor(np.zeros(c, F32)), ops.tensor(np.array([0.0, 1.0], F32)), 1, "none", True)
    got, v = out.view(x.size, (2, c)).numpy().astype(np.float64), float(F32(0.1))
    # as above; a product is a rounding more
    assert np.abs(got[1] / (v * inner) - 1).max() <= 384 * R.E and np.abs(got[0] / (v * v * inner) - 1).max() <= 385 * R.E
