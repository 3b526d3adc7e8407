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
