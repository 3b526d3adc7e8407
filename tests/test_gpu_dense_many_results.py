"""Dense layers of more rows or columns than one side of a launch counts threads for (2^32)."""
import numpy as np
import pytest

from dopt_amd import capi, ops

pytestmark = pytest.mark.gpu
F32 = np.float32


def _whole(r, shape):
    """Small whole numbers: products and sums of a few are exact."""
    return r.integers(-8, 9, shape, np.int8).astype(F32)


def test_a_wavefront_per_result():
    n = (1 << 26) + 5
    r = np.random.default_rng(1)
    v = _whole(r, (n, 2))
    want = (3 * v[:, 0] - 2 * v[:, 1]) + 1
    tv, tw, tb = ops.tensor(v), ops.tensor(np.array([[3.0, -2.0]], F32)), ops.tensor(np.ones(1, F32))
    assert np.array_equal(ops.dense_act(tv, tw, tb).numpy()[:, 0], want)
    assert np.array_equal(ops.dense_act(tw, tv, act="relu").numpy()[0], np.maximum(want - 1, 0))
    assert np.array_equal(ops.matmul_t(tv, tw, False, True).numpy()[:, 0], want - 1)


@pytest.mark.parametrize("rows", [1, 3])
def test_column_sums(rows):
    n = (1 << 27) + 3
    dy = _whole(np.random.default_rng(2), (rows, n))
    td, out = ops.tensor(dy), ops.tensor(np.full(n + 8, 99.0, F32))
    capi.check(capi.load().dopt_hip_dense_act_grad(rows, n, 1, 0, td.ptr, None, None, None, None, None, out.ptr))
    got = out.numpy()
    assert np.array_equal(got[:n], dy.sum(0)) and (got[n:] == 99.0).all()
