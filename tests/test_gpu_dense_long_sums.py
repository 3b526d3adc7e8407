"""Dense layers whose sums are long and of one sign: what every rounding adds shows there, where signs that vary hide it."""
import numpy as np
import pytest

from dopt_amd import capi, core, ops

pytestmark = pytest.mark.gpu
F32 = np.float32
E = 2.0 ** -24

# A sum of at most 4096 steps is formed by three instructions for every sixteen of them, each of which adds its products in two halves: 1536
# roundings of partial sums that grow evenly.  One is off by a value spread evenly over half a step either way (1 / sqrt(3) of it), half a
# step is E of a value between powers of two (0.74 of E in the root mean square), and evenly growing sums carry 1 / sqrt(3) of what
# the last one would: 0.58 x 0.74 x sqrt(1536 / 3) = 9.6 E in the root mean square.  Further parts of a sum only average.
RMS = 10 * E
# The instruction rounds down what lies below its guard bits; products of 16-bit values may drift by so much over 4096 steps
# (what the products of plain matrices are held to).
DRIFT = 2e-7


def _operand(r, shape, kind):
    v = r.random(shape, F32) if kind == "uniform" else np.maximum(r.standard_normal(shape, F32), 0)
    return np.ascontiguousarray(v, F32)


def _held(got, want, what):
    off = got.astype(np.float64) / want - 1
    mean, rms = off.mean(), np.sqrt((off * off).mean())
    assert abs(mean) <= DRIFT and rms <= RMS, "%s: off by %.3g on average, %.3g in the root mean square" % (what, mean, rms)


# both kinds of tiles: [2400 x 2411] and [4100 x 4096] are large ones, the others small
@pytest.mark.parametrize("kind", ["uniform", "relu"])
@pytest.mark.parametrize("size", [(2400, 2411, 1000), (2400, 2411, 17001), (4100, 4096, 8190), (2000, 2000, 4097), (2000, 2000, 20000), (1100, 1030, 9000),
                                  (700, 701, 1003)], ids=str)
def test_forward(size, kind):
    m, n, k = size
    r = np.random.default_rng(m + k)
    x, w = _operand(r, (m, k), kind), _operand(r, (n, k), kind)
    y = ops.dense_act(ops.tensor(x), ops.tensor(w)).numpy()
    _held(y, x.astype(np.float64) @ w.astype(np.float64).T, "y")


@pytest.mark.parametrize("kind", ["uniform", "relu"])
@pytest.mark.parametrize("size", [(2400, 9000, 2411), (9001, 2400, 2411), (20000, 2000, 1999), (1999, 20000, 2000), (1000, 1777, 1111)], ids=str)
def test_gradients(size, kind):
    m, n, k = size
    r = np.random.default_rng(m + n)
    dy, x, w = _operand(r, (m, n), kind), _operand(r, (m, k), kind), _operand(r, (n, k), kind)
    dx, dw, db = (t.numpy() for t in ops.dense_act_grad(ops.tensor(dy), ops.tensor(x), ops.tensor(w)))
    dy, x, w = (t.astype(np.float64) for t in (dy, x, w))
    _held(dx, dy @ w, "dx")
    _held(dw, dy.T @ x, "dw")
    _held(db, dy.sum(0), "dbias")


@pytest.mark.parametrize("size", [(1 << 18, 8192), (1 << 20, 1001), (1 << 20, 3)], ids=str)
def test_column_sums_of_equal_values(size):
    """Each column of one value, whose roundings all go the same way: chains of 64, 64 and 64 additions, each off by half a step of its sum."""
    m, n = size
    v = np.random.default_rng(3).uniform(0.05, 1.0, n).astype(F32)
    td = ops.tensor(np.broadcast_to(v, (m, n)))
    db = ops.Tensor((n,))
    capi.check(capi.load().dopt_hip_dense_act_grad(m, n, 1, 0, td.ptr, None, None, None, None, None, db.ptr))
    off = db.numpy().astype(np.float64) / (v.astype(np.float64) * m) - 1
    assert np.abs(off).max() <= 192 * E, np.abs(off).max()


@pytest.mark.parametrize("size", [(2400, 2411, 5000), (2001, 2000, 9001)], ids=str)
def test_values_that_are_not_finite(size):
    """They reach their row and column whichever pass they are in, and no others."""
    m, n, k = size
    r = np.random.default_rng(5)
    x, w = _operand(r, (m, k), "uniform"), _operand(r, (n, k), "uniform")
    # no zeros for an infinity to meet
    x[:, 4500], w[:, k - 1] = np.maximum(x[:, 4500], F32(1e-3)), np.maximum(w[:, k - 1], F32(1e-3))
    clean = ops.dense_act(ops.tensor(x), ops.tensor(w), act="relu").numpy()
    x[7, 3], x[m - 1, k - 1], w[n - 1, 4500] = np.nan, np.inf, np.inf
    y = ops.dense_act(ops.tensor(x), ops.tensor(w), act="relu").numpy()
    nan, inf = np.zeros((m, n), bool), np.zeros((m, n), bool)
    inf[m - 1], inf[:, n - 1] = True, True
    inf[7], nan[7] = False, True
    assert np.array_equal(np.isnan(y), nan) and np.array_equal(np.isposinf(y), inf)
    rest = ~(nan | inf)
    assert np.array_equal(y[rest], clean[rest])


@pytest.mark.parametrize("size", [(2400, 2411, 5000), (2000, 2000, 9001)], ids=str)
def test_recorded_passes(size):
    """Replays, with other users of the workspace between them, give the bits of the call."""
    m, n, k = size
    r = np.random.default_rng(6)
    x, w = _operand(r, (m, k), "relu"), _operand(r, (n, k), "uniform")
    vx, vw = core.float32([m, k]), core.float32([n, k], w)
    plan = core.compile([core.denseAct(vx, vw, None, None, "silu")], core.PLAN_VIEWS | core.PLAN_FUSE | core.PLAN_GRAPH)
    out = ops.tensor(np.full(m * n + 64, 3.0, F32))
    dev = {vx: ops.tensor(x)}
    want = ops.dense_act(dev[vx], ops.tensor(w), act="silu").numpy()
    for _ in range(4):
        out.set(np.full(out.shape, 3.0, F32))
        plan.execute(dev, [out.view(0, (m, n))])
        got = out.numpy()
        assert np.array_equal(got[:m * n].reshape(m, n), want) and (got[m * n:] == 3.0).all()
        ops.dense_act(ops.tensor(x[:900]), ops.tensor(w[:900]))
    assert plan.recordings()["replays"] >= 2
