"""Group norm, dense layer with activation and orthogonalised update on the device against their float64 forms."""
import ctypes as C
import math

import numpy as np
import pytest

import norm_dense_muon as R
from dopt_amd import capi, core, nnet, online, ops

pytestmark = pytest.mark.gpu
F32 = np.float32
E_TINY = 2.0 ** -149   # the last place of the smallest values


def _f(a):
    return np.asarray(a, F32)


def _off_grid(a):
    """A device copy that starts four bytes behind a 16-byte boundary."""
    t = ops.Tensor((a.size + 1,))
    v = t.view(1, a.shape)
    return v.set(a)


# ------------------------------------------------------------------------------------------------ group norm

# n, c, h, w, groups
NORMS = [(1, 1, 1, 1, 1), (1, 64, 8, 8, 8), (3, 6, 1, 1, 2), (2, 32, 1, 1, 1), (4, 12, 5, 7, 3), (2, 96, 4, 4, 32), (5, 7, 3, 11, 7), (5, 7, 3, 11, 1),
         (37, 40, 9, 3, 8), (1, 64, 64, 64, 2), (1, 16, 128, 129, 1), (2, 160, 32, 32, 32), (2, 640, 8, 8, 16), (3, 33, 31, 17, 3),
         (2, 1024, 2, 2, 4), (1, 2, 200, 200, 2), (300, 8, 2, 2, 4), (2, 24, 16, 17, 8), (1, 4, 300, 301, 1), (3, 200, 29, 33, 25)]


def _norm_case(n, c, h, w, last, seed, offset=0.5):
    r = np.random.default_rng(seed)
    shape, per = ((n, h, w, c), (1, 1, 1, c)) if last else ((n, c, h, w), (1, c, 1, 1))
    x = _f(r.standard_normal(shape) * (0.5 + r.random(per)) + offset * r.standard_normal(per))
    return x, _f(1 + 0.2 * r.standard_normal(c)), _f(0.2 * r.standard_normal(c)), _f(r.standard_normal(shape))


def _check_norm(x, scale, bias, groups, name, last, up=ops.tensor, eps=1e-5):
    got = ops.group_norm(up(x), up(scale), up(bias), groups, eps, name, last).numpy()
    y, mean, rstd = R.group_norm(x, scale, bias, groups, eps, name, last)
    s = x.shape[0] * groups
    R.close(got[:x.size], (y[0].ravel(), y[1].ravel()), "y")
    R.close(got[x.size:x.size + s], mean, "mean")
    R.close(got[x.size + s:], rstd, "rstd")
    return got[x.size:]


def _check_norm_grad(dy, x, scale, bias, groups, name, last, up=ops.tensor, eps=1e-5):
    _, (mean, _), (rstd, _) = R.group_norm(x, scale, bias, groups, eps, name, last)
    stats = _f(np.concatenate([mean, rstd]))
    s = len(mean)
    if name == "relu":   # where z is within a rounding of zero either answer is one
        z = R.group_norm(x, scale, bias, groups, eps, "none", last)[0][0]
        dy = np.where(np.abs(z) < 1e-3, F32(0), dy)
    got = ops.group_norm_grad(up(dy), up(x), up(scale), up(bias), up(stats), groups, name, last).numpy()
    c = len(scale)
    dx, ds, db = R.group_norm_grad(dy, x, scale, bias, stats[:s], stats[s:], groups, name, last)
    R.close(got[:x.size], (dx[0].ravel(), dx[1].ravel()), "dx")
    R.close(got[x.size:x.size + c], ds, "dscale")
    R.close(got[x.size + c:], db, "dbias")


@pytest.mark.parametrize("last", [False, True], ids=["first", "last"])
@pytest.mark.parametrize("size", NORMS, ids=lambda s: "x".join(map(str, s)))
def test_group_norm(size, last):
    n, c, h, w, groups = size
    x, scale, bias, dy = _norm_case(n, c, h, w, last, sum(size))
    name = R.ACTS[sum(size) % 4]
    _check_norm(x, scale, bias, groups, name, last)
    _check_norm_grad(dy, x, scale, bias, groups, name, last)


# groups of a power of two of channels, on both sides of what a workgroup holds of them forward (32768 values) and backward (16384)
HELD = [(2, 64, 30, 31, 8), (3, 48, 13, 19, 3), (2, 64, 11, 23, 2), (2, 128, 9, 29, 2), (3, 24, 1, 2, 3), (1, 8, 63, 65, 1), (2, 16, 45, 45, 2),
        (9, 8, 3, 3, 1), (2, 16, 64, 65, 2), (2, 16, 40, 45, 1), (2, 20, 16, 16, 1), (1, 12, 37, 37, 1),
        (2, 30, 39, 28, 3), (1, 40, 39, 28, 1), (1, 1, 100, 101, 1), (2, 6, 50, 52, 2), (3, 4, 63, 51, 2), (2, 64, 32, 33, 1),
        (2, 3, 40, 41, 3), (1, 520, 9, 7, 130), (40, 99, 1, 3, 3),
        (2, 8448, 9, 15, 12)]


@pytest.mark.parametrize("last", [False, True], ids=["first", "last"])
@pytest.mark.parametrize("size", HELD, ids=lambda s: "x".join(map(str, s)))
def test_group_norm_of_groups_that_a_workgroup_holds(size, last):
    n, c, h, w, groups = size
    x, scale, bias, dy = _norm_case(n, c, h, w, last, sum(size))
    for name, up in (("silu", ops.tensor), ("gelu", _off_grid)):
        _check_norm(x, scale, bias, groups, name, last, up)
        _check_norm_grad(dy, x, scale, bias, groups, name, last, up)


# one launch counts 2^32 threads along a side of its grid: whole groups, held ones, runs of pixels, rows, and the rest
@pytest.mark.parametrize("size,last", [((2 ** 20 + 3, 2, 2, 2, 1), False), ((2 ** 20 + 9, 8, 1, 2, 1), True), ((2 ** 20 + 5, 4, 1, 3, 1), True),
                                       ((2 ** 22 + 7, 8, 1, 1, 1), False), ((2 ** 20 + 5, 4, 1, 2, 1), False)], ids=str)
def test_group_norm_of_more_groups_than_a_row_of_a_grid(size, last):
    n, c, h, w, groups = size
    x, scale, bias, dy = _norm_case(n, c, h, w, last, 18)
    _check_norm(x, scale, bias, groups, "none", last)
    _check_norm_grad(dy, x, scale, bias, groups, "none", last)


def test_group_norm_gradient_of_more_than_the_caches_hold():
    x, scale, bias, dy = _norm_case(54, 256, 32, 64, True, 9)
    _check_norm_grad(dy, x, scale, bias, 32, "none", True)


@pytest.mark.parametrize("name", R.ACTS)
@pytest.mark.parametrize("last", [False, True], ids=["first", "last"])
def test_group_norm_activations_and_alignment(name, last):
    x, scale, bias, dy = _norm_case(3, 24, 6, 10, last, 5)
    scale[3], bias[3] = 0.0, -40.0   # a channel far below every activation's knee
    for up in (ops.tensor, _off_grid):
        _check_norm(x, scale, bias, 4, name, last, up)
        _check_norm_grad(dy, x, scale, bias, 4, name, last, up)


@pytest.mark.parametrize("last", [False, True], ids=["first", "last"])
def test_group_norm_of_values_far_from_zero_and_of_constants(last):
    x, scale, bias, dy = _norm_case(2, 16, 12, 12, last, 6)
    _check_norm(_f(x + 1000.0), scale, bias, 4, "silu", last)
    same = np.full_like(x, 3.0)   # variance zero: y = act(bias), dx of order 1 / sqrt(eps)
    got = ops.group_norm(ops.tensor(same), ops.tensor(scale), ops.tensor(bias), 4, 1e-5, "none", last).numpy()
    y = got[:x.size].reshape(x.shape)
    want = bias if last else bias[:, None, None]
    assert np.array_equal(y, np.broadcast_to(want, x.shape))
    _check_norm(_f(x * 1e-18), scale, bias, 4, "none", last)
    _check_norm(_f(x * 1e17), scale, bias, 4, "none", last)


@pytest.mark.parametrize("last", [False, True], ids=["first", "last"])
@pytest.mark.parametrize("size", [(4, 16, 8, 8, 4), (3, 16, 100, 101, 2)], ids=["small", "large"])
def test_group_norm_keeps_what_is_not_finite_in_its_group(size, last):
    n, c, h, w, groups = size
    x, scale, bias, _ = _norm_case(n, c, h, w, last, 7)
    clean = ops.group_norm(ops.tensor(x), ops.tensor(scale), ops.tensor(bias), groups, 1e-5, "relu", last).numpy()
    v = x.copy()
    at = (1, h - 1, w - 1, c - 1) if last else (1, c - 1, h - 1, w - 1)   # the last group of sample 1
    v[at] = np.nan
    got = ops.group_norm(ops.tensor(v), ops.tensor(scale), ops.tensor(bias), groups, 1e-5, "relu", last).numpy()
    hit = np.zeros((n, groups, c // groups * h * w), bool)
    hit[1, groups - 1] = True
    ids = R.ungrouped(hit, x.shape, last).ravel()
    assert np.isnan(got[:x.size][ids]).all() and np.array_equal(got[:x.size][~ids], clean[:x.size][~ids])


def test_group_norm_without_pixels_or_samples():
    z = ops.tensor(np.zeros((0,), F32).reshape(0, 8, 3))
    one, grad = ops.tensor(np.ones(8, F32)), ops.tensor(np.full(16, 7.0, F32))
    ops.group_norm_grad(z, z, one, one, ops.Tensor((0,)), 2, out=grad)
    assert np.array_equal(grad.numpy(), np.zeros(16, F32))   # dscale and dbias are sums of nothing
    assert ops.group_norm(z, one, one, 2).size == 0
    z = ops.Tensor((3, 8, 0))
    got = ops.group_norm(z, one, one, 2, 0.25).numpy()
    assert np.array_equal(got, np.repeat(_f([0.0, 2.0]), 6))


def test_group_norm_twice_and_beside_its_neighbours():
    """The same bits again, and nothing written behind the result."""
    for size, last in (((2, 32, 20, 20, 8), False), ((2, 32, 20, 20, 8), True), ((1, 8, 150, 150, 1), False), ((1, 8, 150, 150, 1), True)):
        n, c, h, w, groups = size
        x, scale, bias, dy = _norm_case(n, c, h, w, last, 8)
        tx, ts, tb, td = (ops.tensor(t) for t in (x, scale, bias, dy))
        pad = 64
        a = ops.tensor(np.full(x.size + 2 * n * groups + pad, 5.0, F32))
        ops.group_norm(tx, ts, tb, groups, 1e-5, "gelu", last, out=a.view(0, (a.size - pad,)))
        first = a.numpy()
        stats = ops.tensor(first[x.size:a.size - pad])
        b = ops.tensor(np.full(x.size + 2 * c + pad, 5.0, F32))
        ops.group_norm_grad(td, tx, ts, tb, stats, groups, "gelu", last, out=b.view(0, (b.size - pad,)))
        second = b.numpy()
        assert (first[-pad:] == 5.0).all() and (second[-pad:] == 5.0).all()
        ops.group_norm(tx, ts, tb, groups, 1e-5, "gelu", last, out=a.view(0, (a.size - pad,)))
        ops.group_norm_grad(td, tx, ts, tb, stats, groups, "gelu", last, out=b.view(0, (b.size - pad,)))
        assert np.array_equal(first, a.numpy()) and np.array_equal(second, b.numpy())


@pytest.mark.parametrize("last", [False, True], ids=["first", "last"])
def test_group_norm_past_32_bits(last):
    """A tensor of 2^31 values and more: its last sample, whose offsets do not fit 31 bits, against the sample by itself."""
    n, c, inner, groups = 65, 32, (1 << 20) + 3, 4
    x = ops.Tensor((n, inner, c) if last else (n, c, inner))
    capi.check(capi.load().dopt_hip_uniform(5, 0, x.size, x.ptr))
    r = np.random.default_rng(9)
    ts, tb = ops.tensor(_f(1 + 0.1 * r.standard_normal(c))), ops.tensor(_f(0.1 * r.standard_normal(c)))
    out = ops.Tensor((x.size + 2 * n * groups,))
    ops.group_norm(x, ts, tb, groups, 1e-5, "silu", last, out=out)
    one = c * inner
    for k in (0, n - 1):
        alone = ops.group_norm(x.view(k * one, (1,) + x.shape[1:]), ts, tb, groups, 1e-5, "silu", last)
        a, b = alone.view(0, (one,)), out.view(k * one, (one,))
        # another number of samples may cut the sums of a group elsewhere: 2^-20 of values near one
        assert ops.max_element(ops.pointwise("abs", ops.pointwise("sub", a, b))).numpy() < 1e-6
    stats = out.view(x.size, (2 * n * groups,))
    assert np.isfinite(stats.numpy()).all()
    g = ops.Tensor((x.size + 2 * c,))
    ops.group_norm_grad(x, x, ts, tb, stats, groups, "silu", last, out=g)
    s = stats.numpy().reshape(2, n, groups)[:, n - 1].ravel()
    last_x = x.view((n - 1) * one, (1,) + x.shape[1:])
    alone = ops.group_norm_grad(last_x, last_x, ts, tb, ops.tensor(s), groups, "silu", last)
    a, b = alone.view(0, (one,)), g.view((n - 1) * one, (one,))
    assert ops.max_element(ops.pointwise("abs", ops.pointwise("sub", a, b))).numpy() < 1e-4   # values to 12, 2^-18 of them


def test_group_norm_refusals():
    x, s = ops.Tensor((2, 6, 4)), ops.Tensor((6,))
    for bad in (lambda: ops.group_norm(x, s, s, 4), lambda: ops.group_norm(x, s, ops.Tensor((5,)), 3), lambda: ops.group_norm(s, s, s, 1),
                lambda: ops.group_norm(x, s, s, 3, act="tanh"), lambda: ops.group_norm(x, s, s, 3, out=x),
                lambda: ops.group_norm_grad(x, x, s, s, s, 3), lambda: ops.group_norm_grad(ops.Tensor((2, 6, 3)), x, s, s, ops.Tensor((12,)), 3),
                lambda: ops.group_norm(ops.Tensor((2, 6, 4), np.int32), s, s, 3)):
        with pytest.raises(capi.HipError):
            bad()


# ------------------------------------------------------------------------------------------------ dense

# m, n, k
DENSES = [(1, 1, 1), (1, 10, 16), (1, 4096, 512), (1, 333, 1025), (2, 3, 5), (7, 64, 100), (33, 65, 127), (64, 512, 784), (130, 70, 1), (256, 10, 512),
          (300, 1, 77), (129, 257, 130), (512, 512, 512), (1000, 130, 260), (257, 300, 2050), (64, 2000, 1030), (520, 1030, 1500), (1024, 1024, 512), (1030, 1100, 530),
          (1300, 1281, 1111), (2560, 2304, 512), (2497, 2370, 131), (2370, 2497, 400),
          (1024, 1024, 2100), (300, 2001, 2000)]


def _dense_case(m, n, k, seed):
    r = np.random.default_rng(seed)
    return (_f(r.standard_normal((m, k))), _f(r.standard_normal((n, k)) * math.sqrt(2.0 / k)), _f(r.standard_normal(n)),
            _f(r.standard_normal((m, n))), _f(r.standard_normal((m, n))))


@pytest.mark.parametrize("size", DENSES, ids=lambda s: "x".join(map(str, s)))
def test_dense_act(size):
    m, n, k = size
    x, w, b, res, dy = _dense_case(m, n, k, sum(size))
    for i, name in enumerate(R.ACTS):
        bias, residual = (b if i != 1 else None), (res if i % 2 else None)
        up = _off_grid if i == 3 else ops.tensor
        pre = ops.Tensor((m, n)) if i else None
        y = ops.dense_act(up(x), up(w), None if bias is None else up(bias), None if residual is None else up(residual), name, pre=pre)
        want_y, want_pre = R.dense_act(x, w, bias, residual, name)
        R.close(y.numpy(), want_y, name + " y")
        if pre is None:
            continue
        kept = pre.numpy()
        R.close(kept, want_pre, name + " pre")
        again = ops.dense_act(up(x), up(w), None if bias is None else up(bias), None if residual is None else up(residual), name)
        assert np.array_equal(again.numpy(), y.numpy())   # whether pre is kept changes nothing
        g = np.where(np.abs(kept) < 1e-3, F32(0), dy) if name == "relu" else dy
        got = ops.dense_act_grad(up(g), up(x), up(w), up(kept), name)
        for t, v, what in zip(got, R.dense_act_grad(g, x, w, kept, name), ("dx", "dw", "dbias")):
            R.close(t.numpy(), v, name + " " + what)
    got = ops.dense_act_grad(ops.tensor(dy), ops.tensor(x), ops.tensor(w))
    for t, v, what in zip(got, R.dense_act_grad(dy, x, w, None, "none"), ("dx", "dw", "dbias")):
        R.close(t.numpy(), v, what)


def test_dense_act_parts_of_the_gradient_and_neighbours():
    m, n, k = 140, 90, 200
    x, w, b, res, dy = _dense_case(m, n, k, 11)
    tx, tw, td, tp = (ops.tensor(t) for t in (x, w, dy, res))
    whole = [t.numpy() for t in ops.dense_act_grad(td, tx, tw, tp, "silu")]
    lib, act = capi.load(), capi.ACTIVATIONS["silu"]
    for i, shape in enumerate(((m, k), (n, k), (n,))):
        size = int(np.prod(shape))
        out = ops.tensor(np.full(size + 16, 3.0, F32))
        ptrs = [out.ptr if j == i else None for j in range(3)]
        capi.check(lib.dopt_hip_dense_act_grad(m, n, k, act, td.ptr, tp.ptr, tx.ptr if i == 1 else None, tw.ptr if i == 0 else None, *ptrs))
        got = out.numpy()
        assert np.array_equal(got[:size].reshape(shape), whole[i]) and (got[size:] == 3.0).all()
    y = ops.tensor(np.full(m * n + 16, 3.0, F32))
    pre = ops.tensor(np.full(m * n + 16, 3.0, F32))
    ops.dense_act(tx, tw, ops.tensor(b), tp, "gelu", out=y.view(0, (m, n)), pre=pre.view(0, (m, n)))
    assert (y.numpy()[m * n:] == 3.0).all() and (pre.numpy()[m * n:] == 3.0).all()


def test_dense_act_of_nothing():
    b, res = _f([1.0, -2.0, 3.0]), _f(np.arange(6).reshape(2, 3))
    y = ops.dense_act(ops.Tensor((2, 0)), ops.Tensor((3, 0)), ops.tensor(b), ops.tensor(res), "relu")
    assert np.array_equal(y.numpy(), np.maximum(b, 0) + res)
    assert ops.dense_act(ops.Tensor((0, 4)), ops.Tensor((3, 4))).size == 0
    dx, dw, db = ops.dense_act_grad(ops.Tensor((0, 3)), ops.Tensor((0, 4)), ops.Tensor((3, 4)), dw=ops.tensor(np.full((3, 4), 2.0, F32)),
                                    dbias=ops.tensor(np.full(3, 2.0, F32)))
    assert dx.size == 0 and not dw.numpy().any() and not db.numpy().any()


@pytest.mark.parametrize("size", [(1, 64, 300), (40, 50, 300), (300, 300, 300), (300, 520, 1200), (1030, 1100, 530), (1030, 1100, 1000), (2500, 2403, 140)], ids=str)
def test_dense_act_with_values_that_are_not_finite(size):
    m, n, k = size
    x, w, b, res, _ = _dense_case(m, n, k, 12)
    x[m - 1, 3], w[5, 7], res[0, 9] = np.nan, np.inf, -np.inf
    x[:, 7] = np.abs(x[:, 7]) + 0.1
    y = ops.dense_act(ops.tensor(x), ops.tensor(w), ops.tensor(b), ops.tensor(res), "relu").numpy()
    clean = R.dense_act(np.nan_to_num(x), np.where(np.isinf(w), 0, w), b, np.where(np.isinf(res), 0, res), "relu")
    want = clean[0][0].copy()
    want[:, 5] = np.inf
    want[0, 9] = -np.inf
    want[m - 1] = np.nan
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(y), np.isnan(want)) and np.array_equal(y[np.isinf(want)], want[np.isinf(want)])
    R.close(y[fine], (want[fine], clean[0][1][fine]), "finite values")


def test_dense_act_of_large_layers_with_rows_of_any_size():
    """Rows 2^160 apart, rows of zeros, and rows whose largest value meets zeros only: what is below 2^-40 of it may be lost."""
    m, n, k = 2401, 2562, 640
    r = np.random.default_rng(14)
    x, w, _, _, _ = _dense_case(m, n, k, 13)
    x = _f(x * 2.0 ** r.integers(-80, 41, (m, 1)))
    w = _f(w * 2.0 ** r.integers(-40, 41, (n, 1)))
    x[3], w[7] = 0.0, 0.0
    y = ops.dense_act(ops.tensor(x), ops.tensor(w), act="none").numpy()
    want, bound = R.product(x, w)
    R.close(y, (want, bound + E_TINY), "rows of any size")
    x[:, 5], w[:, 5] = np.abs(x).max(1) * F32(2.0 ** 26), 0.0
    y = ops.dense_act(ops.tensor(x), ops.tensor(w), act="none").numpy()
    want, bound = R.product(x, w)
    top = np.outer(np.abs(x).max(1).astype(np.float64), np.abs(w).max(1).astype(np.float64))
    R.close(y, (want, bound + 2.0 ** -39 * k * top + E_TINY), "rows of small values and a large one")


def test_dense_act_of_long_rows():
    m, n, k = 2368, 2504, 17001
    x, w, b, _, _ = _dense_case(m, n, k, 15)
    x[:, 17000] += F32(300.0)   # the largest value is the last one
    y = ops.dense_act(ops.tensor(x), ops.tensor(w), ops.tensor(b), act="silu").numpy()
    R.close(y, R.dense_act(x, w, b, None, "silu")[0], "y")


@pytest.mark.parametrize("size", [(2400, 2411, 2421), (2563, 300, 2500), (2499, 2305, 130), (1000, 1777, 1111)], ids=str)
def test_dense_act_gradient_of_large_layers(size):
    m, n, k = size
    x, w, _, pre, dy = _dense_case(m, n, k, 16)
    x = _f(x * 2.0 ** np.random.default_rng(17).integers(-20, 21, (1, k)))   # each column of its own size
    for name, up in (("silu", ops.tensor), ("none", _off_grid)):
        got = ops.dense_act_grad(up(dy), up(x), up(w), up(pre), name)
        for t, v, what in zip(got, R.dense_act_grad(dy, x, w, pre, name), ("dx", "dw", "dbias")):
            R.close(t.numpy(), v, name + " " + what)
    x[5, 7], dy[9, 11] = np.inf, np.nan
    dy[5] = np.abs(dy[5]) + F32(0.1)
    with np.errstate(invalid="ignore"):
        dx, dw = (t.numpy() for t in ops.dense_act_grad(ops.tensor(dy), ops.tensor(x), ops.tensor(w))[:2])
    want_x, want_w = np.zeros((m, k), bool), np.zeros((n, k), bool)
    want_x[9], want_w[11] = True, True
    assert np.array_equal(np.isnan(dx), want_x) and np.array_equal(np.isnan(dw), want_w)
    want_w[:, 7] ^= True
    want_w[11] = False
    assert np.array_equal(np.isposinf(dw), want_w) and not np.isinf(dx).any()


def test_dense_act_refusals():
    x, w, y = ops.Tensor((4, 6)), ops.Tensor((5, 6)), ops.Tensor((4, 5))
    for bad in (lambda: ops.dense_act(x, ops.Tensor((5, 7))), lambda: ops.dense_act(x, w, ops.Tensor((4,))), lambda: ops.dense_act(x, w, None, x),
                lambda: ops.dense_act(x, w, None, y, out=y), lambda: ops.dense_act(x, w, act="elu"), lambda: ops.dense_act(x, w, out=ops.Tensor((4, 4))),
                lambda: ops.dense_act_grad(y, x, w, None, "gelu"), lambda: ops.dense_act_grad(x, x, w),
                lambda: ops.dense_act(ops.Tensor((4, 6), np.int32), w), lambda: ops.dense_act(x, w, pre=ops.Tensor((4, 4)))):
        with pytest.raises(capi.HipError):
            bad()


# ------------------------------------------------------------------------------------------------ muon

def _matrix(r, shape, kind="plain"):
    g = r.standard_normal(shape)
    if kind == "weak":     # rank 2, and the rest a millionth of it
        v = g.reshape(shape[0], -1)
        u, s, vt = np.linalg.svd(v, full_matrices=False)
        s[2:] *= 1e-6
        g = ((u * s) @ vt).reshape(shape)
    return _f(1e-3 * g)


def _run_muon(shapes, iterations, nesterov=True, seed=0, kind="plain", up=ops.tensor):
    """w starts at zero and lr is one, so the new w is the orthogonalised matrix and its bound holds for w itself."""
    r = np.random.default_rng(seed)
    g, m = [_matrix(r, s, kind) for s in shapes], [_matrix(r, s, kind) for s in shapes]
    w = [np.zeros(s, F32) for s in shapes]
    tw, tg, tm = ([up(t) for t in v] for v in (w, g, m))
    opt = ops.MuonOptimizer(tw, tg, tm)
    opt.step(1.0, 0.75, nesterov, 0.0, iterations)
    for i, s in enumerate(shapes):
        want, mom, o = R.muon(w[i], g[i], m[i], 1.0, 0.75, nesterov, 0.0, iterations)
        R.close(tm[i].numpy(), (mom, 2 * R.E * (np.abs(0.75 * m[i].astype(float)) + np.abs(mom))), "momentum of %s" % (s,))
        off = np.linalg.norm(tw[i].numpy().astype(np.float64) - want) / max(np.linalg.norm(o), 1e-300)
        assert off <= R.muon_bound(iterations), (s, off, R.muon_bound(iterations))
        assert np.array_equal(tg[i].numpy(), g[i])


MUONS = [[(1, 1)], [(1, 7)], [(9, 1)], [(2, 3)], [(64, 576)], [(576, 64)], [(64, 27)], [(10, 512)], [(33, 65), (65, 33), (31, 31)], [(130, 1030)],
         [(300, 257), (16, 16), (1, 5), (512, 10)], [(64, 3, 3, 3), (64, 64, 3, 3), (128, 64)], [(640, 320), (20, 5000)], [(1030, 700)]]


@pytest.mark.parametrize("iterations", [0, 1, 5])
@pytest.mark.parametrize("shapes", MUONS, ids=lambda s: ",".join("x".join(map(str, t)) for t in s))
def test_muon(shapes, iterations):
    _run_muon(shapes, iterations, seed=len(shapes) + iterations)


@pytest.mark.parametrize("iterations", [1, 2, 3, 5])
def test_muon_of_many_matrices(iterations):
    """More tiles than compute units, of matrices of many sizes; each moves as it does alone."""
    shapes = [(64, 27), (64, 576), (128, 576), (256, 1152), (256, 2304), (512, 600), (512, 512), (10, 512)] + [(64, 130)] * 200 + [(200, 130)] * 20
    _run_muon(shapes, iterations, seed=iterations)


def test_muon_of_large_matrices():
    """More tiles of X than compute units: sides of odd numbers of 128 rows, and a side of at most 64 among them."""
    _run_muon([(300, 9000), (9000, 700), (40, 5001), (515, 900), (64, 64), (1000, 130)], 5, seed=11)
    _run_muon([(300, 9000), (9001, 700), (40, 5000)], 2, False, 12, up=_off_grid)


@pytest.mark.parametrize("kind", ["plain", "weak"])
@pytest.mark.parametrize("nesterov", [False, True])
def test_muon_momenta_alignment_and_weak_directions(nesterov, kind):
    _run_muon([(96, 200), (70, 35)], 3, nesterov, 4, kind)
    _run_muon([(96, 200), (70, 35)], 3, nesterov, 4, kind, up=_off_grid)


def test_muon_scales_decay_and_steps():
    """Three steps with decay, gradients of many sizes: their squares may leave the range of float32."""
    r = np.random.default_rng(5)
    shapes = [(40, 60), (60, 40), (24, 24)]
    for size in (1e-30, 1e-9, 1.0, 1e30):
        w, g = [_f(r.standard_normal(s)) for s in shapes], [_f(r.standard_normal(s) * size) for s in shapes]
        m = [np.zeros(s, F32) for s in shapes]
        tw, tg, tm = ([ops.tensor(t) for t in v] for v in (w, g, m))
        opt = ops.MuonOptimizer(tw, tg, tm)
        ref, mom = [t.astype(np.float64) for t in w], [t.astype(np.float64) for t in m]
        for _ in range(3):
            opt.step(0.1, 0.5, True, 0.2, 5)
            for i in range(3):
                ref[i], mom[i], _ = R.muon(ref[i], g[i], mom[i], 0.1, 0.5, True, 0.2, 5)
        for i in range(3):
            off = np.linalg.norm(tw[i].numpy() - ref[i])
            # three updates of norm 0.1 |O|, |O| at most 1.3 sqrt(24..40 directions) sqrt(1.5), plus the roundings of w
            assert off <= 3 * 0.1 * R.muon_bound(5) * 1.3 * math.sqrt(60) * 1.3 + 12 * R.E * np.linalg.norm(w[i]), (size, shapes[i], off)


def test_muon_of_zero_and_of_nan():
    r = np.random.default_rng(6)
    shapes = [(20, 30), (20, 30), (50, 20)]
    w, g, m = [_f(r.standard_normal(s)) for s in shapes], [_f(r.standard_normal(s)) for s in shapes], [np.zeros(s, F32) for s in shapes]
    g[0][:] = 0.0
    g[1][3, 4] = np.nan
    tw, tg, tm = ([ops.tensor(t) for t in v] for v in (w, g, m))
    ops.MuonOptimizer(tw, tg, tm).step(0.1, 0.9, True)
    assert np.array_equal(tw[0].numpy(), w[0])          # no gradient: no step
    assert np.isnan(tw[1].numpy()).all()                # one NaN reaches every direction of its matrix
    want = R.muon(w[2], g[2], m[2], 0.1, 0.9, True, 0.0, 5)[0]
    assert np.linalg.norm(tw[2].numpy() - want) <= 0.1 * R.muon_bound(5) * 1.3 * math.sqrt(20 * 2.5) + 4 * R.E * np.linalg.norm(w[2])


def test_muon_of_nothing_twice_and_beside_others():
    ops.MuonOptimizer([], [], []).step()
    empty = [ops.Tensor((0, 5))]
    ops.MuonOptimizer(empty, [ops.Tensor((0, 5))], [ops.Tensor((0, 5))]).step()
    # the same bits again, whether a matrix is updated alone or in a set
    r = np.random.default_rng(7)
    shapes = [(128, 300), (300, 128), (64, 64), (5, 900)]
    w, g = [_f(r.standard_normal(s)) for s in shapes], [_f(r.standard_normal(s)) for s in shapes]

    def run(which):
        tw, tg, tm = [ops.tensor(w[i]) for i in which], [ops.tensor(g[i]) for i in which], [ops.Tensor(shapes[i]) for i in which]
        opt = ops.MuonOptimizer(tw, tg, tm)
        opt.step()
        opt.step()
        opt.close()
        return [t.numpy() for t in tw]
    a, b = run([0, 1, 2, 3]), run([0, 1, 2, 3])
    assert all(np.array_equal(p, q) for p, q in zip(a, b))


def test_muon_refusals():
    w, g, m = ops.Tensor((4, 4)), ops.Tensor((4, 4)), ops.Tensor((4, 4))
    for bad in (lambda: ops.MuonOptimizer([w], [w], [m]), lambda: ops.MuonOptimizer([w, w], [g, g], [m, m]),
                lambda: ops.MuonOptimizer([w], [g], []), lambda: ops.MuonOptimizer([ops.Tensor((4,))], [ops.Tensor((4,))], [ops.Tensor((4,))]),
                lambda: ops.MuonOptimizer([w], [ops.Tensor((4, 3))], [m])):
        with pytest.raises(capi.HipError):
            bad()
    opt = ops.MuonOptimizer([w], [g], [m])
    with pytest.raises(capi.HipError, match="iterations"):
        opt.step(iterations=-1)


# ------------------------------------------------------------------------------------------------ together, through graphs and plans

REWRITES = core.PLAN_VIEWS | core.PLAN_FUSE


def _block(seed, batch=48, width=96):
    """A residual block of dense layers between a stem and a head: (loss, predictions, parameters, placeholders)."""
    feats, labels = core.float32([batch, 30]), core.float32([batch, 10])
    init = nnet.Init(seed)
    stem = nnet.denseAct(nnet.dataSource(feats), width, init)
    h = nnet.groupNorm(stem, 8, "silu")
    h = nnet.denseAct(h, 2 * width, init, "gelu")
    h = nnet.denseAct(h, width, init, residual=stem)
    preds = nnet.softmax(nnet.dense(nnet.groupNorm(h, 4, "relu"), 10, init))
    net = nnet.DAGNetwork([feats], [preds])
    loss = nnet.crossEntropy(preds.trainOutput, labels) + net.paramLoss
    r = np.random.default_rng(seed + 1)
    for p in net.params:
        if p.rank == 1:
            p.set_value(_f(1 + 0.1 * r.standard_normal(p.shape)))
    y = np.eye(10, dtype=F32)[r.integers(0, 10, batch)]
    return loss, preds, net.params, {feats: _f(r.standard_normal((batch, 30))), labels: y}


def _block64(params, x, y):
    """The block's loss in float64, from its parameters' values."""
    def norm(v, p, groups, name):
        return R.group_norm(v, p[0], p[1], groups, 1e-5, name, False)[0][0]
    p = [np.asarray(v, np.float64) for v in params]
    stem = x @ p[0].T + p[1]
    h = norm(stem, p[2:4], 8, "silu")
    h = R.act(h @ p[4].T + p[5], "gelu")
    h = h @ p[6].T + p[7] + stem
    z = norm(h, p[8:10], 4, "relu") @ p[10].T + p[11]
    z = np.exp(z - z.max(1, keepdims=True))
    return -(y * np.log(z / z.sum(1, keepdims=True) + 1e-6)).sum() / len(x)


@pytest.mark.parametrize("flags", [0, REWRITES, REWRITES | core.PLAN_GRAPH, REWRITES | core.PLAN_OVERLAP], ids=["plain", "fused", "graph", "overlap"])
def test_a_blocks_gradients_against_differences(flags):
    loss, preds, params, args = _block(3)
    x, y = (np.asarray(v, np.float64) for v in args.values())
    dev = {k: ops.tensor(v) for k, v in args.items()}
    plan = core.compile([loss] + core.grad(loss, params), flags)
    outs = [ops.Tensor(o.shape) for o in plan.outputs]
    values = [p.value.astype(np.float64) for p in params]
    base = _block64(values, x, y)
    results = []
    for _ in range(4):   # recorded the second time, replayed from then on, with eager work between
        plan.execute(dev, outs)
        results.append([t.numpy() for t in outs])
        ops.group_norm(ops.tensor(np.ones((64, 128, 40), F32)), ops.tensor(np.ones(128, F32)), ops.tensor(np.ones(128, F32)), 4)
        ops.dense_act_grad(ops.Tensor((300, 200)), ops.Tensor((300, 100)), ops.Tensor((200, 100)), ops.Tensor((300, 200)), "gelu")
    for again in results[1:]:
        for a, b in zip(results[0], again):
            assert np.array_equal(a, b)
    if flags & core.PLAN_GRAPH:
        assert plan.recordings()["replays"] >= 2
    got = results[0]
    assert abs(got[0].item() - base) <= 1e-5 * (1 + abs(base))
    r, h = np.random.default_rng(4), 1e-6
    for i, g in enumerate(got[1:]):
        d = r.standard_normal(g.shape)
        up, down = list(values), list(values)
        up[i], down[i] = values[i] + h * d, values[i] - h * d
        slope, want = (_block64(up, x, y) - _block64(down, x, y)) / (2 * h), float((g * d).sum())
        # float32 gradients: a thousand roundings of what is added up; differences: h^2, and 1e-16 / h
        assert abs(slope - want) <= 1000 * R.E * np.abs(g * d).sum() + 1e-8, (i, params[i].shape, slope, want)


@pytest.mark.parametrize("flags", [0, REWRITES], ids=["plain", "fused"])
def test_a_block_is_trained_alike_by_the_graph_form_and_the_fused_one(flags):
    """Two steps: the update's bound for matrices (after one step both forms start the next from weights that far apart)."""
    runs = []
    for make in (online.muon, online.fused_muon):
        loss, preds, params, args = _block(5)
        start = [p.value.copy() for p in params]
        up = make([loss, preds.trainOutput], params, None, learningRate=0.02, momentumRate=0.5, decay=0.1, restRate=0.05, flags=flags)
        dev = {k: ops.tensor(v) for k, v in args.items()}
        up(dev)
        runs.append(([p.value.copy() for p in params], start))
    for a, b, s in zip(runs[0][0], runs[1][0], runs[0][1]):
        assert np.abs(a - s).max() > 1e-4
        moved = np.linalg.norm(a - s)
        # both are within the bound of the exact update, from gradients that agree to 1e-5
        assert np.linalg.norm(a - b) <= (2 * R.muon_bound(5) + 1e-3) * moved + 4 * R.E * np.linalg.norm(s), s.shape


def test_inference_of_the_block_matches_its_training_pass():
    loss, preds, params, args = _block(7)
    dev = {k: v for k, v in args.items()}
    a, b = core.compile([preds.output, preds.trainOutput], REWRITES).execute(dev)
    assert np.array_equal(a, b)   # neither norm nor dense layer depends on the batch or on what is kept


@pytest.mark.parametrize("size", [(1100, 1203, 1000), (2600, 2304, 2500)], ids=str)
def test_a_recorded_plan_of_a_large_layer(size):
    """Replays, with other users of the workspace between them, give the bits of the entry points called one by one."""
    m, n, k = size
    x, w, b, _, dy = _dense_case(m, n, k, 19)
    vx, vt, vw, vb = core.float32([m, k]), core.float32([m, n]), core.float32([n, k], w), core.float32([n], b)
    y = core.denseAct(vx, vw, vb, None, "gelu")
    plan = core.compile([y] + core.grad(core.sum(y * vt), [vw, vb, vx]), REWRITES | core.PLAN_GRAPH)
    outs = [ops.Tensor(o.shape) for o in plan.outputs]
    dev = {vx: ops.tensor(x), vt: ops.tensor(dy)}
    tw, pre = ops.tensor(w), ops.Tensor((m, n))
    want = [ops.dense_act(dev[vx], tw, ops.tensor(b), None, "gelu", pre=pre).numpy()]
    dx, dw, db = ops.dense_act_grad(dev[vt], dev[vx], tw, pre, "gelu")
    want += [dw.numpy(), db.numpy(), dx.numpy()]
    for _ in range(4):
        for t in outs:
            t.set(np.full(t.shape, 7.0, F32))
        plan.execute(dev, outs)
        for a, t in zip(want, outs):
            assert np.array_equal(a, t.numpy().reshape(a.shape))
        ops.dense_act(ops.tensor(dy), ops.tensor(np.ascontiguousarray(dy[:900])))
    assert plan.recordings()["replays"] >= 2


def test_two_plans_share_the_workspace():
    """Two recorded plans and eager calls that need scratch memory, one after the other: every replay gives the eager values."""
    blocks = [_block(8, 48, 96), _block(9, 130, 64)]
    plans, outs, devs, first = [], [], [], []
    for loss, preds, params, args in blocks:
        plans.append(core.compile([loss] + core.grad(loss, params), REWRITES | core.PLAN_GRAPH))
        outs.append([ops.Tensor(o.shape) for o in plans[-1].outputs])
        devs.append({k: ops.tensor(v) for k, v in args.items()})
        plans[-1].execute(devs[-1], outs[-1])
        first.append([t.numpy() for t in outs[-1]])
    for _ in range(3):
        for p, d, o, f in zip(plans, devs, outs, first):
            p.execute(d, o)
            assert all(np.array_equal(t.numpy(), v) for t, v in zip(o, f))
        ops.dense_act_grad(ops.Tensor((700, 900)), ops.Tensor((700, 100)), ops.Tensor((900, 100)), ops.Tensor((700, 900)), "gelu")   # grows it
