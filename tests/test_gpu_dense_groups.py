"""Dense layers of groups of rows on the device against their float64 form."""
import numpy as np
import pytest

import dense_groups as D
import norm_dense_muon as R
from dopt_amd import capi, core, nnet, online, ops

pytestmark = pytest.mark.gpu
F32 = np.float32


def _f(a):
    return np.asarray(a, F32)


def _off_grid(a):
    """A device copy that starts four bytes behind a 16-byte boundary."""
    return ops.Tensor((a.size + 1,), a.dtype).view(1, a.shape).set(a)


def _case(sizes, n, k, seed, before=0, after=0):
    r = np.random.default_rng(seed)
    m, g = before + sum(sizes) + after, len(sizes)
    offsets = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32) + np.int32(before)
    return {"offsets": offsets, "x": _f(r.standard_normal((m, k))), "w": _f(r.standard_normal((g, n, k)) * np.sqrt(2.0 / max(k, 1))),
            "bias": _f(0.3 * r.standard_normal((g, n))), "dy": _f(r.standard_normal((m, n))), "pre": _f(1.4 * r.standard_normal((m, n)))}


def _place(shape, up):
    """A result buffer that holds something already."""
    return up(np.full(shape, 7, F32))


def _parts(t):
    """Whether the products may be of two fp16 parts: all but the small ones, counted in whole tiles."""
    (m, k), (g, n) = t["x"].shape, t["w"].shape[:2]
    return max(m, 32 * g) * n * k >= 10000000


def _check(t, name, up=ops.tensor, keep=True, bias=True):
    d = {k: up(v) for k, v in t.items()}
    (m, k), (g, n) = t["x"].shape, t["w"].shape[:2]
    y, pre = _place((m, n), up), _place((m, n), up) if keep else None
    ops.dense_groups(d["x"], d["w"], d["offsets"], d["bias"] if bias else None, name, out=y, pre=pre)
    want = D.forward(t["x"], t["w"], t["bias"] if bias else None, t["offsets"], name, _parts(t))
    R.close(y.numpy(), want[0], "y")
    if keep:
        R.close(pre.numpy(), want[1], "pre")
    _check_grad(t, name, d, up)


def _check_grad(t, name, d=None, up=ops.tensor):
    d = d or {k: up(v) for k, v in t.items()}
    p = t["pre"] if name != "none" else None
    got = ops.dense_groups_grad(d["dy"], d["x"], d["w"], d["offsets"], d["pre"] if name != "none" else None, name, dx=_place(t["x"].shape, up),
                                dw=_place(t["w"].shape, up), dbias=_place(t["w"].shape[:2], up))
    want = D.backward(t["dy"], t["x"], t["w"], p, t["offsets"], name, _parts(t))
    for a, b, what in zip(got, want, ("dx", "dw", "dbias")):
        R.close(a.numpy(), b, what)
    return got


SIZES = [[1], [0], [5], [0, 0, 3, 0], [31, 32, 33], [9, 0, 17, 3, 11, 8, 14, 2], [64] * 4, [130, 1, 0, 77], [200, 63, 65], [1] * 70, [0] * 64 + [5] + [0] * 70 + [3]]


@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: "%dx%d" % (len(s), sum(s)))
@pytest.mark.parametrize("n,k", [(1, 1), (3, 5), (32, 32), (33, 65), (10, 200), (129, 31), (70, 128)])
def test_sizes(sizes, n, k):
    name = R.ACTS[(len(sizes) + n) % 4]
    _check(_case(sizes, n, k, n + k), name, up=_off_grid if k % 2 else ops.tensor, keep=n % 2 == 0, bias=n != 10)


@pytest.mark.parametrize("name", R.ACTS)
def test_rows_of_no_group(name):
    for before, after in ((3, 0), (0, 70), (40, 33)):
        t = _case([20, 0, 45], 50, 40, 3, before, after)
        t["x"][:before], t["dy"][:before], t["pre"][:before] = np.nan, np.inf, np.nan
        if after:
            t["x"][-after:], t["dy"][-after:], t["pre"][-after:] = np.inf, np.nan, np.nan
        _check(t, name)


@pytest.mark.parametrize("offsets", [[0, 0, 0, 0], [7, 7, 7, 7], [-5, 3, 9, 40], [0, 10, 4, 30], [50, 20, 30, 40], [0, 30, 30, 2 ** 31 - 1], [-2 ** 31, 5, -1, 29],
                                     [60, 60, 60, 60], [100, 200, 300, 400], [30, 20, 10, 0]])
def test_offsets_of_any_value(offsets):
    """Boundaries beyond the rows and ones that fall are taken as the rules say; nothing outside the operands is read or written."""
    t = _case([10, 20, 30], 24, 36, 4)
    t["offsets"] = np.asarray(offsets, np.int32)
    _check(t, "silu")


def test_no_groups_and_no_rows():
    t = _case([5], 8, 12, 1)
    y = ops.tensor(np.full((5, 8), 3, F32))
    lib = capi.load()
    x, w, o = ops.tensor(t["x"]), ops.tensor(t["w"]), ops.tensor(t["offsets"])
    capi.check(lib.dopt_hip_dense_groups(0, 5, 8, 12, 0, None, x.ptr, None, None, y.ptr, None))
    assert not y.numpy().any()
    dx, dw, db = ops.tensor(np.ones((5, 12), F32)), ops.tensor(np.ones((1, 8, 12), F32)), ops.tensor(np.ones((1, 8), F32))
    capi.check(lib.dopt_hip_dense_groups_grad(0, 5, 8, 12, 0, None, y.ptr, None, x.ptr, None, dx.ptr, None, None))
    assert not dx.numpy().any()
    capi.check(lib.dopt_hip_dense_groups_grad(1, 0, 8, 12, 0, o.ptr, None, None, None, None, None, dw.ptr, db.ptr))
    assert not dw.numpy().any() and not db.numpy().any()
    capi.check(lib.dopt_hip_dense_groups(1, 5, 8, 0, 0, o.ptr, None, None, ops.tensor(t["bias"]).ptr, y.ptr, None))
    assert np.array_equal(y.numpy(), np.tile(t["bias"], (5, 1)))
    db.set(np.ones((1, 8), F32))
    capi.check(lib.dopt_hip_dense_groups_grad(1, 5, 8, 0, 0, o.ptr, ops.tensor(t["dy"]).ptr, None, None, None, None, None, db.ptr))
    R.close(db.numpy(), D.backward(t["dy"], t["x"], t["w"], None, t["offsets"], "none")[2], "dbias")


def test_some_of_the_gradients():
    t = _case([33, 0, 50, 12], 45, 70, 6, 2, 5)
    d = {k: ops.tensor(v) for k, v in t.items()}
    whole = [v.numpy() for v in _check_grad(t, "gelu", d)]
    for want in range(1, 8):
        out = [ops.Tensor(v.shape) if want >> i & 1 else None for i, v in enumerate(whole)]
        capi.check(capi.load().dopt_hip_dense_groups_grad(4, len(t["x"]), 45, 70, 2, d["offsets"].ptr, d["dy"].ptr, d["pre"].ptr,
                                                          d["x"].ptr if want & 2 else None, d["w"].ptr if want & 1 else None, *[o.ptr if o else None for o in out]))
        assert all(o is None or np.array_equal(o.numpy(), v) for o, v in zip(out, whole))


# reductions over many rows, in parts and by many groups; sizes of training
@pytest.mark.parametrize("sizes,n,k", [([3000, 1, 700], 40, 24), ([20000], 17, 33), ([9000, 0, 9000], 64, 64), ([512, 311, 905, 77], 256, 200),
                                       ([131, 0, 77, 200, 1, 64, 0, 45, 150, 33, 9, 120, 101], 333, 231), ([40] * 200, 64, 48), ([1024, 700, 90], 520, 384),
                                       ([700, 1300], 1030, 260), ([300, 0, 5, 1500], 512, 1040)])
def test_training_sizes(sizes, n, k):
    t = _case(sizes, n, k, n, 1, 9)
    _check(t, R.ACTS[n % 4])


def test_a_group_that_is_not_finite_is_alone():
    t = _case([40, 200, 30], 70, 90, 8)
    clean = [ops.dense_groups(*[ops.tensor(t[k]) for k in ("x", "w", "offsets", "bias")], "gelu").numpy()] + [v.numpy() for v in _check_grad(t, "gelu")]
    t["x"][50, 3], t["w"][1, 5, 7], t["dy"][60, 9] = np.nan, np.inf, -np.inf
    d = {k: ops.tensor(v) for k, v in t.items()}
    y = ops.dense_groups(d["x"], d["w"], d["offsets"], d["bias"], "gelu").numpy()
    dx, dw, db = (v.numpy() for v in ops.dense_groups_grad(d["dy"], d["x"], d["w"], d["offsets"], d["pre"], "gelu"))
    others = np.r_[0:40, 240:270]
    assert np.array_equal(y[others], clean[0][others]) and np.array_equal(dx[others], clean[1][others])
    assert np.array_equal(dw[[0, 2]], clean[2][[0, 2]]) and np.array_equal(db[[0, 2]], clean[3][[0, 2]])
    assert np.isnan(y[50]).all() and not np.isfinite(y[40:240, 5]).any()


def test_many_equal_values():
    """A column of 0.1 summed over 100000 rows, and its products with ones: sums of at most 64 and 1024 values in a row."""
    t = _case([100000, 5], 8, 8, 1)
    t["dy"][:], t["x"][:] = 0.1, 1.0
    dx, dw, db = (v.numpy() for v in ops.dense_groups_grad(*[ops.tensor(t[k]) for k in ("dy", "x", "w", "offsets")]))
    assert np.abs(db[0] / (100000 * np.float64(F32(0.1))) - 1).max() <= 100 * R.E
    assert np.abs(dw[0] / (100000 * np.float64(F32(0.1))) - 1).max() <= 600 * R.E


def test_repeated_calls_give_the_same_bits():
    t = _case([300, 1, 0, 512, 90], 200, 150, 2)
    d = {k: ops.tensor(v) for k, v in t.items()}
    first = [v.numpy() for v in _check_grad(t, "silu", d)]
    for _ in range(5):
        again = ops.dense_groups_grad(d["dy"], d["x"], d["w"], d["offsets"], d["pre"], "silu")
        assert all(np.array_equal(a, b.numpy()) for a, b in zip(first, again))


# ------------------------------------------------------------------------------------------------ in graphs

FLAGS = [0, core.PLAN_VIEWS | core.PLAN_FUSE, core.PLAN_VIEWS | core.PLAN_FUSE | core.PLAN_GRAPH, core.PLAN_VIEWS | core.PLAN_OVERLAP]


@pytest.mark.parametrize("flags", FLAGS)
@pytest.mark.parametrize("name", R.ACTS)
def test_in_a_graph(name, flags):
    """The same plan with offsets that change from step to step: what no group has is zero each time."""
    t = _case([10, 5, 0, 25], 30, 20, 5, 0, 8)
    f = {k: core.float32(t[k].shape) for k in ("x", "w", "bias", "dy")}
    o = core.int32(t["offsets"].shape)
    y = core.denseGroups(f["x"], f["w"], o, f["bias"], name)
    wrt = [f[k] for k in ("x", "w", "bias")]
    outputs = [y] + core.grad(core.sum(y * f["dy"], [0, 1]).reshape([]), wrt)
    plan = core.compile(outputs, flags)
    rets = [ops.Tensor(v.shape) for v in outputs]
    args = {f[k]: ops.tensor(t[k]) for k in f}
    args[o] = ops.tensor(t["offsets"])
    for offsets in ([0, 10, 15, 15, 40], [3, 3, 20, 48, 48], [0, 10, 15, 15, 40], [0, 0, 0, 0, 0], [0, 12, 24, 36, 48]):
        t["offsets"] = np.asarray(offsets, np.int32)
        args[o].set(t["offsets"])
        plan.execute(args, rets)
        got = [r.numpy() for r in rets]
        (want, bound), (pre, _) = D.forward(t["x"], t["w"], t["bias"], t["offsets"], name)
        R.close(got[0], (want, bound), "y")
        if name == "relu":   # (where pre is within a rounding of zero either gradient is one)
            assert np.abs(pre[want > 0]).min(initial=1.0) > 1e-5
        _, p = ops.dense_groups(*[args[f[k]] for k in ("x", "w")], args[o], args[f["bias"]], name), ops.Tensor(want.shape)
        ops.dense_groups(*[args[f[k]] for k in ("x", "w")], args[o], args[f["bias"]], name, pre=p)
        grads = D.backward(t["dy"], t["x"], t["w"], p.numpy() if name != "none" else None, t["offsets"], name)
        for a, b, what in zip(got[1:], grads, ("dx", "dw", "dbias")):
            R.close(a, b, what)


def test_a_network_of_blocks_with_groups_trains():
    """Norms around blocks of two layers of groups, gradients clipped: with and without rewrites the same losses, and the clipped norm is as asked."""
    losses = []
    for flags in (0, core.PLAN_VIEWS | core.PLAN_FUSE | core.PLAN_GRAPH):
        init = nnet.Init(3)
        x, y, o = core.float32([60, 24]), core.float32([60, 24]), core.int32([5])
        stream = nnet.dataSource(x)
        _, h = nnet.residualNorm(stream, pre="rms")
        for _ in range(2):
            body = nnet.denseGroups(nnet.denseGroups(h, o, 4, 48, init, "gelu"), o, 4, 24, init)
            stream, h = nnet.residualNorm(stream, body, gate=0.5, post="layer", pre="rms")
        net = nnet.DAGNetwork([x], [h])
        d = h.trainOutput - y
        loss = core.sum(d * d, [0, 1]).reshape([])
        up = online.fused_adam([loss], net.params, net.paramProj, flags=flags, maxNorm=2.0)
        r = np.random.default_rng(2)
        feed = {x: ops.tensor(_f(r.standard_normal((60, 24)))), y: ops.tensor(_f(r.standard_normal((60, 24)))), o: ops.tensor(np.asarray([0, 9, 9, 40, 57], np.int32))}
        run = []
        for _ in range(5):
            run.append(float(up(feed)[0]))
            norm, factor = up.norm.numpy()
            assert norm > 2.0 and abs(factor * norm / 2.0 - 1) < 4 * R.E
        losses.append(run)
    assert np.array_equal(*losses) and np.isfinite(losses).all()


# ------------------------------------------------------------------------------------------------ large products

LARGE = [([512, 311, 905, 77, 640, 388, 1001, 262], 1024, 300), ([1300, 0, 200, 3000], 700, 513), ([4200, 5000], 300, 384), ([128] * 40, 520, 530),
         ([2000, 1], 1030, 1100), ([300, 256, 255, 257, 1], 1500, 1024)]


@pytest.mark.parametrize("sizes,n,k", LARGE, ids=lambda v: "%dx%d" % (len(v), sum(v)) if isinstance(v, list) else str(v))
def test_large(sizes, n, k):
    for i, (before, after) in enumerate(((0, 0), (5, 300))):
        t = _case(sizes, n, k, n + i, before, after)
        _check(t, R.ACTS[(n + i) % 4], up=_off_grid if i else ops.tensor, keep=i == 0, bias=i == 0)


FEW = [([0, 0, 1], 300, 4097), ([1], 10, 5), ([1, 0, 2, 0], 129, 2048), ([1] * 64, 40, 1030), ([3, 0, 1, 4], 515, 1027), ([0, 2, 0, 0, 0, 0, 0, 0], 9, 1),
       ([7, 5, 9, 0, 6, 8], 33, 1500), ([0, 1, 0, 0, 0, 0, 1, 0], 1024, 4096), ([2], 1000, 1023), ([4] * 8, 70, 2051)]


@pytest.mark.parametrize("sizes,n,k", FEW, ids=lambda v: "%dx%d" % (len(v), sum(v)) if isinstance(v, list) else str(v))
def test_single_tokens(sizes, n, k):
    for i, (before, after) in enumerate(((0, 0), (2, 3))):
        t = _case(sizes, n, k, n + i, before, after)
        _check(t, R.ACTS[(n + i) % 4], up=_off_grid if i else ops.tensor, keep=i == 0, bias=i == 0)


def test_single_tokens_with_values_that_are_not_finite():
    t = _case([1, 0, 2, 1], 40, 1500, 1)
    clean = ops.dense_groups(*[ops.tensor(t[c]) for c in ("x", "w", "offsets")]).numpy()
    t["x"][1, 1499], t["w"][2, 7, 3], t["w"][1], t["x"][3, 1024] = np.nan, np.inf, np.nan, -np.inf
    y = ops.dense_groups(*[ops.tensor(t[c]) for c in ("x", "w", "offsets")]).numpy()
    cols = np.delete(np.arange(40), 7)
    assert np.isnan(y[1]).all() and np.isinf(y[2, 7]) and np.isinf(y[3]).all()
    assert np.array_equal(y[0], clean[0]) and np.array_equal(y[2, cols], clean[2, cols])


MIDDLE = [([9, 0, 170, 3, 110, 80, 14, 200], 512, 512), ([70, 600, 1, 333], 300, 1111), ([200, 31, 257, 64, 90], 777, 200), ([500], 1024, 1024),
          ([3000, 100, 2500], 96, 130), ([16] * 64, 520, 260), ([1, 2, 3, 60], 2050, 1030), ([6000, 900, 0, 2000], 12, 1561), ([5000, 1000], 5, 830),
          ([7000], 31, 717), ([1200, 20, 4000], 48, 819), ([108], 367, 2458), ([40, 0, 60, 1], 130, 5001), ([64, 64], 1024, 4096), ([300], 70, 20000),
          ([5, 23, 13, 0, 46, 10], 2573, 1017), ([83, 190, 109, 13], 2857, 265), ([40], 9000, 70)]


@pytest.mark.parametrize("sizes,n,k", MIDDLE, ids=lambda v: "%dx%d" % (len(v), sum(v)) if isinstance(v, list) else str(v))
def test_middle(sizes, n, k):
    for i, (before, after) in enumerate(((0, 0), (5, 100))):
        t = _case(sizes, n, k, n + i, before, after)
        _check(t, R.ACTS[(n + i) % 4], up=_off_grid if i else ops.tensor, keep=i == 0, bias=i == 0)


def test_middle_with_a_long_reduction():
    """More steps than one accumulator takes, of every product; groups of more rows than a part of a reduction."""
    _check(_case([40, 100], 300, 4200, 1), "gelu")
    _check(_case([30, 70], 4300, 100, 2), "silu")
    _check(_case([9000, 300], 100, 64, 3), "gelu")


@pytest.mark.parametrize("offsets", [[0, 0, 0, 0], [400, 400, 400, 400], [-5, 100, 300, 5000], [0, 300, 100, 330], [500, 20, 30, 40], [7000, 1, 1, 1]])
def test_middle_with_offsets_of_any_value(offsets):
    t = _case([100, 200, 100], 400, 300, 4, 0, 50)
    t["offsets"] = np.asarray(offsets, np.int32)
    _check(t, "silu")


@pytest.mark.parametrize("sizes,n,k", [([150, 0, 250, 100], 300, 500), ([600, 900, 20, 800], 300, 500), ([20, 0, 30, 10], 150, 3000), ([20, 0, 30, 10], 2500, 150)])
def test_middle_with_values_that_are_not_finite(sizes, n, k):
    """One NaN or infinity in a chunk at the end or the beginning of its reduction, in each operand: it reaches what depends on it alone, as a sum of
    products does."""
    t = _case(sizes, n, k, 9, 10, 20)
    clean = [ops.dense_groups(*[ops.tensor(t[c]) for c in ("x", "w", "offsets")]).numpy()] + [v.numpy() for v in _check_grad(t, "none")]
    a, b = t["offsets"][2], t["offsets"][3]
    t["x"][a + 3, k - 1], t["x"][a + 7, 0], t["w"][2, 5, 7], t["dy"][b - 1, 9] = np.nan, np.inf, -np.inf, np.inf
    t["x"][:10], t["x"][-20:], t["w"][1] = np.nan, np.inf, np.where(sizes[1], t["w"][1], np.nan)
    d = {c: ops.tensor(v) for c, v in t.items()}
    got = [ops.dense_groups(d["x"], d["w"], d["offsets"]).numpy()] + [v.numpy() for v in ops.dense_groups_grad(d["dy"], d["x"], d["w"], d["offsets"])]
    with np.errstate(invalid="ignore"):
        x, w, dy = t["x"][a:b].astype(np.float64), t["w"][2].astype(np.float64), t["dy"][a:b].astype(np.float64)
        want = [clean[0].astype(np.float64), clean[1].astype(np.float64), clean[2].astype(np.float64)]
        for i, (rows, v) in enumerate((((slice(a, b), slice(None)), np.array([[np.sum(p * q) for q in w] for p in x])),
                                       ((slice(a, b), slice(None)), np.array([[np.sum(p * q) for q in w.T] for p in dy])),
                                       ((2, slice(None), slice(None)), np.array([[np.sum(p * q) for q in x.T] for p in dy.T])))):
            odd = ~np.isfinite(v)
            want[i][rows] = np.where(odd, v, want[i][rows])
    for g, v, what in zip(got, want, ("y", "dx", "dw")):
        odd = ~np.isfinite(v)
        assert odd.any() and np.array_equal(g[odd], v[odd].astype(F32), equal_nan=True), what
        assert np.array_equal(g[~odd], v[~odd].astype(F32)), what


def test_middle_values_over_many_orders():
    """Rows that grow and fall along their reduction by far more than fp16 holds, of zeros up to their end, of the smallest and the largest values."""
    m, n, k = 300, 200, 640
    t = _case([100, 200], n, k, 3)
    r = np.random.default_rng(5)
    grow = np.linspace(-25, 25, k)
    t["x"][:40] *= _f(2.0 ** grow)
    t["x"][40:80] *= _f(2.0 ** grow[::-1])
    t["x"][80:90, :-1] = 0
    t["x"][90:95], t["x"][95:100] = 0, t["x"][95:100] * F32(1e-38)
    t["x"][100:110] *= F32(2.0 ** 100)
    t["x"][110:120] *= F32(2.0 ** -100)
    t["x"][120:] *= _f(2.0 ** r.integers(-30, 30, (180, 1)))
    t["w"] *= _f(2.0 ** r.integers(-20, 0, t["w"].shape))
    t["w"][0, :20] *= _f(2.0 ** grow)
    y = ops.dense_groups(*[ops.tensor(t[c]) for c in ("x", "w", "offsets")]).numpy()
    for g, s in enumerate((slice(0, 100), slice(100, 300))):
        x, w = t["x"][s].astype(np.float64), t["w"][g].astype(np.float64)
        bound = (k * 2.0 ** -24 + 2.0 ** -20) * (np.abs(x) @ np.abs(w).T) + 2.0 ** -37 * k * np.outer(np.abs(x).max(1), np.abs(w).max(1)) + 2.0 ** -149
        assert (np.abs(y[s] - x @ w.T) <= bound).all()


def test_middle_in_a_recorded_plan():
    t = _case([100, 0, 250, 60], 320, 384, 5, 0, 60)
    f = {c: core.float32(t[c].shape) for c in ("x", "w", "bias", "dy")}
    o = core.int32(t["offsets"].shape)
    y = core.denseGroups(f["x"], f["w"], o, f["bias"], "gelu")
    outputs = [y] + core.grad(core.sum(y * f["dy"], [0, 1]).reshape([]), [f[c] for c in ("x", "w", "bias")])
    plan = core.compile(outputs, core.PLAN_VIEWS | core.PLAN_FUSE | core.PLAN_GRAPH)
    rets = [ops.Tensor(v.shape) for v in outputs]
    args = {f[c]: ops.tensor(t[c]) for c in f}
    args[o] = ops.tensor(t["offsets"])
    for offsets in ([0, 100, 100, 350, 410], [3, 3, 300, 400, 470], [0, 0, 0, 0, 0], [0, 100, 100, 350, 410]):
        args[o].set(np.asarray(offsets, np.int32))
        pre = ops.Tensor(y.shape)
        want = [ops.dense_groups(args[f["x"]], args[f["w"]], args[o], args[f["bias"]], "gelu", pre=pre).numpy()]
        want += [v.numpy() for v in ops.dense_groups_grad(args[f["dy"]], args[f["x"]], args[f["w"]], args[o], pre, "gelu")]
        plan.execute(args, rets)
        assert all(np.array_equal(r.numpy(), v) for r, v in zip(rets, want))
    assert plan.stats()["kernels"] and plan.recordings()["replays"] > 0


def test_large_with_a_long_reduction():
    """More steps than one accumulator takes, of every product."""
    _check(_case([5000, 300, 4500], 200, 4600, 1), "gelu")
    _check(_case([300, 700], 5000, 260, 2), "silu")


@pytest.mark.parametrize("offsets", [[0, 0, 0, 0, 0], [2000, 2000, 2000, 2000, 2000], [-5, 300, 900, 5000, 700], [0, 1500, 400, 3000, 2900],
                                     [900, 100, 300, 200, 2 ** 31 - 1], [7000, 1, 1, 1, 1]])
def test_large_with_offsets_of_any_value(offsets):
    t = _case([500, 500, 500, 500], 800, 640, 4, 0, 100)
    t["offsets"] = np.asarray(offsets, np.int32)
    _check(t, "silu")


def test_large_with_values_that_are_not_finite():
    t = _case([600, 0, 900, 500], 700, 640, 9, 10, 20)
    clean = [ops.dense_groups(*[ops.tensor(t[k]) for k in ("x", "w", "offsets", "bias")], "gelu").numpy()] + [v.numpy() for v in _check_grad(t, "gelu")]
    t["x"][700, 3], t["x"][900, 5], t["w"][2, 5, 7], t["dy"][1000, 9] = np.nan, np.inf, np.inf, -np.inf
    t["x"][:10], t["x"][-20:], t["w"][1] = np.nan, np.inf, np.nan
    d = {k: ops.tensor(v) for k, v in t.items()}
    y = ops.dense_groups(d["x"], d["w"], d["offsets"], d["bias"], "gelu").numpy()
    dx, dw, db = (v.numpy() for v in ops.dense_groups_grad(d["dy"], d["x"], d["w"], d["offsets"], d["pre"], "gelu"))
    others = np.r_[0:610, 1510:2030]
    assert np.array_equal(y[others], clean[0][others]) and np.array_equal(dx[others], clean[1][others])
    assert np.array_equal(dw[[0, 1, 3]], clean[2][[0, 1, 3]]) and np.array_equal(db[[0, 1, 3]], clean[3][[0, 1, 3]])
    assert np.isnan(y[700]).all() and not np.isfinite(y[610:1510, 5]).any()
    fine = np.delete(np.arange(610, 1510), [90, 290])
    cols = np.delete(np.arange(700), 5)
    assert np.array_equal(y[np.ix_(fine, cols)], clean[0][np.ix_(fine, cols)])
    assert not np.isfinite(dw[2][:, [3, 5]]).any() and not np.isfinite(dw[2][9]).any() and not np.isfinite(db[2, 9])
    rows, cols = np.delete(np.arange(700), 9), np.delete(np.arange(640), [3, 5])
    assert np.array_equal(dw[2][np.ix_(rows, cols)], clean[2][2][np.ix_(rows, cols)])
    assert not np.isfinite(dx[1000]).any() and not np.isfinite(dx[610:1510, 7]).any()


def test_large_some_of_the_gradients():
    t = _case([600, 300, 900], 600, 640, 6, 2, 5)
    d = {k: ops.tensor(v) for k, v in t.items()}
    for name in ("gelu", "none"):
        whole = [v.numpy() for v in _check_grad(t, name, d)]
        for want in range(1, 8):
            out = [ops.Tensor(v.shape) if want >> i & 1 else None for i, v in enumerate(whole)]
            capi.check(capi.load().dopt_hip_dense_groups_grad(3, len(t["x"]), 600, 640, capi.ACTIVATIONS[name], d["offsets"].ptr, d["dy"].ptr,
                                                              d["pre"].ptr if name != "none" else None, d["x"].ptr if want & 2 else None,
                                                              d["w"].ptr if want & 1 else None, *[o.ptr if o else None for o in out]))
            for o, v, what in zip(out, whole, ("dx", "dw", "dbias")):
                if o is not None and what == "dbias":   # (alone its sums go by other runs)
                    R.close(o.numpy(), D.backward(t["dy"], t["x"], t["w"], t["pre"] if name != "none" else None, t["offsets"], name)[2], what)
                elif o is not None:
                    assert np.array_equal(o.numpy(), v) or np.abs(o.numpy() - v).max() <= 2.0 ** -18 * np.abs(v).max(), what


def test_large_values_over_many_orders():
    """Rows whose largest values differ by 2^60, and values far below their row's largest: each keeps 22 bits, or 2^-38 of that."""
    t = _case([500, 700], 600, 640, 3)
    r = np.random.default_rng(4)
    t["x"] *= _f(2.0 ** r.integers(-30, 30, (1200, 1)))
    t["w"] *= _f(2.0 ** r.integers(-20, 0, t["w"].shape))
    y = ops.dense_groups(*[ops.tensor(t[k]) for k in ("x", "w", "offsets")]).numpy()
    for g, s in enumerate((slice(0, 500), slice(500, 1200))):
        x, w = t["x"][s].astype(np.float64), t["w"][g].astype(np.float64)
        bound = (640 * 2.0 ** -24 + 2.0 ** -20) * (np.abs(x) @ np.abs(w).T) + 2.0 ** -37 * 640 * np.outer(np.abs(x).max(1), np.abs(w).max(1))
        assert (np.abs(y[s] - x @ w.T) <= bound).all()


def test_large_in_a_recorded_plan():
    t = _case([700, 0, 900, 300], 512, 640, 5, 0, 60)
    f = {k: core.float32(t[k].shape) for k in ("x", "w", "bias", "dy")}
    o = core.int32(t["offsets"].shape)
    y = core.denseGroups(f["x"], f["w"], o, f["bias"], "silu")
    outputs = [y] + core.grad(core.sum(y * f["dy"], [0, 1]).reshape([]), [f[k] for k in ("x", "w", "bias")])
    plan = core.compile(outputs, core.PLAN_VIEWS | core.PLAN_FUSE | core.PLAN_GRAPH)
    rets = [ops.Tensor(v.shape) for v in outputs]
    args = {f[k]: ops.tensor(t[k]) for k in f}
    args[o] = ops.tensor(t["offsets"])
    for offsets in ([0, 700, 700, 1600, 1900], [3, 3, 1200, 1480, 1960], [0, 0, 0, 0, 0], [0, 700, 700, 1600, 1900]):
        args[o].set(np.asarray(offsets, np.int32))
        pre = ops.Tensor(y.shape)
        want = [ops.dense_groups(args[f["x"]], args[f["w"]], args[o], args[f["bias"]], "silu", pre=pre).numpy()]
        want += [v.numpy() for v in ops.dense_groups_grad(args[f["dy"]], args[f["x"]], args[f["w"]], args[o], pre, "silu")]
        plan.execute(args, rets)
        assert all(np.array_equal(r.numpy(), w) for r, w in zip(rets, want))
    assert plan.stats()["kernels"] and plan.recordings()["replays"] > 0


@pytest.mark.parametrize("k", [1, 4])
def test_gradients_of_more_rows_than_two_to_the_thirty(k):
    """As many rows as the forward pass takes.  All but some rows are zero, so that sums have a term for each of those alone."""
    m, n = (1 << 30) + 64, 4
    offsets = np.array([0, (1 << 29) + 7, (1 << 30) + 40], np.int32)
    places = [0, 5, (1 << 29) + 6, (1 << 29) + 7, (1 << 30) - 1, 1 << 30, (1 << 30) + 39, (1 << 30) + 40, m - 1]
    r = np.random.default_rng(k)
    dy_of, x_of = _f(r.standard_normal((len(places), n))), _f(r.standard_normal((len(places), k)))
    w = _f(r.standard_normal((2, n, k)))
    dy, x, dx = ops.Tensor((m, n)), ops.Tensor((m, k)), ops.Tensor((m, k))
    for p, a, b in zip(places, dy_of, x_of):
        dy.view(p * n, (n,)).set(a)
        x.view(p * k, (k,)).set(b)
        dx.view(p * k, (k,)).set(np.full(k, 7, F32))
    _, dw, db = ops.dense_groups_grad(dy, x, ops.tensor(w), ops.tensor(offsets), dx=dx)
    at = [0, 3, 7]   # places of the groups; the last two belong to none
    want = D.backward(dy_of, x_of, w, None, at, "none", True)
    R.close(np.stack([dx.view(p * k, (k,)).numpy() for p in places]), want[0], "dx")
    R.close(dw.numpy(), want[1], "dw")
    R.close(db.numpy(), want[2], "dbias")


@pytest.mark.parametrize("n", [70001, 1 << 20])
def test_many_equal_values_of_a_row(n):
    """dx of layers of so many columns and two inputs: products of 0.1 and one.  At most 1024 of them follow each other, whose sums of one sign are off by half
    of that many roundings, then up to 128 such sums and eight wavefronts'."""
    dy, w = np.full((40, n), 0.1, F32), np.ones((2, n, 2), F32)
    offsets = ops.tensor(np.array([0, 33, 40], np.int32))
    dx = ops.Tensor((40, 2))
    capi.check(capi.load().dopt_hip_dense_groups_grad(2, 40, n, 2, 0, offsets.ptr, ops.tensor(dy).ptr, None, None, ops.tensor(w).ptr, dx.ptr, None, None))
    assert np.abs(dx.numpy() / (n * np.float64(F32(0.1))) - 1).max() <= 600 * R.E


def test_many_equal_values_of_a_long_reduction():
    """The same forward, of rows enough that they go by tiles."""
    m, n, k = 7000, 2, 65536
    x, w = np.full((m, k), 0.1, F32), np.ones((1, n, k), F32)
    y = ops.dense_groups(ops.tensor(x), ops.tensor(w), ops.tensor(np.array([0, m], np.int32)))
    assert np.abs(y.numpy() / (k * np.float64(F32(0.1))) - 1).max() <= 600 * R.E


def _spread(g, m, seed):
    """Sizes of g groups with m rows in all, of which every third on average has none."""
    r = np.random.default_rng(seed)
    weight = r.random(g) * (r.random(g) < 0.67)
    weight[g // 2] += 1
    return np.bincount(np.searchsorted(np.cumsum(weight / weight.sum()), r.random(m) * 0.999999), minlength=g)


# more than a piece of 64 groups, and more than 256, whose searches begin at a piece: sizes of single rows, small, split and wide products and gradients
@pytest.mark.parametrize("g,m,n,k", [(100, 700, 33, 20), (100, 50, 300, 2000), (100, 2000, 100, 200), (100, 30000, 320, 128), (100, 40000, 128, 1024),
                                     (257, 700, 33, 20), (300, 50, 300, 2000), (300, 3000, 40, 60), (300, 5000, 200, 3000), (257, 60000, 192, 128), (257, 100000, 128, 1024),
                                     (4096, 4000, 24, 64), (5000, 20000, 64, 64), (70000, 50000, 16, 16), (1 << 20, 5000, 4, 4), (1 << 20, 5000, 3, 2)])
@pytest.mark.parametrize("falling", [False, True])
def test_long_lists_of_groups(g, m, n, k, falling):
    """Groups at borders of pieces, the last ones and some others against their definition; what has no rows, or no group, is zero."""
    before, after = 37, 70
    t = _case(_spread(g, m, g + m), n, k, 11, before, after)
    m = len(t["x"])
    name = R.ACTS[n % 4]
    if falling:   # (rows of the next group that does not fall)
        r = np.random.default_rng(5)
        low = r.choice(np.arange(1, g), g // 5, replace=False)
        t["offsets"][low] -= r.integers(0, m, g // 5).astype(np.int32)
    at = D.bounds(t["offsets"], m)
    d = {key: ops.tensor(v) for key, v in t.items()}
    y, pre = _place((m, n), ops.tensor), _place((m, n), ops.tensor)
    ops.dense_groups(d["x"], d["w"], d["offsets"], d["bias"], name, out=y, pre=pre)
    plain = name == "none"
    grads = ops.dense_groups_grad(d["dy"], d["x"], d["w"], d["offsets"], None if plain else d["pre"], name, dx=_place((m, k), ops.tensor),
                                  dw=_place((g, n, k), ops.tensor), dbias=_place((g, n), ops.tensor))
    y, pre, dx, dw, db = (v.numpy() for v in (y, pre) + tuple(grads))
    sizes = np.diff(at)
    some = np.random.default_rng(1).choice(np.flatnonzero(sizes), min(30, np.count_nonzero(sizes)), replace=False)
    border = [b for b in (0, 1, 62, 63, 64, 65, 127, 128, 1023, 1024, 4095, 4096, 65535, 65536, g - 66, g - 2, g - 1) if 0 <= b < g]
    for i in sorted(set(some) | set(border)):
        s, one, local = slice(at[i], at[i + 1]), slice(i, i + 1), [0, sizes[i]]
        if not sizes[i]:
            continue
        of = {key: t[key][s] for key in ("x", "dy", "pre")}
        want = D.forward(of["x"], t["w"][one], t["bias"][one], local, name, True)
        R.close(y[s], want[0], "y of group %d" % i)
        R.close(pre[s], want[1], "pre of group %d" % i)
        want = D.backward(of["dy"], of["x"], t["w"][one], None if plain else of["pre"], local, name, True)
        for a, b, what in zip((dx[s], dw[one], db[one]), want, ("dx", "dw", "dbias")):
            R.close(a, b, "%s of group %d" % (what, i))
    assert not dw[sizes == 0].any() and not db[sizes == 0].any()
    for a in (y, pre, dx):
        assert not a[:at[0]].any() and not a[at[-1]:].any()


@pytest.mark.parametrize("flags", FLAGS)
def test_long_lists_in_a_graph(flags):
    """As test_in_a_graph, of 300 groups whose sizes change from step to step."""
    n, k, g, m = 20, 30, 300, 900
    t = _case(_spread(g, m, 3), n, k, 5)
    f = {key: core.float32(t[key].shape) for key in ("x", "w", "bias", "dy")}
    o = core.int32(t["offsets"].shape)
    y = core.denseGroups(f["x"], f["w"], o, f["bias"], "gelu")
    outputs = [y] + core.grad(core.sum(y * f["dy"], [0, 1]).reshape([]), [f[key] for key in ("x", "w", "bias")])
    plan = core.compile(outputs, flags)
    rets = [ops.Tensor(v.shape) for v in outputs]
    args = {f[key]: ops.tensor(t[key]) for key in f}
    args[o] = ops.tensor(t["offsets"])
    for seed in (3, 4, 5, 3):
        t["offsets"] = np.concatenate([[0], np.cumsum(_spread(g, m, seed))]).astype(np.int32)
        args[o].set(t["offsets"])
        plan.execute(args, rets)
        p = ops.Tensor((m, n))
        want = [ops.dense_groups(args[f["x"]], args[f["w"]], args[o], args[f["bias"]], "gelu", pre=p)]
        want += ops.dense_groups_grad(args[f["dy"]], args[f["x"]], args[f["w"]], args[o], p, "gelu")
        for a, b in zip(rets, want):
            assert np.array_equal(a.numpy().reshape(b.shape), b.numpy())
        (whole, bound), _ = D.forward(t["x"], t["w"], t["bias"], t["offsets"], "gelu", True)
        R.close(rets[0].numpy(), (whole, bound), "y")
