"""The residual norm and its gradient on the device against their float64 forms."""
import os
import subprocess
import sys

import numpy as np
import pytest

import residual_norm as R
from dopt_amd import capi, core, nnet, online, ops

pytestmark = pytest.mark.gpu
F32 = np.float32
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _f(a):
    return np.asarray(a, F32)


def _off_grid(a):
    """A device copy that starts four bytes behind a 16-byte boundary."""
    return ops.Tensor((a.size + 1,)).view(1, a.shape).set(a)


def _case(rows, cols, gates, post, pre, seed, offset=0.3):
    r = np.random.default_rng(seed)
    t = {"x": 2 * r.standard_normal((rows, cols)) + r.standard_normal((rows, 1)),
         "branch": r.standard_normal((rows, cols)) * (0.3 + r.random((rows, 1))) + offset,
         "gate": r.standard_normal((gates, cols)) if gates else None}
    for n in R.NAMES:
        kind = {"post": post, "pre": pre}[n.split("_")[0]]
        there = kind != "none" and (n.endswith("scale") or kind == "layer")
        t[n] = (n.endswith("scale") + 0.2 * r.standard_normal(cols)) if there else None
    t["dy"], t["dh"] = r.standard_normal((rows, cols)), r.standard_normal((rows, cols))
    return {k: None if v is None else _f(v) for k, v in t.items()}


def _up(t, up=ops.tensor):
    return {k: None if v is None else up(v) for k, v in t.items()}


def _check_forward(t, post, pre, scale, eps=1e-5, up=ops.tensor, **where):
    d = _up(t, up)
    vectors = {n: t[n] for n in R.NAMES}
    y, h, stats = ops.residual_norm(d["x"], d["branch"], d["gate"], post, d["post_scale"], d["post_bias"], pre, d["pre_scale"], d["pre_bias"],
                                    scale, eps, **{k: d[v] if isinstance(v, str) else v for k, v in where.items()})
    got = y.numpy()
    want = R.forward(t["x"], t["branch"], t["gate"], post, pre, vectors, scale, eps, y=got)
    R_close(got, want["y"], "y")
    if pre != "none":
        R_close(h.numpy(), want["h"], "h")
    R_close(stats.numpy(), want["stats"], "stats")
    return got, stats.numpy()


def R_close(got, want_and_bound, what):
    from norm_dense_muon import close
    close(got, want_and_bound, what)


def _check_backward(t, y, stats, post, pre, scale, up=ops.tensor, with_dy=True):
    t = dict(t, y=y, stats=stats, dh=t["dh"] if pre != "none" else None, dy=t["dy"] if with_dy or pre == "none" else None)
    d = _up(t, up)
    got = ops.residual_norm_grad(d["dy"], d["dh"], d["y"] if pre != "none" else None, d["branch"], d["stats"], d["gate"], post, d["post_scale"],
                                 d["post_bias"], pre, d["pre_scale"], d["pre_bias"], scale)
    want = R.backward(t["dy"], t["dh"], y, t["branch"], t["gate"], stats, post, pre, {n: t[n] for n in R.NAMES}, scale)
    expected = {"dx"} | {"d" + k for k in ("branch", "gate") + R.NAMES if t[k] is not None}
    assert set(got) == expected
    for k, v in got.items():
        R_close(v.numpy(), want[k], k)
    return got


KINDS = [("layer", "layer"), ("rms", "rms"), ("rms", "layer"), ("none", "layer"), ("layer", "none"), ("none", "rms"), ("none", "none")]
COLS = [1, 2, 3, 4, 5, 31, 63, 64, 65, 127, 128, 129, 255, 257, 511, 512, 513, 777, 1023, 1024, 1025, 1111, 2048, 2050, 4096, 4099, 8191, 8192, 8193,
        12289, 16383, 16384, 16385, 20001]


@pytest.mark.parametrize("cols", COLS)
def test_lengths_of_rows(cols):
    for i, (rows, gates) in enumerate([(1, 1), (7, 0), (12, 4), (9, 9)]):
        post, pre = KINDS[(cols + i) % len(KINDS)]
        t = _case(rows, cols, gates, post, pre, cols + i)
        up = _off_grid if i % 2 else ops.tensor
        y, stats = _check_forward(t, post, pre, 0.7, up=up)
        _check_backward(t, y, stats, post, pre, 0.7, up=up, with_dy=i != 2)


@pytest.mark.parametrize("post,pre", KINDS)
@pytest.mark.parametrize("cols", [10, 200, 640, 1500, 9000, 17000])
def test_norms_and_gates(post, pre, cols):
    for rows, gates in [(60, 0), (60, 1), (60, 3), (60, 20), (60, 30), (60, 60)]:
        t = _case(rows, cols, gates, post, pre, rows + gates)
        y, stats = _check_forward(t, post, pre, 1.0)
        _check_backward(t, y, stats, post, pre, 1.0)


@pytest.mark.parametrize("rows,cols,gates", [(4107, 111, 37), (4107, 111, 1), (20000, 16, 5000), (20000, 16, 10), (70001, 40, 0), (3000, 1000, 2), (3000, 1000, 1500),
                                             (2500, 4096, 1), (1111, 1777, 11), (600, 8192, 6), (300, 16000, 3), (130, 18000, 2), (130, 18000, 65)])
def test_many_rows(rows, cols, gates):
    post, pre = KINDS[rows % 3]
    t = _case(rows, cols, gates, post, pre, rows)
    y, stats = _check_forward(t, post, pre, 0.9)
    _check_backward(t, y, stats, post, pre, 0.9)


@pytest.mark.parametrize("cols,per_gate", [(10, 15), (100, 3), (200, 7), (640, 5), (1500, 1), (1500, 3), (5000, 2), (9000, 3), (16390, 1)])
def test_many_gates_of_few_rows(cols, per_gate):
    """More gates than are shared by a workgroup's teams each."""
    post, pre = KINDS[(cols + per_gate) % len(KINDS)]
    t = _case(600 * per_gate, cols, 600, post, pre, cols)
    y, stats = _check_forward(t, post, pre, 0.7)
    _check_backward(t, y, stats, post, pre, 0.7)


@pytest.mark.parametrize("per_gate,cols", [(16, 2), (40, 1)])
def test_gates_beyond_the_workgroups_of_a_launch(per_gate, cols):
    """2^22 gates of more rows than a workgroup takes several gates of.  Single rows and gates as the definition has them at some thousand places; the scale's and
    bias' gradients over all rows: a gate's rows and up to eight gates by a team, at most 48 teams, runs of those by 32 lanes in pieces of 64 are under 256
    additions that follow each other."""
    gates = 1 << 22
    rows = gates * per_gate
    r = np.random.default_rng(per_gate)
    branch, dy = (r.standard_normal((rows, cols), F32) for _ in range(2))
    branch += F32(0.5)
    gate, scale = r.standard_normal((gates, cols), F32), _f(1 + 0.2 * r.standard_normal(cols))
    d = [ops.tensor(a) for a in (dy, branch, gate, scale)]
    y, _, stats = ops.residual_norm(None, d[1], d[2], "rms", d[3])
    got = ops.residual_norm_grad(d[0], None, None, d[1], stats, d[2], "rms", d[3], out={n: ops.Tensor(s) for n, s in (
        ("dbranch", (rows, cols)), ("dgate", (gates, cols)), ("dpost_scale", (cols,)))})
    y, stats, got = y.numpy(), stats.numpy(), {k: v.numpy() for k, v in got.items()}
    some = np.unique(np.r_[0, gates - 1, r.integers(0, gates, 3000)])
    at = (some[:, None] * per_gate + np.arange(per_gate)).reshape(-1)
    v = dict(dict.fromkeys(R.NAMES), post_scale=scale)
    want = R.forward(None, branch[at], gate[some], "rms", "none", v, 1.0, 1e-5)
    R_close(y[at], want["y"], "y")
    R_close(stats[at], want["stats"], "stats")
    want = R.backward(dy[at], None, None, branch[at], gate[some], stats[at], "rms", "none", v, 1.0)
    R_close(got["dbranch"][at], want["dbranch"], "dbranch")
    R_close(got["dgate"][some], want["dgate"], "dgate")
    total = size = 0.0
    for g in range(0, gates, 1 << 18):
        s = slice(g * per_gate, (g + (1 << 18)) * per_gate)
        q = dy[s].astype(np.float64) * branch[s] * stats[s, None] * np.repeat(gate[g:g + (1 << 18)], per_gate, 0)
        total, size = total + q.sum(0), size + np.abs(q).sum(0)
    R_close(got["dpost_scale"], (total, (256 + 8) * 2.0 ** -24 * size), "dpost_scale")


def test_gates_of_long_rows_beyond_the_workgroups_of_a_launch():
    """As many gates of four rows, of 65 workgroups' columns each, as a launch has no workgroups for.  All but some rows are zero; the gradient of y, the branch and the gate
    lie in the same memory."""
    gates, cols = (1 << 24) // 65 + 1, 16640
    big, dgate = ops.Tensor((4 * gates, cols)), ops.Tensor((gates, cols))
    r = np.random.default_rng(2)
    places = [0, 31, 32, 1000, gates - 1]
    values = _f(r.standard_normal((len(places), 4, cols)))
    for p, v in zip(places, values):
        big.view(4 * p * cols, (4, cols)).set(v)
        dgate.view(p * cols, (cols,)).set(v[0])
    dgate.view(5 * cols, (cols,)).set(values[0, 0])
    ops.residual_norm_grad(big, None, None, big, None, big.view(0, (gates, cols)), out={"dgate": dgate})
    for p, v in zip(places, values):   # three sums of four squares
        want = (v.astype(np.float64) ** 2).sum(0)
        R_close(dgate.view(p * cols, (cols,)).numpy(), (want, 8 * 2.0 ** -24 * want), "dgate")
    assert not dgate.view(5 * cols, (cols,)).numpy().any()


def test_rows_beyond_thirty_two_bits_of_values():
    """2^32 values and more: rows before and behind that border, of which the others are zero."""
    rows, cols = (1 << 21) + 5, 2048 + 4
    assert rows * cols > 1 << 32
    big = ops.Tensor((rows, cols))
    r = np.random.default_rng(1)
    places = [0, 12345, (1 << 32) // cols - 1, (1 << 32) // cols, (1 << 32) // cols + 1, rows - 1]
    values = _f(r.standard_normal((len(places), cols)))
    for p, v in zip(places, values):
        big.view(p * cols, (cols,)).set(v)
    y = ops.Tensor((rows, cols))
    _, _, stats = ops.residual_norm(None, big, post="rms", y=y)
    want = R.forward(None, values, None, "rms", "none", dict.fromkeys(R.NAMES), 1.0, 1e-5)
    R_close(np.stack([y.view(p * cols, (cols,)).numpy() for p in places]), want["y"], "y")
    rstd = stats.numpy()
    R_close(rstd[places], want["stats"], "stats")
    assert np.all(np.delete(rstd, places) == rstd[1])
    # the gradient of the branch, with the gradient of y in y's own values
    db = ops.Tensor((rows, cols))
    ops.residual_norm_grad(y, None, None, big, stats, post="rms", out={"dbranch": db})
    want = R.backward(np.stack([y.view(p * cols, (cols,)).numpy() for p in places]), None, None, values, None, rstd[places], "rms", "none",
                      dict.fromkeys(R.NAMES), 1.0)
    R_close(np.stack([db.view(p * cols, (cols,)).numpy() for p in places]), want["dbranch"], "dbranch")


@pytest.mark.parametrize("cols", [48, 700, 5000, 17001])
def test_operands_that_are_missing(cols):
    t = _case(24, cols, 0, "layer", "layer", 3)
    only = dict.fromkeys(t)
    # a norm of the stream alone, as before a network's first block
    first = dict(only, x=t["x"], pre_scale=t["pre_scale"], dh=t["dh"], dy=t["dy"])
    y, stats = _check_forward(first, "none", "layer", 1.0)
    assert np.array_equal(y, t["x"])
    _check_backward(first, y, stats, "none", "layer", 1.0)
    # the branch alone, without scales
    alone = dict(only, branch=t["branch"], dy=t["dy"], dh=t["dh"])
    y, stats = _check_forward(alone, "rms", "layer", 1.0)
    _check_backward(alone, y, stats, "rms", "layer", 1.0, with_dy=False)
    # nothing but the scaled sum
    y, stats = _check_forward(dict(t, post_scale=None, post_bias=None, pre_scale=None, pre_bias=None), "none", "none", -0.5)
    assert stats.size == 0
    # some of the gradients give what all of them give
    y, stats = _check_forward(t, "layer", "layer", 0.6)
    every = {k: v.numpy() for k, v in _check_backward(t, y, stats, "layer", "layer", 0.6).items()}
    d = _up(dict(t, y=y, stats=stats))
    for names in (["dx"], ["dbranch"], ["dpre_bias"], ["dpost_scale", "dx"], ["dpost_bias", "dpre_scale"], []):
        out = {n: ops.Tensor(every[n].shape) for n in names}
        got = ops.residual_norm_grad(d["dy"], d["dh"], d["y"], d["branch"], d["stats"], None, "layer", d["post_scale"], d["post_bias"], "layer",
                                     d["pre_scale"], d["pre_bias"], 0.6, out=out)
        assert set(got) == set(names) and all(np.array_equal(got[n].numpy(), every[n]) for n in names)


@pytest.mark.parametrize("cols", [33, 900, 3001, 17001])
@pytest.mark.parametrize("place", [{"y": "x"}, {"y": "branch"}, {"h": "x"}, {"h": "branch"}, {"y": "x", "h": "branch"}, {"y": "branch", "h": "x"}],
                         ids=lambda p: ",".join("%s=%s" % i for i in p.items()))
def test_results_in_the_place_of_operands(place, cols):
    t = _case(50, cols, 5, "layer", "rms", 4)
    plain = [v.numpy() for v in ops.residual_norm(**_operands(t, "layer", "rms"))]
    o = _operands(t, "layer", "rms")
    got = ops.residual_norm(**o, **{k: o[v] for k, v in place.items()})
    assert all(np.array_equal(a, b.numpy()) for a, b in zip(plain, got))


def _operands(t, post, pre):
    d = _up(t)
    return dict({k: d[k] for k in ("x", "branch", "gate") + R.NAMES}, post=post, pre=pre)


@pytest.mark.parametrize("cols", [40, 1000, 4000, 17001])
def test_inference_needs_neither_statistics_nor_y(cols):
    t = _case(30, cols, 3, "layer", "layer", 6)
    y, h, _ = ops.residual_norm(**_operands(t, "layer", "layer"))
    d = _up(t)
    only = ops.Tensor(t["x"].shape)
    desc = capi.ResidualNormDesc(30, cols, 3, 1, 1, 1e-5, 1.0)
    capi.check(capi.load().dopt_hip_residual_norm(desc, *[d[k].ptr for k in ("x", "branch", "gate") + R.NAMES], None, only.ptr, None))
    assert np.array_equal(only.numpy(), h.numpy())


@pytest.mark.parametrize("cols", [16, 900, 2500, 17001])
@pytest.mark.parametrize("post,pre", KINDS[:3])
def test_rows_far_from_zero_and_without_spread(post, pre, cols):
    t = _case(20, cols, 1, post, pre, 8, offset=300.0)
    t["branch"][3] = 0.25
    t["x"][5], t["gate"][:], t["branch"][5] = 1.0, 1.0, 0.0
    t["x"][6], t["branch"][6] = 0.0, 0.0
    y, stats = _check_forward(t, post, pre, 1.0)
    assert np.isfinite(y).all() and np.isfinite(stats).all()


@pytest.mark.parametrize("cols", [24, 800, 3333, 17001])
def test_a_row_that_is_not_finite_is_alone(cols):
    t = _case(40, cols, 0, "layer", "layer", 9)
    clean = [v.numpy() for v in ops.residual_norm(**_operands(t, "layer", "layer"))]
    for bad, value in ((7, np.nan), (11, np.inf), (30, -np.inf)):
        t["branch"][bad, cols // 2] = value
    got = [v.numpy() for v in ops.residual_norm(**_operands(t, "layer", "layer"))]
    others = [i for i in range(40) if i not in (7, 11, 30)]
    for a, b in zip(clean[:2], got[:2]):
        assert np.array_equal(a[others], b[others]) and not np.isfinite(b[[7, 11, 30]]).any()
    d = _up(dict(t, y=got[0], stats=got[2]))
    g = ops.residual_norm_grad(d["dy"], d["dh"], d["y"], d["branch"], d["stats"], None, "layer", d["post_scale"], d["post_bias"], "layer",
                               d["pre_scale"], d["pre_bias"])
    dx = g["dx"].numpy()
    assert np.isfinite(dx[others]).all() and np.isnan(dx[[7, 11, 30]]).all()
    assert np.isnan(g["dpost_scale"].numpy()).all()


def test_no_rows():
    d = capi.ResidualNormDesc(0, 8, 0, 1, 2, 1e-5, 1.0)
    lib = capi.load()
    capi.check(lib.dopt_hip_residual_norm(d, *[None] * 10))
    out = [ops.tensor(np.full(8, 7, F32)) for _ in range(4)]
    capi.check(lib.dopt_hip_residual_norm_grad(d, None, None, None, out[0].ptr, None, None, None, None, None, None, None, None, *[o.ptr for o in out]))
    assert all(not o.numpy().any() for o in out)


def test_repeated_calls_give_the_same_bits():
    t = _case(999, 777, 27, "layer", "layer", 5)
    y, stats = _check_forward(t, "layer", "layer", 1.0)
    first = {k: v.numpy() for k, v in _check_backward(t, y, stats, "layer", "layer", 1.0).items()}
    for _ in range(5):
        again = _check_backward(t, y, stats, "layer", "layer", 1.0)
        assert all(np.array_equal(first[k], again[k].numpy()) for k in first)


_ORDER = """
import hashlib, sys
import numpy as np
from dopt_amd import ops
for cols in [int(c) for c in sys.argv[1:]]:
    rows = 1 << 19 - cols.bit_length()
    r = np.random.default_rng(cols)
    x, b, dh = (ops.tensor(r.standard_normal((rows, cols), np.float32)) for _ in range(3))
    gate, scale = ops.tensor(r.standard_normal((4, cols), np.float32)), ops.tensor(r.standard_normal(cols, np.float32))
    y, h, stats = ops.residual_norm(x, b, gate, "none", None, None, "layer", scale, scale)
    g = ops.residual_norm_grad(None, dh, y, b, stats, gate, "none", None, None, "layer", scale, scale)
    out = b"".join(g[k].numpy().tobytes() for k in sorted(g))
    print(cols, hashlib.sha256(out).hexdigest(), flush=True)
"""


def test_the_bits_do_not_depend_on_the_calls_before():
    lengths = ["48", "128", "512", "1024", "2048", "4096"]
    runs = [sorted(subprocess.run([sys.executable, "-c", _ORDER] + order, cwd=ROOT, capture_output=True, text=True, timeout=100, check=True)
                   .stdout.splitlines()) for order in (lengths, lengths[::-1])]
    assert len(runs[0]) == len(lengths) and runs[0] == runs[1]


def test_sums_of_many_equal_rows():
    """A million rows whose gradients are alike: sums of at most 128 additions of one value and its multiples in a row."""
    rows, cols = 1 << 20, 12
    dy = np.full((rows, cols), 0.1, F32)
    branch = np.tile(_f(np.linspace(-1, 1, cols)), (rows, 1))
    t = dict.fromkeys(("x", "gate", "dh") + R.NAMES)
    t.update(dy=dy, branch=branch, x=branch, post_scale=np.ones(cols, F32), post_bias=np.zeros(cols, F32), gate=np.ones((1, cols), F32))
    y, stats = _check_forward(t, "layer", "none", 1.0)
    got = _check_backward(t, y, stats, "layer", "none", 1.0)
    assert np.abs(got["dpost_bias"].numpy() / (rows * np.float64(F32(0.1))) - 1).max() < 200 * R.E


# ------------------------------------------------------------------------------------------------ in graphs

FLAGS = [0, core.PLAN_VIEWS | core.PLAN_FUSE, core.PLAN_VIEWS | core.PLAN_FUSE | core.PLAN_GRAPH, core.PLAN_VIEWS | core.PLAN_OVERLAP]


@pytest.mark.parametrize("flags", FLAGS)
@pytest.mark.parametrize("post,pre", KINDS[:5])
def test_in_a_graph(post, pre, flags):
    t = _case(24, 50, 6, post, pre, 11)
    names = [k for k in ("x", "branch", "gate") + R.NAMES if t[k] is not None]
    f = {k: core.float32(t[k].shape) for k in names}
    y, h = core.residualNorm(f["x"], f["branch"], f["gate"], post, f.get("post_scale"), f.get("post_bias"), pre, f.get("pre_scale"), f.get("pre_bias"), 0.8)
    cy, ch = core.float32(t["dy"].shape), core.float32(t["dh"].shape)
    loss = core.sum(y * cy, [0, 1]).reshape([])
    if pre != "none":
        loss = loss + core.sum(h * ch, [0, 1]).reshape([])
    outputs = [y] + ([h] if pre != "none" else []) + core.grad(loss, [f[k] for k in names])
    plan = core.compile(outputs, flags)
    args = dict({f[k]: ops.tensor(t[k]) for k in names}, **{})
    args[cy] = ops.tensor(t["dy"])
    if pre != "none":
        args[ch] = ops.tensor(t["dh"])
    rets = [ops.Tensor(o.shape) for o in outputs]
    for _ in range(4):
        plan.execute(args, rets)
        got = [r.numpy() for r in rets]
        vectors = {n: t[n] for n in R.NAMES}
        want = R.forward(t["x"], t["branch"], t["gate"], post, pre, vectors, 0.8, 1e-5, y=got[0])
        R_close(got[0], want["y"], "y")
        if pre != "none":
            R_close(got[1], want["h"], "h")
        _, _, stats = ops.residual_norm(**_operands(t, post, pre), residual_scale=0.8)
        grads = R.backward(t["dy"], t["dh"] if pre != "none" else None, got[0], t["branch"], t["gate"], stats.numpy(), post, pre, vectors, 0.8)
        for k, g in zip(names, got[-len(names):]):
            R_close(g, grads["d" + k], "d" + k)


def test_a_residual_network_trains_the_same_with_and_without_rewrites():
    losses = []
    for flags in (0, core.PLAN_VIEWS | core.PLAN_FUSE | core.PLAN_GRAPH):
        init = nnet.Init(3)
        x, y = core.float32([40, 24]), core.float32([40, 24])
        stream = nnet.dataSource(x)
        _, h = nnet.residualNorm(stream, pre="rms")
        for _ in range(3):
            body = nnet.denseAct(nnet.denseAct(h, 48, init, "gelu"), 24, init)
            stream, h = nnet.residualNorm(stream, body, gate=0.5, post="layer", pre="rms")
        net = nnet.DAGNetwork([x], [h])
        d = h.trainOutput - y
        loss = core.sum(d * d, [0, 1]).reshape([])
        up = online.fused_adam([loss], net.params, net.paramProj, flags=flags, maxNorm=5.0)
        r = np.random.default_rng(2)
        feed = {x: ops.tensor(_f(r.standard_normal((40, 24)))), y: ops.tensor(_f(r.standard_normal((40, 24))))}
        losses.append([float(up(feed)[0]) for _ in range(5)])
    assert np.array_equal(*losses)
