"""The norm of a set of gradients, clipping, and updates that take its factor, on the device.

Squares and sums are formed in 64 bits, so the norm and the factor are a rounding to 32 bits (2^-24 of them) from their definition, and
a hundredth of that for what 64 bits leave; a clipped gradient is the product of two float32 values, rounded once."""
import numpy as np
import pytest

import norm_dense_muon as R
from dopt_amd import capi, core, nnet, online, ops

pytestmark = pytest.mark.gpu
F32 = np.float32
E = 1.01 * 2.0 ** -24

SIZES = [[1], [4095], [4096], [4097], [3, 0, 5], [0], [], [1] * 300, [27 * 64, 64, 64, 576 * 64, 10, 5130], [4096 * 9 + 3, 1, 2, 7, 70001],
         [1 << 24, 1 << 20, 12345], [4096 * 256 * 8 + 1, 4096]]


def _gradients(sizes, seed=0, scale=1.0):
    r = np.random.default_rng(seed)
    return [(r.standard_normal(n) * scale * 10.0 ** (i % 4 - 2)).astype(F32) for i, n in enumerate(sizes)]


def _norm64(grads):
    return np.sqrt(sum(float((g.astype(np.float64) ** 2).sum()) for g in grads))


def _up(a, shift):
    """On the device, `shift` values behind a boundary of 16 bytes."""
    return ops.Tensor((a.size + shift,)).view(shift, a.shape).set(a) if shift else ops.tensor(a)


def _check(grads, most, tensors, outs=None, place=None):
    n = ops.GradientNorm(tensors, outs)
    norm, factor = n.norm(most, place).numpy() if outs is None else n.clip(most, place).numpy()
    want, most = _norm64(grads), float(F32(most))   # the largest norm is an argument of 32 bits (1e-38 there is off by 2^-23 of itself)
    by = 1.0 if want <= most else most / want
    assert (norm == np.inf if want > 3.403e38 else abs(norm - want) <= E * want) and abs(factor - by) <= E * by
    return norm, factor


@pytest.mark.parametrize("shift", [0, 1, 3])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: "%dx%d" % (len(s), sum(s)))
def test_norm_and_clipping(sizes, shift):
    grads = _gradients(sizes, len(sizes))
    tensors = [_up(g, shift if i % 2 else 0) for i, g in enumerate(grads)]
    norm = _norm64(grads)
    for most in (0.5 * norm + 0.1 * (norm == 0), 2.0 * norm + 1, float("inf"), 0.0):
        _check(grads, most, tensors)
    outs = [_up(np.full(g.shape, 7, F32), (shift + i) % 3) for i, g in enumerate(grads)]
    for most in (0.25 * norm, 2.0 * norm):
        _, factor = _check(grads, most, tensors, outs)
        for g, o, t in zip(grads, outs, tensors):
            assert np.array_equal(o.numpy(), g * factor) and np.array_equal(t.numpy(), g)
    for most in (2.0 * norm, 0.25 * norm):
        _, factor = _check(grads, most, tensors, tensors)
        for g, t in zip(grads, tensors):
            assert np.array_equal(t.numpy(), g * factor)


def test_what_lies_between_the_tensors_is_left():
    flat = np.arange(1, 10000, dtype=F32)
    t = ops.tensor(flat)
    parts = [(1, 5), (7, 4097), (4200, 4096), (9000, 17)]
    views = [t.view(a, (n,)) for a, n in parts]
    norm, factor = _check([flat[a:a + n] for a, n in parts], 3.0, views, views)
    want = flat.copy()
    for a, n in parts:
        want[a:a + n] *= factor
    assert np.array_equal(t.numpy(), want)


@pytest.mark.parametrize("scale", [1e-38, 1e-30, 1e30, 3e37])
def test_squares_outside_the_range_of_floats(scale):
    grads = [np.full(1000, scale, F32), np.full(77, -scale, F32), np.full(3, F32(scale) / 2, F32)]
    _check(grads, scale, [ops.tensor(g) for g in grads])


def test_many_equal_values():
    grads = [np.full(1 << 25, 0.1, F32)]
    _check(grads, 1.0, [ops.tensor(g) for g in grads])


def test_infinities_and_nan():
    g = _gradients([5000, 3])
    g[0][4321] = np.inf
    t = [ops.tensor(a) for a in g]
    outs = [ops.Tensor(a.shape) for a in g]
    result = ops.GradientNorm(t, outs).clip(1.0).numpy()
    assert result[0] == np.inf and result[1] == 0
    got = outs[0].numpy()
    assert np.isnan(got[4321]) and not np.delete(got, 4321).any() and not outs[1].numpy().any()
    g[1][1] = np.nan
    t[1].set(g[1])
    assert np.isnan(ops.GradientNorm(t, outs).clip(1.0).numpy()).all()
    assert np.isnan(outs[0].numpy()).all() and np.isnan(outs[1].numpy()).all()


def test_a_gradient_listed_twice_counts_twice():
    g = _gradients([3000])
    t = ops.tensor(g[0])
    _check(g * 2, 1.0, [t, t])


def test_clipping_needs_places():
    n = ops.GradientNorm([ops.tensor(np.ones(4, F32))])
    with pytest.raises(capi.HipError, match="no place"):
        n.clip(1.0)
    for bad in (-1.0, float("nan")):
        with pytest.raises(capi.HipError, match="largest norm"):
            n.norm(bad)
    with pytest.raises(capi.HipError, match="wrong size"):
        ops.GradientNorm([ops.Tensor((4,))], [ops.Tensor((5,))])
    with pytest.raises(capi.HipError, match="wrong size or type"):
        ops.GradientNorm([ops.Tensor((4,), np.int32)])


def test_the_norms_place_is_apart_from_the_gradients():
    g, out = ops.tensor(np.arange(9, dtype=np.float32)), ops.Tensor((9,))
    n = ops.GradientNorm([g], [out])
    for t in (g, out):
        for call in (n.norm, n.clip):
            with pytest.raises(capi.HipError, match="lies in a gradient"):
                call(1.0, out=t.view(7, (2,)))
    assert not out.numpy().any() and np.array_equal(g.numpy(), np.arange(9))


def test_repeated_calls_give_the_same_bits():
    grads = _gradients([1 << 20, 333, 70000], 4)
    n = ops.GradientNorm([ops.tensor(g) for g in grads])
    first = n.norm(1.0).numpy()
    place = ops.Tensor((2,))
    for _ in range(20):
        assert np.array_equal(n.norm(1.0, place).numpy(), first)


# ------------------------------------------------------------------------------------------------ updates

SHAPES = [(64, 27), (64,), (130, 70), (1, 5), (4097,), (2, 3, 5, 7), (40, 200)]


def _state(seed):
    r = np.random.default_rng(seed)
    return [[r.standard_normal(s).astype(F32) for s in SHAPES] for _ in range(3)] + [
        [(r.standard_normal(s).astype(F32)) ** 2 for s in SHAPES] for _ in range(2)]


@pytest.mark.parametrize("rule", ["sgd", "nesterov", "adam", "amsgrad", "muon"])
@pytest.mark.parametrize("most", [0.5, 1e9])
def test_updates_read_gradients_as_if_clipped(rule, most):
    results = []
    for scaled in (True, False):
        w, g, m, v, vhat = [[ops.tensor(a) for a in s] for s in _state(3)]
        result = ops.Tensor((2,))
        norm = ops.GradientNorm(g, g)
        if rule == "muon":
            mats = [i for i, s in enumerate(SHAPES) if len(s) > 1 and s[0] > 1]
            opt = ops.MuonOptimizer(*[[t[i] for i in mats] for t in (w, g, m)])
        else:
            opt = ops.FusedOptimizer(w, g, m, v, vhat)
        for step in range(3):
            if scaled:
                norm.norm(most, result)
                factor = result.view(1, (1,))
            else:
                for t, a in zip(g, _state(3)[1]):
                    t.set(a)
                norm.clip(most, result)
                factor = None
            if rule == "muon":
                opt.step(0.02, 0.9, True, 0.01, 5, factor=factor)
            elif rule in ("sgd", "nesterov"):
                opt.sgd(0.1, 0.9, rule == "nesterov", factor=factor)
            else:
                getattr(opt, rule)(1e-3, 0.9, 0.99, 1e-8, factor=factor)
        results.append([t.numpy() for s in (w, m, v, vhat) for t in s])
    for a, b in zip(*results):
        assert np.array_equal(a, b)


def test_a_factor_is_one_value():
    w, g, m, v, vhat = [[ops.tensor(a) for a in s] for s in _state(3)]
    opt = ops.FusedOptimizer(w, g, m, v, vhat)
    with pytest.raises(capi.HipError, match="one float32 value"):
        opt.sgd(0.1, factor=ops.Tensor((2,)))


def _network(rule, most, fused):
    init = nnet.Init(5)
    x, y = core.float32([32, 20]), core.float32([32, 7])
    body = nnet.denseAct(nnet.dataSource(x), 24, init, "gelu")
    preds = nnet.denseAct(body, 7, init)
    net = nnet.DAGNetwork([x], [preds])
    d = preds.trainOutput - y
    loss = core.sum(d * d, [0, 1]).reshape([])
    make = getattr(online, ("fused_" if fused else "") + rule)
    args = {}
    if rule == "sgd":
        args = {"learningRate": 0.05} if fused else {"learningRate": core.float32([], [0.05])}
    up = make([loss], net.params, net.paramProj, maxNorm=most, flags=core.PLAN_VIEWS | core.PLAN_FUSE | (core.PLAN_GRAPH if fused else 0), **args)
    r = np.random.default_rng(8)
    feed = {x: ops.tensor(r.standard_normal((32, 20)).astype(F32)), y: ops.tensor(r.standard_normal((32, 7)).astype(F32))}
    return up, net, feed


@pytest.mark.parametrize("rule", ["sgd", "adam", "amsgrad", "muon"])
def test_updaters_clip(rule):
    """One step of the fused form and of the graph's.  Their factors are sums of some 700 squares in 64 and in 32 bits, within 32 roundings
    of each other, and so are the gradients of the two plans relative to a tensor's largest (sums of at most 32 terms).  SGD's step is
    the gradient's, 2^-18 of it; ADAM's first one is the learning rate times g / |g|, whatever the scale, but for gradients as small as
    its eps, 1e-8 (there 2^-18 of it as well); the orthogonalised matrix is within muon_bound of its definition each time.  What is added is seen behind the rounding
    of a parameter below two."""
    most = 0.3
    state = []
    for fused in (True, False):
        up, net, feed = _network(rule, most, fused)
        before = [p.value.astype(np.float64) for p in net.params]
        up(feed)
        state.append([p.value - b for p, b in zip(net.params, before)])
        assert all(np.abs(b).max() < 2 for b in before)
        if fused:
            norm, factor = up.norm.numpy()
            assert norm > most and abs(factor - most / norm) <= 2.1 * E * factor
    for a, b in zip(*state):
        assert np.abs(a).max() > 0
        if rule == "muon" and a.ndim > 1:
            assert np.linalg.norm(a - b) <= 2 * R.muon_bound(5) * np.linalg.norm(b) + a.size ** 0.5 * 2.0 ** -22
        else:
            assert np.abs(a - b).max() <= 2.0 ** -18 * np.abs(b).max() + 2.0 ** -22


def test_sgd_moves_by_the_clipped_gradients():
    moved = []
    for most in (None, 0.3):
        up, net, feed = _network("sgd", most, True)
        before = [p.value.astype(np.float64) for p in net.params]
        up(feed)
        moved.append([p.value.astype(np.float64) - b for p, b in zip(net.params, before)])
    norm, factor = up.norm.numpy()
    for a, b, w in zip(*moved, before):
        # each is lr g of its gradient and a rounding of the parameter, whose size is under four
        assert np.abs(a * float(factor) - b).max() <= 4 * np.abs(a).max() * 2.0 ** -24 + 2 * (np.abs(w).max() + np.abs(a).max()) * 2.0 ** -24
    total = np.sqrt(sum((m ** 2).sum() for m in moved[1])) / 0.05
    assert abs(total - 0.3) < 1e-4


@pytest.mark.parametrize("most", [0.0, 1e-3, 1.0, 5.0])
@pytest.mark.parametrize("size", [0.0, 1e-24, 1.0, 1e20, 1e37])
def test_a_graph_clips_gradients_of_any_size(size, most):
    """As tests/test_gradient_norm_cpu.py has it, compiled for the device, with the same bound for each result; and the fused updates' factor, which is formed in
    64 bits and rounded once, is within 20 roundings of the graph's."""
    r = np.random.default_rng(7)
    values = [(size * r.uniform(-9, 9, s)).astype(F32) for s in ((3, 4), (5,), (2, 2, 2))]
    norm = np.sqrt(sum((v.astype(np.float64) ** 2).sum() for v in values))
    factor = 1.0 if norm <= most else most / norm
    g = [core.float32(v.shape) for v in values]
    got = core.evaluate(online.clipped(g, most), dict(zip(g, values)))
    for a, v in zip(got, values):
        want = v.astype(np.float64) * factor
        assert np.isfinite(a).all()
        assert (np.abs(a - want) <= 21 * 2.0 ** -24 * np.abs(want) + np.abs(v) * 2.0 ** -149 + 2.0 ** -149).all()
    fused = float(ops.GradientNorm([ops.tensor(v) for v in values]).norm(most).numpy()[1])
    for a, v in zip(got, values):
        assert (np.abs(a - v.astype(np.float64) * fused) <= 22 * 2.0 ** -24 * np.abs(v) * fused + np.abs(v) * 2.0 ** -148 + 2.0 ** -149).all()


@pytest.mark.parametrize("rule", ["sgd", "adam", "amsgrad", "muon"])
@pytest.mark.parametrize("most", [1.0, 5.0])
def test_a_step_without_gradients_moves_nothing(rule, most):
    """Zero gradients: both forms leave the parameters as they are, to the bit."""
    for fused in (True, False):
        w, x = core.float32([6, 5]), core.float32([6, 5])
        start = np.random.default_rng(3).standard_normal((6, 5)).astype(F32)
        w.set_value(start)
        loss = core.sum(w * x, [0, 1]).reshape([])
        up = getattr(online, ("fused_" if fused else "") + rule)([loss], [w], maxNorm=most)
        for _ in range(2):
            up({x: ops.tensor(np.zeros((6, 5), F32))})
        assert np.array_equal(w.value, start)
