"""Group norm, dense layer with activation, orthogonalised update: what is refused before the device is touched, what the graph
operations are, and the float64 forms that the device tests compare with, against differences."""
import ctypes as C

import numpy as np
import pytest

import norm_dense_muon as R
from dopt_amd import capi, core, nnet

P = C.c_void_p


def _addr(n):
    """Addresses that nobody reads: the calls below end before a kernel is launched."""
    return P(n << 24)


def _norm(N=2, Cc=8, inner=4, groups=2, act=0, x=1, scale=2, bias=3, packed=4):
    return capi.load().dopt_hip_group_norm(N, Cc, inner, groups, 0, 1e-5, act, _addr(x), _addr(scale), _addr(bias), _addr(packed))


def _norm_grad(N=2, Cc=8, inner=4, groups=2, act=0, dy=5, x=1, scale=2, bias=3, stats=6, packed=4):
    return capi.load().dopt_hip_group_norm_grad(N, Cc, inner, groups, 0, act, *[_addr(p) for p in (dy, x, scale, bias, stats, packed)])


def _dense(M=4, N=8, K=16, act=0, x=1, w=2, bias=3, residual=4, y=5, pre=6):
    return capi.load().dopt_hip_dense_act(M, N, K, act, *[_addr(p) for p in (x, w, bias, residual, y, pre)])


def _dense_grad(M=4, N=8, K=16, act=2, dy=1, pre=2, x=3, w=4, dx=5, dw=6, dbias=7):
    return capi.load().dopt_hip_dense_act_grad(M, N, K, act, *[_addr(p) for p in (dy, pre, x, w, dx, dw, dbias)])


@pytest.mark.parametrize("call, text", [
    (lambda: _norm(groups=0), b"0 groups"), (lambda: _norm(groups=3), b"parted into 3"), (lambda: _norm(act=4), b"activation 4"),
    (lambda: _norm(act=-1), b"activation -1"), (lambda: _norm(x=0), b"null"), (lambda: _norm(packed=0), b"null"),
    (lambda: _norm(packed=1), b"overlaps"), (lambda: _norm(packed=3), b"overlaps"), (lambda: _norm(N=1 << 31), b"too large"),
    (lambda: _norm(N=1 << 20, Cc=1 << 12), b"too large"),
    (lambda: _norm_grad(groups=5), b"parted into 5"), (lambda: _norm_grad(act=9), b"activation 9"), (lambda: _norm_grad(dy=0), b"null"),
    (lambda: _norm_grad(stats=0), b"null"), (lambda: _norm_grad(packed=5), b"overlaps"), (lambda: _norm_grad(packed=6), b"overlaps"),
    (lambda: _dense(act=4), b"activation 4"), (lambda: _dense(x=0), b"null"), (lambda: _dense(y=0), b"null"),
    (lambda: _dense(y=4), b"overlaps"), (lambda: _dense(pre=1), b"overlaps"), (lambda: _dense(pre=5), b"y and pre"),
    (lambda: _dense(M=1 << 30), b"too large"),
    (lambda: _dense_grad(pre=0), b"null"), (lambda: _dense_grad(dy=0), b"null"), (lambda: _dense_grad(w=0), b"needs w"),
    (lambda: _dense_grad(x=0), b"needs x"), (lambda: _dense_grad(dx=1), b"overlaps"), (lambda: _dense_grad(dw=5), b"two results"),
    (lambda: _dense_grad(act=7), b"activation 7"),
])
def test_refusals(call, text):
    assert call() == 1
    assert text in capi.load().dopt_hip_last_error(), capi.load().dopt_hip_last_error()


def _muon(*matrices):
    refs = (capi.MatrixRef * max(1, len(matrices)))(*[capi.MatrixRef(w << 24, g << 24, m << 24, r, c) for w, g, m, r, c in matrices])
    h = C.c_void_p(7)
    rc = capi.load().dopt_hip_muon_create(len(matrices), refs, C.byref(h))
    assert not h.value
    return rc


@pytest.mark.parametrize("matrices, text", [
    ([(1, 0, 3, 4, 4)], b"null"), ([(1, 2, 1, 4, 4)], b"share"), ([(1, 1, 3, 4, 4)], b"share"),
    ([(1, 2, 3, 4, 4), (1, 5, 6, 4, 4)], b"0 and 1 share"), ([(1, 2, 3, 4, 4), (4, 3, 6, 4, 4)], b"0 and 1 share"),
    ([(1, 2, 3, 4, 4), (4, 5, 2, 4, 4)], b"0 and 1 share"), ([(1, 2, 3, 20000, 20000)], b"too large"), ([(1, 2, 3, 1 << 60, 16)], b"too large"),
])
def test_muon_refusals(matrices, text):
    assert _muon(*matrices) == 1
    assert text in capi.load().dopt_hip_last_error(), capi.load().dopt_hip_last_error()


def test_muon_step_needs_a_handle():
    lib = capi.load()
    assert lib.dopt_hip_muon_step(None, 0.1, 0.9, 1, 0.0, 5) == 1 and b"handle" in lib.dopt_hip_last_error()
    assert lib.dopt_hip_muon_create(1, None, C.byref(C.c_void_p())) == 1
    assert lib.dopt_hip_muon_destroy(None) == 0


def test_graph_operations_are_verified():
    f = core.float32
    x, s = f([2, 6, 3, 3]), f([6])
    y, mean, rstd = core.groupNorm(x, s, s, 3)
    assert y.shape == (2, 6, 3, 3) and mean.shape == rstd.shape == (6,)
    assert core.groupNorm(f([2, 3, 3, 6]), s, s, 3, channelsLast=True)[1].shape == (6,)
    for bad in (lambda: core.groupNorm(x, s, s, 4), lambda: core.groupNorm(x, f([5]), s, 3), lambda: core.groupNorm(f([6]), s, s, 3),
                lambda: core.groupNorm(x, s, s, 0), lambda: core.groupNorm(core.int32([2, 6]), s, s, 3),
                lambda: core.denseAct(f([2, 3]), f([4, 5])), lambda: core.denseAct(f([2, 3]), f([4, 3]), f([3])),
                lambda: core.denseAct(f([2, 3]), f([4, 3]), None, f([2, 3])), lambda: core.denseAct(f([2, 3, 1]), f([4, 3]))):
        with pytest.raises(core.VerificationError):
            bad()
    for bad in (lambda: core.groupNorm(x, s, s, 3, activation="tanh"), lambda: core.denseAct(f([2, 3]), f([4, 3]), activation="tanh")):
        with pytest.raises(ValueError, match="no activation"):
            bad()
    assert core.denseAct(f([2, 3]), f([4, 3]), f([4]), f([2, 4]), "gelu").shape == (2, 4)


def test_gradients_have_their_operands_shapes():
    f = core.float32
    x, gamma, beta, w, b = f([5, 8]), f([8]), f([8]), f([8, 8]), f([8])
    h = core.groupNorm(x, gamma, beta, 2, activation="silu")[0]
    y = core.denseAct(h, w, b, x, "gelu")
    for g, v in zip(core.grad(core.sum(y * y, [0, 1]).reshape([]), [x, gamma, beta, w, b]), (x, gamma, beta, w, b)):
        assert g.shape == v.shape
    with pytest.raises(ValueError, match="keepPre"):
        core.grad(core.sum(core.denseAct(x, w, b, None, "gelu", keepPre=False), [0, 1]).reshape([]), [w])


def test_layers():
    f, init = core.float32([4, 16]), nnet.Init(0)
    body = nnet.groupNorm(nnet.dataSource(f), 4, "silu")
    body = nnet.denseAct(body, 16, init, "gelu", residual=nnet.dataSource(f), weight_decay=1e-4)
    net = nnet.DAGNetwork([f], [body])
    assert [p.shape for p in net.params] == [(16,), (16,), (16, 16), (16,)]
    assert body.output.shape == body.trainOutput.shape == (4, 16)


# ------------------------------------------------------------------------------------------------ the float64 forms

@pytest.mark.parametrize("name", R.ACTS)
@pytest.mark.parametrize("last", [False, True])
def test_group_norm_gradient_against_differences(name, last):
    r = np.random.default_rng(1)
    shape = (3, 2, 5, 6) if last else (3, 6, 2, 5)
    x, dy = r.standard_normal(shape) + 0.3, r.standard_normal(shape)
    scale, bias = 1 + 0.3 * r.standard_normal(6), 0.3 * r.standard_normal(6)
    groups, eps = 3, 1e-5

    def loss(x, scale, bias):
        return float((R.group_norm(x, scale, bias, groups, eps, name, last)[0][0] * dy).sum())
    (_, (mean, _), (rstd, _)) = R.group_norm(x, scale, bias, groups, eps, name, last)
    grads = [v for v, _ in R.group_norm_grad(dy, x, scale, bias, mean, rstd, groups, name, last)]
    _differences(loss, [x, scale, bias], grads, r)


@pytest.mark.parametrize("name", R.ACTS)
def test_dense_gradient_against_differences(name):
    r = np.random.default_rng(2)
    x, w, b, dy = r.standard_normal((4, 7)), r.standard_normal((5, 7)), r.standard_normal(5), r.standard_normal((4, 5))

    def loss(x, w, b):
        return float((R.dense_act(x, w, b, dy, name)[0][0] * dy).sum())
    grads = [v for v, _ in R.dense_act_grad(dy, x, w, R.dense_act(x, w, b, None, name)[1][0], name)]
    _differences(loss, [x, w, b], grads, r)


def _differences(loss, at, grads, r):
    """Central differences along random directions; their error is of second order in h: 1e-5 of values near one, 1e-10 / 1e-5 of rounding."""
    h = 1e-5
    for i, g in enumerate(grads):
        d = r.standard_normal(g.shape)
        up, down = list(at), list(at)
        up[i], down[i] = at[i] + h * d, at[i] - h * d
        slope, want = (loss(*up) - loss(*down)) / (2 * h), float((g * d).sum())
        assert abs(slope - want) <= 1e-6 * (1 + np.abs(g * d).sum()), (i, slope, want)


def test_muon_brings_singular_values_near_one():
    r = np.random.default_rng(3)
    w, g = np.zeros((12, 30)), r.standard_normal((12, 30))
    for shape in ((12, 30), (30, 12)):
        _, m, o = R.muon(w.reshape(shape), g.reshape(shape), 0 * g.reshape(shape), 1.0, 0.9, False, 0.0, 5)
        s = np.linalg.svd(o, compute_uv=False) / max(1.0, shape[0] / shape[1]) ** 0.5
        assert 0.6 < s.min() and s.max() < 1.25 and np.array_equal(m, g.reshape(shape))
