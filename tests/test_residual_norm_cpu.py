"""The residual norm: what is refused before the device is touched, what the graph operation is, and its float64 form against
differences."""
import ctypes as C
import re

import numpy as np
import pytest

import residual_norm as R
from dopt_amd import capi, core, nnet

P = C.c_void_p


def _addr(n):
    return P(n << 24) if n else None


def _desc(rows=6, cols=8, gates=2, post=1, pre=2, eps=1e-5, scale=1.0):
    return capi.ResidualNormDesc(rows, cols, gates, post, pre, eps, scale)


def _forward(x=1, branch=2, gate=3, ps=4, pb=5, qs=6, qb=7, y=8, h=9, stats=10, **desc):
    return capi.load().dopt_hip_residual_norm(C.byref(_desc(**desc)), *[_addr(p) for p in (x, branch, gate, ps, pb, qs, qb, y, h, stats)])


def _backward(dy=1, dh=2, y=3, branch=4, gate=5, ps=6, pb=7, qs=8, stats=9, dx=10, db=11, dg=12, dps=13, dpb=14, dqs=15, dqb=16, **desc):
    return capi.load().dopt_hip_residual_norm_grad(C.byref(_desc(**desc)), *[_addr(p) for p in (
        dy, dh, y, branch, gate, ps, pb, qs, stats, dx, db, dg, dps, dpb, dqs, dqb)])


@pytest.mark.parametrize("call, text", [
    (lambda: _forward(post=3), b"norm 3"), (lambda: _forward(pre=-1), b"norm -1"), (lambda: _forward(gates=4), b"share 4"),
    (lambda: _forward(gates=7), b"share 7"), (lambda: _forward(gates=0), b"0 gates, and an operand"), (lambda: _forward(gate=0), b"no operand"),
    (lambda: _forward(eps=-1.0), b"eps"), (lambda: _forward(eps=float("nan")), b"eps"), (lambda: _forward(post=0), b"not there"),
    (lambda: _forward(pre=0, h=0), b"not there"), (lambda: _forward(branch=0), b"branch that is not there"),
    (lambda: _forward(x=0, branch=0, gate=0, gates=0, post=0, ps=0, pb=0), b"neither"), (lambda: _forward(h=0), b"belong together"),
    (lambda: _forward(pre=0, qs=0, qb=0), b"belong together"), (lambda: _forward(y=0, h=0, pre=0, qs=0, qb=0), b"no result"),
    (lambda: _forward(y=3), b"overlaps an operand"), (lambda: _forward(h=7), b"overlaps an operand"), (lambda: _forward(stats=1), b"overlaps an operand"),
    (lambda: _forward(y=9), b"two results"), (lambda: _forward(stats=8), b"two results"), (lambda: _forward(rows=1 << 21, cols=8), b"two results overlap"),
    (lambda: _forward(rows=1 << 32), b"too large"), (lambda: _forward(cols=1 << 30), b"too large"),
    (lambda: _backward(dh=0), b"gradient of h"), (lambda: _backward(y=0), b"gradient of h"), (lambda: _backward(pre=0, qs=0), b"gradient of h"),
    (lambda: _backward(dy=0, dh=0, pre=0, qs=0, dqs=0, dqb=0), b"gradient of h"), (lambda: _backward(stats=0), b"statistics"),
    (lambda: _backward(branch=0, gates=0, gate=0, post=0, ps=0, pb=0, dg=0, dps=0, dpb=0), b"branch that is not there"),
    (lambda: _backward(gates=0, gate=0), b"gate that is not there"), (lambda: _backward(post=0, ps=0, pb=0), b"norm that is not there"),
    (lambda: _backward(dx=1), b"overlaps an operand"), (lambda: _backward(dg=12, dps=12), b"two results"), (lambda: _backward(dqb=9), b"overlaps an operand"),
])
def test_refusals(call, text):
    assert call() == 1
    assert text in capi.load().dopt_hip_last_error(), capi.load().dopt_hip_last_error()


def test_null_descriptor():
    lib = capi.load()
    assert lib.dopt_hip_residual_norm(None, *[None] * 10) == 1 and lib.dopt_hip_residual_norm_grad(None, *[None] * 16) == 1


def test_graph_operation_is_verified():
    f = core.float32
    x, b, c = f([2, 3, 8]), f([2, 3, 8]), f([8])
    y, h = core.residualNorm(x, b, f([2, 8]), "layer", c, c, "rms", c)
    assert y.shape == h.shape == (2, 3, 8)
    assert core.residualNorm(x, b)[1] is None and core.residualNorm(x, pre="layer")[1].shape == (2, 3, 8)
    assert core.residualNorm(x, b, f([6, 8]), pre="rms")[0].shape == (2, 3, 8)
    for bad in (lambda: core.residualNorm(x, f([2, 3, 4])), lambda: core.residualNorm(x, f([3, 2, 8])), lambda: core.residualNorm(x, b, f([4, 8])),
                lambda: core.residualNorm(x, b, f([7])), lambda: core.residualNorm(x, None, c), lambda: core.residualNorm(x, b, post="rms", postScale=f([4])),
                lambda: core.residualNorm(x, b, postScale=c), lambda: core.residualNorm(x, b, preBias=c), lambda: core.residualNorm(x, post="rms"),
                lambda: core.residualNorm(core.int32([2, 8])), lambda: core.residualNorm(f([]), pre="rms")):
        with pytest.raises(core.VerificationError):
            bad()
    with pytest.raises(ValueError, match="no norm"):
        core.residualNorm(x, b, post="batch")
    with pytest.raises(ValueError, match="stream or a branch"):
        core.residualNorm()


def test_gradients_have_their_operands_shapes_and_no_padding():
    f = core.float32
    x, b, gate, c = f([4, 3, 8]), f([4, 3, 8]), f([4, 8]), [f([8]) for _ in range(4)]
    y, h = core.residualNorm(x, b, gate, "layer", c[0], c[1], "layer", c[2], c[3])
    loss = core.sum(y * y, [0, 1, 2]).reshape([]) + core.sum(h * h, [0, 1, 2]).reshape([])
    grads = core.grad(loss, [x, b, gate] + c)
    for g, v in zip(grads, [x, b, gate] + c):
        assert g.shape == v.shape
    join = [o for o in core.topological_sort(grads) if o.opType == "residualNormGrad"]
    assert len(join) == 1 and join[0].attributes["hasDy"] == 1
    assert not [o for o in core.topological_sort(grads) if o.opType == "pad"]
    only_h = core.grad(core.sum(h * h, [0, 1, 2]).reshape([]), [x])
    assert [o.attributes["hasDy"] for o in core.topological_sort(only_h) if o.opType == "residualNormGrad"] == [0]
    core.grad(core.sum(y * y, [0, 1, 2]).reshape([]), [x, c[2]])


def test_layers():
    f, init = core.float32([4, 16]), nnet.Init(0)
    stream = nnet.dataSource(f)
    _, h = nnet.residualNorm(stream, pre="rms")
    body = nnet.denseAct(h, 16, init, "gelu")
    stream, h = nnet.residualNorm(stream, body, gate=0.1, post="layer", pre="layer", residual_scale=0.9, scale_decay=1e-4)
    out, same = nnet.residualNorm(stream, nnet.denseAct(h, 16, init), nnet.denseAct(nnet.dataSource(f), 16, init))
    assert out is same
    net = nnet.DAGNetwork([f], [out])
    assert sorted(p.shape for p in net.params) == sorted([(16,)] + [(16, 16), (16,)] * 3 + [(16,)] * 5)
    assert out.output.shape == out.trainOutput.shape == (4, 16)


@pytest.mark.parametrize("post", R.NORMS)
@pytest.mark.parametrize("pre", R.NORMS)
@pytest.mark.parametrize("gates", [0, 1, 3, 6])
def test_gradient_against_differences(post, pre, gates):
    r = np.random.default_rng(7)
    rows, cols, scale, eps = 6, 9, 0.7, 1e-5
    at = {"x": r.standard_normal((rows, cols)), "branch": r.standard_normal((rows, cols)) + 0.3}
    if gates:
        at["gate"] = r.standard_normal((gates, cols))
    at.update({n: 1 + 0.3 * r.standard_normal(cols) for n in R.NAMES if {"post": post, "pre": pre}[n.split("_")[0]] != "none"})
    cy, ch = r.standard_normal((rows, cols)), r.standard_normal((rows, cols))

    def value(a):
        return R.forward(a["x"], a["branch"], a.get("gate"), post, pre, {n: a.get(n) for n in R.NAMES}, scale, eps)

    def loss(a):
        f = value(a)
        return float((f["y"][0] * cy).sum() + ((f["h"][0] * ch).sum() if pre != "none" else 0.0))
    f = value(at)
    grads = R.backward(cy, ch if pre != "none" else None, f["y"][0], at["branch"], at.get("gate"), f["stats"][0], post, pre,
                       {n: at.get(n) for n in R.NAMES}, scale)
    step = 1e-5
    for name, v in at.items():
        g = grads["d" + name][0]
        d = r.standard_normal(v.shape)
        up, down = dict(at), dict(at)
        up[name], down[name] = v + step * d, v - step * d
        slope, want = (loss(up) - loss(down)) / (2 * step), float((g * d).sum())
        assert abs(slope - want) <= 1e-6 * (1 + np.abs(g * d).sum()), (name, slope, want)


def test_the_library_holds_no_gradient_that_no_call_reaches():
    """A wavefront's lanes have one quad of a row backward; longer rows go to whole wavefronts."""
    names = set(re.findall(rb"join_grad_kILi(\d+)ELi(\d+)E", open(capi.LIB_PATH, "rb").read()))
    assert names == {(b"16", b"1"), (b"32", b"1"), (b"64", b"1"), (b"0", b"2"), (b"0", b"4")}
