"""Dense layers of groups of rows: what is refused before the device is touched, what the graph operation is, and the float64 form's
gradients against differences."""
import ctypes as C

import numpy as np
import pytest

import dense_groups as D
from dopt_amd import capi, core, nnet

P = C.c_void_p


def _addr(n):
    return P(n << 24) if n else None


def _forward(G=3, M=4, N=8, K=16, act=0, o=1, x=2, w=3, bias=4, y=5, pre=6):
    return capi.load().dopt_hip_dense_groups(G, M, N, K, act, *[_addr(p) for p in (o, x, w, bias, y, pre)])


def _backward(G=3, M=4, N=8, K=16, act=2, o=1, dy=2, pre=3, x=4, w=5, dx=6, dw=7, dbias=8):
    return capi.load().dopt_hip_dense_groups_grad(G, M, N, K, act, *[_addr(p) for p in (o, dy, pre, x, w, dx, dw, dbias)])


@pytest.mark.parametrize("call, text", [
    (lambda: _forward(act=4), b"activation 4"), (lambda: _forward(act=-1), b"activation -1"), (lambda: _forward(o=0), b"null"),
    (lambda: _forward(x=0), b"null"), (lambda: _forward(w=0), b"null"), (lambda: _forward(y=0), b"null"), (lambda: _forward(y=1), b"overlaps"),
    (lambda: _forward(y=4), b"overlaps"), (lambda: _forward(pre=2), b"overlaps"), (lambda: _forward(pre=5), b"two results"),
    (lambda: _forward(M=1 << 31), b"too large"), (lambda: _forward(N=1 << 21), b"too large"), (lambda: _forward(K=1 << 21), b"too large"),
    (lambda: _forward(N=1 << 15, K=1 << 15), b"too large"), (lambda: _forward(G=(1 << 20) + 1), b"too large"),
    (lambda: _backward(act=9), b"activation 9"), (lambda: _backward(o=0), b"null"), (lambda: _backward(dy=0), b"null"), (lambda: _backward(pre=0), b"null"),
    (lambda: _backward(w=0), b"needs w"), (lambda: _backward(x=0), b"needs x"), (lambda: _backward(dx=2), b"overlaps"), (lambda: _backward(dw=1), b"overlaps"),
    (lambda: _backward(dw=6), b"two results"), (lambda: _backward(M=1 << 20, N=1 << 20), b"too large"),
])
def test_refusals(call, text):
    assert call() == 1
    assert text in capi.load().dopt_hip_last_error(), capi.load().dopt_hip_last_error()


def test_graph_operation_is_verified():
    f, i = core.float32, core.int32
    x, w, o = f([5, 6]), f([3, 4, 6]), i([4])
    assert core.denseGroups(x, w, o).shape == core.denseGroups(x, w, o, f([3, 4]), "gelu").shape == (5, 4)
    for bad in (lambda: core.denseGroups(x, w, i([3])), lambda: core.denseGroups(x, w, f([4])), lambda: core.denseGroups(x, f([4, 6]), o),
                lambda: core.denseGroups(f([5, 7]), w, o), lambda: core.denseGroups(x, w, o, f([3, 3])), lambda: core.denseGroups(x, w, o, f([4, 3])),
                lambda: core.denseGroups(i([5, 6]), w, o), lambda: core.denseGroups(f([5]), w, o)):
        with pytest.raises(core.VerificationError):
            bad()
    with pytest.raises(ValueError, match="no activation"):
        core.denseGroups(x, w, o, activation="tanh")


def test_gradients_have_their_operands_shapes():
    f = core.float32
    x, w, o, b = f([5, 6]), f([3, 4, 6]), core.int32([4]), f([3, 4])
    for y in (core.denseGroups(x, w, o, b, "gelu"), core.denseGroups(x, w, o, b), core.denseGroups(x, w, o)):
        wrt = [x, w] + ([b] if len(core.topological_sort([y])) > 5 else [])
        loss = core.sum(y * y, [0, 1]).reshape([])
        wrt = [v for v in (x, w, b) if v in core.topological_sort([y])]
        for g, v in zip(core.grad(loss, wrt), wrt):
            assert g.shape == v.shape
        with pytest.raises(ValueError, match="Could not find"):
            core.grad(loss, [o])
    with pytest.raises(ValueError, match="keepPre"):
        core.grad(core.sum(core.denseGroups(x, w, o, b, "gelu", keepPre=False), [0, 1]).reshape([]), [w])


def test_layer():
    f, o, init = core.float32([5, 6]), core.int32([4]), nnet.Init(0)
    body = nnet.denseGroups(nnet.dataSource(f), o, 3, 8, init, "silu", weight_decay=1e-3)
    body = nnet.denseGroups(body, o, 3, 2, init, use_bias=False)
    net = nnet.DAGNetwork([f], [body])
    assert [p.shape for p in net.params] == [(3, 8, 6), (3, 8), (3, 2, 8)]
    assert body.output.shape == body.trainOutput.shape == (5, 2)


def test_boundaries():
    assert D.bounds([3, 1, 7, 5, 9], 8).tolist() == [3, 3, 7, 7, 8]
    assert D.bounds([-5, 2, -1, 100], 8).tolist() == [0, 2, 2, 8]


@pytest.mark.parametrize("name", ("none", "relu", "gelu", "silu"))
def test_gradient_against_differences(name):
    r = np.random.default_rng(2)
    offsets = [1, 4, 4, 7]
    x, w, b, dy = r.standard_normal((8, 6)), r.standard_normal((3, 5, 6)), r.standard_normal((3, 5)), r.standard_normal((8, 5))
    pre = D.forward(x, w, b, offsets, name)[1][0]

    def loss(x, w, b):
        return float((D.forward(x, w, b, offsets, name)[0][0] * dy).sum())
    grads = [v for v, _ in D.backward(dy, x, w, pre, offsets, name)]
    at, h = [x, w, b], 1e-5
    for i, g in enumerate(grads):
        d = r.standard_normal(g.shape)
        up, down = list(at), list(at)
        up[i], down[i] = at[i] + h * d, at[i] - h * d
        slope, want = (loss(*up) - loss(*down)) / (2 * h), float((g * d).sum())
        assert abs(slope - want) <= 1e-6 * (1 + np.abs(g * d).sum()), (i, slope, want)
