"""The orthogonalised update's kernels that few sets of matrices reach, with two and three iterations: five leave a bound in which one of the three
16-bit products of a value could be missing (a product of a [64 x 64] matrix without it is 2e-4 off after three, the bound 1.6e-4)."""
import numpy as np
import pytest

import norm_dense_muon as R
from dopt_amd import core, nnet, online, ops
from test_gpu_norm_dense_muon import _run_muon

pytestmark = pytest.mark.gpu
F32 = np.float32


# 272, 273 and 272 tiles of 128 x 128 on and below the diagonals of the square matrices: from one per compute unit (256) on they are multiplied
# as such, 64 x 64 tiles of a narrow matrix beside them
SQUARES = {"two": [(2000, 2100), (2100, 1999)], "thirteen": [(700, 800)] * 7 + [(801, 699)] * 6, "mixed": [(2048, 2048), (40, 300), (1920, 2500), (130, 131),
                                                                                                         (576, 64), (500, 641), (641, 129)]}


@pytest.mark.parametrize("iterations", [1, 2, 3])
@pytest.mark.parametrize("which", SQUARES)
def test_large_tiles_of_square_products(which, iterations):
    _run_muon(SQUARES[which], iterations, seed=iterations)


def test_large_tiles_of_square_products_of_weak_directions_off_the_grid():
    from test_gpu_norm_dense_muon import _off_grid
    _run_muon(SQUARES["thirteen"], 2, False, 4, "weak", _off_grid)


# every shorter side at most 64: a group's square products in one workgroup
@pytest.mark.parametrize("iterations", [2, 3, 4])
@pytest.mark.parametrize("shapes", [[(64, 576)], [(576, 63)], [(33, 65), (65, 33), (31, 31)], [(64, 64), (5, 900), (4000, 64), (1, 9), (17, 3, 3, 3)]], ids=str)
def test_square_products_of_small_matrices(shapes, iterations):
    _run_muon(shapes, iterations, seed=iterations)
    _run_muon(shapes, iterations, False, iterations, "weak")


def test_a_matrix_moves_in_a_set_as_it_does_alone():
    """Within the bound of each: a set's size decides where sums are cut."""
    r = np.random.default_rng(7)
    shapes = [(128, 300), (300, 128), (64, 64), (5, 900), (2000, 2100), (2100, 1999)]
    w, g = [r.standard_normal(s, F32) for s in shapes], [r.standard_normal(s, F32) for s in shapes]

    def run(which):
        tw, tg, tm = [ops.tensor(w[i]) for i in which], [ops.tensor(g[i]) for i in which], [ops.Tensor(shapes[i]) for i in which]
        opt = ops.MuonOptimizer(tw, tg, tm)
        opt.step(0.1, 0.9, True, 0.0, 2)
        return [t.numpy().astype(np.float64) for t in tw]
    for which in ([0, 1, 2, 3], [0, 1, 2, 3, 4, 5]):
        for i, a in zip(which, run(which)):
            b = run([i])[0]
            moved = np.linalg.norm(b - w[i])
            assert np.linalg.norm(a - b) <= 2 * R.muon_bound(2) * moved + 4 * R.E * np.linalg.norm(w[i]), shapes[i]


@pytest.mark.parametrize("make", [online.muon, online.fused_muon], ids=["graph", "fused"])
@pytest.mark.parametrize("nesterov", [False, True])
def test_three_steps_of_a_network_follow_the_formula(make, nesterov):
    """Each step against the formula in float64, from the weights and gradients before it: momenta of matrices and of the rest are
    carried from step to step."""
    lr, mu, decay, rest, iterations = 0.02, 0.5, 0.1, 0.05, 2
    feats, labels = core.float32([32, 20]), core.float32([32, 10])
    init = nnet.Init(3)
    h = nnet.groupNorm(nnet.denseAct(nnet.dataSource(feats), 48, init), 6, "silu")
    preds = nnet.softmax(nnet.dense(nnet.denseAct(h, 30, init, "gelu"), 10, init))
    net = nnet.DAGNetwork([feats], [preds])
    loss = nnet.crossEntropy(preds.trainOutput, labels) + net.paramLoss
    r = np.random.default_rng(4)
    dev = {feats: ops.tensor(r.standard_normal((32, 20), F32)), labels: ops.tensor(np.eye(10, dtype=F32)[r.integers(0, 10, 32)])}
    grads = core.compile(core.grad(loss, net.params))
    step = make([loss], net.params, None, learningRate=lr, momentumRate=mu, nesterov=nesterov, decay=decay, restRate=rest, iterations=iterations)
    matrix = [p.rank >= 2 and p.shape[0] > 1 and p.volume > p.shape[0] for p in net.params]
    assert any(matrix) and not all(matrix)
    mom = [np.zeros(p.shape) for p in net.params]
    # two plans' gradients agree to 1000 roundings of their norms; two iterations enlarge that by their slopes, 3.4445^2 at most
    off = 1000 * R.E
    for _ in range(3):
        before = [p.value.astype(np.float64) for p in net.params]
        g = [np.asarray(v, np.float64) for v in grads.execute(dev)]
        step(dev)
        for i, p in enumerate(net.params):
            if matrix[i]:
                want, mom[i], o = R.muon(before[i], g[i], mom[i], lr, mu, nesterov, decay, iterations)
                bound = lr * (R.muon_bound(iterations) + 12 * off) * np.linalg.norm(o)
            else:
                mom[i] = mu * mom[i] + rest * g[i]
                want, bound = before[i] - mom[i], off * np.linalg.norm(mom[i])
            assert np.linalg.norm(p.value - want) <= bound + 4 * R.E * np.linalg.norm(want), (i, p.shape)


@pytest.mark.parametrize("make", [online.muon, online.fused_muon], ids=["graph", "fused"])
@pytest.mark.parametrize("which", ["matrices", "rest", "projected"])
def test_sets_without_a_rest_or_without_matrices(make, which):
    """Only matrices, none at all, and two whose projections change the updated value and replace it."""
    r = np.random.default_rng(8)
    lr, mu, rest, iterations = 0.1, 0.5, 0.2, 2
    shapes = {"matrices": [(6, 9), (12, 5)], "rest": [(7,), (1, 9), (5, 1)], "projected": [(6, 9), (8, 4), (4,)]}[which]
    start, targets = [r.standard_normal(s, F32) for s in shapes], [r.standard_normal(s, F32) for s in shapes]
    ps = [core.float32(list(s), v) for s, v in zip(shapes, start)]
    ts = [core.float32(list(s)) for s in shapes]
    loss = None
    for p, t in zip(ps, ts):
        d = p - t
        term = core.sum(d * d).reshape([])
        loss = term if loss is None else loss + term
    projs = {ps[0]: lambda v: 0.5 * v, ps[1]: lambda ignored: 2.0 * ts[1]} if which == "projected" else {}
    step = make([loss], ps, projs, learningRate=lr, momentumRate=mu, nesterov=False, restRate=rest, iterations=iterations)
    dev = {t: ops.tensor(v) for t, v in zip(ts, targets)}
    want, mom = [s.astype(np.float64) for s in start], [np.zeros(s) for s in shapes]
    for _ in range(3):
        step(dev)
        for i, s in enumerate(shapes):
            g = 2 * (want[i] - targets[i])
            if len(s) > 1 and s[0] > 1 and np.prod(s) > s[0]:
                new, mom[i], o = R.muon(want[i], g, mom[i], lr, mu, False, 0.0, iterations)
                bound = lr * (R.muon_bound(iterations) + 12 * 64 * R.E) * np.linalg.norm(o)
            else:
                mom[i] = mu * mom[i] + rest * g
                new, bound = want[i] - mom[i], 64 * R.E * np.linalg.norm(mom[i])
            if which == "projected" and i < 2:
                new = 0.5 * new if i == 0 else 2.0 * targets[1].astype(np.float64)
            got = ps[i].value.astype(np.float64)
            assert np.linalg.norm(got - new) <= bound + 8 * R.E * np.linalg.norm(new), (i, s)
            want[i] = got   # (the next step starts from the values that are there)
