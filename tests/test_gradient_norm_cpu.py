"""The norm of a set of gradients and clipping: what is refused before the device is touched."""
import ctypes as C

import numpy as np
import pytest

from dopt_amd import capi, core, online
from oracle import evaluator

P = C.c_void_p


def _create(*tensors):
    """tensors: (gradient, result, size) with addresses that nobody reads."""
    refs = (capi.GradientRef * max(1, len(tensors)))(*[capi.GradientRef(g << 24 or None, out << 24 or None, n) for g, out, n in tensors])
    h = P(7)
    rc = capi.load().dopt_hip_gradient_norm_create(len(tensors), refs, C.byref(h))
    assert not h.value
    return rc


@pytest.mark.parametrize("tensors, text", [
    ([(0, 0, 4)], b"tensor 0 is null"), ([(1, 0, 4), (0, 2, 4)], b"tensor 1 is null"), ([(1, 0, 1 << 41)], b"too large"),
    ([(1, 2, 4), (3, 2, 4)], b"overlaps"), ([(1, 1, 4), (1, 1, 4)], b"overlaps"), ([(1, 2, 4), (2, 3, 4)], b"overlaps"),
    ([(1, 1, 4), (1, 2, 4)], b"overlaps"), ([(1, 2, (1 << 22) + 1)], b"overlaps"), ([(2, 1, (1 << 22) + 1)], b"overlaps"),
    ([(5, 6, 1), (1, 1, (5 << 22) + 1)], b"overlaps"),
])
def test_refusals(tensors, text):
    assert _create(*tensors) == 1
    assert text in capi.load().dopt_hip_last_error(), capi.load().dopt_hip_last_error()


def test_calls_need_a_handle():
    lib = capi.load()
    for call in (lib.dopt_hip_gradient_norm, lib.dopt_hip_gradient_clip):
        assert call(None, 1.0, P(1 << 24)) == 1 and b"handle" in lib.dopt_hip_last_error()
    assert lib.dopt_hip_gradient_norm_create(1, None, C.byref(P())) == 1
    assert lib.dopt_hip_gradient_norm_create(-1, None, C.byref(P())) == 1
    assert lib.dopt_hip_gradient_norm_create(0, None, None) == 1
    assert lib.dopt_hip_gradient_norm_destroy(None) == 0
    assert lib.dopt_hip_sgd_step_scaled(None, 0.1, 0.9, 0, None) == 1 and b"handle" in lib.dopt_hip_last_error()
    assert lib.dopt_hip_muon_step_scaled(None, 0.1, 0.9, 1, 0.0, 5, None) == 1 and b"handle" in lib.dopt_hip_last_error()


def test_gradients_in_a_graph():
    g = [core.float32([3, 4]), core.float32([5])]
    assert online.clipped(g, None) == g and online.clipped(g, float("inf")) == g and online.clipped([], 1.0) == []
    assert [c.shape for c in online.clipped(g, 1.0)] == [(3, 4), (5,)]
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="largest norm"):
            online.clipped(g, bad)


@pytest.mark.parametrize("rule", ["fused_sgd", "fused_adam", "fused_amsgrad", "fused_muon"])
def test_fused_updaters_refuse_a_norm_that_is_none(rule):
    x = core.float32([3])
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="largest norm"):
            getattr(online, rule)([core.sum(x * x)], [x], maxNorm=bad)


def _clipped(values, most):
    """The graph's gradients as the oracle's evaluator has them."""
    g = [core.float32(v.shape) for v in values]
    return evaluator.evaluate(online.clipped(g, most), dict(zip(g, values)))


@pytest.mark.parametrize("most", [0.0, 1e-30, 1.0, 4.0, 5.0, 1e3, 3e38, 1e39])
@pytest.mark.parametrize("value", [0.0, 1e-24])
def test_a_norm_of_zero_in_a_graph(value, most):
    """Gradients of a step without any stay what they are: their norm is in bounds wherever it is not the largest one that is nothing, and then what
    is left of them is nothing as well."""
    values = [np.full((3, 4), value, np.float32), np.full(5, -value, np.float32)]
    for got, v in zip(_clipped(values, most), values):
        assert np.isfinite(got).all()
        if most >= 1.0 or not value:
            assert np.array_equal(got, v)


@pytest.mark.parametrize("most", [0.5, 5.0, 12.9, 13.1, 1e39])
def test_norms_of_ordinary_size_in_a_graph(most):
    """3, 4 and 12 of two gradients: the norm is 13.  The factor is off by the roundings of four squares, their three sums, the root, the quotient: under
    nine halves of a last place, and the product's."""
    values = [np.array([[3.0, 4.0]], np.float32), np.array([0.0, -12.0], np.float32)]
    for got, v in zip(_clipped(values, most), values):
        want = v.astype(np.float64) * min(1.0, most / 13.0)
        assert np.abs(got - want).max() <= 10 * 2.0 ** -24 * 12 and (most < 13 or np.array_equal(got, v))


@pytest.mark.parametrize("most", [0.0, 1e-25, 1e-3, 1.0, 5.0, 1e18, 1e22])
@pytest.mark.parametrize("size", [1e-44, 1e-38, 1e-30, 1e-24, 1e-19, 1.0, 1e18, 1e20, 1e37])
def test_gradients_of_any_size_in_a_graph(size, most):
    """Against the definition in 64 bits.  A square over the largest one is off by three roundings of values over the largest, the sums of under thirty
    values by thirty, the root halves that: the norm is within 18 roundings, the quotients add two, the product one.  A quotient or product
    below the smallest normal number is off by up to 2^-149."""
    r = np.random.default_rng(7)
    values = [(size * r.uniform(-9, 9, s)).astype(np.float32) for s in ((3, 4), (5,), (2, 2, 2))]
    norm = np.sqrt(sum((v.astype(np.float64) ** 2).sum() for v in values))
    factor = 1.0 if norm <= most else most / norm
    for got, v in zip(_clipped(values, most), values):
        want = v.astype(np.float64) * factor
        assert np.isfinite(got).all()
        assert (np.abs(got - want) <= 21 * 2.0 ** -24 * np.abs(want) + np.abs(v) * 2.0 ** -149 + 2.0 ** -149).all()


def test_gradients_that_are_not_finite_in_a_graph():
    ordinary = np.array([1.0, -2.0], np.float32)
    for most in (0.5, 5.0):
        got = _clipped([ordinary, np.array([np.inf, 3.0], np.float32)], most)
        assert not got[0].any() and np.isnan(got[1][0]) and got[1][1] == 0
        got = _clipped([ordinary, np.array([np.nan, 3.0], np.float32)], most)
        assert np.isnan(got[0]).all() and np.isnan(got[1]).all()
