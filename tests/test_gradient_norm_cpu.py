"""The norm of a set of gradients and clipping: what is refused before the device is touched."""
import ctypes as C

import pytest

from dopt_amd import capi, core, online

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
