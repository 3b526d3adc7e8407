"""Dense layer with activation: operands that hold as many values as they should in another shape."""
import numpy as np
import pytest

from dopt_amd import capi, core, ops

f = core.float32


class _Shaped:
    """A tensor as far as the checks look at one; the calls below end before its memory is."""

    def __init__(self, *shape):
        self.shape, self.dtype, self.size, self.ptr = shape, np.dtype("float32"), int(np.prod(shape)), 1 << 24


@pytest.mark.parametrize("make", [
    lambda: core.denseAct(f([2, 3]), f([4, 3]), None, f([4, 2])), lambda: core.denseAct(f([2, 3]), f([4, 3]), f([4]), f([4, 2]), "gelu"),
    lambda: core.denseAct(f([]), f([4, 3])), lambda: core.denseAct(f([2, 3]), f([])), lambda: core.denseAct(f([3]), f([4, 3])),
    lambda: core.Operation("denseActGrad", [f([4, 2]), f([2, 3]), f([4, 3])], {"activation": 0}),
    lambda: core.Operation("denseActGrad", [f([2, 4]), f([2, 3]), f([4, 3]), f([4, 2])], {"activation": 2}),
    lambda: core.Operation("denseActGrad", [f([2, 4]), f([]), f([4, 3])], {"activation": 0})])
def test_graph_operations_refuse(make):
    with pytest.raises(core.VerificationError):
        make()


def test_rows_of_images_and_flat_values_are_taken():
    assert core.denseAct(f([2, 3]), f([4, 3]), None, f([2, 2, 2])).shape == (2, 4)
    assert core.denseAct(f([2, 3]), f([4, 3]), f([4]), f([8])).shape == (2, 4)


@pytest.mark.parametrize("call, what", [
    (lambda t: ops.dense_act(t(2, 3), t(4, 3), None, t(4, 2), out=t(2, 4)), "residual"), (lambda t: ops.dense_act(t(2, 3), t(4, 3), out=t(2, 4), pre=t(4, 2)), "pre"),
    (lambda t: ops.dense_act_grad(t(4, 2), t(2, 3), t(4, 3), None, "none", t(2, 3), t(4, 3), t(4)), "dy"),
    (lambda t: ops.dense_act_grad(t(2, 4), t(2, 3), t(4, 3), t(4, 2), "silu", t(2, 3), t(4, 3), t(4)), "pre")])
def test_calls_refuse(call, what):
    with pytest.raises(capi.HipError, match="%s has the wrong size" % what):
        call(_Shaped)
