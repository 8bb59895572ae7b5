"""What the Python surface of the block-scaled operators promises or refuses, without a device."""
import pytest

from nervanagpu_amd import NervanaGPU
from test_mx_host import calls, fake, fake_mx  # noqa: F401

FAR = [2 ** 31, 2 ** 32 + 64]


@pytest.mark.parametrize("far", FAR)
def test_extents_that_do_not_fit_an_int_are_refused(calls, far):  # noqa: F811
    """extents travel as ints: 2^32 + 64 rows would arrive as 64, and the rest would be left as it was"""
    ng = NervanaGPU()
    for shape in ((far, 32), (32, far), (far, 1), (1, far)):
        for axis in (0, 1):
            with pytest.raises(AssertionError, match="2\\^31"):
                fake_mx(ng, shape, axis=axis)
        with pytest.raises(AssertionError, match="2\\^31"):
            ng.fprop_act("relu", fake(ng, shape), fake(ng, shape))
    left, right = fake_mx(ng, (8, 32)), fake_mx(ng, (32, 8), axis=0)
    for A, B, C in ((fake(ng, (far, 32)), right, fake(ng, (far, 8))), (left, fake(ng, (32, far)), fake(ng, (8, far))),
                    (left, fake(ng, (far, 32)).T, fake(ng, (far, 8)).T)):
        with pytest.raises(AssertionError, match="2\\^31"):
            ng.mx_dot(A, B, C)
    assert not calls


def test_rectifier_below_a_layer_without_saved_input_is_refused():
    """relu_below reads the saved input: without one the derivative of the layer below would be left out unseen"""
    import numpy as np
    from nervanagpu_amd.layers import FullLayer
    layer = FullLayer(NervanaGPU(), np.float16, 32, 64, 16)
    layer.relu_below = layer.relu_done_above = True
    with pytest.raises(AssertionError, match="save8"):
        layer.bprop(None)
