"""Block-scaled operators where ordinary inputs do not look: what is not finite, the tails of the activation
functions, the border of the 8-bit codes.  Through the package's public entry points, against the definitions in 64 bits."""
import numpy as np
import pytest

import oracle as orc

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("shape", [(2, 64), (3, 45)])
def test_relu_keeps_what_is_not_a_number(ng, dtype, shape):
    """forward: NaN stays NaN, infinities are themselves; backward: every value of a block that is marked NaN has a NaN
    derivative, as with the other functions, so that one overflowed activation cannot silence its 31 neighbours"""
    z = np.full(shape, 1.5, dtype=dtype)
    z[:, ::2] = -2.0
    z[0, 3], z[0, 4], z[1, 40], z[1, 41] = np.nan, -np.inf, np.inf, -0.0
    Y, Q = ng.empty(shape, dtype=dtype), ng.mx_empty(shape, "int8", rounding=0)
    ng.fprop_act("relu", ng.array(z, dtype=dtype), Y, saved=Q)
    assert np.array_equal(Y.get(), np.maximum(z, 0), equal_nan=True)
    bad = np.isnan(Q.get())
    assert bad[0, :32].all() and bad[1, 32:].all() and not bad[0, 32:].any() and not bad[1, :32].any()
    G = ng.ones(shape, dtype=dtype)
    ng.bprop_act("relu", Q, G, G)
    assert np.array_equal(G.get(), np.where(bad, np.nan, z > 0), equal_nan=True)


def test_relu_below_a_dense_layer_keeps_what_is_not_a_number(ng):
    """the same through FullLayer.relu_below: an infinity in the saved input marks its block of the error passed down"""
    from nervanagpu_amd.layers import FullLayer
    nin, nout, N = 40, 33, 48
    rng = np.random.default_rng(1)
    x = np.abs(rng.standard_normal((nin, N))).astype(np.float16) + np.float16(0.5)
    layer = FullLayer(ng, np.float16, N, nin, nout, save8=True)
    layer.init_activations()
    layer.init_deltas()
    layer.init_weights()
    layer.relu_below, layer.relu_done_above = True, True
    layer.fprop(ng.array(x))
    layer.fprop_in.set(np.where(np.arange(nin * N).reshape(nin, N) == 5 * N + 7, np.inf, x))
    ng.mx_quantize(layer.fprop_in, layer.saved_in)
    dx = layer.bprop(ng.array(rng.standard_normal((nout, N)).astype(np.float16))).get()
    bad = np.isnan(dx)
    assert bad[5, :32].all() and bad.sum() == 32
