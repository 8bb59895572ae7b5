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


@pytest.mark.parametrize("kinds", ["44", "4h", "h4", "8h", "h8"])
@pytest.mark.parametrize("m,n,k", [(40, 24, 200), (35, 21, 200), (40, 1, 200), (33, 40, 2600), (70, 9, 2600)])
@pytest.mark.parametrize("out,rounding", [(np.float16, 0), (np.float16, 10), (np.float32, 0)])
def test_rectified_products_keep_what_is_not_a_number(ng, kinds, m, n, k, out, rounding):
    """a row of A and a column of B whose block is NaN reach the result with relu as they do without; the rest is
    the rectified product of small integers, which every store and its roundings hold exactly"""
    rng = np.random.default_rng(m + n)
    a = rng.integers(-2, 3, (m, k)).astype(np.float16)
    b = (rng.integers(-2, 3, (k, n)) * (rng.random((k, n)) < 0.1)).astype(np.float16)
    ref = np.maximum(a.astype(np.float64) @ b.astype(np.float64), 0)
    assert ref.max() < 2048
    ref[m // 2] = np.nan
    a[m // 2, k - 1] = np.nan
    if n > 1:
        ref[:, n - 1] = np.nan
        b[3, n - 1] = np.nan
    side = {"h": lambda x, axis: ng.array(x), "4": lambda x, axis: ng.mx_array(x, "fp4", axis, rounding=0),
            "8": lambda x, axis: ng.mx_array(x, "int8", axis, rounding=0)}
    A, B = side[kinds[0]](a, 1), side[kinds[1]](b, 0)
    for beta in (0.0, 1.0):
        C = ng.ones((m, n), dtype=out)
        C.rounding = rounding
        ng.mx_dot(A, B, C, beta=beta, relu=True)
        assert np.array_equal(C.get(), (ref + beta).astype(out), equal_nan=True)
