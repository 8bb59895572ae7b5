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


EPS32, HALF16 = 2.0 ** -24, 2.0 ** -11


def _close(got, ref, tol, what):
    """within tol, and for fp16 half a unit of the result (2^-11 of its value, 2^-25 among the subnormal numbers); tol and
    the reference are in 64 bits and both have the result's own magnitude, however small that is"""
    if got.dtype == np.float16:
        tol = tol * (1 + HALF16) + np.maximum(np.abs(ref) * HALF16, 2.0 ** -25)
    else:
        tol = tol + np.maximum(np.abs(ref) * EPS32, 2.0 ** -149)
    off = np.abs(got.astype(np.float64) - ref)
    worst = np.argmax(off - tol)
    assert np.all(off <= tol), "%s: %g instead of %g, %g allowed" % (what, got.flat[worst], ref.flat[worst], tol.flat[worst])


def _all_halves(lo, hi):
    h = np.arange(65536, dtype=np.uint16).view(np.float16)
    h = h[np.isfinite(h)]
    h = np.sort(h[(h >= lo) & (h <= hi)])
    return np.concatenate([h, np.zeros(-len(h) % 96, dtype=np.float16)]).reshape(-1, 96)


def _checkpoints(top):
    """values that 8-bit codes hold exactly: lines of one block, codes -127 .. 127 of every scale, to nearly twice `top`"""
    codes = np.concatenate([np.arange(-127, 128), [127]])
    rows = [np.append(part[:-1], 127) * 2.0 ** e for e in range(int(np.log2(top)) - 6, -12, -1) for part in codes.reshape(-1, 32)]
    return np.array(rows, dtype=np.float32)


# Bounds in units of 2^-24 of the value.  fp16 operands: the tail Phi(-x) is a bell times a polynomial's quotient.  The quotient is off by
# its fit (2.4e-6: 40 units), the argument t of its polynomial (3 units, which count 2.7-fold at most) and 6 steps of it (8); the bell by the
# exponential (2) and by its argument's two roundings (z^2); three products: 61 + z^2 in all.  fp32 operands: erfc 16 ulp (32 units),
# its argument's two roundings (2 z^2), two products.  The tail's complement adds one rounding of a value above 1/2.
def _gelu_units(z, dtype):
    return 61 + z * z if dtype == np.float16 else 35 + 2 * z * z


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_gelu_keeps_the_digits_of_its_left_tail(ng, dtype):
    """every fp16 argument up to where the result vanishes, and for fp32 as far as the result is a normal number: the bound follows
    the result itself"""
    z = _all_halves(-6.5, 20) if dtype == np.float16 else np.linspace(-12.5, 12.5, 96 * 40, dtype=np.float32).reshape(-1, 96)
    Y = ng.empty(z.shape, dtype=dtype)
    ng.fprop_act("gelu", ng.array(z, dtype=dtype), Y)
    zd = z.astype(np.float64)
    ref = orc.ref_act("gelu", zd)
    _close(Y.get(), ref, _gelu_units(zd, dtype) * EPS32 * np.abs(ref), "gelu")


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("error", [1.0, 1024.0])
def test_gelu_slope_keeps_the_digits_of_its_left_tail(ng, dtype, error):
    """Phi(z) + z phi(z): each of the two to its own digits (they cancel near z = -0.75 alone), then one sum and one product"""
    z = _checkpoints(8.0)
    q = ng.mx_array(z, "int8", rounding=0)
    assert np.array_equal(q.get(), z)
    G = ng.empty(z.shape, dtype=dtype)
    ng.bprop_act("gelu", q, ng.array(np.full(z.shape, error, dtype=dtype), dtype=dtype), G)
    zd = z.astype(np.float64)
    parts = orc.ref_act("gelu", -np.abs(zd)) / np.where(zd == 0, -1, -np.abs(zd)) * (zd != 0) + 0.5 * (zd == 0) \
        + np.abs(zd) * np.exp(-0.5 * zd * zd) / np.sqrt(2 * np.pi)
    ref = error * orc.ref_act_slope("gelu", zd)
    tol = EPS32 * (error * _gelu_units(zd, dtype) * parts + 3 * np.abs(ref))
    # beyond |z| = 13 the tail and the density are subnormal numbers, off by up to a unit of 2^-149, which |z| and the error multiply
    tol += error * (1 + np.abs(zd)) * 2.0 ** -149
    _close(G.get(), ref, tol, "slope of gelu")


# Units of 2^-24 of the slope.  With t = e^-|z| (tanh: e^-2|z|) and r = 1 / (1 + t) the slopes are t r r and 4 t r r.  fp32 operands: exp
# 3 ulp (6 units); of it r takes at most half, its sum and quotient 1 + 5, twice; two products: 26.  fp16 operands: exp and reciprocal 1 ulp
# (2 units) and the two roundings of the exponent (2 units a unit of its argument, of which r's take at most half, twice): 12 + 4 |z|.
def _saturated_units(op, z, dtype):
    if dtype == np.float32:
        return 26 + 0 * z
    return 12 + 4 * np.abs(z) * (2 if op == "tanh" else 1)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("op", ["sig", "tanh"])
@pytest.mark.parametrize("error", [1.0, -1024.0])
def test_slopes_of_saturated_functions(ng, dtype, op, error):
    """sig' and tanh' fall like e^-|z| and e^-2|z| on both sides: the bound follows them"""
    z = _checkpoints(16.0)
    q = ng.mx_array(z, "int8", rounding=0)
    assert np.array_equal(q.get(), z)
    G = ng.empty(z.shape, dtype=dtype)
    ng.bprop_act(op, q, ng.array(np.full(z.shape, error, dtype=dtype), dtype=dtype), G)
    zd = z.astype(np.float64)
    t = np.exp(-np.abs(zd) * (2 if op == "tanh" else 1))
    ref = error * (4 if op == "tanh" else 1) * t / (1 + t) ** 2
    _close(G.get(), ref, (_saturated_units(op, zd, dtype) + 1) * EPS32 * np.abs(ref), op)


@pytest.mark.parametrize("op", ["sig", "silu"])
def test_logistic_functions_keep_their_left_tail(ng, op):
    """fp32, as far as the value is a normal number (e^-87): e^z (1 + e^z)^-1 needs no e^-z, which leaves the range of fp32 there.
    exp 3 ulp (6 units), a sum and a quotient (6 and at most half of exp's), two products; what underflows on the way is off by 2^-149,
    times z for silu"""
    z = np.linspace(-103.0, 30.0, 96 * 40, dtype=np.float32).reshape(-1, 96)
    Y = ng.empty(z.shape, dtype=np.float32)
    ng.fprop_act(op, ng.array(z, dtype=np.float32), Y)
    zd = z.astype(np.float64)
    ref = orc.ref_act(op, zd)
    tol = 18 * EPS32 * np.abs(ref) + 3 * 2.0 ** -149 * (np.abs(zd) if op == "silu" else 1)
    _close(Y.get(), ref, tol, op)
    q = ng.mx_array(np.tile(np.arange(-103, -71, dtype=np.float32), (2, 1)), "int8", rounding=0)
    if op == "silu":
        G = ng.ones((2, 32), dtype=np.float32)
        ng.bprop_act(op, q, G, G)
        zq = q.get().astype(np.float64)
        ref = orc.ref_act_slope(op, zq)
        _close(G.get(), ref, 18 * EPS32 * np.abs(ref) + 3 * 2.0 ** -149 * np.abs(zq), "slope of silu")


@pytest.mark.parametrize("axis", [0, 1])
@pytest.mark.parametrize("top", [127.0, 127.5, 127.984375])
def test_stochastic_int8_is_right_on_average_up_to_its_last_code(ng, axis, top):
    """units of the block are 1 here (its largest value lies in 64 .. 128).  Up to 127 units the mean of n draws is right: between
    neighbours 1 apart its variance is at most 1 / 4n, 6 sigma are 3 / sqrt(n), and the 16 bits of the definition add 2^-16.  Above there
    is no code: such values become 127 in every draw, stochastic or not"""
    n = 4096
    row = np.zeros(32, dtype=np.float32)
    row[:9] = [top, 126.75, -126.25, 100.5, -64.1, 12.3, 0.4, -0.03, -top]
    x = np.tile(row, (n, 1)) if axis == 1 else np.tile(row[:, None], (1, n))
    q = ng.mx_empty(x.shape, "int8", axis, rounding=1)
    got = ng.mx_quantize(ng.array(x, dtype=np.float32), q).get().astype(np.float64)
    got = got if axis == 1 else got.T
    below = np.abs(row) <= 127
    assert np.all(np.abs(got.mean(axis=0) - row)[below] <= 3 / np.sqrt(n) + 2.0 ** -16)
    assert np.all(got[:, ~below] == np.sign(row[~below]) * 127)
    nearest = ng.mx_quantize(ng.array(x, dtype=np.float32), ng.mx_empty(x.shape, "int8", axis, rounding=0)).get()
    assert np.array_equal((nearest if axis == 1 else nearest.T)[0][~below], np.sign(row[~below]) * 127)
