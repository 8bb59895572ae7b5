"""Block-scaled matrices (4 and 8 bits), their products, and activation checkpoints, through the package's
public entry points against the 64-bit definitions in oracle/ref_mx.py.

Tolerances.  Codes, scales and values are compared exactly: scaling by powers of two and the comparisons of
the rounding are exact in fp32.  Products: the operands' values are exact, fp32 accumulation errs by at most
sqrt(k) 2^-24 sum|a||b| (util.assert_fp32_sum_close, which says why), an fp16 result by half a unit more.
Activation functions: the bounds are counted at ACT_BOUND."""
import ctypes

import numpy as np
import pytest

import oracle as orc
from util import EPS32, assert_fp16_within_ulp, assert_fp32_sum_close

pytestmark = pytest.mark.gpu

SHAPES = [(1, 1), (1, 31), (2, 32), (3, 33), (64, 64), (5, 257), (130, 100), (33, 1030), (67, 130)]


def _mixed(rng, shape, dtype):
    """normal values under very different row strengths, with zeros, ties, subnormals and large magnitudes"""
    x = rng.standard_normal(shape) * np.exp2(rng.integers(-9, 10, (shape[0], 1)))
    pick = rng.random(shape)
    x = np.where(pick < 0.1, 0.0, x)
    x = np.where((pick > 0.1) & (pick < 0.3), rng.integers(-32, 33, shape) / 4.0, x)      # ties of both formats
    x[0, : shape[1] // 2] = 0.0
    if shape[0] > 2:
        x[1] = rng.integers(-3, 4, shape[1]) * 2.0 ** -24                                   # fp16 subnormals
        x[2] = np.where(rng.random(shape[1]) < 0.5, 65504.0, -60000.0)
    return x.astype(dtype)


def _check(q, x, stochastic=None):
    """a converted tensor against the definition: values, and the scales of every block"""
    seed, stream = stochastic or (None, None)
    codes, scales, values = orc.ref_mx_round(x, q.fmt, q.axis, seed, stream)
    data, sc = q.codes.get(), q.scales.get()
    nb = scales.shape[1]
    assert np.array_equal(sc[:, :nb], scales)
    got = orc.ref_mx_values(data, sc, q.fmt, q.shape, q.axis)
    assert np.array_equal(got, values, equal_nan=True)
    # what lies behind the last value of a line is zero
    full = orc.ref_mx_values(data, np.where(sc == 255, 127, sc), q.fmt, (q.lines, nb * 32), 1)
    assert not full[:, q.depth:].any()
    return values


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("fmt", ["fp4", "int8"])
@pytest.mark.parametrize("axis", [0, 1])
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_quantize_and_back(ng, shape, fmt, axis, dtype):
    rng = np.random.default_rng(shape[0] * 7 + shape[1] + axis)
    x = _mixed(rng, shape, dtype)
    dX = ng.array(x, dtype=dtype)
    q = ng.mx_quantize(dX, ng.mx_empty(shape, fmt, axis))
    values = _check(q, x)
    assert np.array_equal(q.get(), values.astype(np.float32))
    h = ng.empty(shape, dtype=np.float16)
    h.fill(3)
    with np.errstate(over="ignore"):
        assert np.array_equal(ng.mx_dequantize(q, h).get(), values.astype(np.float16))
    # the same matrix through its transposes
    t = ng.mx_quantize(dX.T, ng.mx_empty(shape[::-1], fmt, 1 - axis))
    assert np.array_equal(t.codes.get(), q.codes.get())
    back = ng.empty(shape[::-1], dtype=np.float32)
    assert np.array_equal(ng.mx_dequantize(q.T, back).get(), values.T.astype(np.float32))


@pytest.mark.parametrize("shape", [(1, 1), (3, 33), (5, 257), (130, 100)])
@pytest.mark.parametrize("fmt", ["fp4", "int8"])
@pytest.mark.parametrize("axis", [0, 1])
def test_stochastic_quantize_follows_the_stream(shape, fmt, axis):
    from nervanagpu_amd import NervanaGPU
    ng = NervanaGPU(stochastic_round=True, seed=11)
    rng = np.random.default_rng(shape[1])
    x = _mixed(rng, shape, np.float32)
    dX = ng.array(x, dtype=np.float32)
    for _ in range(2):          # another stream every call
        q = ng.mx_quantize(dX, ng.mx_empty(shape, fmt, axis))
        assert q.rounding
        _check(q, x, (ng.rng_seed, ng.rng_counter))


@pytest.mark.parametrize("fmt", ["fp4", "int8"])
def test_many_blocks_across_the_rows(ng, fmt):
    """large enough for the kernel that puts four blocks together (on a device), ragged at both ends"""
    rng = np.random.default_rng(14)
    x = rng.standard_normal((525, 8200)).astype(np.float16)
    q = ng.mx_quantize(ng.array(x), ng.mx_empty(x.shape, fmt, 0))
    got = q.get()
    for cols in (slice(0, 5), slice(4000, 4006), slice(8190, 8200)):
        _, scales, values = orc.ref_mx_round(x[:, cols], fmt, 0)
        assert np.array_equal(got[:, cols], values.astype(np.float32))
        assert np.array_equal(q.scales.get()[cols, :scales.shape[1]], scales)


def test_stochastic_quantize_is_right_on_average(ng):
    """mean of n draws of a value between neighbours u apart: its variance is at most u^2 / 4n, so 6 sigma of the
    mean are 3 u / sqrt(n); the fixed point of the definition adds at most 2^-14 of a unit"""
    n = 4096
    row = np.zeros(32, dtype=np.float32)
    row[:8] = [5.9, 4.5, 3.2, 2.9, 1.7, 0.6, 0.1, -5.1]
    x = np.tile(row, (n, 1))
    q = ng.mx_empty(x.shape, rounding=1)
    ng.mx_quantize(ng.array(x, dtype=np.float32), q)
    unit = np.where(np.abs(row) < 2, 0.5, np.where(np.abs(row) < 4, 1.0, 2.0))
    assert np.all(np.abs(q.get().astype(np.float64).mean(axis=0) - row) <= unit * (3 / np.sqrt(n) + 2.0 ** -14))


@pytest.mark.parametrize("fmt", ["fp4", "int8"])
@pytest.mark.parametrize("axis", [0, 1])
def test_views_and_what_lies_around_them(ng, fmt, axis):
    """a window of a larger matrix, at every alignment, is read alone; dequantize writes only its window"""
    rng = np.random.default_rng(5)
    big = rng.standard_normal((70, 203)).astype(np.float16)
    big[:, :3] = np.nan
    big[:, 100:] = np.inf
    dB = ng.array(big)
    for lo, hi in ((3, 100), (8, 72), (3, 4)):
        x = big[2:69, lo:hi]
        q = ng.mx_quantize(dB[2:69, lo:hi], ng.mx_empty(x.shape, fmt, axis))
        values = _check(q, x)
        out = ng.ones((70, 203), dtype=np.float32)
        ng.mx_dequantize(q, out[2:69, lo:hi])
        expect = np.ones((70, 203), dtype=np.float32)
        expect[2:69, lo:hi] = values
        assert np.array_equal(out.get(), expect)


@pytest.mark.parametrize("fmt", ["fp4", "int8"])
@pytest.mark.parametrize("axis", [0, 1])
def test_blocks_with_infinities_become_nan(ng, fmt, axis):
    rng = np.random.default_rng(6)
    x = rng.standard_normal((66, 70)).astype(np.float32)
    x[1, 2], x[40, 64], x[65, 69], x[33, 33] = np.inf, np.nan, -np.inf, np.nan
    for dtype in (np.float16, np.float32):
        q = ng.mx_quantize(ng.array(x, dtype=dtype), ng.mx_empty(x.shape, fmt, axis))
        _check(q, x.astype(dtype))
        assert np.isnan(q.get()).any()


@pytest.mark.parametrize("fmt", ["fp4", "int8"])
def test_fp32_range(ng, fmt):
    """the whole range of fp32, subnormal numbers included"""
    x = np.zeros((6, 64), dtype=np.float32)
    for i, m in enumerate((3.4e38, 2.0 ** 120, 2.0 ** -100, 2.0 ** -126, 2.0 ** -140, 2.0 ** -149)):
        x[i] = (np.linspace(-1, 1, 64) * m).astype(np.float32)
    q = ng.mx_quantize(ng.array(x, dtype=np.float32), ng.mx_empty(x.shape, fmt))
    _check(q, x)


# ---- products ---------------------------------------------------------------------------------

def _operand(ng, rng, shape, fmt, axis, scale=1.0):
    """a block-scaled operand and its values"""
    x = (rng.standard_normal(shape) * scale * np.exp2(rng.integers(-3, 4, (shape[0], 1)))).astype(np.float16)
    q = ng.mx_quantize(ng.array(x), ng.mx_empty(shape, fmt, axis))
    return q, orc.ref_mx_values(q.codes.get(), q.scales.get(), fmt, shape, axis)


def _check_product(out, a, b, what, alpha=1.0, beta=0.0, c0=None, relu=False):
    k = a.shape[1]
    ref = alpha * (a @ b)
    if relu:
        ref = np.maximum(ref, 0)
    absdot = abs(alpha) * (np.abs(a) @ np.abs(b))
    if beta:
        ref = ref + beta * c0.astype(np.float64)
        absdot = absdot + abs(beta * c0.astype(np.float64))
    # alpha, beta * C and their sum round once each
    terms = k + (0 if alpha == 1.0 and not beta else 9)
    if out.dtype == np.float32:
        tol = np.sqrt(float(max(terms, 1))) * EPS32 * absdot + EPS32 * np.abs(ref)
        bad = np.abs(out - ref) > tol
        assert not bad.any(), "%s: %d of %d, worst %g" % (what, bad.sum(), bad.size, np.abs(out - ref).max())
    else:
        assert_fp16_within_ulp(out, ref, 0.5, what, np.sqrt(float(max(terms, 1))) * EPS32 * absdot)


DOT_SIZES = [(1, 1, 1), (5, 3, 31), (33, 65, 32), (64, 1, 200), (1, 130, 97), (128, 128, 128), (130, 257, 513),
             (300, 70, 1000), (17, 19, 4099), (257, 136, 64)]


@pytest.mark.parametrize("m,n,k", DOT_SIZES)
@pytest.mark.parametrize("out", [np.float16, np.float32])
def test_fp4_product(ng, m, n, k, out):
    rng = np.random.default_rng(m + n + k)
    A, a = _operand(ng, rng, (m, k), "fp4", 1, 0.25)
    B, b = _operand(ng, rng, (k, n), "fp4", 0)
    C = ng.empty((m, n), dtype=out)
    C.fill(7)
    ng.mx_dot(A, B, C, relu=m % 2 == 0)
    _check_product(C.get(), a, b, "fp4 %s" % ((m, n, k),), relu=m % 2 == 0)


@pytest.mark.parametrize("kinds", ["44", "4h", "h4", "8h", "h8"])
@pytest.mark.parametrize("m,n,k", [(520, 264, 264), (530, 1030, 1100), (2900, 3080, 300)])
def test_larger_products(ng, kinds, m, n, k):
    """several tiles in both directions, ragged; the second fills the chip"""
    rng = np.random.default_rng(k)
    def side(kind, shape, axis):
        if kind == "h":
            x = rng.standard_normal(shape).astype(np.float16)
            return ng.array(x), x
        return _operand(ng, rng, shape, "fp4" if kind == "4" else "int8", axis)
    A, a = side(kinds[0], (m, k), 1)
    B, b = side(kinds[1], (k, n), 0)
    for out in (np.float16, np.float32):
        C = ng.empty((m, n), dtype=out)
        ng.mx_dot(A, B, C)
        _check_product(C.get(), a.astype(np.float64), b.astype(np.float64), kinds)


MIX = [("fp4", "left"), ("fp4", "right"), ("int8", "left"), ("int8", "right")]


@pytest.mark.parametrize("m,n,k", DOT_SIZES + [(70, 2, 300), (50, 3, 256), (40, 8, 1024), (200, 16, 96), (31, 17, 520),
                                              (48, 33, 160)])
@pytest.mark.parametrize("fmt,side", MIX)
@pytest.mark.parametrize("order", ["rows", "columns"])
def test_mixed_product(ng, m, n, k, fmt, side, order):
    """one block-scaled operand, the other fp16 with either axis contiguous"""
    rng = np.random.default_rng(m + n + k)
    if side == "left":
        A, a = _operand(ng, rng, (m, k), fmt, 1, 0.25)
        b = rng.standard_normal((k, n)).astype(np.float16)
        B = ng.array(b) if order == "rows" else ng.array(np.ascontiguousarray(b.T)).T
    else:
        B, b = _operand(ng, rng, (k, n), fmt, 0, 0.25)
        a = rng.standard_normal((m, k)).astype(np.float16)
        A = ng.array(a) if order == "rows" else ng.array(np.ascontiguousarray(a.T)).T
    for out in (np.float16, np.float32):
        C = ng.empty((m, n), dtype=out)
        C.fill(7)
        ng.mx_dot(A, B, C)
        _check_product(C.get(), a.astype(np.float64), b.astype(np.float64), "%s %s %s" % (fmt, side, (m, n, k)))


@pytest.mark.parametrize("kinds", ["44", "4h", "h8"])
@pytest.mark.parametrize("m,n,k", [(40, 24, 96), (130, 1, 520), (70, 200, 2048)])
def test_alpha_beta_relu_and_transposed_result(ng, kinds, m, n, k):
    rng = np.random.default_rng(k)
    if kinds[0] == "4":
        A, a = _operand(ng, rng, (m, k), "fp4", 1, 0.25)
    else:
        a = rng.standard_normal((m, k)).astype(np.float16)
        A = ng.array(a)
    if kinds[1] == "h":
        b = rng.standard_normal((k, n)).astype(np.float16)
        B = ng.array(b)
    else:
        B, b = _operand(ng, rng, (k, n), "int8" if kinds[1] == "8" else "fp4", 0)
    a, b = a.astype(np.float64), b.astype(np.float64)
    c0 = rng.standard_normal((m, n)).astype(np.float16)
    for out in (np.float16, np.float32):
        C = ng.array(c0, dtype=out)
        ng.mx_dot(A, B, C, alpha=0.3, beta=-1.5, relu=True)
        _check_product(C.get(), a, b, kinds, float(np.float32(0.3)), -1.5, c0, True)
        # a result whose columns are contiguous, inside a larger matrix that stays as it was
        T = ng.ones((n + 2, m + 3), dtype=out)
        ng.mx_dot(A, B, T[1:n + 1, 2:m + 2].T)
        got = T.get()
        _check_product(np.ascontiguousarray(got[1:n + 1, 2:m + 2].T), a, b, kinds + " transposed")
        got[1:n + 1, 2:m + 2] = 1
        assert np.all(got == 1)


def test_stochastic_result(ng):
    """small integers: the product is exact, so the stored halves follow the stream bit for bit"""
    from nervanagpu_amd import NervanaGPU
    sg = NervanaGPU(stochastic_round=True, seed=3)
    rng = np.random.default_rng(8)
    m, n, k = 50, 72, 640
    a = rng.integers(-4, 5, (m, k)).astype(np.float16)
    b = rng.integers(-4, 5, (k, n)).astype(np.float16)
    A = ng.mx_array(a)
    B = ng.mx_array(b, axis=0)
    assert np.array_equal(A.get(), a) and np.array_equal(B.get(), b)
    exact = (a.astype(np.float32) @ b.astype(np.float32)) * np.float32(1.0 / 3.0)
    r = lambda count: orc.rand_sr16(3, sg.rng_counter, np.arange(count, dtype=np.uint32)).reshape(m, n)
    for left, right in ((A, B), (A, ng.array(b))):
        C = sg.empty((m, n))
        sg.mx_dot(left, right, C, alpha=1.0 / 3.0)
        expect = orc.round_stochastic_fp16(exact, 10, r(m * n))
        assert np.array_equal(C.get().view(np.uint16), expect.view(np.uint16))


@pytest.mark.parametrize("fmt,side", MIX)
@pytest.mark.parametrize("order", ["rows", "columns"])
@pytest.mark.parametrize("count", [1, 3, 40, 72])
def test_windows_as_dense_operands(ng, fmt, side, order, count):
    """a dense operand inside a matrix of NaN, at aligned and odd places; results inside another that stays as it was"""
    rng = np.random.default_rng(15)
    other, k = 70, 200
    d = rng.standard_normal((k, count)).astype(np.float16)
    X, x = _operand(ng, rng, (other, k), fmt, 1, 0.25)
    for off in (8, 3):
        big = np.full((k + 16, count + 16) if order == "rows" else (count + 16, k + 16), np.nan, dtype=np.float16)
        big[off:off + k, off:off + count] = d if order == "rows" else big[off:off + k, off:off + count]
        if order != "rows":
            big[off:off + count, off:off + k] = d.T
        D = ng.array(big)
        D = D[off:off + k, off:off + count] if order == "rows" else D[off:off + count, off:off + k].T
        if side == "left":
            T = ng.ones((other + 9, count + 11), dtype=np.float32)
            C = T[off:off + other, off:off + count]
            ng.mx_dot(X, D, C)
            got = T.get()
            _check_product(np.ascontiguousarray(got[off:off + other, off:off + count]), x, d.astype(np.float64), "window")
            got[off:off + other, off:off + count] = 1
        else:
            T = ng.ones((count + 9, other + 11), dtype=np.float32)
            ng.mx_dot(D.T, X.T, T[off:off + count, off:off + other])
            got = T.get()
            _check_product(np.ascontiguousarray(got[off:off + count, off:off + other]), d.T.astype(np.float64), x.T, "window")
            got[off:off + count, off:off + other] = 1
        assert np.all(got == 1)


def test_nan_blocks_reach_their_row_alone(ng):
    rng = np.random.default_rng(9)
    m, n, k = 40, 24, 200
    a = rng.standard_normal((m, k)).astype(np.float16)
    a[3, 190] = np.inf
    b = rng.standard_normal((k, n)).astype(np.float16)
    A = ng.mx_array(a)
    for B in (ng.mx_array(b, axis=0), ng.array(b)):
        C = ng.empty((m, n), dtype=np.float32)
        ng.mx_dot(A, B, C)
        bad = np.isnan(C.get())
        assert bad[3].all() and bad.sum() == n
    # and infinities of the dense operand are not hidden by zero codes
    z = ng.mx_array(np.zeros((m, k), dtype=np.float16))
    b[7, 5] = np.inf
    C = ng.empty((m, n), dtype=np.float32)
    ng.mx_dot(z, ng.array(b), C)
    bad = np.isnan(C.get())
    assert bad[:, 5].all() and bad.sum() == m


def test_padding_bytes_do_not_matter(ng):
    """scales behind the last block may hold anything, NaN's 255 among it"""
    rng = np.random.default_rng(10)
    m, n, k = 70, 40, 300
    A, a = _operand(ng, rng, (m, k), "fp4", 1)
    B, b = _operand(ng, rng, (k, n), "fp4", 0)
    X, x = _operand(ng, rng, (n, k), "int8", 1)
    for t in (A, B, X):
        s = t.scales.get()
        s[:, 10:] = 255
        t.scales.set(s)
    h = rng.standard_normal((k, n)).astype(np.float16)
    C = ng.empty((m, n), dtype=np.float32)
    _check_product(ng.mx_dot(A, B, C).get(), a, b, "fp4 padding")
    _check_product(ng.mx_dot(A, ng.array(h), C).get(), a, h.astype(np.float64), "mixed padding")
    e = rng.standard_normal((m, k)).astype(np.float16)
    _check_product(ng.mx_dot(ng.array(e), X.T, C).get(), e.astype(np.float64), x.T, "int8 padding")


def test_scales_outside_the_fp16_range(ng):
    """beside a dense operand the values are fp16 first: the far ones overflow or vanish as an fp16 store would"""
    m, k = 10, 64
    for fmt in ("fp4", "int8"):
        x = np.outer(np.exp2(np.array([-40.0, -30, -26, -25, -24, -16, 10, 13, 14, 20])), np.linspace(0.25, 1.0, k)).astype(np.float32)
        q = ng.mx_array(x, fmt)
        vals = orc.ref_mx_values(q.codes.get(), q.scales.get(), fmt, (m, k))
        with np.errstate(over="ignore"):
            half = vals.astype(np.float16).astype(np.float64)
        eye = np.eye(k, dtype=np.float16)
        C = ng.empty((m, k), dtype=np.float32)
        ng.mx_dot(q, ng.array(eye), C)
        with np.errstate(invalid="ignore"):
            ref = half @ eye.astype(np.float64)
        assert np.array_equal(C.get(), ref.astype(np.float32), equal_nan=True), fmt


@pytest.mark.parametrize("k", [0, 40])
def test_empty_extents(ng, k):
    A, B = ng.mx_empty((5, k), axis=1), ng.mx_empty((k, 7), axis=0)
    C = ng.ones((5, 7), dtype=np.float32)
    if k == 0:
        ng.mx_dot(A, B, C, beta=0.5)          # an empty sum
        assert np.all(C.get() == 0.5)
        ng.mx_dot(A, ng.empty((0, 7)), C)
        assert not C.get().any()
    q = ng.mx_empty((0, k))
    ng.mx_quantize(ng.empty((0, k)), q)
    ng.mx_dot(q, ng.mx_empty((k, 3), axis=0), ng.empty((0, 3)))


def test_scratch_is_refused_when_too_small(ng):
    from nervanagpu_amd import _lib
    A, B = ng.mx_empty((64, 4096), axis=1), ng.mx_empty((4096, 64), axis=0)
    C = ng.ones((64, 64), dtype=np.float32)
    a, b = A.operand(), B.operand()
    need = _lib.load().ng_mx_gemm_workspace_bytes(1, 64, 64, 4096, a, b)
    if need:
        with pytest.raises(_lib.NervanaGPUError, match="workspace"):
            _lib.call("ng_mx_gemm", 1, 64, 64, 4096, a, b, C.ptr, 64, 1.0, 0.0, 0, 0, 0, None, 0, None)
    assert np.all(C.get() == 1)


# ---- activation functions and their checkpoint -----------------------------------------------------

ACTS = ["relu", "sig", "tanh", "silu", "gelu"]


def _act_bound(op, z, back):
    """Bound on the fp32 evaluation, in units of 2^-24.  The library's functions (fp32 operands) keep the OpenCL limits:
    exp 3 ulp (6 units), erfc 16 (32), tanh 5 (10); the hardware's exponential and reciprocal (fp16 operands) are good to
    one ulp (2 units) and the polynomial of the normal distribution to 7.5e-8 (2 units); every other operation adds 1.
    A rounded argument moves exp(-z^2/2) and erfc(-z/sqrt 2) by about z^2 (relative)."""
    z = np.abs(z)
    if op == "relu":
        return 0 * z
    if op == "tanh":
        return 0 * z + 22 if back else 10 * np.tanh(z)
    if op == "gelu":
        if back:
            return (36 + z * z) * (1.0 + z * np.exp(-0.5 * z * z) * 0.4) + 2
        return (34 + z * z) * np.maximum(np.abs(orc.ref_act("gelu", z)), np.abs(orc.ref_act("gelu", -z)))
    if op == "sig":
        return 10 + 0 * z if back else 9 + 0 * z
    return 10 * z + 12 if back else 10 * z


@pytest.mark.parametrize("op", ACTS)
@pytest.mark.parametrize("shape", [(1, 1), (3, 33), (64, 128), (5, 1030), (130, 40)])
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_activation_and_checkpoint(ng, op, shape, dtype):
    rng = np.random.default_rng(shape[1])
    z = (rng.standard_normal(shape) * 4).astype(dtype)
    dZ = ng.array(z, dtype=dtype)
    Y, Q = ng.empty(shape, dtype=dtype), ng.mx_empty(shape, "int8")
    ng.fprop_act(op, dZ, Y, saved=Q)
    vals = _check(Q, z)
    zd = z.astype(np.float64)
    ref = orc.ref_act(op, zd)
    tol = _act_bound(op, zd, False) * EPS32

    def compare(got, ref, tol):
        if dtype == np.float16:
            assert_fp16_within_ulp(got, ref, 0.5, op, tol + 2.0 ** -149)
        else:
            assert np.all(np.abs(got - ref) <= tol + EPS32 * np.abs(ref) + 2.0 ** -149), op

    compare(Y.get(), ref, tol)
    Y2 = ng.empty(shape, dtype=dtype)
    assert np.array_equal(ng.fprop_act(op, dZ, Y2).get(), Y.get())     # without a checkpoint
    Q2, Z2 = ng.mx_empty(shape, "int8"), ng.array(z, dtype=dtype)
    assert np.array_equal(ng.fprop_act(op, Z2, Z2, saved=Q2).get(), Y.get())   # in place
    assert np.array_equal(Q2.codes.get(), Q.codes.get()) and np.array_equal(Q2.get(), Q.get())
    e = rng.standard_normal(shape).astype(dtype)
    G = ng.array(e, dtype=dtype)
    ng.bprop_act(op, Q, G, G)                                            # in place
    slope = orc.ref_act_slope(op, vals)
    compare(G.get(), e.astype(np.float64) * slope,
            np.abs(e.astype(np.float64)) * (_act_bound(op, vals, True) + 1) * EPS32)


@pytest.mark.parametrize("op", ACTS)
def test_slope_is_the_difference_quotient(ng, op):
    """d/dz by central differences of the forward pass: third derivatives are below 1, so a step h = 2^-6 leaves
    h^2 / 6 < 4.1e-5, and fp32 forward values of at most 4 (off by 64 units of 2^-24 of that) 64 * 4 * 2^-24 / h < 1e-3"""
    z = np.arange(-127, 128, 2, dtype=np.float32).reshape(4, 32) / 32.0      # multiples of 1/32 below 4: exact codes
    h = np.float32(2.0 ** -6)
    up, down = ng.empty(z.shape, dtype=np.float32), ng.empty(z.shape, dtype=np.float32)
    ng.fprop_act(op, ng.array(z + h, dtype=np.float32), up)
    ng.fprop_act(op, ng.array(z - h, dtype=np.float32), down)
    q = ng.mx_array(z, "int8")
    assert np.array_equal(q.get(), z)
    G = ng.empty(z.shape, dtype=np.float32)
    ng.bprop_act(op, q, ng.ones(z.shape, dtype=np.float32), G)
    quotient = (up.get().astype(np.float64) - down.get()) / (2 * h)
    assert np.abs(quotient - G.get()).max() <= 1.1e-3


def test_activation_views_leave_their_surroundings(ng):
    rng = np.random.default_rng(12)
    big = rng.standard_normal((20, 90)).astype(np.float16)
    dB = ng.array(big)
    out = ng.ones((20, 90))
    q = ng.mx_empty((15, 70), "int8")
    ng.fprop_act("silu", dB[3:18, 5:75], out[3:18, 5:75], saved=q)
    _check(q, big[3:18, 5:75])
    got = out.get()
    assert np.abs(got[3:18, 5:75] - orc.ref_act("silu", big[3:18, 5:75])).max() < 0.01
    got[3:18, 5:75] = 1
    assert np.all(got == 1)


def test_non_finite_activations(ng):
    z = np.full((2, 64), 1.5, dtype=np.float32)
    z[0, 3], z[1, 40] = np.inf, np.nan
    for op in ACTS:
        Y, Q = ng.empty(z.shape, dtype=np.float32), ng.mx_empty(z.shape, "int8")
        ng.fprop_act(op, ng.array(z, dtype=np.float32), Y, saved=Q)
        bad = np.isnan(Q.get())
        assert bad[0, :32].all() and bad[1, 32:].all() and bad.sum() == 64
        G = ng.ones(z.shape, dtype=np.float32)
        ng.bprop_act(op, Q, G, G)
        if op != "relu":
            assert np.array_equal(np.isnan(G.get()), bad)


# ---- together --------------------------------------------------------------------------------------

@pytest.mark.parametrize("mx4,save8,fold", [(True, False, False), (False, True, False), (True, True, True)])
def test_dense_layers_of_a_network(ng, mx4, save8, fold):
    """FullLayer with 4-bit products and 8-bit saved inputs, built and run by the network driver: each layer's three
    products against the values of its own block-scaled tensors, the rectifier derivative below, the update"""
    from nervanagpu_amd import convnet_benchmarks as cb
    from nervanagpu_amd.layers import DataLayer, FullLayer
    confs = [{"layer": DataLayer, "N": 40, "C": 70, "H": 1, "W": 1}] + \
            [{"layer": FullLayer, "nOut": n, "mx4": mx4, "save8": save8} for n in (136, 96, 33)]
    layers = cb.build_network(ng, confs, np.float16, seed=2, fold_relu=fold)
    layers[1].init_deltas()
    assert [l.relu_done_above for l in layers[1:]] == [fold, fold, False]
    y = None
    for l in layers:
        x = y
        y = l.fprop(y)
        if type(l) is FullLayer:
            w, xin = (l._mx["W"].get(), l._mx["x"].get()) if mx4 else (l.weights.get(), x.get().reshape(l.dimI))
            _check_product(y.get(), w.astype(np.float64), xin.astype(np.float64), "fprop", relu=True)
            if save8:
                assert np.array_equal(l.saved_in.get(), orc.ref_mx_round(x.get().reshape(l.dimI), "int8")[2].astype(np.float32))
    rng = np.random.default_rng(3)
    err = ng.array(rng.standard_normal(layers[-1].dimO).astype(np.float16))
    for l in layers[:0:-1]:
        e = err.get().reshape(l.dimO).astype(np.float64)
        if not l.relu_done_above:
            e = e * (l.fprop_out.get() > 0)
        w0 = l.weights.get()
        l.learning_rate = 0.0
        err = l.bprop(err)
        dx = err.get()
        e16 = e.astype(np.float16).astype(np.float64)
        if mx4:
            wt, eq = l._mx["W^T"].get().T.astype(np.float64), l._mx["e"].get().astype(np.float64)
            assert np.array_equal(eq, orc.ref_mx_round(e16, "fp4", 0)[2])
        else:
            wt, eq = w0.T.astype(np.float64), e16
        xs = l.saved_in.get().astype(np.float64) if save8 else l.fprop_in.get().astype(np.float64)
        if l.relu_below:
            assert not dx[xs <= 0].any()
            ref = wt @ eq
            assert_fp16_within_ulp(dx, np.where(xs > 0, ref, 0.0), 0.5, "dx", np.sqrt(w0.shape[0]) * EPS32 * (np.abs(wt) @ np.abs(eq)))
        else:
            _check_product(dx, wt, eq, "dx")
        _check_product(l.updat_out.get(), e16, xs.T, "dw")


def test_shared_activation_buffers(ng):
    """with 8-bit saved inputs two activation buffers serve a chain: the gradients are those of separate buffers"""
    from nervanagpu_amd.layers import FullLayer
    rng = np.random.default_rng(4)
    N, sizes = 24, (64, 48, 80, 40)
    x0, top = rng.standard_normal((sizes[0], N)).astype(np.float16), rng.standard_normal((sizes[-1], N)).astype(np.float16)
    ws = [(rng.standard_normal((b, a)) * 0.2).astype(np.float16) for a, b in zip(sizes, sizes[1:])]
    grads = []
    for share in (False, True):
        buffers = [ng.empty((max(sizes), N)) for _ in range(2)]
        layers, y = [], ng.array(x0)
        for w in ws:
            l = FullLayer(ng, np.float16, N, w.shape[1], w.shape[0], save8=True)
            l.init_activations(shared=buffers if share else None)
            l.init_deltas()
            l.init_weights()
            l.weights.set(w)
            if layers:
                l.relu_below = layers[-1].relu_done_above = True
            y = l.fprop(y)
            layers.append(l)
        e = ng.array(top)
        got = []
        for l in layers[::-1]:
            e = l.bprop(e)
            got += [e.get(), l.updat_out.get()]
        grads.append(got)
    for a, b in zip(*grads):
        assert np.array_equal(a, b)


def test_dense_layer_step_in_few_bits(ng):
    """forward, data gradient and weight gradient of a dense layer as a training program chains them"""
    rng = np.random.default_rng(13)
    nin, nout, N = 200, 136, 72
    w = (rng.standard_normal((nout, nin)) * 0.1).astype(np.float16)
    x = rng.standard_normal((nin, N)).astype(np.float16)
    e = rng.standard_normal((nout, N)).astype(np.float16)
    W, X, E = ng.array(w), ng.array(x), ng.array(e)
    Wf = ng.mx_quantize(W, ng.mx_empty(w.shape, axis=1))        # for y = W x
    Wb = ng.mx_quantize(W, ng.mx_empty(w.shape, axis=0))        # for dx = W^T e
    Xf = ng.mx_quantize(X, ng.mx_empty(x.shape, axis=0))
    Y, A = ng.empty((nout, N)), ng.empty((nout, N))
    ng.mx_dot(Wf, Xf, Y)
    _check_product(Y.get(), Wf.get().astype(np.float64), Xf.get().astype(np.float64), "y")
    Q, X8 = ng.mx_empty((nout, N), "int8"), ng.mx_quantize(X, ng.mx_empty(x.shape, "int8"))
    ng.fprop_act("gelu", Y, A, saved=Q)
    G = ng.empty((nout, N))
    ng.bprop_act("gelu", Q, E, G)
    g = G.get().astype(np.float64)
    G4 = ng.mx_quantize(G, ng.mx_empty((nout, N), axis=0))
    dX, dW = ng.empty((nin, N)), ng.empty((nout, nin), dtype=np.float32)
    ng.mx_dot(Wb.T, G4, dX)
    _check_product(dX.get(), Wb.get().T.astype(np.float64), G4.get().astype(np.float64), "dx")
    ng.mx_dot(G, X8.T, dW)
    _check_product(dW.get(), g, X8.get().T.astype(np.float64), "dw")
    # the checkpoint is close to what it stands for: half a unit of 1/64 .. 1/127 of the block's largest value (one
    # unit where that one saturates)
    assert np.abs(X8.get() - x).max() <= np.abs(x).max() / 64


# ---- streams, graphs, far offsets -----------------------------------------------------------------

def _emulated():
    from nervanagpu_amd import _lib
    return "emulation" in _lib.device_name()


def _chain(ng, t):
    """every operator once, on the tensors of `t`"""
    ng.mx_quantize(t["x"], t["x4"])
    ng.mx_dot(t["w4"], t["x4"], t["y"])
    ng.fprop_act("silu", t["y"], t["a"], saved=t["q"])
    ng.mx_dequantize(t["q"], t["z"])
    ng.bprop_act("silu", t["q"], t["a"], t["g"])
    ng.mx_dot(t["g"], t["q"].T, t["dw"])
    ng.mx_dot(t["w4"], t["x"], t["y2"])
    ng.mx_dot(t["w4"], t["few"], t["y3"])


def _chain_tensors(ng, seed):
    rng = np.random.default_rng(seed)
    n, k, m = 72, 1000, 136
    f = lambda *shape: ng.empty(shape)
    return {"x": ng.array(rng.standard_normal((k, n)).astype(np.float16)), "x4": ng.mx_empty((k, n), axis=0, rounding=0),
            "w4": ng.mx_array((rng.standard_normal((m, k)) * 0.1).astype(np.float16), rounding=0), "few": ng.array(rng.standard_normal((k, 3)).astype(np.float16)),
            "y": f(m, n), "a": f(m, n), "z": f(m, n), "g": f(m, n), "q": ng.mx_empty((m, n), "int8", rounding=0),
            "dw": ng.empty((m, m), dtype=np.float32), "y2": f(m, n), "y3": f(m, 3)}


_CHAIN_OUT = ("y", "a", "z", "g", "dw", "y2", "y3")


def test_on_a_stream_of_its_own(ng):
    from nervanagpu_amd import NervanaGPU, _lib
    t = _chain_tensors(ng, 21)
    _chain(ng, t)
    expect = {k: t[k].get() for k in _CHAIN_OUT}
    stream = ctypes.c_void_p()
    _lib.call("ng_stream_create", ctypes.byref(stream))
    other = NervanaGPU(seed=1)
    other.stream = stream
    u = _chain_tensors(other, 21)
    _lib.stream_sync(None)
    for _ in range(3):
        _chain(other, u)
    for k in _CHAIN_OUT:
        assert np.array_equal(u[k].get(), expect[k]), k
    _lib.stream_sync(stream)
    _lib.call("ng_stream_destroy", stream)


def test_captured_and_replayed():
    """the calls record nothing but kernels: a graph of all of them, replayed with new inputs between eager work"""
    from nervanagpu_amd import NervanaGPU, _lib
    if _emulated():
        pytest.skip("graphs are a device matter")
    hip = _lib.load()           # its own HIP runtime answers for the graph calls
    vp = ctypes.c_void_p

    def ok(status):
        assert status == 0, "HIP status %d" % status

    ng = NervanaGPU(seed=1)
    stream, graph, run = vp(), vp(), vp()
    _lib.call("ng_stream_create", ctypes.byref(stream))
    ng.stream = stream
    t = _chain_tensors(ng, 22)
    _chain(ng, t)                       # the arena is there before the capture
    _lib.stream_sync(stream)
    ok(hip.hipStreamBeginCapture(stream, 0))
    _chain(ng, t)
    ok(hip.hipStreamEndCapture(stream, ctypes.byref(graph)))
    ok(hip.hipGraphInstantiate(ctypes.byref(run), graph, None, None, ctypes.c_size_t(0)))
    rng = np.random.default_rng(23)
    for _ in range(3):
        t["x"].set(rng.standard_normal(t["x"].shape).astype(np.float16))
        _chain(ng, t)
        expect = {k: t[k].get() for k in _CHAIN_OUT}
        for k in _CHAIN_OUT:
            t[k].fill(9)
        _lib.stream_sync(stream)
        ok(hip.hipGraphLaunch(run, stream))
        _lib.stream_sync(stream)
        for k in _CHAIN_OUT:
            assert np.array_equal(t[k].get(), expect[k]), k
    ok(hip.hipGraphExecDestroy(run))
    ok(hip.hipGraphDestroy(graph))
    _lib.call("ng_stream_destroy", stream)


def test_reruns_are_bit_identical(ng):
    rng = np.random.default_rng(24)
    A, _ = _operand(ng, rng, (200, 4096), "fp4", 1)
    B, _ = _operand(ng, rng, (4096, 100), "fp4", 0)
    h = ng.array(rng.standard_normal((4096, 100)).astype(np.float16))
    for right in (B, h, h[:, :9]):
        C = ng.empty((200, right.shape[1]), dtype=np.float32)
        first = ng.mx_dot(A, right, C).get()
        for _ in range(3):
            assert np.array_equal(ng.mx_dot(A, right, C).get(), first)


def test_far_offsets(ng):
    """rows 2^20 elements apart: the last ones lie beyond 2^32 elements and 2^33 bytes from the first"""
    from nervanagpu_amd import _lib
    if _emulated():
        pytest.skip("needs 9 GB")
    rows, pitch, cols = 4104, 1 << 20, 96
    rng = np.random.default_rng(25)
    big = ng.empty((rows, pitch))
    w = big[:, 64:64 + cols]
    checked = [0, 1, 2047] + list(range(4096, rows))
    x = {r: rng.standard_normal(cols).astype(np.float16) for r in checked}
    for r in checked:
        _lib.memcpy_htod(w.ptr + 2 * r * pitch, x[r])
    q = ng.mx_quantize(w, ng.mx_empty((rows, cols), "int8"))
    got = q.get()
    for r in checked:
        assert np.array_equal(got[r], orc.ref_mx_round(x[r][None], "int8")[2][0].astype(np.float32))
    tail = np.stack([x[r] for r in range(4096, rows)])
    q0 = ng.mx_quantize(w, ng.mx_empty((rows, cols), "fp4", 0))
    assert np.array_equal(q0.get()[4096:], orc.ref_mx_round(tail, "fp4", 0)[2].astype(np.float32))
    # written back and read as a dense operand in place
    ng.mx_dequantize(q, w)
    back = np.empty(cols, dtype=np.float16)
    for r in checked:
        _lib.memcpy_dtoh(back, w.ptr + 2 * r * pitch)
        assert np.array_equal(back, got[r].astype(np.float16))
    ng.fprop_act("relu", w, w)
    for r in checked:
        _lib.memcpy_dtoh(back, w.ptr + 2 * r * pitch)
        assert np.array_equal(back, np.maximum(got[r], 0).astype(np.float16))
    E = ng.mx_array(np.eye(cols, dtype=np.float16), axis=0)
    C = ng.empty((rows, cols))
    ng.mx_dot(w, E, C)
    out = C.get()
    for r in checked:
        assert np.array_equal(out[r], np.maximum(got[r], 0).astype(np.float16))
