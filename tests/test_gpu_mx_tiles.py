"""Products of block-scaled matrices on every kernel and tile that a size can be sent to, against the product of the operands'
values in 64 bits (tolerances as in test_gpu_mx.py).  Which kernel a size takes is asserted in test_mx_tiles_host.py."""
import numpy as np
import pytest

from test_gpu_mx import _check_product, _operand

pytestmark = pytest.mark.gpu

MIXED = ["4h", "4h across", "h4", "8h", "h8"]
# (kinds of the operands, m, n, k, kernel on 256 CUs, whether the contraction is cut into slices).  "across": the
# dense operand's rows lie along the columns of the result, and are read in place
DEVICE = [
    ("44", 2900, 3080, 770, "mx44_kernel<256, 256,", False),
    ("44", 1500, 1601, 770, "mx44_kernel<128, 128,", False),
    ("44", 1111, 777, 700, "mx44_kernel<64, 64,", False),
    ("44", 200, 301, 5000, "mx44_kernel<64, 64,", True),
] + [case for kinds in MIXED for case in [
    (kinds, 2900, 3080, 770, "256, 256, 4, 2, 3,", False),
    (kinds, 1500, 1600, 770, "128, 128, 4, 2, 3,", False),
    (kinds, 1500, 1600, 100, "128, 128, 2, 2, 2,", False),
    (kinds, 600, 904, 8011, "128, 128, 4, 2, 3,", True),
    (kinds, 300, 504, 601, "64, 64, 2, 1, 4,", False),
    (kinds, 257, 136, 3001, "64, 64, 2, 1, 4,", True),
]] + [
    ("4h", 300, 1, 5000, "<X_IS_A, 1, 16, false,", False),
    ("4h", 300, 1, 5003, "<X_IS_A, 1, 16, false,", False),
    ("h4", 1, 301, 5003, "<X_IS_A, 1, 16, false,", False),
    ("4h", 300, 1, 600, "<X_IS_A, 1, 4, false,", False),
    ("4h", 301, 9, 5000, "<X_IS_A, 1, 16, true,", False),
    ("h4", 16, 300, 600, "<X_IS_A, 1, 4, true,", False),
    ("4h across", 301, 30, 5003, "<X_IS_A, 2, 8, true,", False),
    ("h4", 32, 301, 601, "<X_IS_A, 2, 4, true,", False),
]
# the larger tiles on emulated chips of 2 and 8 CUs, which small outputs fill
SMALL = [("44", 300, 520, 770, "mx44_kernel<256, 256,", False, 2)] + [case for kinds in MIXED for case in [
    (kinds, 257, 136, 330, "128, 128, 4, 2, 3,", False, 2),
    (kinds, 257, 136, 100, "128, 128, 2, 2, 2,", False, 2),
    (kinds, 129, 136, 1100, "128, 128, 4, 2, 3,", True, 8),
]]


def check(ng, kinds, m, n, k, outs=(np.float16, np.float32)):
    rng = np.random.default_rng(m + n + k)

    def side(kind, shape, axis):
        if kind != "h":
            return _operand(ng, rng, shape, "fp4" if kind == "4" else "int8", axis, 0.25)
        x = rng.standard_normal(shape).astype(np.float16)
        # rows contiguous for an "across" right operand; else the contraction
        if axis == 1 or "across" in kinds:
            return ng.array(x), x
        return ng.array(np.ascontiguousarray(x.T)).T, x

    A, a = side(kinds[0], (m, k), 1)
    B, b = side(kinds[1], (k, n), 0)
    a, b = a.astype(np.float64), b.astype(np.float64)
    for out in outs:
        C = ng.empty((m, n), dtype=out)
        C.fill(7)
        ng.mx_dot(A, B, C)
        _check_product(C.get(), a, b, "%s %s" % (kinds, (m, n, k)))


@pytest.mark.parametrize("kinds,m,n,k,kernel,slices", DEVICE)
def test_every_kernel(ng, kinds, m, n, k, kernel, slices):
    from nervanagpu_amd import _lib
    if "emulation" in _lib.device_name():
        pytest.skip("sizes for a whole chip")
    check(ng, kinds, m, n, k)


@pytest.mark.parametrize("kinds,m,n,k,kernel,slices,cus", SMALL)
def test_large_tiles_on_few_units(ng, kinds, m, n, k, kernel, slices, cus):
    """a device takes other tiles for these sizes; they are as good there"""
    import os
    from nervanagpu_amd import _lib
    if "emulation" in _lib.device_name() and os.environ.get("EMU_CUS") != str(cus):
        pytest.skip("for %d CUs" % cus)
    check(ng, kinds, m, n, k, outs=(np.float16,) if m > 257 else (np.float32,))


def test_codes_beyond_32_bits_of_offset(ng):
    """a matrix of 65600 lines of 131072 values: 4.3 GB of 4-bit codes, 8.6 GB of 8-bit ones, 17 GB of fp16.  The lines checked are the
    first, those around 2^31 and 2^32 bytes, and the last; the others hold what the memory held (a line's products are its own)"""
    import oracle as orc
    from nervanagpu_amd import _lib
    if "emulation" in _lib.device_name():
        pytest.skip("needs 30 GB")
    lines, depth = 65600, 131072
    rng = np.random.default_rng(30)
    big = ng.empty((lines, depth))
    checked = [0, 8191, 8192, 16384, 32767, 32768, 65535, 65536, lines - 1]
    x = (rng.standard_normal((len(checked), depth)) * np.exp2(rng.integers(-3, 4, (len(checked), 1)))).astype(np.float16)
    for r, row in zip(checked, x):
        _lib.memcpy_htod(big.ptr + 2 * r * depth, row)
    dense = rng.standard_normal((depth, 40)).astype(np.float16)
    back = np.empty(depth, dtype=np.float16)
    for fmt in ("fp4", "int8"):
        q = ng.mx_quantize(big, ng.mx_empty((lines, depth), fmt, rounding=0))
        _, _, v = orc.ref_mx_round(x, fmt)
        for count in (1, 16, 40) if fmt == "fp4" else (40,):
            C = ng.empty((lines, count), dtype=np.float32)
            ng.mx_dot(q, ng.array(dense[:, :count]), C)
            _check_product(C.get()[checked], v, dense[:, :count].astype(np.float64), "%s by %d" % (fmt, count))
        if fmt == "fp4":
            few = ng.mx_array(dense, axis=0, rounding=0)
            ng.mx_dot(q, few, C)
            _check_product(C.get()[checked], v, few.get().astype(np.float64), "fp4 by fp4")
        ng.mx_dequantize(q, big)
        for r, row in zip(checked, v):
            _lib.memcpy_dtoh(back, big.ptr + 2 * r * depth)
            assert np.array_equal(back, row.astype(np.float16)), r
        for r, row in zip(checked, x):
            _lib.memcpy_htod(big.ptr + 2 * r * depth, row)
    # in place, with a checkpoint that lies as far
    ng.fprop_act("relu", big, big, saved=q)
    ng.bprop_act("relu", q, big, big)
    for r, row, value in zip(checked, x, v):
        _lib.memcpy_dtoh(back, big.ptr + 2 * r * depth)
        assert np.array_equal(back, np.where(value > 0, np.maximum(row, 0), 0)), r
