"""Block-scaled tensors on the CPU: shapes and refusals of the Python surface and the C ABI (no device call is made), and
the GPU tests of the conversions and products run on the lane-level CPU emulation."""
import ctypes
import os
import subprocess
import sys

import numpy as np
import pytest

import oracle as orc
from nervanagpu_amd import GPUTensor, MXTensor, NervanaGPU, _lib
from nervanagpu_amd.mx import code_pitch, scale_pitch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def fake(ng, shape, dtype=np.float16, addr=0x100000, **kw):
    return GPUTensor(ng, shape, dtype, gpudata=addr, **kw)


def fake_mx(ng, shape, fmt="fp4", axis=1, **kw):
    lines, depth = shape[1 - axis], shape[axis]
    return MXTensor(ng, shape, fmt, axis, codes=fake(ng, (lines, code_pitch(fmt, depth)), np.uint8),
                    scales=fake(ng, (lines, scale_pitch(depth)), np.uint8, 0x200000), **kw)


@pytest.fixture
def calls(monkeypatch):
    """the library calls a Python method would make, instead of making them"""
    made = []
    monkeypatch.setattr(_lib, "call", lambda name, *args: made.append((name,) + args))
    return made


def test_layout():
    assert [code_pitch("fp4", d) for d in (0, 1, 32, 33, 100)] == [0, 16, 16, 32, 64]
    assert [code_pitch("int8", d) for d in (1, 64, 65)] == [32, 64, 96]
    assert [scale_pitch(d) for d in (0, 1, 256, 257)] == [0, 8, 8, 16]
    ng = NervanaGPU()
    q = fake_mx(ng, (5, 70), axis=0)
    assert (q.lines, q.depth) == (70, 5) and q.codes.shape == (70, 16) and q.scales.shape == (70, 8)
    with pytest.raises(AttributeError):
        q.codes = q.scales          # the memory is fixed
    t = q.T
    assert t.shape == (70, 5) and t.axis == 1 and t.codes is q.codes and len(t) == 70 and t.nbytes == q.nbytes


def test_tensor_refusals():
    ng = NervanaGPU()
    with pytest.raises(ValueError):
        fake_mx(ng, (4, 4)).__class__(ng, (4, 4), "fp6")
    with pytest.raises(ValueError):
        MXTensor(ng, (4, 4), axis=2)
    with pytest.raises(AssertionError):
        MXTensor(ng, (4, 4, 4))
    good = fake(ng, (4, 16), np.uint8), fake(ng, (4, 8), np.uint8)
    MXTensor(ng, (4, 4), codes=good[0], scales=good[1])
    for codes, scales in ((good[0], None), (None, good[1]), (fake(ng, (4, 8), np.uint8), good[1]),
                          (fake(ng, (4, 16), np.int8), good[1]), (fake(ng, (4, 16), np.uint8, 0x100008), good[1]),
                          (fake(ng, (16, 4), np.uint8).T, good[1])):
        with pytest.raises(AssertionError):
            MXTensor(ng, (4, 4), codes=codes, scales=scales)


def test_quantize_refusals(calls):
    ng = NervanaGPU()
    q = fake_mx(ng, (8, 64))
    for bad in (fake(ng, (8, 63)), fake(ng, (64, 8)), fake(ng, (16, 128))[::2, ::2], fake(ng, (8, 65))[:, ::-1][:, :64]):
        with pytest.raises(AssertionError):
            ng.mx_quantize(bad, q)
        with pytest.raises(AssertionError):
            ng.mx_dequantize(q, bad)
    with pytest.raises(TypeError):
        ng.mx_quantize(fake(ng, (8, 64), np.int8), q)
    with pytest.raises(TypeError):
        ng.mx_dequantize(q, fake(ng, (8, 64), np.int32))
    with pytest.raises(AssertionError):
        ng.mx_quantize(fake(ng, (8, 64)), fake(ng, (8, 64)))
    index = fake(ng, (8,), np.int32)
    with pytest.raises(AssertionError):
        ng.mx_quantize(fake(ng, (20, 64)).take(index, 0), q)
    assert not calls
    ng.mx_quantize(fake(ng, (8, 100))[:, 3:67], q)
    ng.mx_quantize(fake(ng, (64, 9)).T[1:9], q)
    assert [c[0] for c in calls] == ["ng_mx_quantize"] * 2
    assert calls[0][4:8] == (100, 1, 8, 64) and calls[1][4:8] == (9, 0, 8, 64)


def test_random_stream_is_taken_only_when_rounding(calls):
    ng = NervanaGPU(seed=5)
    ng.mx_quantize(fake(ng, (8, 64)), fake_mx(ng, (8, 64)))
    assert ng.rng_counter == 0
    ng.mx_quantize(fake(ng, (8, 64)), fake_mx(ng, (8, 64), rounding=1))
    assert ng.rng_counter == 1 and calls[1][-4:-1] == (_lib.FLAG_SR, 5, 1)


def test_dot_refusals(calls):
    ng = NervanaGPU()
    A, B, C = fake_mx(ng, (8, 64)), fake_mx(ng, (64, 16), axis=0), fake(ng, (8, 16))
    a16, b16 = fake(ng, (8, 64)), fake(ng, (64, 16))
    with pytest.raises(TypeError):
        ng.mx_dot(a16, b16, C)
    with pytest.raises(ValueError):
        ng.mx_dot(fake_mx(ng, (8, 64), axis=0), B, C)
    with pytest.raises(ValueError):
        ng.mx_dot(A, fake_mx(ng, (64, 16), axis=1), C)
    for left, right in ((fake_mx(ng, (8, 64), "int8"), B), (A, fake_mx(ng, (64, 16), "int8", 0)),
                        (fake_mx(ng, (8, 64), "int8"), fake_mx(ng, (64, 16), "int8", 0))):
        with pytest.raises(TypeError):
            ng.mx_dot(left, right, C)
    with pytest.raises(TypeError):
        ng.mx_dot(A, B, fake(ng, (8, 16), np.int32))
    for args in ((A, fake(ng, (64, 16), np.float32), C), (A, B, fake(ng, (16, 8))), (A, fake_mx(ng, (32, 16), axis=0), C),
                 (A, B, fake(ng, (16, 32))[::2, ::2]), (A, fake(ng, (128, 32))[::2, ::2], C)):
        with pytest.raises(AssertionError):
            ng.mx_dot(*args)
    assert not calls


def test_result_with_rows_too_far_apart_is_refused(calls):
    """the pitch of C travels as an int: 2^32 + 16 would arrive as 16"""
    ng = NervanaGPU()
    A, B = fake_mx(ng, (8, 64)), fake_mx(ng, (64, 16), axis=0)
    for wide in (fake(ng, (8, 2 ** 32 + 16))[:, :16], fake(ng, (16, 2 ** 31))[:, :8].T):
        with pytest.raises(AssertionError, match="apart"):
            ng.mx_dot(A, B, wide)
    assert not calls


def test_activation_refusals(calls):
    ng = NervanaGPU()
    z, q = fake(ng, (8, 64)), fake_mx(ng, (8, 64), "int8")
    with pytest.raises(ValueError):
        ng.fprop_act("softplus", z, z)
    with pytest.raises(ValueError):
        ng.bprop_act("softplus", q, z, z)
    for bad in (fake_mx(ng, (8, 64)), fake_mx(ng, (8, 64), "int8", 0)):
        with pytest.raises(ValueError):
            ng.fprop_act("relu", z, z, saved=bad)
        with pytest.raises(ValueError):
            ng.bprop_act("relu", bad, z, z)
    for bad in (fake(ng, (8, 63)), fake(ng, (64, 8)).T, fake(ng, (8, 64), np.float32)):
        with pytest.raises(AssertionError):
            ng.fprop_act("relu", z, bad)
        with pytest.raises(AssertionError):
            ng.bprop_act("relu", q, z, bad)
    with pytest.raises(TypeError):
        ng.fprop_act("relu", fake(ng, (8, 64), np.int8), fake(ng, (8, 64), np.int8))
    with pytest.raises(AssertionError):
        ng.fprop_act("relu", fake(ng, (8, 63)), fake(ng, (8, 63)), saved=q)
    assert not calls


def test_c_abi_refusals():
    """every refused call returns a status before anything is launched (no device is needed to be refused)"""
    lib = _lib.load()
    vp = ctypes.c_void_p
    P = vp(0x100000)

    def operand(fmt, along=1, ld=0, codes=0x100000, scales=0x100000):
        return _lib.MxOperand(fmt, along, ld, codes, scales)

    four, half = operand(1), operand(0, 1, 64)
    quant = lambda *a: lib.ng_mx_quantize(*a)
    assert quant(1, 0, P, 64, 1, 0, 64, None, None, 0, 0, 0, None) == 0             # nothing to do
    assert quant(3, 0, P, 64, 1, 4, 64, P, P, 0, 0, 0, None) < 0                     # unknown format
    assert quant(1, 2, P, 64, 1, 4, 64, P, P, 0, 0, 0, None) < 0                     # bytes are not quantized
    assert quant(1, 0, None, 64, 1, 4, 64, P, P, 0, 0, 0, None) < 0
    assert quant(1, 0, P, 63, 1, 4, 64, P, P, 0, 0, 0, None) < 0                     # rows overlap
    assert quant(1, 0, P, 3, 0, 4, 64, P, P, 0, 0, 0, None) < 0
    assert quant(1, 0, P, 64, 1, -4, 64, P, P, 0, 0, 0, None) < 0
    assert quant(1, 0, P, 64, 1, 4, 64, None, P, 0, 0, 0, None) < 0
    assert quant(1, 0, P, 64, 1, 4, 64, vp(0x100004), P, 0, 0, 0, None) < 0
    assert quant(1, 0, P, 1 << 20, 1, 1 << 20, 1 << 20, P, P, 0, 0, 0, None) < 0     # 2^40 values
    assert lib.ng_mx_dequantize(1, P, P, 4, 64, 2, P, 64, 1, None) < 0
    assert lib.ng_mx_dequantize(1, None, P, 4, 64, 0, P, 64, 1, None) < 0
    assert lib.ng_act_fprop(9, 0, 4, 64, P, 64, P, 64, None, None, None) < 0
    assert lib.ng_act_fprop(0, 0, 4, 64, P, 64, P, 60, None, None, None) < 0
    assert lib.ng_act_fprop(0, 0, 4, 64, P, 64, P, 64, P, None, None) < 0
    assert lib.ng_act_bprop(0, 0, 4, 64, None, None, P, 64, P, 64, None) < 0

    def gemm(a, b, m=4, n=4, k=64, c=0x100000, ldc=4, dtype=0, ws=None, nbytes=0):
        return lib.ng_mx_gemm(dtype, m, n, k, a, b, vp(c), ldc, 1.0, 0.0, 0, 0, 0, ws, nbytes, None)

    assert gemm(four, four, m=0) == 0
    assert gemm(four, four, dtype=2) < 0
    assert gemm(half, half) < 0 and gemm(operand(2), operand(2)) < 0 and gemm(operand(2), four) < 0
    assert gemm(operand(5), half) < 0
    assert gemm(None, four) < 0
    assert gemm(four, four, m=-1) < 0
    assert gemm(four, four, c=0) < 0
    assert gemm(four, four, ldc=3) < 0
    assert gemm(operand(1, codes=0), half) < 0 and gemm(operand(1, scales=0), half) < 0
    assert gemm(operand(1, codes=0x100004), half) < 0
    assert gemm(four, operand(0, 1, 60)) < 0 and gemm(four, operand(0, 0, 3)) < 0
    assert gemm(four, half, k=1 << 21) < 0
    assert gemm(four, half, m=1 << 26) < 0
    assert gemm(four, four, m=1 << 17, n=1 << 16, ldc=1 << 16) < 0
    # a dense operand that has to be copied first needs room
    odd = operand(0, 1, 65, 0x100002)
    need = lib.ng_mx_gemm_workspace_bytes(0, 4, 4, 65, four, odd)
    assert need >= 4 * 65 * 2 or need == 0
    if need:
        assert gemm(four, odd, k=65) < 0
        assert gemm(four, odd, k=65, ws=vp(0x100008), nbytes=need) < 0


@pytest.mark.parametrize("along", [0, 1])
@pytest.mark.parametrize("extents", [(2 ** 31 - 1, 1), (1, 2 ** 31 - 1), (2 ** 31 - 256, 1)])
def test_extents_that_round_up_past_an_int_are_refused(along, extents):
    """rounding such an extent up to whole blocks or workgroups leaves the range of int"""
    lib = _lib.load()
    P = ctypes.c_void_p(0x100000)
    lines, depth = extents
    ld, want = max(extents), -87
    assert lib.ng_mx_quantize(1, 0, P, ld, along, lines, depth, P, P, 0, 0, 0, None) == want
    assert lib.ng_mx_dequantize(1, P, P, lines, depth, 0, P, ld, along, None) == want
    if along:
        assert lib.ng_act_fprop(0, 0, lines, depth, P, ld, P, ld, None, None, None) == want
        assert lib.ng_act_bprop(0, 0, lines, depth, P, P, P, ld, P, ld, None) == want


@pytest.mark.parametrize("fmt,steps", [("fp4", None), ("int8", 1.0)])
def test_oracle_rounds_to_the_nearest(fmt, steps):
    """the oracle itself: no value of the format is nearer, and packing loses nothing"""
    rng = np.random.default_rng(1)
    x = rng.standard_normal((7, 75)) * np.exp2(rng.integers(-5, 6, (7, 1)))
    codes, scales, v = orc.ref_mx_round(x, fmt)
    data, sc = orc.ref_mx_pack(codes, scales, fmt)
    assert np.array_equal(orc.ref_mx_values(data, sc, fmt, x.shape), v)
    e = scales.astype(np.float64) - 127 - (0 if fmt == "fp4" else 6)
    grid = np.array([0, .5, 1, 1.5, 2, 3, 4, 6]) if fmt == "fp4" else np.arange(128.0)
    for i in range(7):
        for j in range(75):
            best = np.abs(grid * 2.0 ** e[i, j // 32] - abs(x[i, j])).min()
            assert abs(v[i, j] - x[i, j]) <= best


def _emulate(expr, cus="8"):
    cmd = [sys.executable, os.path.join(ROOT, "tests", "emu", "run_on_emulator.py"), os.path.join(ROOT, "tests", "test_gpu_mx.py"),
           "-x", "-q", "-p", "no:cacheprovider", "-k", expr]
    done = subprocess.run(cmd, cwd=ROOT, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, timeout=1500,
                          env=dict(os.environ, EMU_CUS=cus))
    tail = done.stdout.decode("utf-8", "replace")[-3000:]
    assert done.returncode == 0, tail
    assert " passed" in tail and "failed" not in tail, tail


def test_conversions_on_the_emulator():
    _emulate("quantize_and_back or views or infinities or follows_the_stream or activation_and or fp32_range")


def test_products_on_the_emulator():
    _emulate("dense_layer or padding or nan_blocks or alpha_beta or empty or stochastic_result or outside or shared or stream_of")


def test_large_tiles_on_the_emulator():
    """on a chip of two CUs the 256x256 tiles cover it"""
    _emulate("larger and 520", "2")
