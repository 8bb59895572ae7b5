"""Which kernel a product of block-scaled matrices takes, by the host code's own choice on an emulated chip (launches are listed,
not run): the sizes of test_gpu_mx_tiles.py reach the kernels they are there for.  And the larger tiles run on the emulation."""
import ctypes
import os
import sys

import numpy as np
import pytest

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "emu"))

import emu  # noqa: E402
from nervanagpu_amd import _lib  # noqa: E402
from test_gpu_mx_tiles import DEVICE, SMALL  # noqa: E402
from test_mx_emulated import _emulate  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def built():
    emu.build()


def launches(kinds, m, n, k, cus, out=np.float16):
    """the launches of a product on a chip of that many CUs, a line each"""
    lib = emu.load()
    lib.emu_launches.restype = ctypes.c_char_p
    lib.ng_mx_gemm.argtypes = _lib._SIGNATURES["ng_mx_gemm"][1]
    lib.ng_mx_gemm_workspace_bytes.restype, lib.ng_mx_gemm_workspace_bytes.argtypes = _lib._SIGNATURES["ng_mx_gemm_workspace_bytes"]

    def side(kind, lines, across):
        if kind == "h":
            return _lib.MxOperand(0, 0 if across else 1, lines if across else k, 0x100000, None)
        return _lib.MxOperand(1 if kind == "4" else 2, 1, 0, 0x100000, 0x200000)

    a, b = side(kinds[0], m, False), side(kinds[1], n, "across" in kinds)
    code = 0 if out is np.float16 else 1
    lib.emu_set_cus(cus)
    lib.emu_set_dry(1)
    try:
        need = lib.ng_mx_gemm_workspace_bytes(code, m, n, k, a, b)
        assert lib.ng_mx_gemm(code, m, n, k, a, b, 0x300000, n, 1.0, 0.0, 0, 0, 0, 0x400000, need, None) == 0
        return lib.emu_launches().decode().splitlines()
    finally:
        lib.emu_set_dry(0)


def assert_takes(kinds, m, n, k, kernel, slices, cus):
    lines = launches(kinds, m, n, k, cus)
    products = [l for l in lines if "mx44_kernel" in l or "mxmix_kernel" in l or "mx_skinny_kernel" in l]
    assert len(products) == 1 and kernel in products[0], lines
    assert any("splitk_reduce" in l for l in lines) == slices, lines
    if "mxmix" in products[0]:
        across = "across" in kinds and kinds[0] == "4"
        for said in ("FMT = %d" % (1 if "4" in kinds else 2), "X_IS_A = %s" % ("true" if kinds[0] != "h" else "false"),
                     "ACROSS = %s" % ("true" if across else "false")):
            assert said in products[0], lines


@pytest.mark.parametrize("kinds,m,n,k,kernel,slices", DEVICE)
def test_device_sizes_take_their_kernel(kinds, m, n, k, kernel, slices):
    assert_takes(kinds, m, n, k, kernel, slices, 256)


@pytest.mark.parametrize("kinds,m,n,k,kernel,slices,cus", SMALL)
def test_small_sizes_take_large_tiles_of_a_small_chip(kinds, m, n, k, kernel, slices, cus):
    assert_takes(kinds, m, n, k, kernel, slices, cus)


@pytest.mark.parametrize("cus", ["2", "8"])
def test_large_tiles_on_the_emulator(cus):
    _emulate("test_gpu_mx_tiles.py", "few_units", cus)
