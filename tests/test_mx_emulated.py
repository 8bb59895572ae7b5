"""The tests of tests/test_gpu_mx_*.py that say something without a device, on the lane-level CPU emulation."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _emulate(name, expr, cus="8"):
    cmd = [sys.executable, os.path.join(ROOT, "tests", "emu", "run_on_emulator.py"), os.path.join(ROOT, "tests", name),
           "-x", "-q", "-p", "no:cacheprovider", "-k", expr]
    done = subprocess.run(cmd, cwd=ROOT, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, timeout=1500,
                          env=dict(os.environ, EMU_CUS=cus))
    tail = done.stdout.decode("utf-8", "replace")[-3000:]
    assert done.returncode == 0, tail
    assert " passed" in tail and "failed" not in tail, tail


@pytest.mark.parametrize("expr", ["relu", "rectified", "gelu", "saturated", "logistic", "int8"])
def test_values_on_the_emulator(expr):
    _emulate("test_gpu_mx_values.py", expr)
