"""What a failed or refused call of a device operator leaves behind, each in a process of its own."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEAD = r"""
import ctypes as C, sys
sys.path[:0] = [%r]
import torch
from poorgrad_b200 import abi, backend, operators
lib = abi.load_library()

def code_of(call):
    try:
        call()
    except backend.BackendError as error:
        return error.code
    return 0
""" % ROOT


def child(text):
    out = subprocess.run([sys.executable, "-c", HEAD + text], capture_output=True, text=True, timeout=600)
    assert out.returncode == 0, out.stderr[-2000:]
    return out.stdout.split()


def test_a_failure_poisons_a_library_that_was_never_asked_for_its_state(device):
    assert child(r"""
lib.tbx_scan_wait_limit.argtypes = [C.c_int64]
lib.tbx_scan_wait_limit(0)
x = torch.randn(8, 1024, 768, device="cuda").bfloat16()
operators.gated_scan(x, x)
print(code_of(operators.synchronize), code_of(lambda: operators.gated_scan(x, x)), backend.status()[0])
""") == ["7", "4", "4"]
