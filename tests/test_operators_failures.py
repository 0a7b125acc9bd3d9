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


def test_a_capture_that_takes_no_work_is_no_failure(device):
    """A call into a capture that an earlier error has ended, and a wait inside one, are refused, and
    later calls are served."""
    out = child(r"""
assert backend.status()[0] == 0
x, at, row = torch.randn(2, 5, 8, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda"), torch.rand(4, device="cuda")
h, final = torch.empty_like(x), torch.empty(2, 8, device="cuda")
q, k, table = torch.randn(1, 3, 2, 8, device="cuda"), torch.randn(1, 3, 1, 8, device="cuda"), torch.rand(3, 8, device="cuda")
calls = [lambda: operators.gated_scan(x, x, out=h, final_state=final),
         lambda: operators.head_rotate(q, k, table, q_out=q, k_out=k)]
for spoil in (torch.cuda.synchronize, operators.synchronize):
    codes = []
    try:
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            try:
                spoil()
            except backend.BackendError as error:
                codes.append(error.code)
            except RuntimeError:
                codes.append("torch")
            codes += [code_of(call) for call in calls]
    except RuntimeError:
        codes.append("lost")
    codes += [code_of(call) for call in calls + [operators.synchronize]] + [backend.status()[0]]
    print(*codes)
""")
    assert out == ["torch", "6", "6", "lost", "0", "0", "0", "0", "6", "6", "6", "lost", "0", "0", "0", "0"]
