"""A wait between the blocks of a scan that runs out: NaN from there on, an error status, nothing hung."""
import os
import subprocess
import sys

import pytest
import torch

from poorgrad_b200 import abi, operators

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CHILD = r"""
import ctypes as C, sys
sys.path[:0] = [%r]
import torch
from poorgrad_b200 import abi, backend, operators
lib = abi.load_library()
lib.tbx_scan_wait_limit.argtypes = [C.c_int64]
assert backend.status()[0] == 0
torch.manual_seed(1)

def scans(size, form, gain=1.0, offsets=None):
    x, gate = (torch.randn(size, device="cuda").to(dtype) for dtype in (torch.bfloat16,) * 2)
    if form == "direct":
        gate = gate.tanh() * gain
    def call():
        h, final = operators.gated_scan(gate, x, form=form, offsets=offsets)
        return (h, final) + operators.gated_scan_backward(x, gate, x, held, form=form, offsets=offsets)
    held = operators.gated_scan(gate, x, form=form, offsets=offsets)[0]
    return call

off = torch.tensor([0, 3, 900, 901, 4000], dtype=torch.int32, device="cuda")
calls = [scans((8, 1024, 768), "sigmoid"), scans((8, 1024, 768), "direct"), scans((8, 1024, 513), "direct"),
         scans((4000, 4096), "direct", offsets=off), scans((8, 1024, 768), "direct", 30.0)]
good = [call() for call in calls]
operators.synchronize()
for limit in (0, 1):  # every wait runs out at once, or where it has to wait at all
    lib.tbx_scan_wait_limit(limit)
    for n, (call, expected) in enumerate(zip(calls, good)):
        got = call()
        torch.cuda.synchronize()
        for name, a, e in zip(("h", "final", "dgate", "dx", "dstate"), got, expected):
            assert bool((a.isnan() | (a == e)).all()), (limit, n, name)
        if limit == 0 and n != 3:  # a block's 64 steps, backwards 32, know what its own warps hand on
            assert bool(got[0][:, 64:].isnan().all()) and bool(got[1].isnan().all())
            assert bool(got[3][:, :-32].isnan().all()) and bool(got[4].isnan().all())
            assert torch.equal(got[0][:, :64], expected[0][:, :64])
            assert torch.equal(got[3][:, -32:], expected[3][:, -32:])
lib.tbx_scan_wait_limit(4000000000)
for call, expected in zip(calls, good):  # nothing is left of it
    assert all(torch.equal(a.nan_to_num(1.5), e.nan_to_num(1.5)) for a, e in zip(call(), expected))
assert lib.tbx_scan_error() == 1
codes = []
for attempt in (operators.synchronize, calls[0]):
    try:
        attempt()
    except backend.BackendError as error:
        codes.append(error.code)
print(*codes)
"""


@pytest.mark.gpu
def test_a_wait_that_runs_out(device):
    out = subprocess.run([sys.executable, "-c", CHILD % ROOT], capture_output=True, text=True, timeout=600)
    assert out.returncode == 0, out.stderr[-2000:]
    runtime, poisoned = (next(c for c, n in abi.STATUS.items() if n == name) for name in ("Runtime", "Poisoned"))
    assert out.stdout.split() == [str(runtime), str(poisoned)]


@pytest.mark.gpu
def test_work_that_went_well(device):
    x = torch.randn(8, 600, 768, device="cuda")
    operators.gated_scan(x, x)
    operators.synchronize()
    operators.synchronize(torch.device("cuda", 0))
    with torch.cuda.stream(torch.cuda.Stream()):
        operators.gated_scan(x, x)
        operators.synchronize()


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the device-less answer")
def test_without_a_device(built):
    assert abi.load_library().tb_operators_synchronize(None) == 2
    with pytest.raises(RuntimeError):
        operators.synchronize()
