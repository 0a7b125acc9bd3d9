"""What the device operators leave in their outputs where no sequence or answer has a row."""
import pytest
import torch

import operator_cases as oc
from operator_cases import TYPES, normal
from poorgrad_b200 import operators
from test_operators import cuda

pytestmark = pytest.mark.gpu


def litter(*arrays):
    """Leaves NaN in blocks of the allocator's cache like these."""
    held = [torch.full_like(a, float("nan")) for a in arrays for _ in range(8)]
    torch.cuda.synchronize()
    del held


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("form", ["direct", "sigmoid"])
@pytest.mark.parametrize("length,channels", [(50, 6), (40, 20001), (60, 20000), (700, 72), (700, 35), (9000, 64)])
@pytest.mark.parametrize("kind", ["inside", "empty", "beyond"])
def test_new_arrays_of_a_packed_scan_are_zero_outside(device, dtype, form, length, channels, kind):
    t = TYPES[dtype]
    offsets = {"inside": [7, 7, length // 2, length - 5], "empty": [9, 9, 9], "beyond": [length, length + 8]}[kind]
    off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    outside = torch.ones(length, dtype=torch.bool, device="cuda")
    outside[offsets[0]:offsets[-1]] = False
    gate, x, dh = (cuda(normal(i, length, channels), t) for i in range(3))
    if form == "direct":
        gate = torch.tanh(gate)
    gate[outside], x[outside] = float("nan"), float("inf")
    dh[outside] = float("nan")
    litter(x)
    h, _ = operators.gated_scan(gate, x, form=form, offsets=off)
    assert bool((h[outside] == 0).all()) and bool(h[~outside].isfinite().all())
    litter(x)
    dgate, dx, _ = operators.gated_scan_backward(dh, gate, x, h, form=form, offsets=off)
    for d in (dgate, dx):
        assert bool((d[outside] == 0).all()) and bool(d[~outside].isfinite().all())
    # an array that the caller gives is left alone there, the other is not
    mark = torch.full_like(x, 5.0)
    litter(x)
    a, b, _ = operators.gated_scan_backward(dh, gate, x, h, form=form, offsets=off, dgate=mark)
    assert bool((a[outside] == 5).all()) and torch.equal(b, dx) and torch.equal(a[~outside], dgate[~outside])
    mark = torch.full_like(x, 5.0)
    litter(x)
    a, b, _ = operators.gated_scan_backward(dh, gate, x, h, form=form, offsets=off, dx=mark)
    assert bool((b[outside] == 5).all()) and torch.equal(a, dgate) and torch.equal(b[~outside], dx[~outside])
    mark = torch.full_like(x, 5.0)
    operators.gated_scan(gate, x, form=form, offsets=off, out=mark)
    assert bool((mark[outside] == 5).all()) and torch.equal(mark[~outside], h[~outside])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [3, 33, 1000, 1027, 5003])
@pytest.mark.parametrize("offsets", [[4, 12, 15], [6, 6, 6], [20, 21, 30]])
def test_new_arrays_of_a_preference_loss_are_zero_outside(device, dtype, vocab, offsets):
    rows = 20
    outside = torch.ones(rows, dtype=torch.bool, device="cuda")
    outside[offsets[0]:offsets[-1]] = False
    z = cuda(normal(1, rows, vocab), TYPES[dtype])
    z[outside] = float("nan")
    at = torch.zeros(rows, dtype=torch.int32, device="cuda")
    off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    ref = cuda(oc.normal(2, rows))
    for gradient in (True, False, z):
        litter(z, ref)
        got = operators.preference_loss(z.clone() if gradient is z else z, at, off, ref,
                                        gradient=z if gradient is z else gradient)
        assert bool((got.logp[outside] == 0).all()) and bool(got.logp[~outside].isfinite().all())
        if gradient is True:
            assert bool((got.gradient[outside] == 0).all())
            assert bool(got.gradient[~outside].isfinite().all())
        elif gradient is z:
            assert bool(z[outside].isnan().all())
