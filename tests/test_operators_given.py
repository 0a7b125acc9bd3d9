"""Arrays that a caller gives the device operators to be written."""
import pytest
import torch

import operator_cases as oc
from poorgrad_b200 import operators
from test_operators import cuda

pytestmark = pytest.mark.gpu


def r(*shape):
    return torch.randn(*shape, device="cuda")


def row(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def loss_rows(rows):
    return torch.zeros(rows, dtype=torch.int32, device="cuda"), r(rows), r(rows), r(rows).abs()


def test_a_written_array_has_another_version(device):
    x, s = r(2, 5, 6), r(2, 6)
    h, _ = operators.gated_scan(x, x)
    table = cuda(oc.table(4, 8))
    q, k = r(1, 4, 3, 8), r(1, 4, 2, 8)
    z = r(4, 9)
    at, old, adv, w = loss_rows(4)
    calls = [
        (lambda o: operators.gated_scan(x, x, out=o), (2, 5, 6)),
        (lambda o: operators.gated_scan(x, x, final_state=o), (2, 6)),
        (lambda o: operators.gated_scan(x, x, state=o, final_state=o), (2, 6)),
        (lambda o: operators.gated_scan_backward(x, x, x, h, dgate=o), (2, 5, 6)),
        (lambda o: operators.gated_scan_backward(x, x, x, h, dx=o), (2, 5, 6)),
        (lambda o: operators.head_rotate(q, k, table, q_out=o), (1, 4, 3, 8)),
        (lambda o: operators.head_rotate(q, k, table, k_out=o), (1, 4, 2, 8)),
        (lambda o: operators.head_rotate_backward(q, k, q, k, table, q_out=o), (1, 4, 3, 8)),
        (lambda o: operators.head_rotate_backward(q, k, q, k, table, k_out=o), (1, 4, 2, 8)),
        (lambda o: operators.policy_loss(z, at, old, adv, w, gradient=o), (4, 9)),
        (lambda o: operators.preference_loss(z, at, row(0, 2, 4), old, gradient=o), (4, 9)),
    ]
    for n, (call, shape) in enumerate(calls):
        o = torch.zeros(shape, device="cuda")
        before = o._version
        call(o)
        assert o._version > before, n
        with torch.inference_mode():
            o = torch.zeros(shape, device="cuda")
        call(o)  # such an array has no version
    for read in (x, s, q, k, z, old):
        assert read._version == 0


def test_a_backward_pass_that_needs_what_was_overwritten_raises(device):
    leaf = r(4, 9).requires_grad_()
    logits = leaf * 1
    (logits * logits).sum().backward(retain_graph=True)
    at, old, adv, w = loss_rows(4)
    kept = (logits * logits).sum()
    operators.preference_loss(logits.detach(), at, row(0, 2, 4), old, gradient=logits.detach())
    with pytest.raises(RuntimeError, match="inplace"):
        kept.backward()
