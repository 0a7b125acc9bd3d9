"""Arrays that a caller gives the device operators to be written: autograd learns of it, and they may not
share memory with what the call still reads or writes."""
import pytest
import torch

import operator_cases as oc
from poorgrad_b200 import operators
from poorgrad_b200.backend import BackendError
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


def test_arrays_that_share_memory_are_refused(device):
    joint = r(3, 7, 12)
    x, g = joint[..., :4], joint[..., 4:8]
    h, d = r(3, 7, 4), r(3, 7, 4)
    flat = r(3 * 7 * 4 + 4)
    ahead, behind = flat[:84].view(3, 7, 4), flat[4:].view(3, 7, 4)
    states = r(4, 4)
    table = cuda(oc.table(7, 8))
    heads = r(1, 7, 6, 8)
    q, k = heads[:, :, :4], heads[:, :, 4:]
    z = r(5, 12)
    at, old, adv, w = loss_rows(5)
    every = r(40 * 3 * 4)
    refused = [
        lambda: operators.gated_scan(g, x, out=joint[..., 3:7]),
        lambda: operators.gated_scan(ahead, d, out=behind), lambda: operators.gated_scan(d, behind, out=ahead),
        lambda: operators.gated_scan(g, x.contiguous()[:1].expand(3, 7, 4), out=x.contiguous()[:1].expand(3, 7, 4)),
        lambda: operators.gated_scan(g, d[:1].expand(3, 7, 4), out=d),
        lambda: operators.gated_scan(g, x, state=states[:3], final_state=states[1:]),
        lambda: operators.gated_scan(d, h, out=every[:84].view(3, 7, 4), final_state=every[72:84].view(3, 4)),
        lambda: operators.gated_scan_backward(d, g, x, h, dgate=ahead, dx=ahead),
        lambda: operators.gated_scan_backward(d, g, x, h, dgate=ahead, dx=behind),
        lambda: operators.gated_scan_backward(d, g, x, h, dgate=d, dx=d),
        lambda: operators.gated_scan_backward(d, g, x, h, dgate=h), lambda: operators.gated_scan_backward(d, g, x, h, dx=h),
        lambda: operators.gated_scan_backward(ahead, g, x, h, dx=behind),
        lambda: operators.gated_scan_backward(d, ahead, x, h, dx=behind),
        lambda: operators.gated_scan_backward(d, g, ahead, h, dgate=behind),
        lambda: operators.head_rotate(q, q, table, q_out=h.new_empty(1, 7, 4, 8), k_out=q),
        lambda: operators.head_rotate(q, k, table, q_out=heads[:, :, 1:5]),
        lambda: operators.head_rotate(q, k, table, q_out=heads[:, :, :4], k_out=heads[:, :, 3:5]),
        lambda: operators.head_rotate_backward(k, k, q[:, :, :2], k, table, q_out=heads[:, :, 3:5]),
        lambda: operators.policy_loss(z[:, :8], at, old, adv, w, gradient=z[:, 1:9]),
        lambda: operators.policy_loss(z[:4], at[:4], old[:4], adv[:4], w[:4], gradient=z[1:]),
        lambda: operators.preference_loss(z[:4], at[:4], row(0, 2, 4), old[:4], gradient=z[1:]),
    ]
    saved = [t.clone() for t in (joint, h, d, flat, states, heads, z, every)]
    for n, call in enumerate(refused):
        with pytest.raises((ValueError, BackendError), match="shares memory|written rows overlap"):
            call()
            print("call", n)
    torch.cuda.synchronize()
    for a, b in zip((joint, h, d, flat, states, heads, z, every), saved):
        assert torch.equal(a, b), "a refused call wrote something"


def test_arrays_side_by_side_in_one_are_accepted(device):
    joint = r(3, 7, 20)
    parts = [joint[..., 4 * i:4 * i + 4] for i in range(5)]
    plain = [p.clone() for p in parts]
    h, final = operators.gated_scan(parts[0], parts[1], out=parts[4])
    e, last = operators.gated_scan(plain[0], plain[1])
    assert torch.equal(h, e) and torch.equal(final, last)
    expected = operators.gated_scan_backward(plain[2], plain[0], plain[1], e)
    got = operators.gated_scan_backward(parts[2], parts[0], parts[1], parts[4], dgate=parts[3], dx=parts[2])
    assert all(torch.equal(a, b) for a, b in zip(got, expected))
    # over what it is made from
    got = operators.gated_scan_backward(plain[2].clone(), parts[0], parts[1], e, dgate=parts[0], dx=parts[1])
    assert all(torch.equal(a, b) for a, b in zip(got, expected))
    heads, table = r(2, 7, 6, 8), cuda(oc.table(7, 8))
    q, k = heads[:, :, :4], heads[:, :, 4:]
    e = operators.head_rotate(q.clone(), k.clone(), table)
    out = torch.empty(2, 6, 7, 8, device="cuda").transpose(1, 2)
    got = operators.head_rotate(q, k, table, q_out=out[:, :, :4], k_out=out[:, :, 4:])
    assert all(torch.equal(a, b) for a, b in zip(got, e))
    # every second token, the others' places kept by the other side
    both = r(1, 8, 2, 8)
    got = operators.head_rotate(both[:, ::2], both[:, 1::2], table, q_out=both[:, ::2], k_out=both[:, 1::2])
    z = r(6, 5)
    at, old, adv, w = loss_rows(3)
    a = operators.policy_loss(z[::2], at, old, adv, w, gradient=z[1::2]).gradient
    assert torch.equal(a, operators.policy_loss(z[::2].clone(), at, old, adv, w).gradient)
    one = operators.gated_scan(r(1, 4, 3), r(1, 4, 3), out=r(1, 4, 3), final_state=r(1, 3))
    assert one[0].shape == (1, 4, 3)
