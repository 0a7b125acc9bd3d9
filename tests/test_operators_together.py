"""The device operators as they are used: around a compiled plan's products, and one after the other
through a decoder step with its backward pass."""
import numpy as np
import pytest
import torch

import operator_cases as oc
from operator_cases import EPS
from poorgrad_b200 import backend, neural, operators
from poorgrad_b200.graph import Dense, Selection, Tape, selection
from poorgrad_b200.plan import Request

pytestmark = pytest.mark.gpu


class DeviceView:
    """A plan's readable value as a torch tensor over the plan's own memory."""

    def __init__(self, pointer, shape):
        self.__cuda_array_interface__ = {"data": (pointer, False), "shape": tuple(shape),
                                         "typestr": "<f4", "version": 3}


def test_policy_training_around_a_compiled_plan(device):
    """Logits from one plan, their gradient from the policy loss on the plan's stream, parameter
    gradients and an optimizer step from a second plan that is fed the logits' gradient."""
    rows, vocab, embed, hidden = 96, 27, 16, 40
    tape = Tape()
    draw = neural.normal(3, 0.4)
    table = tape.parameter(Dense((vocab, embed), draw((vocab, embed))))
    first = neural.Linear(tape, draw((embed, hidden)), np.zeros(hidden, np.float32))
    second = neural.Linear(tape, draw((hidden, vocab)), np.zeros(vocab, np.float32))
    tokens = tape.input(selection(np.zeros(rows, np.int64), vocab))
    upstream = tape.input(Dense((rows, vocab), np.zeros((rows, vocab), np.float32)))
    logits = second.express(first.express(table.gather(tokens)).tanh())
    pulled = (logits * upstream).sum()
    params = [table] + first.parameters() + second.parameters()
    grads = tape.differentiate(pulled, params)
    network = tape.into_network()
    forward = backend.DevicePlan(network.compile(Request([logits])))
    backward = backend.DevicePlan(network.compile(Request([pulled] + list(grads))))
    payloads = network.parameters()
    held = backend.DeviceParameters(forward, payloads)
    rate = 0.25
    optimizer = backend.Optimizer(backward, held, backend.SGD, zip(params, grads), rate)

    ids = neural.integers(5, vocab, rows)
    targets = torch.from_numpy(neural.integers(6, vocab, rows)).int()
    old = (oc.normal(7, rows) - 3).float()
    advantages = oc.normal(8, rows).float()
    weights = torch.full((rows,), 1 / 64)
    weights[64:] = 0.0
    fed = {tokens: Selection(ids, vocab)}
    forward.forward(held, fed)
    with torch.cuda.stream(torch.cuda.ExternalStream(forward.stream())):
        z = torch.as_tensor(DeviceView(forward.device_pointer(logits), (rows, vocab)), device="cuda")
        result = operators.policy_loss(z, targets.cuda(), old.cuda(), advantages.cuda(),
                                       weights.cuda(), clip_low=0.2, clip_high=0.2)
    torch.cuda.synchronize()
    backward.forward(held, {**fed, upstream: ("device", result.gradient.data_ptr(), "dense")}, sync=True)
    got = [backward.of(g) for g in grads]
    del optimizer

    payloads = [np.asarray(p, np.float32).reshape(s) for p, s in zip(payloads, held.shapes)]
    leaves = [torch.from_numpy(p).double().requires_grad_() for p in payloads]
    e, w1, b1, w2, b2 = leaves
    ref = torch.tanh(e[torch.from_numpy(np.asarray(ids)).long()] @ w1 + b1) @ w2 + b2
    logp = torch.log_softmax(ref, 1).gather(1, targets.long()[:, None])[:, 0]
    r = torch.exp(logp - old.double())
    a = advantages.double()
    loss = -(weights.double() * torch.minimum(r * a, r.clamp(0.8, 1.2) * a)).sum()
    loss.backward()
    # two products of up to 96 terms in f32-equivalent arithmetic on each side of the loss, the loss's
    # own steps (about 100), and the ratio's amplification of a log probability's error, below e:
    # 4 * 96 + 3 * 100 steps of the magnitudes, which exceed a gradient's largest element by less than 4
    assert abs(float(result.loss) - float(loss.detach())) <= 700 * 4 * EPS
    for g, leaf, p in zip(got, leaves, range(len(leaves))):
        scale = float(leaf.grad.abs().max())
        assert np.abs(g - leaf.grad.numpy()).max() <= 700 * 4 * EPS * scale
        stepped = payloads[p] - g * np.float32(rate)
        assert np.array_equal(held.download(p), stepped.astype(np.float32))


def test_a_decoder_step_and_its_backward_pass(device):
    """Projection, head norm and rotation, attention, gated scan, vocabulary product, preference loss;
    then back through each operator's gradient, against 64-bit autograd of the formulas."""
    batch, length, heads, shared, dim, width, vocab = 2, 24, 4, 2, 16, 48, 61
    beta = 0.5
    x = oc.normal(1, batch, length, width)
    wp = 0.2 * oc.normal(2, width, (heads + 2 * shared) * dim)
    wg = 0.2 * oc.normal(3, width, heads * dim)
    wo = 0.3 * oc.normal(4, heads * dim, vocab)
    wq, wk = 1 + 0.1 * oc.normal(5, dim), 1 + 0.1 * oc.normal(6, dim)
    table = oc.table(length, dim)
    targets = torch.randint(0, vocab, (batch * length,), generator=torch.Generator().manual_seed(9)).int()
    targets[::5] = -1
    ref = oc.normal(10, batch * length) - 4
    offsets = torch.tensor([0, length, 2 * length], dtype=torch.int32)
    leaves = [v.float().double().requires_grad_() for v in (x, wp, wg, wo, wq, wk)]
    ref = ref.float().double()
    mask = torch.full((length, length), -float("inf")).triu(1)

    def attend(q, k, v):
        k, v = (t.repeat_interleave(heads // shared, 2) for t in (k, v))
        s = torch.einsum("bthd,bshd->bhts", q, k) / dim ** 0.5 + mask.to(q)
        return torch.einsum("bhts,bshd->bthd", torch.softmax(s, -1), v)

    def split(rows):
        q, k, v = rows.split([heads * dim, shared * dim, shared * dim], -1)
        return (t.unflatten(-1, (-1, dim)) for t in (q, k, v))

    # the formulas in 64 bits
    lx, lp, lg, lo, lq, lk = leaves
    q, k, v = split(lx @ lp)
    along = torch.arange(length).expand(batch, -1)
    y = attend(oc.rotate(q, lq, table.double(), along, 1e-5, "halves"),
               oc.rotate(k, lk, table.double(), along, 1e-5, "halves"), v).flatten(2)
    gate = lx @ lg
    a, b = torch.sigmoid(gate), torch.sigmoid(-gate) * y
    h, carried = [], torch.zeros_like(b[:, 0])
    for t in range(length):
        carried = a[:, t] * carried + b[:, t]
        h.append(carried)
    z = (torch.stack(h, 1) @ lo).flatten(0, 1)
    live = targets >= 0
    step = torch.where(live, torch.log_softmax(z, 1).gather(1, targets.long().clamp(min=0)[:, None])[:, 0]
                       - ref, torch.zeros(()).double())
    margin = beta * (step[:length].sum() - step[length:].sum())
    loss = torch.nn.functional.softplus(-margin)
    loss.backward()

    # the operators
    f = [v.detach().float().cuda() for v in leaves]
    rows = f[0] @ f[1]
    q, k, v = split(rows)
    tab = table.cuda()
    qr, kr = operators.head_rotate(q, k, tab, q_weight=f[4], k_weight=f[5])
    parts = [t.detach().requires_grad_() for t in (qr, kr, v)]
    y = attend(*parts)
    flat = y.detach().flatten(2)
    gates = f[0] @ f[2]
    hs, _ = operators.gated_scan(gates, flat)
    z = (hs @ f[3]).flatten(0, 1)
    result = operators.preference_loss(z, targets.cuda(), offsets.cuda(), ref.float().cuda(), beta=beta)
    dz = result.gradient.view(batch, length, vocab)
    dh = dz @ f[3].T
    dgate, dy, _ = operators.gated_scan_backward(dh, gates, flat, hs)
    dqr, dkr, dv = torch.autograd.grad(y, parts, dy.view_as(y))
    dq, dk, dwq, dwk = operators.head_rotate_backward(dqr, dkr, q, k, tab, q_weight=f[4], k_weight=f[5])
    drows = torch.cat([dq.flatten(2), dk.flatten(2), dv.flatten(2)], -1)
    got = [drows @ f[1].T + dgate @ f[2].T, torch.einsum("btw,btr->wr", f[0], drows),
           torch.einsum("btw,btr->wr", f[0], dgate), torch.einsum("btw,btr->wr", hs, dz), dwq, dwk]

    # at most eight stages behind any result, each within 20 * 24 + 3 * 64 steps of the magnitudes
    # that it sums (the scan's 24 steps are the longest); those exceed the largest result by less than 4
    bar = 8 * 4 * (20 * length + 3 * 64) * EPS
    assert abs(float(result.loss) - float(loss.detach())) <= bar * max(1.0, float(loss.detach()))
    for name, g, leaf in zip(("x", "projection", "gate", "vocabulary", "q weight", "k weight"), got, leaves):
        error = float((g.double().cpu() - leaf.grad).abs().max())
        assert error <= bar * float(leaf.grad.abs().max()), name
