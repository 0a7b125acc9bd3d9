"""The device operators against their definitions in 64 bits, at the sizes, strides, masks and
indexes where they can go wrong.

Tolerances count roundings: EPS is a whole f32 step, so one f32 rounding is EPS / 2, and each result
is stored with one rounding of half_step(type).  The fast exponential is off by at most
2 + 1.2 |x| steps, divisions and reciprocal roots by 2."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import operator_cases as oc
from operator_cases import EPS, TYPES, half_step, normal
from poorgrad_b200 import operators
from poorgrad_b200.backend import BackendError

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SENTINEL = -77.0


def cuda(t, dtype=torch.float32):
    return t.to(dtype).cuda()


def within(got, expected, tolerance, what):
    got, expected = got.detach().double().cpu(), expected.double()
    assert got.shape == expected.shape, what
    odd = ~torch.isfinite(expected)
    assert torch.equal(torch.isnan(got), torch.isnan(expected)), f"{what}: other NaN"
    assert torch.equal(got[odd & ~torch.isnan(expected)], expected[odd & ~torch.isnan(expected)]), what
    error = torch.where(odd, torch.zeros_like(got), (got - expected).abs())
    bar = torch.where(odd, torch.zeros_like(got), torch.as_tensor(tolerance).double().expand_as(got))
    bad = error > bar
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off, worst "
                           f"{float((error / bar.clamp(min=1e-300)).max())} of the tolerance")


def laid(t, dtype, layout):
    """A device array holding `t` [batch, length, channels] in one of several layouts."""
    batch, length, channels = t.shape
    if layout == "plain":
        return cuda(t, dtype)
    if layout == "shifted":  # the base one element past an aligned address
        flat = torch.empty(t.numel() + 1, dtype=dtype, device="cuda")[1:].view(t.shape)
    elif layout == "padded":  # rows inside wider rows
        flat = torch.full((batch, length, channels + 5), SENTINEL, dtype=dtype,
                          device="cuda")[:, :, 2:2 + channels]
    elif layout == "aligned":  # rows inside wider rows, whole 16 bytes apart
        flat = torch.full((batch, length, -(-channels // 8) * 8 + 8), SENTINEL, dtype=dtype,
                          device="cuda")[:, :, :channels]
    else:  # time-major
        flat = torch.empty(length, batch, channels, dtype=dtype, device="cuda").transpose(0, 1)
    flat.copy_(t)
    return flat


# ---------------------------------------------------------------- gated scan
def scan_inputs(seed, form, dtype, batch, length, channels, count=None):
    t = TYPES[dtype]
    gate = normal(seed, batch, length, channels) * 2 + (1 if form == "sigmoid" else 0)
    if form == "direct":
        gate = torch.tanh(gate)
    made = [gate, normal(seed + 1, batch, length, channels)]
    made = [v.to(t).double() for v in made]
    return made + [normal(seed + 2, count or batch, channels).float().double()]


def steps_of(batch, length, offsets=None):
    """Steps behind each output, counted from its sequence's start (the longest count there)."""
    n = torch.zeros(batch, length, 1, dtype=torch.float64)
    for _, row, lo, hi in oc.spans_of(offsets, batch, length):
        n[row, lo:hi, 0] = torch.arange(1, hi - lo + 1, dtype=torch.float64)
    return n


# a step rounds twice and carries the gate's error: the form's exponential and division
PER_STEP = {"direct": 2, "sigmoid": 20}

SCAN_SIZES = [(1, 1, 1), (2, 1, 8), (3, 2, 5), (1, 17, 31), (2, 127, 64), (2, 128, 33),
              (1, 129, 66), (3, 257, 40), (1, 700, 2), (5, 65, 130), (1, 1100, 257)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("form", ["direct", "sigmoid"])
@pytest.mark.parametrize("size", SCAN_SIZES)
def test_scan_follows_the_recurrence(device, form, dtype, size):
    batch, length, channels = size
    t = TYPES[dtype]
    gate, x, state = scan_inputs(1, form, dtype, *size)
    h, final, m, fm = oc.scan(form, gate, x, state)
    got, got_final = operators.gated_scan(cuda(gate, t), cuda(x, t), form=form, state=cuda(state))
    n = steps_of(batch, length)
    k = PER_STEP[form]
    within(got, h, (k * n + k) * EPS * m + half_step(t) * h.abs(), "h")
    within(got_final, final, (k * length + k) * EPS * fm, "final state")
    # no state is a state of zeros
    zero = torch.zeros_like(state)
    h, final, m, fm = oc.scan(form, gate, x, zero)
    got, got_final = operators.gated_scan(cuda(gate, t), cuda(x, t), form=form)
    within(got, h, (k * n + k) * EPS * m + half_step(t) * h.abs(), "h without a state")
    within(got_final, final, (k * length + k) * EPS * fm, "final state without a state")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("form", ["direct", "sigmoid"])
@pytest.mark.parametrize("size", SCAN_SIZES)
def test_scan_backward_follows_the_formula(device, form, dtype, size):
    batch, length, channels = size
    t = TYPES[dtype]
    gate, x, state = scan_inputs(3, form, dtype, *size)
    h = oc.scan(form, gate, x, state)[0].to(t).double()
    dh = normal(5, *size).to(t).double()
    dfinal = normal(6, batch, channels).float().double()
    for init, last in ((state, dfinal), (None, None)):
        zero = torch.zeros_like(state)
        expected, sizes = oc.scan_backward(form, dh, gate, x, h, zero if init is None else init,
                                           zero if last is None else last)
        got = operators.gated_scan_backward(
            cuda(dh, t), cuda(gate, t), cuda(x, t), cuda(h, t), form=form,
            state=None if init is None else cuda(init), dfinal=None if last is None else cuda(last))
        k = PER_STEP[form]
        for name, a, e, m, half in zip(("dgate", "dx", "dstate"), got, expected, sizes,
                                       (half_step(t), half_step(t), 0.0)):
            within(a, e, (k * length + 3 * k) * EPS * m + half * e.abs(), name)


OFFSETS = [[0, 9], [0, 0, 9], [0, 3, 3, 3, 9], [0, 1, 2, 9, 9], [2, 5, 8], [0, 130, 131, 300, 555],
           [7, 7, 300, 301, 550], [0, 0, 0], [0, 16, 32, 48, 64, 128, 256, 512, 555]]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("form", ["direct", "sigmoid"])
@pytest.mark.parametrize("offsets", OFFSETS)
@pytest.mark.parametrize("channels", [3, 72])
def test_packed_scan_keeps_sequences_apart(device, form, dtype, offsets, channels):
    t = TYPES[dtype]
    length, count = max(9, 555 if offsets[-1] > 9 else 9), len(offsets) - 1
    gate, x, state = scan_inputs(11, form, dtype, 1, length, channels, count)
    inside = torch.zeros(length, dtype=torch.bool)
    inside[offsets[0]:offsets[-1]] = True
    # what lies outside every sequence must not matter
    gate[0, ~inside], x[0, ~inside] = float("nan"), float("inf")
    h, final, m, fm = oc.scan(form, gate, x, state, offsets)
    off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    out = torch.full((length, channels), SENTINEL, dtype=t, device="cuda")
    got, got_final = operators.gated_scan(cuda(gate[0], t), cuda(x[0], t), form=form,
                                          state=cuda(state), offsets=off, out=out)
    k = PER_STEP[form]
    n = steps_of(1, length, offsets)[0]
    tol = (k * n + k) * EPS * m[0] + half_step(t) * h[0].abs()
    within(got[inside.cuda()], h[0, inside], tol[inside], "h")
    assert bool((got[~inside.cuda()] == SENTINEL).all()), "rows outside every sequence"
    within(got_final, final, (k * length + k) * EPS * fm, "final state")

    h = h.to(t).double()
    h[0, ~inside] = float("nan")
    dh = normal(13, 1, length, channels).to(t).double()
    dh[0, ~inside] = float("nan")
    dfinal = normal(14, count, channels).float().double()
    expected, sizes = oc.scan_backward(form, dh, gate, x, h, state, dfinal, offsets)
    dgate, dx = (torch.full((length, channels), SENTINEL, dtype=t, device="cuda") for _ in range(2))
    got = operators.gated_scan_backward(cuda(dh[0], t), cuda(gate[0], t), cuda(x[0], t),
                                        cuda(h[0], t), form=form, state=cuda(state), offsets=off,
                                        dfinal=cuda(dfinal), dgate=dgate, dx=dx)
    for name, a, e, m in zip(("dgate", "dx"), got, expected, sizes):
        within(a[inside.cuda()], e[0, inside], (k * length + 3 * k) * EPS * m[0, inside]
               + half_step(t) * e[0, inside].abs(), name)
        assert bool((a[~inside.cuda()] == SENTINEL).all()), name
    within(got[2], expected[2], (k * length + 3 * k) * EPS * sizes[2], "dstate")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["shifted", "padded", "aligned", "time-major"])
@pytest.mark.parametrize("channels", [40, 33])
def test_scan_in_other_layouts(device, dtype, layout, channels):
    t = TYPES[dtype]
    size = (3, 50, channels)
    gate, x, state = scan_inputs(21, "sigmoid", dtype, *size)
    plain, final = operators.gated_scan(cuda(gate, t), cuda(x, t), state=cuda(state))
    dh = normal(22, *size).to(t).double()
    grads = operators.gated_scan_backward(cuda(dh, t), cuda(gate, t), cuda(x, t), plain,
                                          state=cuda(state))
    out = laid(torch.full(size, SENTINEL), t, layout)
    got, got_final = operators.gated_scan(laid(gate, t, layout), laid(x, t, layout),
                                          state=cuda(state), out=out)
    # the same recurrence, in whatever order of work the layout selects
    h, _, m, _ = oc.scan("sigmoid", gate, x, state)
    within(got, h, 20 * 51 * EPS * m + half_step(t) * h.abs(), layout)
    within(got_final, final.double().cpu(), 2 * 20 * 51 * EPS * m[:, -1], layout)
    dgate, dx = (laid(torch.full(size, SENTINEL), t, layout) for _ in range(2))
    other = operators.gated_scan_backward(laid(dh, t, layout), laid(gate, t, layout),
                                          laid(x, t, layout), laid(plain.double().cpu(), t, layout),
                                          state=cuda(state), dgate=dgate, dx=dx)
    expected, sizes = oc.scan_backward("sigmoid", dh, gate, x, plain.double().cpu(), state,
                                       torch.zeros_like(state))
    for a, e, m in zip(other, expected, sizes):
        half = half_step(t) if a.dtype == t else 0.0
        within(a, e, 20 * 53 * EPS * m + half * e.abs(), layout)
    for a, b in zip(grads, other):
        assert a.shape == b.shape
    if layout in ("padded", "aligned"):
        base = out._base if out._base is not None else out
        assert int((base == SENTINEL).sum()) == base.numel() - out.numel(), "written between rows"


@pytest.mark.parametrize("length", [0, 1, 40])
def test_scan_in_place_and_as_a_decode_carry(device, length):
    gate, x, state = scan_inputs(31, "direct", "f32", 2, length, 24)
    first, final = operators.gated_scan(cuda(gate), cuda(x), form="direct", state=cuda(state))
    g, v, s = cuda(gate), cuda(x), cuda(state)
    got, carried = operators.gated_scan(g, v, form="direct", state=s, out=v, final_state=s)
    assert got is v and carried is s
    assert torch.equal(got, first) and torch.equal(carried, final)
    got, _ = operators.gated_scan(cuda(gate), cuda(x), form="direct", state=cuda(state), out=g)
    if length == 0:
        assert torch.equal(final, cuda(state))
    # one token at a time gives the recurrence too
    s = cuda(state)
    h, _, m, _ = oc.scan("direct", gate, x, state)
    for t in range(length):
        one, s = operators.gated_scan(cuda(gate[:, t:t + 1]), cuda(x[:, t:t + 1]), form="direct",
                                      state=s, final_state=s)
        within(one[:, 0], h[:, t], (2 * t + 4) * EPS * m[:, t], f"step {t}")
    dh = normal(33, 2, length, 24)
    for into in ("dgate", "dx"):
        d = cuda(dh)
        a = operators.gated_scan_backward(cuda(dh), cuda(gate), cuda(x), first, form="direct")
        b = operators.gated_scan_backward(d, cuda(gate), cuda(x), first, form="direct", **{into: d})
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_scan_gradient_against_differences(device):
    size = (2, 37, 5)
    gate, x, state = scan_inputs(41, "sigmoid", "f32", *size)
    w, wf = normal(42, *size), normal(43, 2, 5)

    def loss(gate, x, state):
        h, final = operators.gated_scan(cuda(gate), cuda(x), state=cuda(state))
        return float((h.double().cpu() * w).sum() + (final.double().cpu() * wf).sum())

    h, _ = operators.gated_scan(cuda(gate), cuda(x), state=cuda(state))
    grads = operators.gated_scan_backward(cuda(w), cuda(gate), cuda(x), h, state=cuda(state),
                                          dfinal=cuda(wf))
    for i, (at, g) in enumerate(zip((gate, x, state), grads)):
        way = normal(44 + i, *at.shape)
        step = 1e-2
        args = [gate, x, state]
        args[i] = at + step * way
        up = loss(*args)
        args[i] = at - step * way
        down = loss(*args)
        slope = float((g.double().cpu() * way).sum())
        # f32 outputs: 370 terms of about 1 with a rounding each over 2 step; the cubic term of
        # the sigmoid is below step^2 of the sum of the magnitudes
        scale = float((g.double().cpu() * way).abs().sum())
        assert abs((up - down) / (2 * step) - slope) <= 370 * 8 * EPS / (2 * step) + step ** 2 * scale


# --------------------------------------------------------------- head rotate
ROTATE = [  # batch, length, q heads, k heads, dim, turned
    (1, 1, 1, 1, 2, 2), (2, 3, 4, 2, 64, 64), (1, 5, 12, 12, 64, 32), (3, 1, 5, 1, 128, 128),
    (1, 7, 3, 3, 80, 80), (2, 2, 2, 1, 34, 16), (1, 3, 2, 2, 96, 0), (1, 2, 3, 1, 256, 256),
    (1, 2, 1, 1, 512, 512), (2, 9, 7, 0, 64, 64), (1, 4, 0, 3, 32, 32), (1, 33, 33, 9, 16, 8),
    (1, 2, 40, 8, 192, 64), (1, 2, 2, 2, 320, 320), (1, 3, 2, 2, 512, 128)]


def rotate_inputs(seed, dtype, batch, length, hq, hk, dim, turned):
    t = TYPES[dtype]
    q, k = (normal(seed + i, batch, length, h, dim).to(t).double() for i, h in enumerate((hq, hk)))
    wq, wk = (1 + 0.3 * normal(seed + 2 + i, dim).float().double() for i in range(2))
    wq, wk = wq.float().double(), wk.float().double()
    table = oc.table(40, turned, first=1000)
    positions = torch.randint(0, 40, (batch, length), generator=torch.Generator().manual_seed(seed))
    return q, k, wq, wk, table, positions


def rotate_bar(x, w, expected, t):
    # the mean of squares: at most 16 terms a lane and 5 tree steps; root, two products, the turn
    n = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-5) * w
    return 48 * EPS * n.abs().amax(-1, keepdim=True) + half_step(t) * expected.abs() if n.numel() \
        else expected


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("style", ["halves", "pairs"])
@pytest.mark.parametrize("size", ROTATE)
def test_rotate_follows_the_formula(device, dtype, style, size):
    t = TYPES[dtype]
    q, k, wq, wk, table, positions = rotate_inputs(51, dtype, *size)
    pos = cuda(positions, torch.int32)
    got = operators.head_rotate(cuda(q, t), cuda(k, t), cuda(table), pos, q_weight=cuda(wq),
                                k_weight=cuda(wk), style=style)
    for a, x, w in zip(got, (q, k), (wq, wk)):
        e = oc.rotate(x, w, table.double(), positions, 1e-5, style)
        within(a, e, rotate_bar(x, w, e, t), "rotate")
    # positions along the length, and no weights
    got = operators.head_rotate(cuda(q, t), cuda(k, t), cuda(table), style=style)
    along = torch.arange(size[1])[None, :].expand(size[0], -1)
    for a, x in zip(got, (q, k)):
        e = oc.rotate(x, torch.ones(size[4]), table.double(), along, 1e-5, style)
        within(a, e, rotate_bar(x, 1.0, e, t), "rotate without weights")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("style", ["halves", "pairs"])
@pytest.mark.parametrize("size", ROTATE)
def test_rotate_backward_follows_the_formula(device, dtype, style, size):
    t = TYPES[dtype]
    q, k, wq, wk, table, positions = rotate_inputs(61, dtype, *size)
    dq, dk = (normal(65 + i, *x.shape).to(t).double() for i, x in enumerate((q, k)))
    got = operators.head_rotate_backward(cuda(dq, t), cuda(dk, t), cuda(q, t), cuda(k, t),
                                         cuda(table), cuda(positions, torch.int32),
                                         q_weight=cuda(wq), k_weight=cuda(wk), style=style)
    bare = operators.head_rotate_backward(cuda(dq, t), cuda(dk, t), cuda(q, t), cuda(k, t),
                                          cuda(table), cuda(positions, torch.int32),
                                          q_weight=cuda(wq), k_weight=cuda(wk), style=style,
                                          weights=False)
    assert bare[2] is None and bare[3] is None
    for i, (x, w, dy) in enumerate(((q, wq, dq), (k, wk, dk))):
        dx, dw, size_w = oc.rotate_backward(dy, x, w, table.double(), positions, 1e-5, style)
        r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-5)
        dn = oc.turn(dy, table.double(), positions, style, True) * w
        inner = (dn * x * r).abs().mean(-1, keepdim=True)
        if x.numel():
            bar = 96 * EPS * r * (dn.abs().amax(-1, keepdim=True)
                                  + (x * r).abs().amax(-1, keepdim=True) * inner)
            # dy enters dn as two products; a turned pair's magnitudes add up
            within(got[i], dx, 2 * bar + half_step(t) * dx.abs(), "dx")
            assert torch.equal(got[i], bare[i])
        heads = x.shape[0] * x.shape[1] * x.shape[2]
        big = oc.turn(dy, table.double(), positions, style, True).abs().amax() if x.numel() else 0
        within(got[2 + i], dw, EPS * ((heads + 64) * size_w + 8 * heads * big), "weight gradient")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 72])
def test_rotate_views_and_in_place(device, dtype, dim):
    """Views of a joint projection, outputs laid out for attention, inputs as outputs."""
    t, batch, length, hq, hk = TYPES[dtype], 2, 11, 6, 2
    joint = cuda(normal(71, batch, length, (hq + 2 * hk) * dim + 3), t)
    for start in (0, 3):  # whole 16-byte rows only at 0, if ever
        rows = joint[..., start:start + (hq + 2 * hk) * dim]
        q = rows[..., :hq * dim].unflatten(-1, (hq, dim))
        k = rows[..., hq * dim:(hq + hk) * dim].unflatten(-1, (hk, dim))
        table = cuda(oc.table(length, dim))
        plain = operators.head_rotate(q.contiguous(), k.contiguous(), table)
        q_out = torch.empty(batch, hq, length, dim, dtype=t, device="cuda").transpose(1, 2)
        k_out = torch.empty(batch, hk, length, dim, dtype=t, device="cuda").transpose(1, 2)
        got = operators.head_rotate(q, k, table, q_out=q_out, k_out=k_out)
        for a, x in zip(got, (q, k)):
            x = x.double().cpu()
            e = oc.rotate(x, torch.ones(dim), table.double().cpu(),
                          torch.arange(length).expand(batch, -1), 1e-5, "halves")
            within(a, e, rotate_bar(x, 1.0, e, t), "view")
        values = rows[..., (hq + hk) * dim:].clone()
        dy = [torch.randn_like(p) for p in plain]
        grads = operators.head_rotate_backward(*dy, q, k, table)
        into = [d.clone() for d in dy]
        again = operators.head_rotate_backward(*into, q, k, table, q_out=into[0], k_out=into[1])
        assert all(torch.equal(a, b) for a, b in zip(grads, again))
        operators.head_rotate(q, k, table, q_out=q, k_out=k)
        assert torch.equal(q, got[0]) and torch.equal(k, got[1])
        assert torch.equal(values, rows[..., (hq + hk) * dim:]), "values were touched"
    flat = operators.head_rotate(q.flatten(0, 1), k.flatten(0, 1), cuda(oc.table(30, dim)),
                                 torch.arange(22, dtype=torch.int32, device="cuda"))
    assert flat[0].shape == (22, hq, dim)


def test_rotate_positions_outside_the_table(device):
    q, k, wq, wk, table, positions = rotate_inputs(81, "f32", 1, 4, 3, 2, 32, 32)
    pos = torch.tensor([[0, 40, 3, -1]], dtype=torch.int32, device="cuda")
    got = operators.head_rotate(cuda(q), cuda(k), cuda(table), pos)
    for a in got:
        assert bool(a[0, [1, 3]].isnan().all()) and not bool(a[0, [0, 2]].isnan().any())


def test_rotate_gradient_against_differences(device):
    q, k, wq, wk, table, positions = rotate_inputs(91, "f32", 2, 3, 2, 1, 16, 16)
    a, b = normal(95, *q.shape), normal(96, *k.shape)
    pos = cuda(positions, torch.int32)

    def loss(q, k, wq, wk):
        y = operators.head_rotate(cuda(q), cuda(k), cuda(table), pos, q_weight=cuda(wq),
                                  k_weight=cuda(wk))
        return float((y[0].double().cpu() * a).sum() + (y[1].double().cpu() * b).sum())

    grads = operators.head_rotate_backward(cuda(a), cuda(b), cuda(q), cuda(k), cuda(table), pos,
                                           q_weight=cuda(wq), k_weight=cuda(wk))
    for i, g in enumerate(grads):
        args = [q, k, wq, wk]
        way, step = normal(97 + i, *args[i].shape), 1e-2
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + step * way, args[i] - step * way
        slope = (loss(*up) - loss(*down)) / (2 * step)
        scale = float((g.double().cpu() * way).abs().sum())
        # 288 outputs of about 1 with 48 steps each over 2 step; the cubic term of a norm is
        # within a few step^2 of the magnitudes
        assert abs(slope - float((g.double().cpu() * way).sum())) <= \
            288 * 48 * EPS / (2 * step) + 8 * step ** 2 * scale


# -------------------------------------------------------------------- losses
VOCABS = [1, 2, 27, 32, 33, 511, 513, 1000, 1025, 4099, 50257]


def loss_inputs(seed, dtype, rows, vocab):
    logits = (2 * normal(seed, rows, vocab)).to(TYPES[dtype]).double()
    targets = torch.randint(0, vocab, (rows,), generator=torch.Generator().manual_seed(seed))
    return logits, targets


def logp_bar(logits, targets, scale):
    """Steps behind a row's log probability and its sum of exponentials: the exponentials' own
    (their arguments weighted by their shares, below log vocab), at most vocab / 32 additions in a
    lane, 20 merges of 4 each."""
    z = scale * logits
    top = z.amax(1)
    vocab = logits.shape[1]
    at = targets.clamp(0, vocab - 1).long()
    steps = 100 + vocab / 32 + 4 * np.log(vocab)
    arg = (z.gather(1, at[:, None])[:, 0] - top).abs()
    return EPS * (steps + 2 * arg + np.log(vocab)), EPS * steps


def gradient_bar(logits, p, slope, slope_bar, scale, sum_bar, t, expected):
    x = (scale * (logits - logits.amax(1, keepdim=True))).abs()
    x = torch.where(torch.isfinite(x), x, torch.zeros_like(x))
    c = (slope.abs() * scale)[:, None]
    return (c * p * (2 * sum_bar + 4 * EPS * (x + 2)) + c * 2 * EPS
            + (slope_bar * scale)[:, None] * 2 + half_step(t) * expected.abs())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("rows,scale", [(1, 1.0), (3, 0.5), (70, 1.25)])
def test_token_logp(device, dtype, vocab, rows, scale):
    logits, targets = loss_inputs(101, dtype, rows, vocab)
    expected = oc.rows(logits, targets, scale)[0]
    got = operators.token_logp(cuda(logits, TYPES[dtype]), cuda(targets, torch.int32), scale=scale)
    within(got, expected, logp_bar(logits, targets, scale)[0], "logp")


def policy_inputs(seed, logits, targets, scale):
    rows = len(targets)
    logp = oc.rows(logits, targets, scale)[0]
    # ratios on both sides of the clipping borders, and on the upper one
    ratio = torch.tensor([0.5, 0.75, 0.85, 1.0, 1.1, 1.25, 2.0], dtype=torch.float64)
    old = (logp - torch.log(ratio[torch.arange(rows) % 7])).float().double()
    ref = (logp + 0.4 * normal(seed + 1, rows)).float().double()
    advantages = normal(seed + 2, rows).float().double()
    weights = (torch.rand(rows, generator=torch.Generator().manual_seed(seed)).double() + 0.1)
    return old, ref, advantages, (weights / rows).float().double()


def check_policy(logits, targets, old, advantages, weights, ref, kl, scale, t, got, rows=None):
    total, token, logp, grad = oc.policy(logits, targets, old, advantages, weights, ref, 0.2, 0.25,
                                         kl, scale)
    bar, sum_bar = logp_bar(logits, targets, scale)
    live = (weights != 0) & (targets >= 0)
    off = bar + EPS * (old.abs() + logp.abs() + 4)  # of the log ratio
    r = torch.exp(logp - old)
    reach = weights.abs() * (r * advantages.abs() + kl * (torch.exp(ref - logp) + 1)) * (
        off + kl * EPS * (ref.abs() + logp.abs()))
    reach = torch.where(live, reach, torch.zeros_like(reach)) * 2
    within(got.logp, logp, torch.where(live, bar, torch.zeros_like(bar)), "logp")
    within(got.token_loss, token, reach + 4 * EPS * token.abs(), "token loss")
    within(got.loss, total, reach.nan_to_num().sum() + 4 * EPS * token.nan_to_num().abs().sum(), "loss")
    if got.gradient is not None:
        zero = torch.zeros_like(r)
        slope = torch.where(live, weights * (r * advantages.abs() + kl * (1 + torch.exp(ref - logp))),
                            zero)
        p = oc.rows(logits, targets, scale)[1]
        # a ratio of 1.25 lies on the upper border: exp(logp - old) is within `off` of it, and on
        # its two sides the clipped term's slope is -r A and 0.  Either is a right answer there, so
        # the slope of such a row may be off by |w r A| (its loss is continuous and may not)
        border = live & ((r - 1.25).abs() <= 1.25 * off)
        reach = reach + torch.where(border, weights * r * advantages.abs(), zero)
        within(got.gradient, grad, gradient_bar(logits, p, slope.abs(), reach, scale, sum_bar, t, grad),
               "gradient")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("rows,scale,kl", [(1, 1.0, 0.0), (9, 0.7, 0.3), (70, 1.0, 0.05)])
def test_policy_loss_and_its_gradient(device, dtype, vocab, rows, scale, kl):
    t = TYPES[dtype]
    logits, targets = loss_inputs(111, dtype, rows, vocab)
    old, ref, advantages, weights = policy_inputs(112, logits, targets, scale)
    weights[::5] = 0.0 if rows > 1 else weights[0]
    args = (cuda(targets, torch.int32), cuda(old), cuda(advantages), cuda(weights))
    named = dict(ref_logp=cuda(ref) if kl else None, kl=kl, scale=scale, clip_low=0.2, clip_high=0.25)
    z = cuda(logits, t)
    got = operators.policy_loss(z, *args, **named)
    check_policy(logits, targets, old, advantages, weights, ref, kl, scale, t, got)
    bare = operators.policy_loss(z, *args, **named, gradient=False)
    assert bare.gradient is None
    for a, b in zip(got[:3], bare[:3]):
        within(a, b.double().cpu(), 2 * 400 * EPS * (1 + b.double().cpu().abs()), "without a gradient")
    # into wider rows, off 16 bytes, and over the logits themselves
    wide = torch.full((rows, vocab + 3), SENTINEL, dtype=t, device="cuda")
    operators.policy_loss(z, *args, **named, gradient=wide[:, 1:1 + vocab])
    check_policy(logits, targets, old, advantages, weights, ref, kl, scale, t,
                 got._replace(gradient=wide[:, 1:1 + vocab]))
    assert bool((wide[:, 0] == SENTINEL).all()) and bool((wide[:, 1 + vocab:] == SENTINEL).all())
    shifted = torch.empty(rows * vocab + 1, dtype=t, device="cuda")[1:].view(rows, vocab).copy_(z)
    over = operators.policy_loss(shifted, *args, **named, gradient=shifted)
    check_policy(logits, targets, old, advantages, weights, ref, kl, scale, t, over)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [5, 64, 2000, 50257])
def test_losses_at_masked_and_hidden_rows(device, dtype, vocab):
    t = TYPES[dtype]
    rows = 10
    logits, targets = loss_inputs(121, dtype, rows, vocab)
    targets = targets.clamp(max=vocab - 2)
    lowest = torch.finfo(t).min
    inf, nan = float("inf"), float("nan")
    logits[1] = -inf                      # nothing is left: hidden
    logits[2] = lowest                    # a uniform row
    logits[3, ::2] = -inf
    logits[3, targets[3]] = 1.0
    logits[4, ::2] = lowest
    logits[4, targets[4]] = 1.0
    logits[5], logits[6] = nan, inf       # hidden by target and by weight
    logits[7, vocab - 1] = nan            # a live row with a NaN
    logits[8, targets[8]] = -inf          # the target itself is masked
    targets[5] = -3
    weights = torch.full((rows,), 0.1, dtype=torch.float64).float().double()
    weights[6] = 0.0
    old = torch.full((rows,), -2.0, dtype=torch.float64)
    advantages = torch.ones(rows, dtype=torch.float64)
    old[6], advantages[6] = nan, inf
    z, at = cuda(logits, t), cuda(targets, torch.int32)
    for scale in (1.0, 2.0):
        got = operators.policy_loss(z, at, cuda(old), cuda(advantages), cuda(weights), scale=scale)
        for n in range(rows):
            g, lp, tl = got.gradient[n].double().cpu(), float(got.logp[n]), float(got.token_loss[n])
            if n in (1, 5, 6):
                assert lp == 0 and tl == 0 and bool((g == 0).all()), n
            elif n == 7:
                assert np.isnan(lp) and np.isnan(tl) and bool(g.isnan().all()), n
            elif n == 8:
                assert lp == -inf and tl == 0 and bool((g == 0).all()), n
            else:
                one = logits[n:n + 1].clamp(min=-1e30)
                one = one - one.amax()    # the scale does not overflow a difference
                e = oc.policy(one, targets[n:n + 1], old[n:n + 1], advantages[n:n + 1],
                              weights[n:n + 1], None, 0.2, 0.2, 0.0, scale)
                within(got.logp[n:n + 1], e[2], logp_bar(one, targets[n:n + 1], scale)[0], n)
                tol = 0.2 * (EPS * 200 + logp_bar(one, targets[n:n + 1], scale)[0]) * (
                    1 + torch.exp(e[2] + 2).abs())
                within(g[None], e[3], 2 * scale * tol[:, None] + half_step(t) * e[3].abs(), n)
        assert np.isnan(float(got.loss))
        logp = operators.token_logp(z, at, scale=scale)
        assert torch.equal(logp[[0, 1, 2, 3, 4, 5, 8, 9]].isnan(), torch.zeros(8, device="cuda") > 0)
        assert float(logp[1]) == 0 and float(logp[5]) == 0 and bool(logp[7].isnan())
    # a token beyond the vocabulary
    at[0] = vocab
    got = operators.policy_loss(z, at, cuda(old), cuda(advantages), cuda(weights))
    assert bool(got.logp[0].isnan()) and bool(got.gradient[0].isnan().all())
    assert bool(operators.token_logp(z, at)[0].isnan())
    pref = operators.preference_loss(z, at, torch.tensor([0, 5, 10], dtype=torch.int32, device="cuda"),
                                     cuda(old))
    assert bool(pref.gradient[0].isnan().all()) and bool(pref.logp[0].isnan())
    assert bool((pref.gradient[1] == 0).all()) and bool((pref.gradient[5] == 0).all())


PAIRS = [([0, 4, 9], 12), ([0, 1, 2, 3, 4], 4), ([2, 2, 9, 20, 31, 40, 40], 50),
         ([0, 0, 0], 3), ([0, 100, 130, 131, 200], 211)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [2, 33, 700, 5003])
@pytest.mark.parametrize("offsets,rows", PAIRS)
@pytest.mark.parametrize("smoothing", [0.0, 0.2])
def test_preference_loss_and_its_gradient(device, dtype, vocab, offsets, rows, smoothing):
    t, beta, scale = TYPES[dtype], 0.3, 0.9
    logits, targets = loss_inputs(131, dtype, rows, vocab)
    targets[::4] = -1
    inside = torch.zeros(rows, dtype=torch.bool)
    inside[offsets[0]:offsets[-1]] = True
    pairs = len(offsets) // 2
    logp0 = oc.rows(logits, targets, scale)[0]
    ref = (logp0 + 0.2 * normal(132, rows)).float().double()
    weights = (0.5 + normal(133, pairs).abs()).float().double()
    total, ratios, logp, grad, slope = oc.preference(logits, targets, offsets, ref, beta, smoothing,
                                                     weights, scale)
    poisoned = logits.clone()
    poisoned[~inside] = float("nan")
    out = torch.full((rows, vocab), SENTINEL, dtype=t, device="cuda")
    off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    z = cuda(poisoned, t)
    got = operators.preference_loss(z, cuda(targets, torch.int32), off, cuda(ref), beta=beta,
                                    smoothing=smoothing, weights=cuda(weights), scale=scale,
                                    gradient=out)
    bar, sum_bar = logp_bar(logits, targets, scale)
    each = bar + EPS * (logp.abs() + 1)
    cut = torch.stack([each[lo:hi].sum() for lo, hi in zip(offsets[:-1], offsets[1:])])
    within(got.ratios, ratios, cut + EPS * ratios.abs(), "ratios")
    margin_bar = beta * (cut[:pairs] + cut[pairs:])
    within(got.loss, total, (weights * margin_bar).sum() + 8 * EPS * total.abs(), "loss")
    here = inside.cuda()
    within(got.logp[here], logp[inside], bar[inside], "logp")
    p = oc.rows(logits, targets, scale)[1]
    slope_bar = torch.full((rows,), float((weights * beta * (margin_bar + 4 * EPS)).max()),
                           dtype=torch.float64)
    bars = gradient_bar(logits, p, slope.abs(), slope_bar, scale, sum_bar, t, grad)
    within(got.gradient[here], grad[inside], bars[inside], "gradient")
    assert bool((out[~here] == SENTINEL).all()), "rows outside every answer"
    if inside.any():
        over = operators.preference_loss(z, cuda(targets, torch.int32), off, cuda(ref), beta=beta,
                                         smoothing=smoothing, weights=cuda(weights), scale=scale,
                                         gradient=z)
        assert torch.equal(over.gradient[here], got.gradient[here])
        assert bool(z[~here].isnan().all())
    # equal pair weights by default
    same = oc.preference(logits, targets, offsets, ref, beta, smoothing,
                         torch.full((pairs,), 1 / pairs), scale)[0]
    bare = operators.preference_loss(cuda(logits, t), cuda(targets, torch.int32), off, cuda(ref),
                                     beta=beta, smoothing=smoothing, scale=scale, gradient=False)
    assert bare.gradient is None
    within(bare.loss, same, margin_bar.sum() / pairs + 8 * EPS * same.abs(), "mean loss")


def test_loss_gradients_against_differences(device):
    rows, vocab = 8, 19
    logits, targets = loss_inputs(141, "f32", rows, vocab)
    old, ref, advantages, weights = policy_inputs(142, logits, targets, 1.0)
    old = oc.rows(logits, targets, 1.0)[0] + 0.05  # away from the clipping borders
    off = torch.tensor([0, 3, 8], dtype=torch.int32, device="cuda")
    at = cuda(targets, torch.int32)

    def policy(z):
        return operators.policy_loss(cuda(z), at, cuda(old), cuda(advantages), cuda(weights),
                                     ref_logp=cuda(ref), kl=0.5)

    def preference(z):
        return operators.preference_loss(cuda(z), at, off, cuda(ref), smoothing=0.1, beta=0.5)

    for call in (policy, preference):
        g = call(logits).gradient.double().cpu()
        way, step = normal(143, rows, vocab), 1e-2
        slope = (float(call(logits + step * way).loss) - float(call(logits - step * way).loss)) / (2 * step)
        scale = float((g * way).abs().sum()) + float(g.abs().sum())
        # the losses are about 1 with a few hundred steps; third derivatives are of the order of
        # the first for steps of a row's logits below 0.1
        assert abs(slope - float((g * way).sum())) <= 400 * EPS / (2 * step) + 20 * step ** 2 * scale


# ------------------------------------------------- streams, graphs, extremes
def everything(inputs):
    """One call of each entry point, as a list of outputs."""
    g, x, s, dh, q, k, tab, z, at, row, off = inputs
    h, final = operators.gated_scan(g, x, state=s)
    out = [h, final, *operators.gated_scan_backward(dh, g, x, h, state=s, dfinal=final)]
    r = operators.head_rotate(q, k, tab)
    out += [*r, *operators.head_rotate_backward(*r, q, k, tab)]
    out += [operators.token_logp(z, at),
            *operators.policy_loss(z, at, row, row, row.abs(), ref_logp=row, kl=0.1),
            *operators.preference_loss(z, at, off, row)]
    return out


def some_inputs(seed):
    torch.manual_seed(seed)

    def r(*shape):
        return torch.randn(*shape, device="cuda")

    z = r(33, 5000)
    return [r(2, 300, 96), r(2, 300, 96), r(2, 96), r(2, 300, 96), r(2, 40, 6, 64), r(2, 40, 2, 64),
            cuda(oc.table(40, 64)), z, torch.randint(0, 5000, (33,), device="cuda").int(), r(33),
            torch.tensor([0, 11, 33], dtype=torch.int32, device="cuda")]


def test_results_do_not_depend_on_the_stream_or_the_run(device):
    inputs = some_inputs(1)
    first = everything(inputs)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    runs = []
    for _ in range(4):
        for st in streams:
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                runs.append(everything(inputs))
    torch.cuda.synchronize()
    for run in runs:
        assert all(torch.equal(a, b) for a, b in zip(first, run))


def test_calls_wait_for_the_work_before_them(device):
    """Inputs that an earlier kernel of the stream is still writing, outputs read right after."""
    inputs = some_inputs(2)
    expected = [t.clone() for t in everything(inputs)]
    for _ in range(3):
        fresh = [torch.zeros_like(t) for t in inputs]
        torch.cuda._sleep(2_000_000)
        for a, b in zip(fresh, inputs):
            a.copy_(b)
        got = [t + 0 for t in everything(fresh)]
        for a in fresh:
            a.zero_()
        assert all(torch.equal(a, b) for a, b in zip(got, expected))


def test_captured_graphs_replay_on_new_inputs(device):
    a, b = some_inputs(3), some_inputs(4)
    expected = [[t.clone() for t in everything(v)] for v in (a, b)]
    graphs = []
    for v in (a, b):  # two graphs alive at once share no scratch
        held = [t.clone() for t in v]
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            out = everything(held)
        graphs.append((graph, held, out))
    for (graph, held, out), other in zip(graphs, (b, a)):
        for t, v in zip(held, other):
            t.copy_(v)
    for graph, _, _ in graphs:
        graph.replay()
    torch.cuda.synchronize()
    for (_, _, out), e in zip(graphs, reversed(expected)):
        assert all(torch.equal(p, q) for p, q in zip(out, e))
    streams = [torch.cuda.Stream() for _ in graphs]
    for (graph, _, _), st in zip(graphs, streams):
        with torch.cuda.stream(st):
            graph.replay()
    torch.cuda.synchronize()
    for (_, _, out), e in zip(graphs, reversed(expected)):
        assert all(torch.equal(p, q) for p, q in zip(out, e))


def test_no_wait_between_blocks_ran_out(device):
    from poorgrad_b200.abi import load_library
    x = torch.randn(8, 2000, 768, device="cuda").bfloat16()
    h, _ = operators.gated_scan(x, x)
    operators.gated_scan_backward(h, x, x, h)
    torch.cuda.synchronize()
    assert load_library().tbx_scan_error() == 0


LARGE_CHILD = r"""
import sys
sys.path[:0] = [%r, %r]
import torch
import operator_cases as oc
from poorgrad_b200 import operators
torch.manual_seed(1)
q, k = (torch.randn(2, 64, h, 128, device="cuda").bfloat16() for h in (8, 2))
x = torch.randn(8, 600, 768, device="cuda").bfloat16()
p = torch.randn(1, 4000, 64, device="cuda")
z = torch.randn(5, 50257, device="cuda")
at, row = torch.randint(0, 50257, (5,), device="cuda").int(), torch.randn(5, device="cuda")
table = torch.from_numpy(operators.rotation_table(64, 128)).cuda()
def calls():
    out = list(operators.head_rotate_backward(q, k, q, k, table))
    out += operators.gated_scan_backward(x, x, x, x)
    out += operators.gated_scan(p, p) + operators.gated_scan(x, x)
    for logits in (z, z.bfloat16()):
        out += operators.policy_loss(logits, at, row, row, row)
    return out
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):   # first calls of kernels with large shared memory, clusters, parts
    out = calls()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(out, calls()))
print("same")
"""


def test_first_calls_of_the_large_kernels_can_be_captured(device):
    out = subprocess.run([sys.executable, "-c", LARGE_CHILD % (ROOT, os.path.join(ROOT, "tests"))],
                         capture_output=True, text=True, timeout=600)
    assert out.returncode == 0 and out.stdout.split() == ["same"], out.stderr[-2000:]


CHILD = r"""
import sys
sys.path[:0] = [%r, %r]
import torch
from test_operators import everything, some_inputs
inputs = some_inputs(5)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):   # the process's first calls are captured
    out = everything(inputs)
graph.replay()
torch.cuda.synchronize()
again = everything(inputs)
assert all(torch.equal(a, b) for a, b in zip(out, again))
print("same")
"""


def test_the_first_calls_of_a_process_can_be_captured(device):
    out = subprocess.run([sys.executable, "-c", CHILD % (ROOT, os.path.join(ROOT, "tests"))],
                         capture_output=True, text=True, timeout=600)
    assert out.returncode == 0 and out.stdout.split() == ["same"], out.stderr[-2000:]


def test_rows_further_apart_than_32_bits_count(device):
    far = (1 << 31) + 64
    flat = torch.empty(far + (1 << 14), dtype=torch.bfloat16, device="cuda")
    z = flat.as_strided((2, 4099), (far, 1))
    logits, targets = loss_inputs(151, "bf16", 2, 4099)
    z.copy_(logits)
    at = cuda(targets, torch.int32)
    near = cuda(logits, torch.bfloat16)
    one = torch.ones(2, device="cuda")
    for a, b in zip(operators.policy_loss(z, at, -one, one, one, gradient=z),
                    operators.policy_loss(near, at, -one, one, one, gradient=near.clone())):
        assert torch.equal(a, b)
    v = flat.as_strided((2, 3, 8), (far, 16, 1))
    g = torch.randn(2, 3, 8, device="cuda").bfloat16()
    v.copy_(g)
    h, _ = operators.gated_scan(v, v, out=v)
    assert torch.equal(h, operators.gated_scan(g, g)[0])
    q = flat.as_strided((2, 3, 2, 8), (far, 16, 8, 1))
    c = torch.randn(2, 3, 2, 8, device="cuda").bfloat16()
    q.copy_(c)
    tab = cuda(oc.table(3, 8))
    y, _ = operators.head_rotate(q, c, tab, q_out=q)
    assert torch.equal(y, operators.head_rotate(c, c, tab)[0])


def test_empty_extents(device):
    def e(*shape):
        return torch.empty(*shape, device="cuda")

    assert operators.gated_scan(e(0, 5, 3), e(0, 5, 3))[1].shape == (0, 3)
    assert operators.gated_scan(e(2, 5, 0), e(2, 5, 0))[0].shape == (2, 5, 0)
    s = torch.randn(2, 3, device="cuda")
    assert torch.equal(operators.gated_scan(e(2, 0, 3), e(2, 0, 3), state=s)[1], s)
    assert torch.equal(operators.gated_scan_backward(e(2, 0, 3), e(2, 0, 3), e(2, 0, 3), e(2, 0, 3),
                                                     dfinal=s)[2], s)
    off = torch.zeros(3, dtype=torch.int32, device="cuda")
    assert torch.equal(operators.gated_scan(e(0, 3), e(0, 3), state=s, offsets=off)[1], s)
    tab = e(4, 8)
    got = operators.head_rotate_backward(*(e(1, 0, 2, 8),) * 4, tab)
    assert bool((got[2] == 0).all()) and bool((got[3] == 0).all())
    assert operators.head_rotate(e(0, 3, 2, 8), e(0, 3, 1, 8), tab)[0].shape == (0, 3, 2, 8)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    assert float(operators.policy_loss(e(0, 7), none, e(0), e(0), e(0)).loss) == 0
    got = operators.preference_loss(e(0, 7), none, off, e(0))
    assert bool((got.ratios == 0).all())
    within(got.loss, torch.tensor(np.log(2.0)), 2 * EPS, "an even pair")
    assert operators.token_logp(e(0, 7), none).shape == (0,)


def test_offsets_that_do_not_rise_stay_in_bounds(device):
    """Unspecified results, but no access outside the arrays: the guards around them stay."""
    torch.manual_seed(7)
    for bad in ([5, 2, 900, -7], [-100, 2000, 3, 3], [2 ** 31 - 1, -2 ** 31, 0, 5]):
        off = torch.tensor(bad, dtype=torch.int32, device="cuda")
        guard = torch.full((60, 8), SENTINEL, device="cuda")
        x = guard[20:40]
        operators.gated_scan(torch.rand(20, 8, device="cuda"), torch.rand(20, 8, device="cuda"),
                             offsets=off, out=x)
        operators.gated_scan_backward(*(torch.rand(20, 8, device="cuda"),) * 4, offsets=off, dgate=x)
        operators.preference_loss(torch.rand(20, 8, device="cuda"),
                                  torch.zeros(20, dtype=torch.int32, device="cuda"), off[:3],
                                  torch.zeros(20, device="cuda"), gradient=x)
        torch.cuda.synchronize()
        assert bool((guard[:20] == SENTINEL).all()) and bool((guard[40:] == SENTINEL).all())


def test_wrappers_refuse_what_does_not_fit(device):
    def r(*shape, dtype=torch.float32):
        return torch.zeros(*shape, device="cuda", dtype=dtype)

    x, off = r(2, 3, 4), torch.zeros(3, dtype=torch.int32, device="cuda")
    i32 = torch.int32
    refused = [
        lambda: operators.gated_scan(r(2, 3, 5), x), lambda: operators.gated_scan(x.bfloat16(), x),
        lambda: operators.gated_scan(x.half(), x.half()), lambda: operators.gated_scan(x, x, form="tanh"),
        lambda: operators.gated_scan(x, x, state=r(3, 4)), lambda: operators.gated_scan(x, x, offsets=off),
        lambda: operators.gated_scan(r(6, 4), r(6, 4)),
        lambda: operators.gated_scan(r(6, 4), r(6, 4), offsets=off.long()),
        lambda: operators.gated_scan(x.cpu(), x), lambda: operators.gated_scan(x, x, state=r(2, 4).double()),
        lambda: operators.gated_scan(x, r(2, 4, 3).transpose(1, 2)),
        lambda: operators.gated_scan(x, x, out=r(2, 1, 4).expand(2, 3, 4)),
        lambda: operators.head_rotate(r(1, 2, 3, 8), r(1, 2, 1, 6), r(4, 8)),
        lambda: operators.head_rotate(r(1, 2, 3, 7), r(1, 2, 1, 7), r(4, 6)),
        lambda: operators.head_rotate(r(1, 2, 3, 8), r(1, 2, 1, 8), r(4, 10)),
        lambda: operators.head_rotate(r(1, 2, 3, 8), r(1, 2, 1, 8), r(4, 8), r(1, 3, dtype=i32)),
        lambda: operators.head_rotate(r(1, 2, 3, 8), r(1, 2, 1, 8), r(4, 8), r(1, 2)),
        lambda: operators.head_rotate(r(1, 2, 3, 8), r(1, 2, 1, 8), r(4, 8), style="both"),
        lambda: operators.head_rotate(r(1, 2, 3, 8), r(1, 2, 1, 8), r(4, 8), q_weight=r(4)),
        lambda: operators.token_logp(r(3, 4), r(3)), lambda: operators.token_logp(r(3, 4), r(2, dtype=i32)),
        lambda: operators.token_logp(r(3, 4), None),
        lambda: operators.policy_loss(r(3, 4), r(3, dtype=i32), r(3), r(3), r(3), kl=0.1),
        lambda: operators.policy_loss(r(3, 4), r(3, dtype=i32), r(3), r(3), r(3), gradient=r(3, 5)),
        lambda: operators.policy_loss(r(3, 4), r(3, dtype=i32), r(3), r(3), r(3), scale=-1.0),
        lambda: operators.preference_loss(r(3, 4), r(3, dtype=i32), r(2, dtype=i32), r(3)),
        lambda: operators.preference_loss(r(3, 4), r(3, dtype=i32), r(3, dtype=i32), r(3), beta=-1.0),
    ]
    for n, call in enumerate(refused):
        with pytest.raises((ValueError, BackendError)) as error:
            call()
        assert not isinstance(error.value, BackendError) or error.value.code == 6, n


# ------------------------------------------------- larger extents, other paths
LONG = [(1, 3000, 64), (2, 2500, 34), (1, 20000, 3), (48, 700, 130), (160, 260, 40), (300, 40, 33),
        (1, 700, 4099), (3, 2049, 67)]


@pytest.mark.parametrize("dtype,form", [("f32", "direct"), ("bf16", "sigmoid")])
@pytest.mark.parametrize("size", LONG)
def test_scan_over_long_and_wide_arrays(device, dtype, form, size):
    batch, length, channels = size
    t, k = TYPES[dtype], PER_STEP[form]
    gate, x, state = scan_inputs(201, form, dtype, *size)
    h, final, m, fm = oc.scan(form, gate, x, state)
    got, got_final = operators.gated_scan(cuda(gate, t), cuda(x, t), form=form, state=cuda(state))
    n = steps_of(batch, length)
    within(got, h, (k * n + k) * EPS * m + half_step(t) * h.abs(), "h")
    within(got_final, final, (k * length + k) * EPS * fm, "final state")
    # the entry state's own array as the final one, however the time axis is cut
    s = cuda(state)
    operators.gated_scan(cuda(gate, t), cuda(x, t), form=form, state=s, final_state=s)
    within(s, final, (k * length + k) * EPS * fm, "carried state")
    h = h.to(t).double()
    dh = normal(203, *size).to(t).double()
    expected, sizes = oc.scan_backward(form, dh, gate, x, h, state, state)
    got = operators.gated_scan_backward(cuda(dh, t), cuda(gate, t), cuda(x, t), cuda(h, t), form=form,
                                        state=cuda(state), dfinal=cuda(state))
    for name, a, e, m, half in zip(("dgate", "dx", "dstate"), got, expected, sizes,
                                   (half_step(t), half_step(t), 0.0)):
        within(a, e, (k * length + 3 * k) * EPS * m + half * e.abs(), name)


@pytest.mark.parametrize("dtype,form", [("f32", "sigmoid"), ("bf16", "direct")])
@pytest.mark.parametrize("length,channels,count", [(5000, 72, 40), (5000, 3, 700), (700, 8200, 9),
                                                   (2049, 330, 300), (900, 66, 900)])
def test_long_packed_batches_keep_sequences_apart(device, dtype, form, length, channels, count):
    t, k = TYPES[dtype], PER_STEP[form]
    cuts = torch.randint(0, length + 1, (count - 1,), generator=torch.Generator().manual_seed(7))
    offsets = [0] + sorted(cuts.tolist()) + [length]
    gate, x, state = scan_inputs(211, form, dtype, 1, length, channels, count)
    # what overflows or is undefined in one sequence stays there
    ill = [i for i in range(count) if offsets[i + 1] > offsets[i]][1::5]
    sane = torch.ones(length, dtype=torch.bool)
    for i in ill:
        x[0, offsets[i]] = float("inf") if i % 2 else float("nan")
        sane[offsets[i]:offsets[i + 1]] = False
    well = torch.tensor([i not in ill for i in range(count)])
    h, final, m, fm = oc.scan(form, gate, x, state, offsets)
    off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    got, got_final = operators.gated_scan(cuda(gate[0], t), cuda(x[0], t), form=form,
                                          state=cuda(state), offsets=off)
    n = steps_of(1, length, offsets)[0]
    tol = (k * n + k) * EPS * m[0] + half_step(t) * h[0].abs()
    within(got[sane.cuda()], h[0, sane], tol[sane], "h")
    within(got_final[well.cuda()], final[well], ((k * length + k) * EPS * fm)[well], "final state")
    for i in ill:
        assert not bool(got[offsets[i]].isfinite().any())
    h = torch.where(sane[None, :, None], h, torch.zeros_like(h)).to(t).double()
    dh = normal(213, 1, length, channels).to(t).double()
    for i in ill:
        dh[0, offsets[i + 1] - 1] = float("nan")
    dfinal = normal(214, count, channels).float().double()
    expected, sizes = oc.scan_backward(form, dh, gate, x, h, state, dfinal, offsets)
    got = operators.gated_scan_backward(cuda(dh[0], t), cuda(gate[0], t), cuda(x[0], t),
                                        cuda(h[0], t), form=form, state=cuda(state), offsets=off,
                                        dfinal=cuda(dfinal))
    for name, a, e, m in zip(("dgate", "dx"), got, expected, sizes):
        within(a[sane.cuda()], e[0, sane], (k * length + 3 * k) * EPS * m[0, sane]
               + half_step(t) * e[0, sane].abs(), name)
    within(got[2][well.cuda()], expected[2][well], ((k * length + 3 * k) * EPS * sizes[2])[well], "dstate")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [1027, 2048, 4101, 20011])
def test_targets_at_every_place_of_a_row(device, dtype, vocab):
    """The first and last elements, which lie before and behind the vectors of a row, and some vectors
    in between, with rows that start at every place of 16 bytes."""
    t = TYPES[dtype]
    places = list(range(20)) + list(range(vocab - 20, vocab)) + list(range(500, 1000, 31))
    rows = len(places)
    logits, _ = loss_inputs(221, dtype, rows, vocab)
    targets = torch.tensor(places)
    old, ref, advantages, weights = policy_inputs(222, logits, targets, 1.0)
    args = (cuda(targets, torch.int32), cuda(old), cuda(advantages), cuda(weights))
    for shift in range(0, 8 if dtype == "bf16" else 4, 3):
        z = torch.empty(rows * vocab + shift, dtype=t, device="cuda")[shift:].view(rows, vocab)
        z.copy_(logits)
        for into in (True, z):
            got = operators.policy_loss(z, *args, clip_low=0.2, clip_high=0.25, gradient=into)
            check_policy(logits, targets, old, advantages, weights, ref, 0, 1.0, t, got)
    z = cuda(logits, t)
    off = torch.tensor([0, rows // 2, rows], dtype=torch.int32, device="cuda")
    got = operators.preference_loss(z, args[0], off, cuda(ref), beta=0.3)
    total, ratios, logp, grad, slope = oc.preference(logits, targets, off.tolist(), ref, 0.3, 0.0,
                                                     torch.ones(1, dtype=torch.float64), 1.0)
    bar, sum_bar = logp_bar(logits, targets, 1.0)
    p = oc.rows(logits, targets, 1.0)[1]
    off_by = torch.full((rows,), 0.3 * float((bar + EPS * (logp.abs() + 1)).sum()), dtype=torch.float64)
    within(got.gradient, grad, gradient_bar(logits, p, slope.abs(), off_by, 1.0, sum_bar, t, grad), "gradient")


@pytest.mark.parametrize("dtype,vocab", [("f32", 60007), ("f32", 130003), ("f32", 500009),
                                         ("bf16", 60007), ("bf16", 130003), ("bf16", 500009)])
def test_losses_over_large_vocabularies(device, dtype, vocab):
    t, rows = TYPES[dtype], 6
    logits, targets = loss_inputs(231, dtype, rows, vocab)
    targets[1], targets[2] = 0, vocab - 1
    old, ref, advantages, weights = policy_inputs(232, logits, targets, 1.0)
    weights[3] = 0.0
    logits[4] = -float("inf")
    args = (cuda(targets, torch.int32), cuda(old), cuda(advantages), cuda(weights))
    keep = torch.tensor([0, 1, 2, 3, 5])
    z = cuda(logits, t)
    got = operators.policy_loss(z, *args, clip_low=0.2, clip_high=0.25)
    assert float(got.logp[4]) == 0 and bool((got.gradient[4] == 0).all())
    sub = [v[keep] for v in (logits, targets, old, advantages, weights, ref)]
    part = got._replace(token_loss=got.token_loss[keep.cuda()], logp=got.logp[keep.cuda()],
                        gradient=got.gradient[keep.cuda()])
    check_policy(*sub, 0, 1.0, t, part)
    over = operators.policy_loss(z, *args, clip_low=0.2, clip_high=0.25, gradient=z)
    assert torch.equal(over.gradient, got.gradient)


def test_many_pairs(device):
    rows, vocab, pairs = 3000, 40, 400
    logits, targets = loss_inputs(241, "f32", rows, vocab)
    cuts = torch.randint(0, rows + 1, (2 * pairs - 1,), generator=torch.Generator().manual_seed(3))
    offsets = [0] + sorted(cuts.tolist()) + [rows]
    ref = (oc.rows(logits, targets, 1.0)[0] + 0.2 * normal(242, rows)).float().double()
    w = torch.full((pairs,), 1 / pairs, dtype=torch.float64)
    total, ratios, logp, grad, slope = oc.preference(logits, targets, offsets, ref, 0.1, 0.0, w, 1.0)
    got = operators.preference_loss(cuda(logits), cuda(targets, torch.int32),
                                    torch.tensor(offsets, dtype=torch.int32, device="cuda"), cuda(ref))
    bar, sum_bar = logp_bar(logits, targets, 1.0)
    each = bar + EPS * (logp.abs() + 1)
    cut = torch.stack([each[lo:hi].sum() for lo, hi in zip(offsets[:-1], offsets[1:])])
    within(got.ratios, ratios, cut + EPS * ratios.abs(), "ratios")
    within(got.loss, total, 0.1 * cut.sum() / pairs + 8 * EPS * total.abs(), "loss")
    p = oc.rows(logits, targets, 1.0)[1]
    off_by = torch.full((rows,), 0.1 * float(cut.max()) / pairs * 2 + EPS, dtype=torch.float64)
    within(got.gradient, grad, gradient_bar(logits, p, slope.abs(), off_by, 1.0, sum_bar,
                                            torch.float32, grad), "gradient")


def test_rotate_over_many_tokens(device):
    """Warps that take several tokens, weight gradients summed over blocks."""
    q, k, wq, wk, _, _ = rotate_inputs(251, "bf16", 3, 1500, 5, 2, 64, 64)
    table = oc.table(2000, 64)
    positions = torch.randint(0, 2000, (3, 1500), generator=torch.Generator().manual_seed(5))
    t = torch.bfloat16
    named = dict(q_weight=cuda(wq), k_weight=cuda(wk))
    pos = cuda(positions, torch.int32)
    got = operators.head_rotate(cuda(q, t), cuda(k, t), cuda(table), pos, **named)
    dq, dk = (normal(255 + i, *v.shape).to(t).double() for i, v in enumerate((q, k)))
    back = operators.head_rotate_backward(cuda(dq, t), cuda(dk, t), cuda(q, t), cuda(k, t),
                                          cuda(table), pos, **named)
    for i, (x, w, dy) in enumerate(((q, wq, dq), (k, wk, dk))):
        e = oc.rotate(x, w, table.double(), positions, 1e-5, "halves")
        within(got[i], e, rotate_bar(x, w, e, t), "rotate")
        dx, dw, size_w = oc.rotate_backward(dy, x, w, table.double(), positions, 1e-5, "halves")
        heads = x.shape[0] * x.shape[1] * x.shape[2]
        big = float(oc.turn(dy, table.double(), positions, "halves", True).abs().amax())
        # a lane adds heads / (8 * 148) terms, then 3 shuffles, 8 warps and 37 + 8 blocks
        within(back[2 + i], dw, EPS * ((heads / 1000 + 80) * size_w + 8 * heads * big), "weight gradient")
        r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-5)
        dn = oc.turn(dy, table.double(), positions, "halves", True) * w
        inner = (dn * x * r).abs().mean(-1, keepdim=True)
        bar = 192 * EPS * r * (dn.abs().amax(-1, keepdim=True) + (x * r).abs().amax(-1, keepdim=True) * inner)
        within(back[i], dx, bar + half_step(t) * dx.abs(), "dx")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [500, 4000, 15001])
def test_long_answers_add_up_no_error_of_one_sign(vocab, dtype):
    rows, t = 8192, TYPES[dtype]
    z = (2 * torch.randn(rows, vocab, generator=torch.Generator().manual_seed(vocab))).to(t)
    at = torch.multinomial(torch.softmax(z.float(), -1), 1, generator=torch.Generator().manual_seed(1))
    exact = (z.double().gather(1, at) - torch.logsumexp(z.double(), -1, keepdim=True))[:, 0]
    ref = (exact - 0.1).float()
    got = operators.preference_loss(cuda(z, t), cuda(at[:, 0], torch.int32),
                                    torch.tensor([0, rows, rows], dtype=torch.int32, device="cuda"),
                                    cuda(ref))
    # A row's roundings (its terms' arguments and sum, its top's term, the rest of the logarithm, the
    # difference from the reference) go either way and come to 1.5e-7 at most, so their mean over the
    # rows has a deviation of at most 1.5e-7 / sqrt(8192) = 1.7e-9; six of those.  The fast exponential
    # is low by 5e-8 on average, and that must not be left.
    ratio = float((exact - ref.double()).sum())
    within(got.ratios.flatten()[:1], torch.tensor([ratio]), 1e-8 * rows + EPS / 2 * abs(ratio), "log ratio")


@pytest.mark.parametrize("vocab", [40, 5000])
@pytest.mark.parametrize("scale", [1.0, 0.3])
@pytest.mark.parametrize("middle", [1453635.0, -1453635.0, 4845450.0, 1e30, -3e38])
def test_log_probabilities_of_large_logits(middle, scale, vocab):
    # tops on both sides of where k top passes 2^21, and far past it, within a row
    z = (middle + 6 * torch.randn(9, vocab, generator=torch.Generator().manual_seed(vocab))).float()
    z[3] = torch.finfo(torch.float32).min
    at = torch.arange(9) % vocab
    exact = torch.log_softmax(z.double() * scale, -1).gather(1, at[:, None])[:, 0]
    got = operators.token_logp(cuda(z), cuda(at, torch.int32), scale=scale)
    # each term is off by 2 + 1.2 |x| steps, |x| below 40 where it counts, and so is the factor that
    # carries it over where that is rounded, up to 12 times; k by half a step of the differences
    within(got, exact, EPS * (50 * 13 + 2 * exact.abs()), "log probability")
