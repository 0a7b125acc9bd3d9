"""The gated scan against its definition in 64 bits within bounds that the recurrence itself carries on: an
error shrinks with the gates behind it, so that a long array has no wider bound than a short one."""
import pytest
import torch

import operator_cases as oc
from operator_cases import EPS, TYPES, half_step, normal
from poorgrad_b200 import operators
from test_operators import cuda, scan_inputs, within

pytestmark = pytest.mark.gpu

# Half steps of f32 (EPS / 2) that a step adds to its output, relative to the sum of magnitudes there: the fused
# product and sum once; in a map the same again, and the product of gates (the walk of a map adds the two);
# the sigmoid form its a and 1 - a besides, whose exponential is off by 2 + 1.2 |gate| steps for gates below
# 10, by 14 steps, the sum and the reciprocal by 1 and 2, a product by half a step.
PER_STEP = {"direct": 4 * EPS / 2, "sigmoid": (4 + 2 * 2 * 17.5) * EPS / 2}


def walk(a, m, e, first):
    """Bounds e_t = |a_t| e_{t-1} + k m_t over the rows of one sequence."""
    out = torch.zeros_like(m)
    for t in range(len(m)):
        first = a[t].abs() * first + e * m[t]
        out[t] = first
    return out, first


def bounds(form, gate, x, m, fm, offsets, back=False, sizes=None):
    a, _ = oc.gates(form, gate, x)
    k = PER_STEP[form]
    out, last = torch.zeros_like(m), torch.zeros_like(fm)
    for s, row, lo, hi in oc.spans_of(offsets, *m.shape[:2]):
        zero = torch.zeros_like(fm[s])
        if back:  # the carried value is a_t g_t: its error passes through the gate of its own step
            first = zero
            for t in range(hi - 1, lo - 1, -1):
                out[row, t] = first + k * m[row, t]
                first = a[row, t].abs() * (out[row, t] + k * m[row, t])
            last[s] = first
        else:
            out[row, lo:hi], last[s] = walk(a[row, lo:hi], m[row, lo:hi], k, zero)
    return out, last


SIZES = [(1, 20000, 3), (2, 2500, 34), (1, 3000, 64), (48, 700, 130), (8, 1024, 72), (300, 40, 33)]
CASES = [(size, False) for size in SIZES] + [((1, *size[1:]), True) for size in SIZES[:3]]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("form", ["direct", "sigmoid"])
@pytest.mark.parametrize("size,packed", CASES)
def test_errors_shrink_with_the_gates(device, dtype, form, size, packed):
    t = TYPES[dtype]
    batch, length, channels = size
    offsets, count = None, batch
    if packed:
        count = 60
        cuts = torch.randint(0, length + 1, (count - 1,), generator=torch.Generator().manual_seed(3))
        offsets = [0] + sorted(cuts.tolist()) + [length]
    gate, x, state = scan_inputs(301, form, dtype, batch, length, channels, count)
    gate = gate.clamp(-10, 10).to(t).double()
    off = None if offsets is None else torch.tensor(offsets, dtype=torch.int32, device="cuda")

    def given(v, kind=t):
        return cuda(v if offsets is None else v[0], kind)

    h, final, m, fm = oc.scan(form, gate, x, state, offsets)
    bar, last = bounds(form, gate, x, m, fm, offsets)
    got, got_final = operators.gated_scan(given(gate), given(x), form=form, state=cuda(state), offsets=off)
    got = got.reshape(h.shape)
    within(got, h, bar + half_step(t) * (h.abs() + bar), "h")
    within(got_final, final, last + EPS / 2 * fm, "final state")

    h = h.to(t).double()
    dh = normal(305, batch, length, channels).to(t).double()
    dfinal = normal(306, count, channels).float().double()
    expected, sizes = oc.scan_backward(form, dh, gate, x, h, state, dfinal, offsets)
    got = operators.gated_scan_backward(given(dh), given(gate), given(x), given(h), form=form, state=cuda(state),
                                        offsets=off, dfinal=cuda(dfinal))
    # g's own bound, from the magnitudes behind g (those of dx divided by the form's 1 - a)
    a, _ = oc.gates(form, gate, x)
    b = torch.ones_like(a) if form == "direct" else torch.sigmoid(-gate)
    g_bar, first = bounds(form, gate, x, sizes[1] / b, fm, offsets, back=True)
    k = PER_STEP[form]
    # dgate = g times what the step's gate weighs (sizes[0] / sizes[1] b is its magnitude): g's error times it, and
    # a few more products of the step's own
    weight = (sizes[0] / sizes[1] * b).nan_to_num()
    for name, v, e, bound in (("dgate", got[0], expected[0], g_bar * weight + 2 * k * sizes[0]),
                              ("dx", got[1], expected[1], g_bar * b + 2 * k * sizes[1])):
        v = v.reshape(e.shape)
        within(v, e, bound + half_step(t) * (e.abs() + bound), name)
    within(got[2], expected[2], first + EPS / 2 * sizes[2], "dstate")
