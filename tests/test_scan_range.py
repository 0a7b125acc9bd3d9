"""The gated scan where products of direct gates leave the range of 32 bits and the recurrence does not."""
import pytest
import torch

import operator_cases as oc
from operator_cases import EPS, TYPES, half_step, normal
from poorgrad_b200 import operators
from test_operators import cuda, steps_of, within

pytestmark = pytest.mark.gpu

# short; a block a column; clusters, with pairs of channels and single ones; the time axis in parts
SIZES = [(3, 12, 10), (300, 300, 64), (8, 500, 200), (5, 400, 33), (1, 1024, 64), (1, 6000, 66), (2, 5000, 35)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("gate", [2.0, -1e30])
def test_nothing_carried_stays_nothing(device, dtype, size, gate):
    t = TYPES[dtype]
    x = torch.zeros(size, dtype=t, device="cuda")
    x[:, -1] = 1.0
    gates = torch.full_like(x, gate)
    h, final = operators.gated_scan(gates, x, form="direct")
    assert torch.equal(h, x) and bool((final == 1).all())
    dh = x.flip(1)
    dgate, dx, dstate = operators.gated_scan_backward(dh, gates, None, torch.ones_like(x), form="direct")
    assert torch.equal(dx, dh) and bool((dgate == 0).all())
    assert bool((dstate == gates[:, 0].float()).all())


def waves(length):
    """Powers of two whose products grow to 2^200, then fall and rise again by 2^100."""
    steps = torch.tensor([4.0] * 50 + ([-4.0] * 25 + [4.0] * 25) * (length // 50 + 1))[:length]
    return torch.exp2(steps)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", SIZES)
def test_a_small_value_is_carried_through_large_products(device, dtype, size):
    """Every product is a power of two, so any order of work gives the same value."""
    batch, length, channels = size
    t = TYPES[dtype]
    factor = waves(length)
    gates = factor[None, :, None].expand(size).to(t).cuda().contiguous()
    x = torch.zeros_like(gates)
    state = torch.full((batch, channels), 2.0 ** -120, device="cuda")
    state[:, 1::3] = 0.0
    expected = 2.0 ** -120 * torch.exp2(torch.cumsum(torch.log2(factor.double()), 0))
    h, final = operators.gated_scan(gates, x, form="direct", state=state)
    for c, each in ((0, expected), (1, torch.zeros_like(expected)), (channels - 1, None)):
        if each is None:
            each = torch.zeros_like(expected) if (channels - 1) % 3 == 1 else expected
        assert torch.equal(h[:, :, c].double().cpu(), each[None].expand(batch, -1))
        assert bool((final[:, c].double().cpu() == each[-1]).all())
    dfinal = state
    dgate, dx, dstate = operators.gated_scan_backward(
        torch.zeros_like(gates), gates.flip(1).contiguous(), None, torch.ones_like(gates), form="direct",
        dfinal=dfinal)
    # g_t is dfinal times the gates behind t, and dstate times all of them
    each = torch.cat([torch.tensor([2.0 ** -120]).double(), expected]).flip(0)
    assert torch.equal(dx[:, :, 0].double().cpu(), each[None, 1:].expand(batch, -1))
    assert bool((dstate[:, 0].double().cpu() == each[0]).all()) and bool((dstate[:, 1] == 0).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [(8, 2000, 72), (1, 2000, 66), (2, 2100, 35)])
@pytest.mark.parametrize("packed", [False, True])
def test_growing_gates_follow_the_recurrence(device, dtype, size, packed):
    """Gates about 1.1 for thousands of steps, after a long start of zeros; what is not finite stays in
    its channel."""
    batch, length, channels = size
    t = TYPES[dtype]
    if packed:
        batch, offsets = 1, [0, 3, 3, 1500, length]
    else:
        offsets = None
    count = batch if offsets is None else 4
    size = (batch, length, channels)
    gate = (1.1 + 0.05 * normal(1, *size)).to(t).double()
    x = normal(2, *size)
    x[:, :1200] = 0.0
    x = (x * 1e-28).to(t).double()
    state = torch.zeros(count, channels, dtype=torch.float64)
    state[:, 5] = 2.0 ** -140  # below the range of normal numbers
    gate[:, 40, 7], gate[:, 50, 8], gate[:, 60, 9] = float("nan"), float("inf"), 0.0
    h, final, m, fm = oc.scan("direct", gate, x, state, offsets)
    off = None if offsets is None else torch.tensor(offsets, dtype=torch.int32, device="cuda")
    given = [cuda(v if offsets is None else v[0], t) for v in (gate, x)]
    got, got_final = operators.gated_scan(*given, form="direct", state=cuda(state), offsets=off)
    got = got.reshape(size)
    n = steps_of(batch, length, offsets)
    assert bool(h[:, 1400].isnan().sum(-1).eq(2).all()), "the two channels that are not finite"
    keep = torch.ones(channels, dtype=torch.bool)
    keep[5] = False  # its first products are too small for a relative bar
    # two roundings a step, twice over (a map and the walk), relative to the sums of magnitudes; what
    # falls below 2^-126 has half of 2^-149
    floor = 2.0 ** -149 * m / m.clamp(min=1e-300) * 1.2 ** n.clamp(max=400)
    tol = (4 * n + 4) * EPS * m + half_step(t) * h.abs() + floor
    within(got[..., keep], h[..., keep], tol[..., keep], "h")
    within(got_final[:, keep], final[:, keep], ((4 * length + 4) * EPS * fm)[:, keep] + 1e-40, "final state")
    # channel 5 grows by some 1.1^1990 = 2^274, past 2^128 near its end: finite where 32 bits hold it
    assert bool(got[..., 5].isfinite().cpu()[h[..., 5] < 1e38].all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("length,channels", [(700, 20000), (900, 8200), (1500, 72), (1500, 35), (40000, 64)])
def test_many_growing_sequences_with_a_carry_in_place(device, dtype, length, channels):
    """Sequences that begin and end within one round of work, whose final states take the entry states'
    places; products of gates pass 2^128 within a sequence, where 0 is carried, and across borders."""
    t = TYPES[dtype]
    lengths, g = [], torch.Generator().manual_seed(1)
    while sum(lengths) < length:
        lengths.append(300 if len(lengths) % 9 == 4 else int(torch.randint(0, 56, (1,), generator=g)))
    lengths[-1] -= sum(lengths) - length
    offsets = torch.tensor([0] + lengths).cumsum(0)
    first = torch.exp2(-100.0 - torch.arange(len(lengths)) % 20)
    first[torch.tensor(lengths) >= 60] = 0.0
    state = first[:, None].expand(-1, channels).contiguous().cuda()
    gates = torch.full((length, channels), 16.0, dtype=t, device="cuda")
    gates[:, 1::2] = -16.0
    x = torch.zeros_like(gates)
    h, final = operators.gated_scan(gates, x, form="direct", state=state, final_state=state,
                                    offsets=offsets.int().cuda())
    assert final is state
    row = torch.arange(length)
    s = torch.searchsorted(offsets, row, right=True) - 1
    steps = (row - offsets[s] + 1).double()
    expected = torch.where(first[s] == 0, 0.0, first[s].double() * torch.exp2(4 * steps))
    sign = 1 - 2 * (steps % 2)
    assert torch.equal(h[:, 0].double().cpu(), expected) and torch.equal(h[:, 1].double().cpu(), expected * sign)
    assert torch.equal(h[:, 0::2], h[:, :1].expand(-1, (channels + 1) // 2))
    assert torch.equal(h[:, 1::2], h[:, 1:2].expand(-1, channels // 2))
    n = torch.tensor(lengths).double()
    ends = torch.where(first == 0, 0.0, first.double() * torch.exp2(4 * n))
    assert torch.equal(final[:, 0].double().cpu(), ends)
    assert torch.equal(final[:, channels - 1], final[:, (channels - 1) % 2])
