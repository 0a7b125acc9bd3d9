"""Packed scans with more empty sequences than others."""
import time

import pytest
import torch

import operator_cases as oc
from operator_cases import EPS
from poorgrad_b200 import operators
from test_operators import cuda, steps_of, within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("carried", [False, True])
@pytest.mark.parametrize("channels", [3, 72, 20000])
def test_empty_sequences_hand_their_state_on(device, channels, carried):
    rows, count = 300, 2000 if channels < 1000 else 90
    g = torch.Generator().manual_seed(1)
    cuts = torch.sort(torch.randint(0, 12, (count - 1,), generator=g) * (rows // 12))[0]
    offsets = [0] + cuts.tolist() + [rows]
    gate, x = (oc.normal(i, 1, rows, channels).float().double() for i in range(2))
    state = oc.normal(3, count, channels).float().double()
    h, final, m, fm = oc.scan("sigmoid", gate, x, state, offsets)
    off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    s = cuda(state)
    got, last = operators.gated_scan(cuda(gate[0]), cuda(x[0]), state=s, offsets=off,
                                     final_state=s if carried else None)
    n = steps_of(1, rows, offsets)[0]
    within(got, h[0], 20 * (n + 1) * EPS * m[0] + EPS * h[0].abs(), "h")
    length = (off[1:] - off[:-1]).cpu()
    within(last, final, 20 * (length + 1.0)[:, None] * EPS * fm, "final state")
    empty = length == 0
    assert int(empty.sum()) > count / 2 and torch.equal(last.double().cpu()[empty], state[empty])
    d = operators.gated_scan_backward(cuda(x[0]), cuda(gate[0]), cuda(x[0]), got, offsets=off, dfinal=cuda(state))[2]
    assert torch.equal(d.double().cpu()[empty], state[empty])


@pytest.mark.parametrize("carried", [False, True])
def test_millions_of_empty_sequences_are_shared_out(device, carried):
    rows, count, channels = 4096, 4_000_000, 8
    off = torch.zeros(count + 1, dtype=torch.int32, device="cuda")
    off[count // 2:] = rows
    gate, x = (torch.randn(rows, channels, device="cuda") for _ in range(2))
    state = torch.randn(count, channels, device="cuda")

    def call():
        return operators.gated_scan(gate, x, offsets=off, state=state, final_state=state if carried else None)

    expected = state.clone()
    _, final = call()
    expected[count // 2 - 1] = final[count // 2 - 1]
    assert torch.equal(final, expected)
    torch.cuda.synchronize()
    since = time.perf_counter()
    call()
    torch.cuda.synchronize()
    # 256 MB read or written take 40 us; one by one, at two dependent reads each, they took 0.3 s and more
    assert time.perf_counter() - since < 0.05
