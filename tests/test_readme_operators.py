"""The device operators' example in the README, run as it stands."""
import os
import re

import pytest
import torch

import operator_cases as oc
from operator_cases import EPS, normal
from test_operators import cuda, within

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_the_example_computes_the_gradients(device):
    text = open(os.path.join(ROOT, "README.md")).read()
    code = re.search(r"## Device operators\n+```python\n(.*?)```", text, re.S).group(1)
    rows, heads, shared, dim, channels, vocab = 20, 3, 2, 128, 6, 50
    offsets = [0, 1, 8, rows]
    v = dict(q_in=normal(1, rows, heads, dim), k_in=normal(2, rows, shared, dim), dq=normal(3, rows, heads, dim),
             dk=normal(4, rows, shared, dim), wq=1 + 0.1 * normal(5, dim), wk=1 + 0.1 * normal(6, dim),
             gate=normal(7, rows, channels), x=normal(8, rows, channels), dh=normal(9, rows, channels),
             state=normal(10, 3, channels), dfinal=normal(11, 3, channels), logits=normal(12, rows, vocab),
             old_logp=normal(13, rows) - 4, ref_logp=normal(14, rows) - 4, advantages=normal(15, rows),
             weights=torch.full((rows,), 1 / rows))
    v = {k: t.float().double() for k, t in v.items()}
    positions = torch.arange(rows)
    at = torch.randint(0, vocab, (rows,), generator=torch.Generator().manual_seed(1))
    space = {k: cuda(t) for k, t in v.items()}
    space.update(positions=cuda(positions, torch.int32), tokens=cuda(at, torch.int32),
                 offsets=torch.tensor(offsets, dtype=torch.int32, device="cuda"),
                 answers=torch.tensor([0, 9, rows], dtype=torch.int32, device="cuda"))
    exec(code, space)
    for name in ("gate", "x", "state"):  # what the backward pass reads is what the scan read
        assert torch.equal(space[name].double().cpu(), v[name]), name

    h, final, m, fm = oc.scan("sigmoid", v["gate"][None], v["x"][None], v["state"], offsets)
    within(space["h"], h[0], 20 * (rows + 1) * EPS * m[0] + EPS * h[0].abs(), "h")
    within(space["final"], final, 20 * (rows + 1) * EPS * fm, "final state")
    grads, sizes = oc.scan_backward("sigmoid", v["dh"][None], v["gate"][None], v["x"][None], h, v["state"],
                                    v["dfinal"], offsets)
    for name, e, size in zip(("dgate", "dx", "dstate"), grads, sizes):
        # h enters dgate with its own error besides, as many steps of a magnitude within size
        within(space[name], e.reshape(space[name].shape),
               60 * (rows + 3) * EPS * (size.reshape(space[name].shape) + m.max() * float(sizes[1].max())), name)
    table = space["table"].double().cpu()
    for side, weight in (("q", "wq"), ("k", "wk")):
        args = (v[side + "_in"][None], v[weight], table, positions[None], 1e-5, "halves")
        e = oc.rotate(*args)
        within(space[side], e[0], 48 * EPS * 2 * e.abs().max(), side)
        dx, dw, _ = oc.rotate_backward(v["d" + side][None], *args)
        within(space["d%s_in" % side], dx[0], 400 * EPS * dx.abs().max(), "d" + side)
        within(space["dw" + side], dw, 400 * EPS * dw.abs().max() * 4, "dw" + side)
    total, ratios, _, grad, _ = oc.preference(v["logits"], at, [0, 9, rows], v["ref_logp"], 0.1, 0.0,
                                              torch.ones(1, dtype=torch.float64), 1.0)
    r = space["r"]
    assert r.gradient is space["logits"]
    within(r.gradient, grad, 400 * EPS, "preference gradient")
    within(r.ratios, ratios, rows * 200 * EPS, "ratios")
