"""References in 64 bits and inputs for the tests of the device operators.

Each reference follows the operator's definition step by step on the CPU, apart from the kernels'
order of work, and returns next to each result the magnitude that its rounding errors scale with."""
import numpy as np
import torch

EPS = float(np.finfo(np.float32).eps)
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def half_step(t):
    """The largest relative error of one rounding to type t."""
    return torch.finfo(t).eps / 2


def normal(seed, *shape):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g, dtype=torch.float64)


def spans_of(offsets, batch, length):
    """(state row, batch row, first, last) of every sequence."""
    if offsets is None:
        return [(b, b, 0, length) for b in range(batch)]
    return [(s, 0, lo, hi) for s, (lo, hi) in enumerate(zip(offsets[:-1], offsets[1:]))]


def gates(form, gate, x):
    if form == "direct":
        return gate, x
    a = torch.sigmoid(gate)
    return a, torch.sigmoid(-gate) * x


def scan(form, gate, x, state, offsets=None):
    """h, final state, and the sums of magnitudes behind each (the recurrence on |a|, |b|)."""
    a, b = gates(form, gate, x)
    h, size = torch.zeros_like(x), torch.zeros_like(x)
    final, final_size = state.clone(), state.abs()
    for s, row, lo, hi in spans_of(offsets, *x.shape[:2]):
        v, m = state[s], state[s].abs()
        for t in range(lo, hi):
            v, m = a[row, t] * v + b[row, t], a[row, t].abs() * m + b[row, t].abs()
            h[row, t], size[row, t] = v, m
        final[s], final_size[s] = v, m
    return h, final, size, final_size


def scan_backward(form, dh, gate, x, h, state, dfinal, offsets=None):
    a, _ = gates(form, gate, x)
    g, size = torch.zeros_like(h), torch.zeros_like(h)
    before = torch.zeros_like(h)
    dstate, dstate_size = dfinal.clone(), dfinal.abs()
    for s, row, lo, hi in spans_of(offsets, *h.shape[:2]):
        carry, m = dfinal[s], dfinal[s].abs()
        for t in range(hi - 1, lo - 1, -1):
            g[row, t], size[row, t] = dh[row, t] + carry, dh[row, t].abs() + m
            carry, m = a[row, t] * g[row, t], a[row, t].abs() * size[row, t]
            before[row, t] = h[row, t - 1] if t > lo else state[s]
        dstate[s], dstate_size[s] = carry, m
    if form == "direct":
        return (g * before, g, dstate), (size * before.abs(), size, dstate_size)
    b = 1 - a
    return ((g * (before - x) * a * b, g * b, dstate),
            (size * (before.abs() + x.abs()) * a * b, size * b, dstate_size))


def turn(z, table, positions, style, back=False):
    half = table.shape[1] // 2
    cos = table[positions][:, :, None, :half]
    sin = table[positions][:, :, None, half:] * (-1 if back else 1)
    out = z.clone()
    for i in range(half):
        u, v = (i, i + half) if style == "halves" else (2 * i, 2 * i + 1)
        out[..., u] = z[..., u] * cos[..., i] - z[..., v] * sin[..., i]
        out[..., v] = z[..., v] * cos[..., i] + z[..., u] * sin[..., i]
    return out


def rotate(x, w, table, positions, epsilon, style):
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + epsilon) * w
    return turn(y, table, positions, style)


def rotate_backward(dy, x, w, table, positions, epsilon, style):
    """dx, dw and the sum of magnitudes behind dw."""
    r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + epsilon)
    dz = turn(dy, table, positions, style, back=True)
    n = x * r
    dn = dz * w
    dx = r * (dn - n * (dn * n).mean(-1, keepdim=True))
    return dx, (dz * n).sum((0, 1, 2)), (dz * n).abs().sum((0, 1, 2))


def table(rows, turned, first=0):
    from poorgrad_b200.operators import rotation_table
    return torch.from_numpy(rotation_table(rows, turned, first=first))


def rows(logits, targets, scale):
    """log probabilities, softmax, and whether the row counts (in 64 bits)."""
    z = scale * logits
    live = (targets >= 0) & (z > -np.inf).any(1) | torch.isnan(z).any(1) & (targets >= 0)
    safe = torch.where(live[:, None], z, torch.zeros_like(z))
    at = targets.long().clamp(0, logits.shape[1] - 1)
    lse = torch.logsumexp(safe, 1)
    logp = safe.gather(1, at[:, None])[:, 0] - lse
    logp = torch.where(targets >= logits.shape[1], torch.full_like(logp, float("nan")), logp)
    return torch.where(live, logp, torch.zeros_like(logp)), torch.softmax(safe, 1), live, at


def gradient(p, at, slope, scale, live):
    d = -p * (slope * scale)[:, None]
    d[torch.arange(len(at)), at] += slope * scale
    return torch.where(live[:, None], d, torch.zeros_like(d))


def policy(logits, targets, old, advantages, weights, ref, low, high, kl, scale):
    logp, p, live, at = rows(logits, targets, scale)
    live = live & (weights != 0)
    logp = torch.where(live, logp, torch.zeros_like(logp))
    r = torch.exp(logp - old)
    held = r.clamp(1 - low, 1 + high)
    loss, slope = -torch.minimum(r * advantages, held * advantages), -r * advantages
    slope = torch.where(r * advantages <= held * advantages, slope, torch.zeros_like(slope))
    slope = torch.where(torch.isnan(r), r, slope)
    if kl:
        d = ref - logp
        loss = loss + kl * (torch.expm1(d) - d)
        slope = slope + kl * -torch.expm1(d)
    zero = torch.zeros_like(loss)
    token = torch.where(live, weights * loss, zero)
    return token.sum(), token, logp, gradient(p, at, torch.where(live, weights * slope, zero),
                                              scale, live)


def preference(logits, targets, offsets, ref, beta, smoothing, weights, scale):
    logp, p, live, at = rows(logits, targets, scale)
    step = torch.where(live, logp - ref, torch.zeros_like(logp))
    ratios = torch.stack([step[lo:hi].sum() for lo, hi in zip(offsets[:-1], offsets[1:])])
    pairs = len(ratios) // 2
    m = beta * (ratios[:pairs] - ratios[pairs:])
    yes, no = torch.nn.functional.softplus(-m), torch.nn.functional.softplus(m)
    each = weights * ((1 - smoothing) * yes + (smoothing * no if smoothing else 0))
    pull = weights * beta * (smoothing * torch.sigmoid(m) - (1 - smoothing) * torch.sigmoid(-m))
    slope = torch.zeros_like(logp)
    for i in range(pairs):
        slope[offsets[i]:offsets[i + 1]] = pull[i]
        slope[offsets[pairs + i]:offsets[pairs + i + 1]] = -pull[i]
    return each.sum(), ratios, logp, gradient(p, at, slope, scale, live), slope
