"""Cases of the device operators around a decoder's matrix products, each in its plain form
(elementary torch operations in 32 bits) and through the framework's entry points:

- ``scan``: the gated linear recurrence h_t = a_t h_{t-1} + b_t over long, batched or packed
  sequences, its backward pass and its one-token step;
- ``rotate``: the root-mean-square norm of every query and key head with the position rotation,
  forward and backward;
- ``policy``: the clipped policy loss with a KL term over a vocabulary, with its gradient;
- ``preference``: the paired log-ratio loss over packed answers, with its gradient.
"""
import math
import random

import numpy as np
import torch

own = False

_EPSILON = 1e-6
_CLIP = 0.2
_BETA = 0.1
_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


# ------------------------------------------------------------------ cases
def _scan_case(direction, dtype, form, batch, length, channels, sequences=0):
    return {"op": "scan", "direction": direction, "dtype": dtype, "form": form, "batch": batch,
            "length": length, "channels": channels, "sequences": sequences}


def _rotate_case(direction, dtype, batch, length, q_heads, k_heads, dim, turned, style, first):
    return {"op": "rotate", "direction": direction, "dtype": dtype, "batch": batch,
            "length": length, "q_heads": q_heads, "k_heads": k_heads, "dim": dim,
            "turned": turned, "style": style, "first": first}


def _policy_case(dtype, rows, vocab, kl, masked, gradient=True):
    return {"op": "policy", "dtype": dtype, "rows": rows, "vocab": vocab, "kl": kl,
            "masked": masked, "gradient": gradient}


def _preference_case(dtype, rows, vocab, pairs, masked):
    return {"op": "preference", "dtype": dtype, "rows": rows, "vocab": vocab, "pairs": pairs,
            "masked": masked}


def listed():
    return [
        # one decoded token for each of 64 requests: latency
        {"name": "scan-step-bf16", **_scan_case("forward", "bf16", "sigmoid", 64, 1, 768)},
        # a long packed batch of ragged documents, one stream of tokens and few channels
        {"name": "scan-forward-bf16-packed",
         **_scan_case("forward", "bf16", "direct", 1, 131072, 768, 37)},
        # training at the decoder's width, 8 sequences of 1024 tokens
        {"name": "scan-backward-bf16", **_scan_case("backward", "bf16", "sigmoid", 8, 1024, 768)},
        # odd extents, rows that are not 16-byte multiples
        {"name": "scan-backward-f32-odd",
         **_scan_case("backward", "f32", "direct", 3, 2049, 1001)},
        # one decoded token for each of 64 requests, far positions, shared key heads
        {"name": "rotate-decode-bf16",
         **_rotate_case("forward", "bf16", 64, 1, 12, 4, 64, 64, "halves", 100000)},
        # prefill or training of a wide decoder with shared key heads
        {"name": "rotate-forward-bf16",
         **_rotate_case("forward", "bf16", 8, 1024, 32, 8, 128, 128, "halves", 0)},
        {"name": "rotate-backward-bf16",
         **_rotate_case("backward", "bf16", 8, 1024, 32, 8, 128, 128, "halves", 0)},
        # the f32 training path at 12 heads of 64, half of each head turned in adjacent pairs
        {"name": "rotate-backward-f32",
         **_rotate_case("backward", "f32", 8, 1024, 12, 12, 64, 32, "pairs", 0)},
        # a character model's vocabulary
        {"name": "policy-f32-characters", **_policy_case("f32", 16384, 27, 0.04, 0.25)},
        # a whole batch of 8 x 1024 tokens over a byte-pair vocabulary: the largest
        {"name": "policy-f32-50257", **_policy_case("f32", 8192, 50257, 0.04, 0.25)},
        # short answers over a small vocabulary
        {"name": "preference-f32-small", **_preference_case("f32", 1000, 512, 6, 0.3)},
        # 8 pairs of answers, prompts masked
        {"name": "preference-bf16-50257", **_preference_case("bf16", 4099, 50257, 8, 0.3)},
    ]


def _spread(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def _elements(case):
    if case["op"] == "scan":
        return case["batch"] * case["length"] * case["channels"]
    if case["op"] == "rotate":
        heads = case["q_heads"] + case["k_heads"]
        return case["batch"] * case["length"] * heads * case["dim"]
    return case["rows"] * case["vocab"]


def _one(rng):
    dtype = rng.choice(["f32", "bf16"])
    op = rng.choice(["scan", "rotate", "policy", "preference"])
    if op == "scan":
        direction = rng.choice(["forward", "backward"])
        form = rng.choice(["direct", "sigmoid"])
        channels = _spread(rng, 1, 4096)
        if rng.random() < 0.5:  # whole 16-byte rows
            channels = -(-channels // 8) * 8
        if rng.random() < 0.4:
            return _scan_case(direction, dtype, form, 1, _spread(rng, 16, 131072), channels,
                              _spread(rng, 1, 200))
        return _scan_case(direction, dtype, form, _spread(rng, 1, 64), _spread(rng, 1, 16384),
                          channels)
    if op == "rotate":
        dim = rng.choice([32, 64, 80, 96, 128, 192, 256, 34])
        turned = rng.choice([dim, dim, dim // 2 // 2 * 2])
        k_heads = _spread(rng, 1, 16)
        return _rotate_case(rng.choice(["forward", "backward"]), dtype, _spread(rng, 1, 64),
                            _spread(rng, 1, 8192), k_heads * _spread(rng, 1, 8), k_heads, dim,
                            turned, rng.choice(["halves", "pairs"]), rng.choice([0, 5000, 100000]))
    rows, vocab = _spread(rng, 1, 16384), _spread(rng, 2, 130000)
    masked = rng.choice([0.0, 0.25, 0.5])
    if op == "policy":
        return _policy_case(dtype, rows, vocab, rng.choice([0.0, 0.04]), masked,
                            rng.random() < 0.8)
    pairs = _spread(rng, 1, 64)
    return _preference_case(dtype, max(rows, 4 * pairs), vocab, pairs, masked)


def draw(rng):
    while True:
        case = _one(rng)
        # no dearer than the largest listed case, in the bytes and in the elements of its kind
        most = {"scan": 110_000_000, "rotate": 45_000_000, "policy": 400_000_000,
                "preference": 220_000_000}[case["op"]]
        if _elements(case) <= most:
            return case


# ----------------------------------------------------------------- inputs
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 2 + 1)
    return g


def _offsets(seed, rows, sequences, least=0):
    """Ragged lengths that fill `rows`, at least `least` each."""
    r = np.random.RandomState(seed % (1 << 31))
    cuts = np.sort(r.randint(0, rows - least * sequences + 1, sequences - 1))
    ends = np.concatenate([cuts + least * np.arange(1, sequences), [rows]])
    return np.concatenate([[0], ends]).astype(np.int32)


def _prepare_scan(case, seed):
    g, t = _generator(seed), _TYPES[case["dtype"]]
    shape = (case["batch"], case["length"], case["channels"])
    packed = case["sequences"] > 0
    count = case["sequences"] if packed else case["batch"]

    def normal(*size):
        return torch.randn(*size, generator=g, device="cuda")

    gate = normal(*shape) + 2.0  # gates near one, as after training
    if case["form"] == "direct":
        gate = torch.sigmoid(gate)
    s = {"gate": gate.to(t), "x": normal(*shape).to(t),
         "state": normal(count, case["channels"]), "offsets": None}
    if packed:
        s["offsets"] = torch.from_numpy(_offsets(seed, case["length"], count)).cuda()
    if case["direction"] == "backward":
        # the saved outputs have the size of a convex mix of the inputs
        s["h"] = (0.5 * normal(*shape)).to(t)
        s["dh"] = normal(*shape).to(t)
        s["dfinal"] = normal(count, case["channels"])
    if packed:
        for name in ("gate", "x", "h", "dh"):
            if name in s:
                s[name] = s[name][0]
    return s


def _prepare_rotate(case, seed):
    g, t = _generator(seed), _TYPES[case["dtype"]]
    batch, length, hq, hk, d = (case[n] for n in ("batch", "length", "q_heads", "k_heads", "dim"))
    half = case["turned"] // 2
    # the projection's output [tokens, q | k | v]: queries and keys are strided views of it
    rows = torch.randn(batch, length, (hq + 2 * hk) * d, generator=g, device="cuda").to(t)
    s = {"q": rows[..., :hq * d].unflatten(-1, (hq, d)),
         "k": rows[..., hq * d:(hq + hk) * d].unflatten(-1, (hk, d)),
         "wq": 1 + 0.1 * torch.randn(d, generator=g, device="cuda"),
         "wk": 1 + 0.1 * torch.randn(d, generator=g, device="cuda")}
    # cos and sin of the positions first .. first + span, kept by the program
    span = length + 512
    angles = (torch.arange(case["first"], case["first"] + span, dtype=torch.float64)[:, None]
              * 10000.0 ** (-torch.arange(half, dtype=torch.float64) / max(half, 1))[None, :])
    s["table"] = torch.cat([angles.cos(), angles.sin()], 1).float().cuda()
    start = torch.randint(0, span - length, (batch, 1), generator=g, device="cuda")
    s["positions"] = (start + torch.arange(length, device="cuda")).to(torch.int32)
    if case["direction"] == "backward":
        s["dq"] = torch.randn(batch, length, hq, d, generator=g, device="cuda").to(t)
        s["dk"] = torch.randn(batch, length, hk, d, generator=g, device="cuda").to(t)
    return s


def _logits(case, seed):
    g = _generator(seed)
    n, v = case["rows"], case["vocab"]
    logits = torch.empty(n, v, dtype=_TYPES[case["dtype"]], device="cuda")
    logits.normal_(0.0, 2.0, generator=g)
    targets = torch.randint(0, v, (n,), generator=g, device="cuda").to(torch.int32)
    at = targets.long()[:, None]
    # a sampled token is a likely one
    logits.scatter_(1, at, (logits.gather(1, at).float() + 4.0).to(logits.dtype))
    # the target's log probability; what other models gave it is near to it
    step = max(1, 60_000_000 // v)
    lse = torch.cat([torch.logsumexp(logits[i:i + step].float(), 1) for i in range(0, n, step)])
    logp = logits.gather(1, at)[:, 0].float() - lse
    hidden = torch.rand(n, generator=g, device="cuda").argsort()[:int(round(case["masked"] * n))]
    return g, logits, targets, logp, hidden


def _prepare_policy(case, seed):
    g, logits, targets, logp, hidden = _logits(case, seed)
    n = case["rows"]
    noise = 0.3 * torch.randn(2, n, generator=g, device="cuda")
    # no ratio so near to a clipping border that the last bits of a log probability decide
    for border in (math.log(1 - _CLIP), math.log(1 + _CLIP)):
        noise[0] = torch.where((noise[0] + border).abs() < 1e-4, 0.0, noise[0])
    weights = torch.full((n,), 1.0 / max(1, n - len(hidden)), device="cuda")
    weights[hidden] = 0.0
    return {"logits": logits, "targets": targets, "old": logp + noise[0],
            "ref": logp + noise[1] if case["kl"] else None,
            "advantages": torch.randn(n, generator=g, device="cuda") + 0.25, "weights": weights}


def _prepare_preference(case, seed):
    g, logits, targets, logp, hidden = _logits(case, seed)
    targets[hidden] = -1  # the prompts' tokens
    # the answers have become likelier than they were to the reference model
    noise = 0.2 * torch.randn(case["rows"], generator=g, device="cuda")
    return {"logits": logits, "targets": targets, "ref": logp - 0.2 + noise,
            "offsets": torch.from_numpy(
                _offsets(seed, case["rows"], 2 * case["pairs"], 1)).cuda()}


def prepare(case, seed):
    made = {"scan": _prepare_scan, "rotate": _prepare_rotate, "policy": _prepare_policy,
            "preference": _prepare_preference}[case["op"]](case, seed)
    made["case"] = case
    return made


# ------------------------------------------------------------ plain forms
def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t along axis 1, h_{-1} = 0: pairs of steps, then the steps between."""
    length = a.shape[1]
    if length == 1:
        return b
    pairs = length // 2
    first_a, second_a = a[:, 0:2 * pairs:2], a[:, 1:2 * pairs:2]
    seconds = _scan(first_a * second_a, second_a * b[:, 0:2 * pairs:2] + b[:, 1:2 * pairs:2])
    h = torch.empty_like(b)
    h[:, 1:2 * pairs:2] = seconds
    h[:, 0] = b[:, 0]
    h[:, 2::2] = a[:, 2::2] * seconds[:, :(length - 1) // 2] + b[:, 2::2]
    return h


def _boundaries(s):
    """Where the packed sequences start, and which of them hold a token."""
    offsets = s["offsets"].long()
    filled = offsets[1:] > offsets[:-1]
    return offsets, filled


def _plain_scan_forward(s, case):
    gate, x = s["gate"].float(), s["x"].float()
    if s["offsets"] is not None:
        gate, x = gate[None], x[None]
    a = torch.sigmoid(gate) if case["form"] == "sigmoid" else gate
    b = torch.sigmoid(-gate) * x if case["form"] == "sigmoid" else x
    a, b = a.clone(), b.clone()
    if s["offsets"] is None:
        b[:, 0] += a[:, 0] * s["state"]
        a[:, 0] = 0
        h = _scan(a, b)
        return h.to(s["x"].dtype), h[:, -1].clone()
    offsets, filled = _boundaries(s)
    starts, ends = offsets[:-1][filled], offsets[1:][filled] - 1
    b[0, starts] += a[0, starts] * s["state"][filled]
    a[0, starts] = 0
    h = _scan(a, b)
    final = s["state"].clone()
    final[filled] = h[0, ends]
    return h[0].to(s["x"].dtype), final


def _plain_scan_backward(s, case):
    gate, x, h, dh = (s[n].float() for n in ("gate", "x", "h", "dh"))
    if s["offsets"] is not None:
        gate, x, h, dh = gate[None], x[None], h[None], dh[None]
    a = torch.sigmoid(gate) if case["form"] == "sigmoid" else gate
    later, before, dh = torch.zeros_like(a), torch.zeros_like(h), dh.clone()
    later[:, :-1] = a[:, 1:]
    before[:, 1:] = h[:, :-1]
    if s["offsets"] is None:
        before[:, 0] = s["state"]
        dh[:, -1] += s["dfinal"]
    else:
        offsets, filled = _boundaries(s)
        starts, ends = offsets[:-1][filled], offsets[1:][filled] - 1
        later[0, ends] = 0
        before[0, starts] = s["state"][filled]
        dh[0, ends] += s["dfinal"][filled]
    g = _scan(later.flip(1), dh.flip(1)).flip(1)
    if case["form"] == "sigmoid":
        b = torch.sigmoid(-gate)
        dgate, dx = g * (before - x) * a * b, g * b
    else:
        dgate, dx = g * before, g
    if s["offsets"] is None:
        return dgate.to(s["gate"].dtype), dx.to(s["x"].dtype), a[:, 0] * g[:, 0]
    dstate = s["dfinal"].clone()
    dstate[filled] = a[0, starts] * g[0, starts]
    return dgate[0].to(s["gate"].dtype), dx[0].to(s["x"].dtype), dstate


def _turn(z, table, positions, style, back):
    half = table.shape[1] // 2
    rows = table[positions.long()][..., None, :]
    cos, sin = rows[..., :half], rows[..., half:]
    sin = -sin if back else sin
    out = z.clone()
    if style == "halves":
        u, v = z[..., :half], z[..., half:2 * half]
        out[..., :half] = u * cos - v * sin
        out[..., half:2 * half] = v * cos + u * sin
    else:
        u, v = z[..., 0:2 * half:2], z[..., 1:2 * half:2]
        out[..., 0:2 * half:2] = u * cos - v * sin
        out[..., 1:2 * half:2] = v * cos + u * sin
    return out


def _plain_rotate_forward(s, case):
    def one(x, w):
        x32 = x.float()
        n = x32 * torch.rsqrt((x32 * x32).mean(-1, keepdim=True) + _EPSILON)
        return _turn(n * w, s["table"], s["positions"], case["style"], False).to(x.dtype)
    return one(s["q"], s["wq"]), one(s["k"], s["wk"])


def _plain_rotate_backward(s, case):
    def one(x, w, dy):
        x32 = x.float()
        r = torch.rsqrt((x32 * x32).mean(-1, keepdim=True) + _EPSILON)
        n = x32 * r
        dz = _turn(dy.float(), s["table"], s["positions"], case["style"], True)
        dw = (dz * n).sum((0, 1, 2))
        dn = dz * w
        return (r * (dn - n * (dn * n).mean(-1, keepdim=True))).to(x.dtype), dw
    dq, dwq = one(s["q"], s["wq"], s["dq"])
    dk, dwk = one(s["k"], s["wk"], s["dk"])
    return dq, dk, dwq, dwk


def _rows_of(logits, targets):
    """Log probabilities of the targets and the softmax of each row, in 32 bits."""
    z = logits.float()
    z = z - z.amax(1, keepdim=True)
    e = torch.exp(z)
    total = e.sum(1, keepdim=True)
    at = targets.long().clamp(min=0)[:, None]
    logp = (z.gather(1, at) - torch.log(total))[:, 0]
    return logp, e / total, at


def _gradient(p, at, coefficient, dtype):
    d = p * -coefficient[:, None]
    d.scatter_add_(1, at, coefficient[:, None])
    return d.to(dtype)


def _plain_policy(s, case):
    live = s["weights"] != 0
    logp, p, at = _rows_of(s["logits"], s["targets"])
    logp = torch.where(live, logp, torch.zeros_like(logp))
    ratio = torch.exp(logp - s["old"])
    plain, held = ratio * s["advantages"], ratio.clamp(1 - _CLIP, 1 + _CLIP) * s["advantages"]
    loss = -torch.minimum(plain, held)
    slope = torch.where(plain <= held, -plain, torch.zeros_like(plain))
    if case["kl"]:
        d = s["ref"] - logp
        loss = loss + case["kl"] * (torch.expm1(d) - d)
        slope = slope - case["kl"] * torch.expm1(d)
    token_loss = torch.where(live, s["weights"] * loss, torch.zeros_like(loss))
    slope = torch.where(live, s["weights"] * slope, torch.zeros_like(slope))
    total = token_loss.sum(dtype=torch.float64).float()
    if not case["gradient"]:
        return total, token_loss, logp
    return total, token_loss, logp, _gradient(p, at, slope, s["logits"].dtype)


def _plain_preference(s, case):
    live = s["targets"] >= 0
    logp, p, at = _rows_of(s["logits"], s["targets"])
    logp = torch.where(live, logp, torch.zeros_like(logp))
    offsets = s["offsets"].long()
    count = offsets[1:] - offsets[:-1]
    sequence = torch.repeat_interleave(torch.arange(len(count), device="cuda"), count,
                                       output_size=case["rows"])
    # sums over whole answers: the margin is a small difference of large sums
    step = torch.where(live, logp.double() - s["ref"].double(), torch.zeros_like(logp).double())
    ratios = torch.zeros(len(count), dtype=torch.float64, device="cuda").index_add_(0, sequence, step)
    pairs = case["pairs"]
    margin = _BETA * (ratios[:pairs] - ratios[pairs:])
    loss = torch.log1p(torch.exp(-margin.abs())) + (-margin).clamp(min=0)
    slope = -_BETA * torch.sigmoid(-margin) / pairs
    slope = torch.cat([slope, -slope])[sequence].float()
    slope = torch.where(live, slope, torch.zeros_like(slope))
    return (loss.sum() / pairs).float(), ratios.float(), logp, _gradient(
        p, at, slope, s["logits"].dtype)


# -------------------------------------------------------------------- run
def run(s):
    case = s["case"]
    op = case["op"]
    if own:
        from poorgrad_b200 import operators
        if op == "scan":
            if case["direction"] == "forward":
                return operators.gated_scan(s["gate"], s["x"], form=case["form"],
                                            state=s["state"], offsets=s["offsets"])
            return operators.gated_scan_backward(s["dh"], s["gate"], s["x"], s["h"],
                                                 form=case["form"], state=s["state"],
                                                 offsets=s["offsets"], dfinal=s["dfinal"])
        if op == "rotate":
            named = {"q_weight": s["wq"], "k_weight": s["wk"], "epsilon": _EPSILON,
                     "style": case["style"]}
            if case["direction"] == "forward":
                return operators.head_rotate(s["q"], s["k"], s["table"], s["positions"], **named)
            return operators.head_rotate_backward(s["dq"], s["dk"], s["q"], s["k"], s["table"],
                                                  s["positions"], **named)
        if op == "policy":
            r = operators.policy_loss(s["logits"], s["targets"], s["old"], s["advantages"],
                                      s["weights"], ref_logp=s["ref"], kl=case["kl"],
                                      clip_low=_CLIP, clip_high=_CLIP,
                                      gradient=case["gradient"])
            if not case["gradient"]:
                return r.loss, r.token_loss, r.logp
            return r.loss, r.token_loss, r.logp, r.gradient
        r = operators.preference_loss(s["logits"], s["targets"], s["offsets"], s["ref"],
                                      beta=_BETA)
        return r.loss, r.ratios, r.logp, r.gradient
    if op == "scan":
        return (_plain_scan_forward if case["direction"] == "forward"
                else _plain_scan_backward)(s, case)
    if op == "rotate":
        return (_plain_rotate_forward if case["direction"] == "forward"
                else _plain_rotate_backward)(s, case)
    return (_plain_policy if op == "policy" else _plain_preference)(s, case)


# ------------------------------------------------------------------- work
def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    n = _elements(case)
    if case["op"] == "scan":
        states = (case["sequences"] or case["batch"]) * case["channels"] * 4
        if case["direction"] == "forward":
            return {"bytes": 3 * n * size + 2 * states, "flops": 2 * n}
        arrays = 6 if case["form"] == "sigmoid" else 5
        return {"bytes": arrays * n * size + 3 * states, "flops": 4 * n}
    if case["op"] == "rotate":
        tokens = case["batch"] * case["length"]
        table = min(tokens, case["length"] + 512) * case["turned"] * 4
        if case["direction"] == "forward":
            return {"bytes": 2 * n * size + table + 4 * tokens, "flops": 7 * n}
        return {"bytes": 3 * n * size + table + 4 * tokens, "flops": 14 * n}
    # masked rows are written as zeros and need not be read
    read = case["rows"] - int(round(case["masked"] * case["rows"]))
    written = case["rows"] if case.get("gradient", True) else 0
    return {"bytes": (read + written) * case["vocab"] * size + 24 * case["rows"],
            "flops": 6 * read * case["vocab"]}


# ------------------------------------------------------------------ exact
def _exact_scan(case, s):
    gate, x = s["gate"].double(), s["x"].double()
    packed = s["offsets"] is not None
    if packed:
        gate, x = gate[None], x[None]
    a = 1 / (1 + torch.exp(-gate)) if case["form"] == "sigmoid" else gate
    b = x / (1 + torch.exp(gate)) if case["form"] == "sigmoid" else x
    length = x.shape[1]
    state = s["state"].double()
    bounds = s["offsets"].tolist() if packed else [0, length]
    spans = [(i, lo, hi) for i, (lo, hi) in enumerate(zip(bounds[:-1], bounds[1:])) if hi > lo]
    rows = (lambda v, i: v[i:i + 1]) if packed else (lambda v, i: v)
    if case["direction"] == "forward":
        out, final = torch.empty_like(x), state.clone()
        for i, lo, hi in spans:
            h = rows(state, i).clone()
            for t in range(lo, hi):
                h = torch.addcmul(b[:, t], a[:, t], h)
                out[:, t] = h
            rows(final, i).copy_(h)
        return (out[0] if packed else out), final
    h, dh, dfinal = s["h"].double(), s["dh"].double(), s["dfinal"].double()
    if packed:
        h, dh = h[None], dh[None]
    carried, dstate = torch.empty_like(x), dfinal.clone()
    previous = torch.empty_like(h)
    for i, lo, hi in spans:
        carry = rows(dfinal, i)
        for t in range(hi - 1, lo - 1, -1):
            g = dh[:, t] + carry
            carried[:, t] = g
            carry = a[:, t] * g
        rows(dstate, i).copy_(carry)
        previous[:, lo] = rows(state, i)
        previous[:, lo + 1:hi] = h[:, lo:hi - 1]
    if case["form"] == "sigmoid":
        dgate, dx = carried * (previous - x) * a * (1 - a), carried * (1 - a)
    else:
        dgate, dx = carried * previous, carried
    return (dgate[0], dx[0], dstate) if packed else (dgate, dx, dstate)


def _exact_rotate(case, s):
    """The rotation as a product of complex numbers; the gradient of the norm by its Jacobian."""
    half = case["turned"] // 2
    rows = s["table"].double()[s["positions"].long()][:, :, None, :]
    unit = torch.complex(rows[..., :half], rows[..., half:])

    def turned(z, by):
        head = z[..., :2 * half]
        if case["style"] == "halves":
            c = torch.complex(head[..., :half], head[..., half:]) * by
            head = torch.cat([c.real, c.imag], -1)
        else:
            c = torch.view_as_complex(head.unflatten(-1, (half, 2)).contiguous()) * by
            head = torch.view_as_real(c).flatten(-2)
        return torch.cat([head, z[..., 2 * half:]], -1)

    def forward(x, w):
        x = x.double()
        return turned(x / (x.square().mean(-1, keepdim=True) + _EPSILON).sqrt() * w.double(), unit)

    def backward(x, w, dy):
        x, w = x.double(), w.double()
        root = (x.square().mean(-1, keepdim=True) + _EPSILON).sqrt()
        dz = turned(dy.double(), unit.conj())
        inner = (dz * w * x).mean(-1, keepdim=True)
        return dz * w / root - x * inner / root ** 3, (dz * x / root).flatten(0, 2).sum(0)

    if case["direction"] == "forward":
        return forward(s["q"], s["wq"]), forward(s["k"], s["wk"])
    dq, dwq = backward(s["q"], s["wq"], s["dq"])
    dk, dwk = backward(s["k"], s["wk"], s["dk"])
    return dq, dk, dwq, dwk


def _exact_logp(s, live):
    """Log probabilities in 64 bits, a few rows at a time."""
    n, step = len(s["targets"]), max(1, 60_000_000 // s["logits"].shape[1])
    parts = []
    for i in range(0, n, step):
        z = s["logits"][i:i + step].double()
        at = s["targets"][i:i + step].long().clamp(min=0)[:, None]
        parts.append(z.gather(1, at)[:, 0] - torch.logsumexp(z, 1))
    return torch.cat(parts) * live


def _exact_gradient(s, coefficient):
    n, step = len(s["targets"]), max(1, 60_000_000 // s["logits"].shape[1])
    full = torch.empty(s["logits"].shape, dtype=torch.float64, device="cuda")
    for i in range(0, n, step):
        c = coefficient[i:i + step]
        part = torch.softmax(s["logits"][i:i + step].double(), 1).mul_(-c[:, None])
        at = s["targets"][i:i + step].long().clamp(min=0)
        part[torch.arange(len(c), device="cuda"), at] += c
        full[i:i + step] = part
    return full


def _exact_policy(case, s):
    w = s["weights"].double()
    logp = _exact_logp(s, (w != 0).double())
    advantages = s["advantages"].double()
    ratio = (logp - s["old"].double()).exp()
    low, high = 1 - _CLIP, 1 + _CLIP
    cut = ((advantages > 0) & (ratio > high)) | ((advantages < 0) & (ratio < low))
    loss = -torch.where(cut, ratio.clamp(low, high), ratio) * advantages
    slope = torch.where(cut, 0.0, -ratio * advantages)
    if case["kl"]:
        d = s["ref"].double() - logp
        loss = loss + case["kl"] * (d.exp() - 1 - d)
        slope = slope + case["kl"] * (1 - d.exp())
    token_loss = w * loss
    if not case["gradient"]:
        return token_loss.sum(), token_loss, logp
    return token_loss.sum(), token_loss, logp, _exact_gradient(s, w * slope)


def _exact_preference(case, s):
    live = (s["targets"] >= 0).double()
    logp = _exact_logp(s, live)
    bounds = s["offsets"].tolist()
    step = (logp - s["ref"].double()) * live
    ratios = torch.stack([step[lo:hi].sum() for lo, hi in zip(bounds[:-1], bounds[1:])])
    pairs = case["pairs"]
    margin = _BETA * (ratios[:pairs] - ratios[pairs:])
    slope = torch.zeros(case["rows"], dtype=torch.float64, device="cuda")
    pull = -_BETA / (1 + margin.exp()) / pairs
    for i in range(pairs):
        slope[bounds[i]:bounds[i + 1]] = pull[i]
        slope[bounds[pairs + i]:bounds[pairs + i + 1]] = -pull[i]
    loss = -torch.nn.functional.logsigmoid(margin).mean()
    return loss, ratios, logp, _exact_gradient(s, slope * live)


def exact(case, seed):
    s = prepare(case, seed)
    return {"scan": _exact_scan, "rotate": _exact_rotate, "policy": _exact_policy,
            "preference": _exact_preference}[case["op"]](case, s)
