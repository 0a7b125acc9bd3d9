"""Python face of the device operators of ``include/topos_b200.h``: what lies around the matrix
products of a decoder's training and decode steps, on device arrays that the caller holds.

- :func:`gated_scan`, :func:`gated_scan_backward` -- the gated linear recurrence over time
- :func:`head_rotate`, :func:`head_rotate_backward` -- norms of query and key heads with the
  position rotation; :func:`rotation_table` makes its cosines and sines
- :func:`token_logp`, :func:`policy_loss`, :func:`preference_loss` -- losses over a vocabulary
  with their gradients by the logits

Device arrays are torch tensors (float32 or bfloat16), used as memory only: nothing here records
gradients.  Arguments of one call live on one device; the work is enqueued on that device's current
torch stream, and outputs that are not given are allocated by torch on that stream.  A malformed
request raises ``ValueError`` or :class:`~poorgrad_b200.backend.BackendError`; there is no CPU
fallback.
"""
from __future__ import annotations

import struct
from typing import NamedTuple, Optional

import numpy as np
import torch

from .abi import (TbPolicyDesc, TbPreferenceDesc, TbRotateDesc, TbScanDesc, load_library,
                  request_format)
from .backend import BackendError

_ELEMENT = {torch.float32: 0, torch.bfloat16: 1}
_FORM = {"direct": 0, "sigmoid": 1}
_STYLE = {"halves": 0, "pairs": 1}
_scan = struct.Struct(request_format(TbScanDesc)).pack
_rotate = struct.Struct(request_format(TbRotateDesc)).pack
_policy = struct.Struct(request_format(TbPolicyDesc)).pack
_preference = struct.Struct(request_format(TbPreferenceDesc)).pack


def _need(condition, what: str):
    if not condition:
        raise ValueError(what)


# The checks below build their messages only when they fail: a small call costs a few microseconds
# of host time, and its checks are most of them.
def _unfit(t, name: str, device, dtype, shape, more: str):
    got = (t.dtype, tuple(t.shape), t.stride(), t.device) if isinstance(t, torch.Tensor) else type(t)
    raise ValueError(f"{name}: expected {dtype} {tuple(shape)} on {device}, {more}; got {got}")


def _device_of(first, name: str):
    if not (isinstance(first, torch.Tensor) and first.is_cuda and first.dtype in _ELEMENT):
        raise ValueError(f"{name}: a float32 or bfloat16 CUDA tensor is expected")
    return first.device


def _array(t, name: str, device, dtype, shape):
    """(strides, address) of a large array of this type, device and shape whose last axis has
    stride 1."""
    if isinstance(t, torch.Tensor) and t.dtype is dtype and t.shape == shape and t.device == device:
        strides = t.stride()
        if strides[-1] == 1 or shape[-1] <= 1:
            return strides, t.data_ptr()
    _unfit(t, name, device, dtype, shape, "stride 1 along the last axis")


def _words(t, name: str, device, dtype, shape):
    """Address of a contiguous 32-bit array, or 0 for None."""
    if t is None:
        return 0
    if not (isinstance(t, torch.Tensor) and t.dtype is dtype and t.shape == shape
            and t.device == device and t.is_contiguous()):
        _unfit(t, name, device, dtype, shape, "contiguous")
    return t.data_ptr()


def _like(t):
    """A new dense array in the order of t's axes, the last one innermost."""
    made = torch.empty_like(t)
    return made if made.stride(-1) == 1 or t.shape[-1] <= 1 else t.new_empty(t.shape)


_entries: dict = {}
# the stream's handle without a Stream object around it, where this torch has that
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _entry(name: str):
    found = _entries.get(name)
    if found is None:
        found = _entries[name] = getattr(load_library(), name)
    return found


def _call(name: str, device, *arguments):
    entry = _entries.get(name) or _entry(name)
    index = device.index
    if index == torch.cuda.current_device():
        code = entry(*arguments, _raw_stream(index))
    else:  # the entry points launch on the current device
        with torch.cuda.device(device):
            code = entry(*arguments, _raw_stream(index))
    if code != 0:
        raise BackendError(code, name)


# ------------------------------------------------------------------ gated scan
def _scan_extents(x, offsets):
    """(batch, length, channels, sequences, rows of the states)."""
    if offsets is None:
        _need(x.dim() == 3, "x: expected [batch, length, channels], or packed [rows, channels] "
                            "with offsets")
        batch, length, channels = x.shape
        return batch, length, channels, 0, batch
    _need(x.dim() == 2, "x: a packed batch is [rows, channels]")
    _need(isinstance(offsets, torch.Tensor) and offsets.dim() == 1 and offsets.shape[0] >= 2,
          "offsets: expected sequences + 1 row numbers")
    length, channels = x.shape
    return 1, length, channels, offsets.shape[0] - 1, offsets.shape[0] - 1


def _states(like, x, count, channels):
    """A new [count, channels] float32 array (a copy of `like`'s form is the quicker to make)."""
    if like is not None and like.shape == (count, channels) and like.dtype is torch.float32:
        return torch.empty_like(like, memory_format=torch.contiguous_format)
    return x.new_empty((count, channels), dtype=torch.float32)


def _scan_workspace(x, batch, length, channels):
    """(tensor, address, bytes) of the scratch that a long call is cut along time with."""
    size = _entry("tb_gated_scan_workspace")(batch, length, channels) if length >= 256 else 0
    if not size:
        return None, 0, 0
    workspace = x.new_empty((size,), dtype=torch.uint8)
    return workspace, workspace.data_ptr(), size


def gated_scan(gate, x, *, form: str = "sigmoid", state=None, offsets=None, out=None,
               final_state=None):
    """``h_t = a_t h_{t-1} + b_t`` over time; returns ``(h, final_state)``.

    ``form="direct"``: a is ``gate`` and b is ``x``.  ``form="sigmoid"``: a is the sigmoid of
    ``gate`` and b is ``(1 - a) x``.  ``gate`` and ``x`` are ``[batch, length, channels]``, or a
    packed ``[rows, channels]`` whose sequences ``offsets`` (int32, sequences + 1 rising row
    numbers) delimits; rows outside every sequence are left as they were.  ``state`` (float32,
    ``[batch or sequences, channels]``, zeros when None) comes before the first step; the returned
    final state may be written into ``state`` itself (``final_state=state``), as a decode loop
    does.  ``out`` may be ``gate`` or ``x``."""
    device = _device_of(x, "x")
    _need(form in _FORM, "form: 'direct' or 'sigmoid' is expected")
    batch, length, channels, sequences, count = _scan_extents(x, offsets)
    shape, dtype, states = x.shape, x.dtype, (count, channels)
    gate_s, gate_p = _array(gate, "gate", device, dtype, shape)
    x_s, x_p = _array(x, "x", device, dtype, shape)
    if out is None:
        out = _like(x)
    out_s, out_p = _array(out, "out", device, dtype, shape)
    state_p = _words(state, "state", device, torch.float32, states)
    if final_state is None:
        final_state = _states(state, x, count, channels)
        final_p = final_state.data_ptr()
    else:
        final_p = _words(final_state, "final_state", device, torch.float32, states)
    offsets_p = _words(offsets, "offsets", device, torch.int32, (sequences + 1,))
    if sequences:  # packed: no batch axis
        gate_s, x_s, out_s = (0, *gate_s), (0, *x_s), (0, *out_s)
    workspace, scratch, size = _scan_workspace(x, batch, length, channels)
    _call("tb_gated_scan", device,
          _scan(_ELEMENT[dtype], _FORM[form], batch, length, channels, sequences, gate_s[0],
                gate_s[1], x_s[0], x_s[1], out_s[0], out_s[1], 0, 0, 0, 0, 0, 0, gate_p, x_p, out_p,
                offsets_p, state_p, final_p, 0, 0, 0, 0, 0, scratch, size))
    return out, final_state


def gated_scan_backward(dh, gate, x, h, *, form: str = "sigmoid", state=None, offsets=None,
                        dfinal=None, dgate=None, dx=None):
    """Gradients ``(dgate, dx, dstate)`` of :func:`gated_scan` from the gradient ``dh`` of its
    outputs ``h`` and ``dfinal`` of its final state (zeros when None).  ``x`` is read by the
    sigmoid form only.  One of ``dgate`` and ``dx`` may be ``dh``."""
    device = _device_of(dh, "dh")
    _need(form in _FORM, "form: 'direct' or 'sigmoid' is expected")
    batch, length, channels, sequences, count = _scan_extents(dh, offsets)
    shape, dtype, states = dh.shape, dh.dtype, (count, channels)
    if dgate is None:
        dgate = _like(dh)
    if dx is None:
        dx = _like(dh)
    if form == "direct" and x is None:
        x = gate  # not read
    arrays = [_array(t, name, device, dtype, shape)
              for t, name in ((gate, "gate"), (x, "x"), (h, "h"), (dh, "dh"), (dgate, "dgate"),
                              (dx, "dx"))]
    state_p = _words(state, "state", device, torch.float32, states)
    dfinal_p = _words(dfinal, "dfinal", device, torch.float32, states)
    dstate = _states(state, dh, count, channels)
    offsets_p = _words(offsets, "offsets", device, torch.int32, (sequences + 1,))
    workspace, scratch, size = _scan_workspace(dh, batch, length, channels)
    strides = [n for s, _ in arrays for n in ((0, s[0]) if sequences else s[:2])]
    _call("tb_gated_scan_backward", device,
          _scan(_ELEMENT[dtype], _FORM[form], batch, length, channels, sequences, *strides,
                arrays[0][1], arrays[1][1], arrays[2][1], offsets_p, state_p, 0, arrays[3][1],
                dfinal_p, arrays[4][1], arrays[5][1], dstate.data_ptr(), scratch, size))
    return dgate, dx, dstate


# ----------------------------------------------------------------- head rotate
def rotation_table(rows: int, turned: int, base: float = 10000.0, first: int = 0) -> np.ndarray:
    """``[rows, turned]`` float32: cosines, then sines, of ``(first + row) * base^(-2i / turned)``
    for i below turned / 2, computed in 64 bits (a far position's angle needs them)."""
    _need(turned >= 0 and turned % 2 == 0, "turned is even and not negative")
    half = turned // 2
    angles = (np.arange(first, first + rows, dtype=np.float64)[:, None]
              * base ** (-np.arange(half, dtype=np.float64) / max(half, 1))[None, :])
    return np.concatenate([np.cos(angles), np.sin(angles)], axis=1).astype(np.float32)


def _heads(t):
    """A [tokens, heads, dim] array as one batch row."""
    return t.unsqueeze(0) if t.dim() == 3 else t


def _rotate_call(entry, device, q, k, table, positions, q_weight, k_weight, epsilon, style, q_out,
                 k_out, dq, dk, dq_weight, dk_weight, workspace, workspace_bytes):
    q_shape, dtype = q.shape, q.dtype
    batch, length, q_heads, dim = q_shape
    k_heads = k.shape[2]
    k_shape = (batch, length, k_heads, dim)
    f32 = torch.float32
    _need(isinstance(table, torch.Tensor) and table.dim() == 2,
          "table: expected [positions, turned]")
    _need(style in _STYLE, "style: 'halves' or 'pairs' is expected")
    (qb, qt, qh, _), q_p = _array(q, "q", device, dtype, q_shape)
    (kb, kt, kh, _), k_p = _array(k, "k", device, dtype, k_shape)
    (ob, ot, oh, _), o_p = _array(q_out, "q_out", device, dtype, q_shape)
    (pb, pt, ph, _), p_p = _array(k_out, "k_out", device, dtype, k_shape)
    gb = gt = gh = g_p = rb = rt = rh = r_p = 0
    if dq is not None:
        (gb, gt, gh, _), g_p = _array(dq, "dq", device, dtype, q_shape)
        (rb, rt, rh, _), r_p = _array(dk, "dk", device, dtype, k_shape)
    table_shape = table.shape
    _call(entry, device, _rotate(
        _ELEMENT[dtype], _STYLE[style], batch, length, q_heads, k_heads, dim, table_shape[1],
        table_shape[0], qb, qt, qh, kb, kt, kh, ob, ot, oh, pb, pt, ph, gb, gt, gh, rb, rt, rh,
        epsilon, q_p, k_p, _words(table, "table", device, f32, table_shape),
        _words(positions, "positions", device, torch.int32, (batch, length)),
        _words(q_weight, "q_weight", device, f32, (dim,)),
        _words(k_weight, "k_weight", device, f32, (dim,)), o_p, p_p, g_p, r_p, dq_weight, dk_weight,
        workspace, workspace_bytes))


def _rotate_inputs(q, k, positions):
    device = _device_of(q, "q")
    _need(q.dim() in (3, 4) and isinstance(k, torch.Tensor) and k.dim() == q.dim(),
          "q, k: expected [tokens, heads, dim] or [batch, length, heads, dim]")
    if q.dim() == 3 and isinstance(positions, torch.Tensor) and positions.dim() == 1:
        positions = positions.unsqueeze(0)
    return device, positions


def head_rotate(q, k, table, positions=None, *, q_weight=None, k_weight=None,
                epsilon: float = 1e-5, style: str = "halves", q_out=None, k_out=None):
    """Root-mean-square norm of every query and key head, then its rotation by the token's
    position; returns ``(q_out, k_out)``.

    ``q`` and ``k`` are ``[batch, length, heads, dim]`` or ``[tokens, heads, dim]`` with any strides
    but 1 along ``dim`` (views of a joint projection, outputs laid out for attention).  ``table``
    (float32 ``[positions, turned]``, :func:`rotation_table`) turns the first ``turned`` elements of
    each head: element i with i + turned/2 (``style="halves"``) or 2i with 2i + 1 (``"pairs"``).
    ``positions`` (int32, one per token; 0, 1, .. along the length when None) selects the rows; one
    outside the table makes the token's heads NaN.  Weights are float32 ``[dim]``, ones when None.
    The outputs may be the inputs."""
    device, positions = _rotate_inputs(q, k, positions)
    if q_out is None:
        q_out = _like(q)
    if k_out is None:
        k_out = _like(k)
    if q.dim() == 4:
        _rotate_call("tb_head_rotate", device, q, k, table, positions, q_weight, k_weight, epsilon,
                     style, q_out, k_out, None, None, 0, 0, 0, 0)
    else:
        _rotate_call("tb_head_rotate", device, _heads(q), _heads(k), table, positions, q_weight,
                     k_weight, epsilon, style, _heads(q_out), _heads(k_out), None, None, 0, 0, 0, 0)
    return q_out, k_out


def head_rotate_backward(dq, dk, q, k, table, positions=None, *, q_weight=None, k_weight=None,
                         epsilon: float = 1e-5, style: str = "halves", q_out=None, k_out=None,
                         weights: bool = True):
    """Gradients ``(q_grad, k_grad, q_weight_grad, k_weight_grad)`` of :func:`head_rotate` from the
    gradients ``dq`` and ``dk`` of its outputs; the last two are float32 ``[dim]``, or None with
    ``weights=False``.  ``q_out`` and ``k_out`` receive the first two and may be ``dq`` and ``dk``."""
    device, positions = _rotate_inputs(q, k, positions)
    _need(isinstance(dq, torch.Tensor) and isinstance(dk, torch.Tensor)
          and dq.dim() == dk.dim() == q.dim(), "dq, dk: expected the shapes of q and k")
    if q_out is None:
        q_out = _like(q)
    if k_out is None:
        k_out = _like(k)
    dq_weight = dk_weight = workspace = None
    given = (0, 0, 0, 0)
    if weights:
        dim = q.shape[-1]
        dq_weight = q.new_empty((dim,), dtype=torch.float32)
        dk_weight = torch.empty_like(dq_weight)
        size = _entry("tb_head_rotate_workspace")(dim)
        workspace = q.new_empty((size,), dtype=torch.uint8)
        given = dq_weight.data_ptr(), dk_weight.data_ptr(), workspace.data_ptr(), size
    _rotate_call("tb_head_rotate_backward", device, _heads(q), _heads(k), table, positions, q_weight,
                 k_weight, epsilon, style, _heads(q_out), _heads(k_out), _heads(dq), _heads(dk),
                 *given)
    return q_out, k_out, dq_weight, dk_weight


# ---------------------------------------------------------------------- losses
class PolicyLoss(NamedTuple):
    loss: torch.Tensor                  # scalar
    token_loss: torch.Tensor            # [rows], the weighted terms that loss sums
    logp: torch.Tensor                  # [rows]
    gradient: Optional[torch.Tensor]    # [rows, vocab]


class PreferenceLoss(NamedTuple):
    loss: torch.Tensor                  # scalar
    ratios: torch.Tensor                # [2 pairs], sum of logp - ref over each answer
    logp: torch.Tensor                  # [rows]
    gradient: Optional[torch.Tensor]    # [rows, vocab]


def _logits(logits):
    """(device, row stride, address)."""
    device = _device_of(logits, "logits")
    _need(logits.dim() == 2, "logits: expected [rows, vocab]")
    strides, address = _array(logits, "logits", device, logits.dtype, logits.shape)
    return device, strides[0], address


def _gradient_of(logits, gradient, device):
    """(tensor, row stride, address) of a gradient that is wanted (True), given, or neither."""
    if gradient is None or gradient is False:
        return None, 0, 0
    if gradient is True:
        gradient = _like(logits)
    strides, address = _array(gradient, "gradient", device, logits.dtype, logits.shape)
    return gradient, strides[0], address


def token_logp(logits, targets, *, scale: float = 1.0):
    """Float32 log probabilities of ``targets`` (int32 ``[rows]``) under ``softmax(scale * logits)``
    of each row.  A hidden row -- a negative target, or no logit above -inf -- gives 0, a target
    beyond the vocabulary NaN."""
    device, row, pointer = _logits(logits)
    rows, vocab = logits.shape
    _need(targets is not None, "targets: missing")
    logp = logits.new_empty((rows,), dtype=torch.float32)
    _call("tb_token_logp", device, _ELEMENT[logits.dtype], pointer, row,
          _words(targets, "targets", device, torch.int32, (rows,)), rows, vocab, scale,
          logp.data_ptr())
    return logp


def policy_loss(logits, targets, old_logp, advantages, weights, *, ref_logp=None,
                clip_low: float = 0.2, clip_high: float = 0.2, kl: float = 0.0,
                scale: float = 1.0, gradient=True) -> PolicyLoss:
    """Clipped policy loss over sampled tokens, with its gradient by the logits.

    With ``r = exp(logp - old_logp)`` and ``d = ref_logp - logp``, the loss is the sum over rows of
    ``weight * (-min(r A, clamp(r, 1 - clip_low, 1 + clip_high) A) + kl (exp(d) - d - 1))``; the
    weights hold the normalizer (1 / tokens, say) and hide a row where they are 0.  A hidden row,
    also one as in :func:`token_logp`, adds nothing whatever it holds and has a gradient of 0.
    ``gradient`` is True, False, or the array to write, which may be ``logits`` itself."""
    device, row, pointer = _logits(logits)
    rows, vocab = logits.shape
    _need(targets is not None and old_logp is not None and advantages is not None
          and weights is not None and (kl == 0 or ref_logp is not None),
          "targets, old_logp, advantages and weights are needed, and ref_logp where kl is not 0")
    gradient, stride, to = _gradient_of(logits, gradient, device)
    f32, shape = torch.float32, (rows,)
    old = _words(old_logp, "old_logp", device, f32, shape)
    loss, token_loss, logp = (old_logp.new_empty(()), torch.empty_like(old_logp),
                              torch.empty_like(old_logp))
    request = _policy(_ELEMENT[logits.dtype], rows, vocab, row, stride, scale, clip_low,
                      clip_high, kl, pointer,
                      _words(targets, "targets", device, torch.int32, shape),
                      old,
                      _words(ref_logp, "ref_logp", device, f32, shape),
                      _words(advantages, "advantages", device, f32, shape),
                      _words(weights, "weights", device, f32, shape),
                      loss.data_ptr(), token_loss.data_ptr(), logp.data_ptr(), to)
    _call("tb_policy_loss", device, request)
    return PolicyLoss(loss, token_loss, logp, gradient)


def preference_loss(logits, targets, offsets, ref_logp, *, beta: float = 0.1,
                    smoothing: float = 0.0, weights=None, scale: float = 1.0,
                    gradient=True) -> PreferenceLoss:
    """Paired log-ratio loss over packed answers, with its gradient by the logits.

    ``offsets`` (int32, 2 pairs + 1 rising row numbers) delimits the chosen answers, then the
    rejected ones in the same order; ``targets`` is negative at rows that are not scored (prompts);
    ``ref_logp`` holds the reference model's log probability of each row.  With
    ``m = beta (ratio_chosen - ratio_rejected)`` the loss is the weighted sum (``weights`` float32
    per pair, 1 / pairs when None) of ``-(1 - smoothing) log sigmoid(m) - smoothing log sigmoid(-m)``.
    Rows outside every answer are left as they were.  ``gradient`` as in :func:`policy_loss`."""
    device, row, pointer = _logits(logits)
    rows, vocab = logits.shape
    _need(isinstance(offsets, torch.Tensor) and offsets.dim() == 1 and offsets.shape[0] >= 3
          and offsets.shape[0] % 2 == 1, "offsets: expected 2 pairs + 1 row numbers")
    _need(targets is not None and ref_logp is not None, "targets and ref_logp are needed")
    pairs = offsets.shape[0] // 2
    gradient, stride, to = _gradient_of(logits, gradient, device)
    f32 = torch.float32
    ref = _words(ref_logp, "ref_logp", device, f32, (rows,))
    loss, ratios, logp = (ref_logp.new_empty(()), ref_logp.new_empty((2 * pairs,)),
                          torch.empty_like(ref_logp))
    size = _entry("tb_preference_workspace")(rows, pairs)
    workspace = logits.new_empty((size,), dtype=torch.uint8)
    request = (_ELEMENT[logits.dtype], rows, vocab, pairs, row, stride, scale, beta,
            smoothing, pointer, _words(targets, "targets", device, torch.int32, (rows,)),
            _words(offsets, "offsets", device, torch.int32, (2 * pairs + 1,)), ref,
            _words(weights, "weights", device, f32, (pairs,)),
            loss.data_ptr(), ratios.data_ptr(), logp.data_ptr(), to, workspace.data_ptr(), size)
    _call("tb_preference_loss", device, _preference(*request))
    return PreferenceLoss(loss, ratios, logp, gradient)
