"""Python face of the device operators of ``include/topos_b200.h``: what lies around the matrix
products of a decoder's training and decode steps, on device arrays that the caller holds.

- :func:`gated_scan`, :func:`gated_scan_backward` -- the gated linear recurrence over time
- :func:`head_rotate`, :func:`head_rotate_backward` -- norms of query and key heads with the
  position rotation; :func:`rotation_table` makes its cosines and sines
- :func:`token_logp`, :func:`policy_loss`, :func:`preference_loss` -- losses over a vocabulary
  with their gradients by the logits
- :func:`synchronize` -- waits for the work, and raises what went wrong in it

Device arrays are torch tensors (float32 or bfloat16), used as memory only: nothing here records
gradients.  An array that is given to be written counts as changed in place, so that a backward pass
that still needs what it held raises; no two arrays of a call share memory unless one is written over
the other as a function says.  Arguments of one call live on one device; the work is enqueued on that
device's current torch stream, and outputs that are not given are allocated by torch on that stream.  A
malformed request raises ``ValueError`` or :class:`~poorgrad_b200.backend.BackendError`; there is no
CPU fallback.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import numpy as np
import torch

from .abi import library_path, load_library
from .backend import BackendError

try:
    from . import _operators as _native
except ImportError as error:
    raise RuntimeError("the operators' binding is not built beside " + library_path()
                       + "; run __graft_entry__.build()") from error

_native.set_error(BackendError)
_FORM = {"direct": 0, "sigmoid": 1}
_STYLE = {"halves": 0, "pairs": 1}


def _one_of(names: dict, name: str, value):
    code = names.get(value)
    if code is None:
        raise ValueError(f"{name}: one of {sorted(names)} is expected, got {value!r}")
    return code


def synchronize(device=None) -> None:
    """Waits for the current stream of ``device`` (the current one when None), and raises
    :class:`~poorgrad_b200.backend.BackendError` where its work failed or a wait between the blocks of an
    operator ever ran out there."""
    with torch.cuda.device(device):
        code = load_library().tb_operators_synchronize(torch.cuda.current_stream().cuda_stream)
    if code != 0:
        raise BackendError(code, "tb_operators_synchronize")


# ------------------------------------------------------------------ gated scan
def gated_scan(gate, x, *, form: str = "sigmoid", state=None, offsets=None, out=None,
               final_state=None):
    """``h_t = a_t h_{t-1} + b_t`` over time; returns ``(h, final_state)``.

    ``form="direct"``: a is ``gate`` and b is ``x``.  ``form="sigmoid"``: a is the sigmoid of
    ``gate`` and b is ``(1 - a) x``.  ``gate`` and ``x`` are ``[batch, length, channels]``, or a
    packed ``[rows, channels]`` whose sequences ``offsets`` (int32, sequences + 1 rising row
    numbers) delimits; rows outside every sequence are 0, or left as they were in a given array.
    ``state`` (float32, ``[batch or sequences, channels]``, zeros when None) comes before the first
    step; the returned final state may be written into ``state`` itself (``final_state=state``), as a
    decode loop does; over a long sequence of few channels an array of its own is up to four times as
    fast.  ``out`` may be ``gate`` or ``x``."""
    return _native.gated_scan(gate, x, _one_of(_FORM, "form", form), state, offsets, out,
                              final_state)


def gated_scan_backward(dh, gate, x, h, *, form: str = "sigmoid", state=None, offsets=None,
                        dfinal=None, dgate=None, dx=None):
    """Gradients ``(dgate, dx, dstate)`` of :func:`gated_scan` from the gradient ``dh`` of its
    outputs ``h`` and ``dfinal`` of its final state (zeros when None).  ``state`` is what the scan
    began with: a carry that was written in place (``final_state=state``) no longer is.  ``x`` is read by the
    sigmoid form only, and may be None in the direct one.  One of ``dgate`` and ``dx`` may be
    ``dh``.  Rows outside every sequence are as in :func:`gated_scan`."""
    return _native.gated_scan_backward(dh, gate, x, h, _one_of(_FORM, "form", form), state, offsets,
                                       dfinal, dgate, dx)


# ----------------------------------------------------------------- head rotate
def rotation_table(rows: int, turned: int, base: float = 10000.0, first: int = 0) -> np.ndarray:
    """``[rows, turned]`` float32: cosines, then sines, of ``(first + row) * base^(-2i / turned)``
    for i below turned / 2, computed in 64 bits (a far position's angle needs them)."""
    if turned < 0 or turned % 2:
        raise ValueError("turned is even and not negative")
    half = turned // 2
    angles = (np.arange(first, first + rows, dtype=np.float64)[:, None]
              * base ** (-np.arange(half, dtype=np.float64) / max(half, 1))[None, :])
    return np.concatenate([np.cos(angles), np.sin(angles)], axis=1).astype(np.float32)


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
    return _native.head_rotate(q, k, table, positions, q_weight, k_weight, epsilon,
                               _one_of(_STYLE, "style", style), q_out, k_out)


def head_rotate_backward(dq, dk, q, k, table, positions=None, *, q_weight=None, k_weight=None,
                         epsilon: float = 1e-5, style: str = "halves", q_out=None, k_out=None,
                         weights: bool = True):
    """Gradients ``(q_grad, k_grad, q_weight_grad, k_weight_grad)`` of :func:`head_rotate` from the
    gradients ``dq`` and ``dk`` of its outputs; the last two are float32 ``[dim]``, or None with
    ``weights=False``, and NaN where a token's position is outside the table.  ``q_out`` and ``k_out``
    receive the first two and may be ``dq`` and ``dk``."""
    return _native.head_rotate_backward(q, k, table, positions, q_weight, k_weight, epsilon,
                                        _one_of(_STYLE, "style", style), q_out, k_out, dq, dk,
                                        bool(weights))


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


def token_logp(logits, targets, *, scale: float = 1.0):
    """Float32 log probabilities of ``targets`` (int32 ``[rows]``) under ``softmax(scale * logits)``
    of each row.  A hidden row -- a negative target, or no logit above -inf -- gives 0, a target
    beyond the vocabulary NaN."""
    return _native.token_logp(logits, targets, scale)


def policy_loss(logits, targets, old_logp, advantages, weights, *, ref_logp=None,
                clip_low: float = 0.2, clip_high: float = 0.2, kl: float = 0.0,
                scale: float = 1.0, gradient=True) -> PolicyLoss:
    """Clipped policy loss over sampled tokens, with its gradient by the logits.

    With ``r = exp(logp - old_logp)`` and ``d = ref_logp - logp``, the loss is the sum over rows of
    ``weight * (-min(r A, clamp(r, 1 - clip_low, 1 + clip_high) A) + kl (exp(d) - d - 1))``; the
    weights hold the normalizer (1 / tokens, say) and hide a row where they are 0.  A hidden row,
    also one as in :func:`token_logp`, adds nothing whatever it holds and has a gradient of 0.
    ``gradient`` is True, False, or the array to write, which may be ``logits`` itself."""
    return PolicyLoss(*_native.policy_loss(logits, targets, old_logp, advantages, weights, ref_logp,
                                           clip_low, clip_high, kl, scale, gradient))


def preference_loss(logits, targets, offsets, ref_logp, *, beta: float = 0.1,
                    smoothing: float = 0.0, weights=None, scale: float = 1.0,
                    gradient=True) -> PreferenceLoss:
    """Paired log-ratio loss over packed answers, with its gradient by the logits.

    ``offsets`` (int32, 2 pairs + 1 rising row numbers) delimits the chosen answers, then the
    rejected ones in the same order; ``targets`` is negative at rows that are not scored (prompts);
    ``ref_logp`` holds the reference model's log probability of each row.  With
    ``m = beta (ratio_chosen - ratio_rejected)`` the loss is the weighted sum (``weights`` float32
    per pair, 1 / pairs when None) of ``-(1 - smoothing) log sigmoid(m) - smoothing log sigmoid(-m)``.
    Rows outside every answer have a log probability and a gradient of 0; a given gradient array is left
    as it was there (the logits, where it is theirs).  ``gradient`` as in :func:`policy_loss`."""
    return PreferenceLoss(*_native.preference_loss(logits, targets, offsets, ref_logp, beta,
                                                   smoothing, weights, scale, gradient))
