"""The policy loss of a training step, forward and backward, on the GPU.

``policy_loss`` trains policy logits on replay rows: the KL of a target
distribution (``TrainingBatch.policy``, the search's visit shares) to the
softmax over the legal actions, and, where the played actions are at hand, the
clipped ratio loss of policy-gradient training with a KL estimate to a
reference policy. Rows are as short as a board's 82 actions or as long as a
vocabulary. It stands in for the policy part of the loss in the reference's
``train_step`` (python/kingdom_ai/training.py:213-230).
"""

from __future__ import annotations

import math
from numbers import Real
from typing import NamedTuple

import torch

from . import _native as native
from .packing import keep_saved_tensors, packing_active

_operator = None


class PolicyLoss(NamedTuple):
    loss: torch.Tensor               # fp32 scalar
    log_probs: torch.Tensor | None   # fp32 [N], log p of the actions (0 for skipped rows); None without actions


_FLOAT = torch.finfo(torch.float32)  # what the kernels take the weights and the denominator in


def _scalar(name, value, least=None, most=math.inf):
    if isinstance(value, bool) or not isinstance(value, Real):
        raise TypeError(f"{name} must be a real number")
    if not math.isfinite(value) or abs(value) > most or (least is not None and value < least):
        raise ValueError(f"{name} must be finite" + ("" if most == math.inf else " in fp32")
                         + ("" if least is None else f" and at least {least}"))
    return float(value)


def _clip(clip):
    low, high = clip if isinstance(clip, tuple) and len(clip) == 2 else (clip, clip)
    low, high = _scalar("clip", low, 0), _scalar("clip", high, 0)
    return 1.0 - low, 1.0 + high


def policy_loss(logits, *, legal_mask=None, actions=None, old_log_probs=None, advantages=None,
                reference_log_probs=None, target=None, clip=0.2, kl_weight=0.0, target_weight=1.0,
                denominator=None) -> PolicyLoss:
    """Sum over the rows of

    - with ``actions``: ``-min(q A, clip(q, 1 - clip, 1 + clip) A)`` with
      ``q = exp(log p[action] - old_log_probs)`` and ``A`` the ``advantages``;
      ``clip`` may be a pair (below, above);
    - with ``reference_log_probs`` too: ``kl_weight (exp(d) - d - 1)`` with
      ``d = reference - log p[action]``, an estimate of the KL to the reference;
    - with ``target``: ``target_weight * KL(target || p)``

    divided by ``denominator`` (a positive number, or an fp32 tensor of one
    element on the logits' device; the number of rows by default), where ``p``
    is the softmax of a row's ``logits`` over the entries that ``legal_mask``
    leaves.

    ``logits`` are CUDA [N, A] in fp32, bf16 or fp16; ``legal_mask`` bool
    [N, A]; ``actions`` int64 [N]; ``target`` [N, A] in fp32 or the logits'
    type; the others fp32 [N]. A row with action -1 (or below), and a row of
    which nothing is left (no legal entry, or legal logits all -inf), adds
    nothing and gets a zero gradient. Masked logits and targets may hold
    anything. An action that is not legal or past the row makes its row, and
    the loss, NaN: nothing is read on the host. Statistics and sums are fp32 or
    wider whatever the logits' type; only ``logits`` get a gradient. The
    gradient of a row with no target mass and no action is zero.

    The gradient is made with the loss, for an upstream gradient of one, and
    handed out by the first backward pass (any other upstream gradient, a later
    pass over a retained graph, and fp16, whose losses are scaled, form it in
    the backward pass). ``logits`` and the other arguments must not change in
    place before that.

    Second derivatives and forward-mode ones (a tensor that carries a tangent)
    are refused. torch.compile cannot trace the call: keep it outside.

    Rows with unit column stride are read in place; others are copied first.
    Longer rows run fastest where the logits', mask's and target's rows start
    on the same remainders of 16 bytes as the gradient's, which are contiguous:
    a view of a padded vocabulary whose width is no multiple of 8 (fp32: 4) is
    faster copied first.
    """
    global _operator
    if not isinstance(logits, torch.Tensor):
        raise TypeError("logits must be a tensor")
    for name, t in (("legal_mask", legal_mask), ("actions", actions), ("old_log_probs", old_log_probs),
                    ("advantages", advantages), ("reference_log_probs", reference_log_probs), ("target", target)):
        if t is not None and not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a tensor")
    low, high = _clip(clip)
    kl_weight = _scalar("kl_weight", kl_weight, most=_FLOAT.max)
    target_weight = _scalar("target_weight", target_weight, most=_FLOAT.max)
    divisor = 1.0
    if denominator is None:
        divisor = float(max(logits.shape[0], 1)) if logits.dim() else 1.0
    elif not isinstance(denominator, torch.Tensor):
        # From the smallest normal number on, its inverse is finite too.
        divisor, denominator = _scalar("denominator", denominator, _FLOAT.tiny, _FLOAT.max), None
    if _operator is None:
        _operator = native.operators().policy_loss.default
    arguments = (logits, legal_mask, actions, old_log_probs, advantages, reference_log_probs, target, low, high,
                 kl_weight, target_weight, divisor, denominator)
    if packing_active():
        with keep_saved_tensors():
            loss, log_probs = _operator(*arguments)
    else:
        loss, log_probs = _operator(*arguments)
    return PolicyLoss(loss, None if actions is None else log_probs)
