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
from torch.autograd.function import once_differentiable

from . import _native as native
from .packing import keep_saved_tensors

_TYPES = native.TYPES
_MOST_COLUMNS = 1 << 30


class PolicyLoss(NamedTuple):
    loss: torch.Tensor               # fp32 scalar
    log_probs: torch.Tensor | None   # fp32 [N], log p of the actions (0 for skipped rows); None without actions


def _scalar(name, value, least=None):
    if isinstance(value, bool) or not isinstance(value, Real):
        raise TypeError(f"{name} must be a real number")
    if not math.isfinite(value) or (least is not None and value < least):
        raise ValueError(f"{name} must be finite" + ("" if least is None else f" and at least {least}"))
    return float(value)


def _clip(clip):
    low, high = clip if isinstance(clip, tuple) and len(clip) == 2 else (clip, clip)
    low, high = _scalar("clip", low, 0), _scalar("clip", high, 0)
    return 1.0 - low, 1.0 + high


def _column(name, t, rows, dtype, device):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if t.shape != (rows,) or t.dtype != dtype or t.device != device:
        raise ValueError(f"{name} must have shape ({rows},), dtype {dtype} and the logits' device")
    if t.requires_grad:
        raise ValueError(f"{name} must not require a gradient: the loss differentiates by its logits alone")
    return t if t.is_contiguous() else t.contiguous()


def _matrix(name, t, shape, dtypes, device):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if t.shape != shape or t.dtype not in dtypes or t.device != device:
        raise ValueError(f"{name} must have shape {tuple(shape)}, dtype {' or '.join(map(str, dtypes))} "
                         "and the logits' device")
    if t.requires_grad:
        raise ValueError(f"{name} must not require a gradient: the loss differentiates by its logits alone")
    return t if t.stride(1) == 1 and t.stride(0) >= 0 else t.contiguous()


class _Call:
    """One batch's arguments: the C struct and the tensors that it points into."""

    def __init__(self, logits, mask, actions, old, advantages, reference, target, clip, kl_weight, target_weight,
                 denominator):
        n, a = logits.shape
        device = logits.device
        p = native.PolicyLossStruct()
        self.struct, self.rows, self.device = p, n, device
        self.inputs = tuple(t for t in (logits, mask, actions, old, advantages, reference, target)
                            if t is not None)
        p.logits, p.rows, p.cols, p.logits_stride = logits.data_ptr(), n, a, logits.stride(0)
        p.logits_type = _TYPES[logits.dtype]
        if mask is not None:
            p.mask, p.mask_stride = mask.data_ptr(), mask.stride(0)
        if target is not None:
            p.target, p.target_stride, p.target_type = target.data_ptr(), target.stride(0), _TYPES[target.dtype]
            p.target_weight = target_weight
        if actions is not None:
            p.actions, p.old_log_probs, p.advantages = actions.data_ptr(), old.data_ptr(), advantages.data_ptr()
            p.clip_low, p.clip_high = clip
        if reference is not None:
            p.reference_log_probs, p.kl_weight = reference.data_ptr(), kl_weight
        if isinstance(denominator, torch.Tensor):
            p.denominator_ptr = denominator.data_ptr()
            self.inputs += (denominator,)
        else:
            p.denominator = denominator

    def forward(self, with_grad, logits):
        """(loss, log_probs, grad), and the row statistics kept for the backward pass."""
        p, n = self.struct, self.rows
        # Row statistics (four floats a row), then the partial sums (doubles).
        self.workspace = torch.empty(2 * n + native.library().gk_policy_loss_parts(n, p.cols), dtype=torch.float64,
                                     device=self.device)
        base = self.workspace.data_ptr()
        loss = torch.empty((), dtype=torch.float32, device=self.device)
        log_probs = None if not p.actions else torch.empty(n, dtype=torch.float32, device=self.device)
        grad = torch.empty(logits.shape, dtype=logits.dtype, device=self.device) if with_grad else None
        p.stats, p.partials = base, base + 16 * n
        p.loss = loss.data_ptr()
        p.log_probs = None if log_probs is None else log_probs.data_ptr()
        p.grad = None if grad is None else grad.data_ptr()
        native.call("gk_policy_loss_forward", p, native.launch_stream(self.device, self.inputs))
        return loss, log_probs, grad

    def backward(self, upstream, grad, written):
        self.struct.grad = grad.data_ptr()
        # The inputs and the workspace were marked on this stream by the forward pass.
        native.call("gk_policy_loss_backward", self.struct, native.ptr(upstream), written,
                    native.launch_stream(self.device, (upstream,)))


class _PolicyLossFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, call):
        # fp16 training scales its loss, so a gradient for an upstream of one
        # would be computed in vain; the other types get it in the same pass.
        with native.on_device(call.device):
            loss, log_probs, grad = call.forward(logits.dtype != torch.float16, logits)
        ctx.save_for_backward(*call.inputs)
        ctx.call, ctx.grad = call, grad
        if log_probs is not None:
            ctx.mark_non_differentiable(log_probs)
        return loss, log_probs

    @staticmethod
    @once_differentiable
    def backward(ctx, upstream, _):
        logits = ctx.saved_tensors[0]  # raises if an input was modified in place
        grad, ctx.grad = ctx.grad, None
        written = grad is not None
        if not written:
            grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        upstream = upstream.contiguous()
        with native.on_device(logits.device):
            ctx.call.backward(upstream, grad, int(written))
        return grad, None


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

    Rows with unit column stride are read in place; others are copied first.
    """
    if not isinstance(logits, torch.Tensor):
        raise TypeError("logits must be a tensor")
    if logits.device.type != "cuda":
        raise ValueError("policy_loss requires CUDA logits")
    if logits.ndim != 2 or logits.dtype not in _TYPES or not 1 <= logits.shape[1] <= _MOST_COLUMNS:
        raise ValueError("logits must have shape [N, A] with A > 0 and dtype float32, bfloat16 or float16")
    n, device = logits.shape[0], logits.device
    if actions is None:
        if old_log_probs is not None or advantages is not None or reference_log_probs is not None:
            raise ValueError("old_log_probs, advantages and reference_log_probs go with actions")
        if target is None:
            raise ValueError("policy_loss needs actions or a target")
    elif old_log_probs is None or advantages is None:
        raise ValueError("actions go with old_log_probs and advantages")
    clip = _clip(clip)
    kl_weight, target_weight = _scalar("kl_weight", kl_weight), _scalar("target_weight", target_weight)
    if denominator is None:
        denominator = float(max(n, 1))
    elif isinstance(denominator, torch.Tensor):
        if denominator.numel() != 1 or denominator.dtype != torch.float32 or denominator.device != device:
            raise ValueError("denominator must hold one float32 on the logits' device")
        if denominator.requires_grad:
            raise ValueError("denominator must not require a gradient")
    else:
        denominator = _scalar("denominator", denominator)
        if denominator <= 0:
            raise ValueError("denominator must be positive")
    if legal_mask is not None:
        legal_mask = _matrix("legal_mask", legal_mask, logits.shape, (torch.bool,), device)
    if target is not None:
        target = _matrix("target", target, logits.shape,
                         (torch.float32,) if logits.dtype == torch.float32 else (torch.float32, logits.dtype), device)
    if actions is not None:
        actions = _column("actions", actions, n, torch.int64, device)
        old_log_probs = _column("old_log_probs", old_log_probs, n, torch.float32, device)
        advantages = _column("advantages", advantages, n, torch.float32, device)
        if reference_log_probs is not None:
            reference_log_probs = _column("reference_log_probs", reference_log_probs, n, torch.float32, device)
    if logits.stride(1) != 1 or logits.stride(0) < 0:
        logits = logits.contiguous()
    call = _Call(logits.detach(), legal_mask, actions, old_log_probs, advantages, reference_log_probs, target, clip,
                 kl_weight, target_weight, denominator)
    if torch.is_grad_enabled() and logits.requires_grad:
        with keep_saved_tensors():
            return PolicyLoss(*_PolicyLossFunction.apply(logits, call))
    with native.on_device(device):
        return PolicyLoss(*call.forward(False, logits)[:2])
