"""Activations kept in 8 bits between the forward and the backward pass.

A training step's memory is mostly what the forward pass keeps for the
backward pass. Here a kept tensor takes 1 byte and 1/32 a value: e4m3 codes and
one power-of-two scale for every 32 values (``gk_pack``), chosen so that the
block's largest magnitude is not cut off. A held value is off by at most 2^-4
of itself down to 2^-15 of its block's largest, and by 2^-19 of the largest
below (smaller ones become zero). Infinities and NaN come back as NaN.

``packed_activations`` packs what PyTorch operators keep (the trunk of a
training step); ``linear(..., checkpoint="e4m3")`` keeps its own input so.
The reference keeps every activation in fp32 (python/kingdom_ai/training.py:
213-230 under autograd).
"""

from __future__ import annotations

import contextlib
import threading

import torch

from . import _native as native

_PACKED_TYPES = (torch.float32, torch.bfloat16, torch.float16)
_active = threading.local()


class PackedActivation:
    """The 8-bit form of a tensor: ``codes`` (uint8, e4m3) and ``scales``
    (uint8, value 2^(byte - 127)), with the shape and dtype to unpack to."""

    __slots__ = ("codes", "scales", "shape", "dtype")

    def __init__(self, codes, scales, shape, dtype):
        self.codes, self.scales, self.shape, self.dtype = codes, scales, shape, dtype

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()

    def unpack(self, dtype=None) -> torch.Tensor:
        """The held values in the packed tensor's shape and its dtype (or in
        fp32, which holds them all), contiguous."""
        if dtype is None:
            dtype = self.dtype
        elif dtype not in (self.dtype, torch.float32):
            raise ValueError(f"unpack gives {self.dtype} or torch.float32")
        return native.operators().unpack.default(self.codes, self.scales, self.shape, dtype)


def pack_activation(x: torch.Tensor) -> PackedActivation:
    """Pack a CUDA tensor of fp32, bf16 or fp16 values (any shape, none at all
    included). Blocks of 32 run through its values in row-major order; strided
    tensors are made contiguous first, and unpack as contiguous ones."""
    if not isinstance(x, torch.Tensor):
        raise TypeError("pack_activation packs a tensor")
    codes, scales = native.operators().pack.default(x)
    return PackedActivation(codes, scales, x.shape, x.dtype)


class _Kept:
    """A saved tensor as it is. Detached, for an operator's own output would
    keep itself alive; with its version, which autograd does not check where
    hooks save."""

    __slots__ = ("tensor", "version")

    def __init__(self, t):
        self.tensor, self.version = t.detach(), t._version

    def unpack(self) -> torch.Tensor:
        if self.tensor._version != self.version:
            raise RuntimeError(f"a tensor of shape {tuple(self.tensor.shape)} that was kept for the backward pass has "
                               f"been modified by an inplace operation: it is at version {self.tensor._version}, and "
                               f"was kept at version {self.version}")
        return self.tensor


def _is_parameter(t: torch.Tensor) -> bool:
    """A parameter, a leaf that is being trained, a view of one, or one cast to another type (autocast)."""
    base = t if t._base is None else t._base
    if isinstance(base, torch.nn.Parameter) or (base.is_leaf and base.requires_grad):
        return True
    fn = t.grad_fn
    if fn is None or not fn.name().startswith("ToCopyBackward"):
        return False
    source = fn.next_functions[0][0] if fn.next_functions else None
    return source is not None and source.name().endswith("AccumulateGrad")


@contextlib.contextmanager
def packed_activations(min_elements: int = 1 << 16):
    """Within the context, what operators keep for the backward pass is packed:
    CUDA tensors of fp32, bf16 or fp16 with at least ``min_elements`` values,
    parameters excepted (frozen ones, views, and casts of those in training; a
    cast of a frozen weight cannot be told from an activation, so keep such a
    layer outside). Gradients are then those of the held values; the forward
    pass computes with the exact ones. A relu that keeps its output passes no
    gradient where the packed output is zero.
    A tensor that two operators keep (a relu its output, the convolution behind
    it its input) is packed for each of them.
    ``linear`` and ``policy_loss`` keep their tensors as they are (``linear``
    has its own ``checkpoint``)."""
    if isinstance(min_elements, bool) or not isinstance(min_elements, int) or min_elements < 1:
        raise ValueError("min_elements must be a positive integer")

    def pack(t):
        if (t.device.type != "cuda" or t.dtype not in _PACKED_TYPES or t.numel() < min_elements
                or t.layout != torch.strided or _is_parameter(t)):
            return _Kept(t)
        return pack_activation(t)

    depth = getattr(_active, "depth", 0)
    with torch.autograd.graph.saved_tensors_hooks(pack, lambda kept: kept.unpack()):
        _active.depth = depth + 1
        try:
            yield
        finally:
            _active.depth = depth


def packing_active() -> bool:
    """Whether this thread is inside packed_activations."""
    return getattr(_active, "depth", 0) > 0


def keep_saved_tensors():
    """A context in which saved tensors are kept as they are inside packed_activations."""
    return torch.autograd.graph.saved_tensors_hooks(_Kept, lambda kept: kept.unpack())


