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

BLOCK = 32  # values that share a scale
_active = threading.local()


class PackedActivation:
    """The 8-bit form of a tensor: ``codes`` (uint8, e4m3) and ``scales``
    (uint8, value 2^(byte - 127)), with the shape and dtype to unpack to."""

    __slots__ = ("codes", "scales", "shape", "dtype", "rows", "cols")

    def __init__(self, codes, scales, shape, dtype, rows, cols):
        self.codes, self.scales, self.shape, self.dtype = codes, scales, shape, dtype
        self.rows, self.cols = rows, cols

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()

    def unpack(self, dtype=None) -> torch.Tensor:
        """The held values in the packed tensor's shape and its dtype (or in
        fp32, which holds them all), contiguous."""
        if dtype not in (None, self.dtype, torch.float32):
            raise ValueError(f"unpack gives {self.dtype} or torch.float32")
        out = torch.empty(self.shape, dtype=dtype or self.dtype, device=self.codes.device)
        if out.numel():
            with native.on_device(out.device):
                native.call("gk_unpack", native.ptr(self.codes), native.ptr(self.scales), self.rows, self.cols,
                            native.ptr(out), self.cols, native.TYPES[out.dtype],
                            native.launch_stream(out.device, (self.codes, self.scales)))
        return out


def pack_rows(x: torch.Tensor, rows: int, cols: int, stride: int, shape) -> PackedActivation:
    """Pack [rows, cols] of x's memory, rows `stride` elements apart; a block never spans two rows."""
    per_row = -(-cols // BLOCK)
    # Codes and scales in one allocation; the codes start it, so they are aligned.
    buffer = torch.empty(rows * (cols + per_row), dtype=torch.uint8, device=x.device)
    codes, scales = buffer[:rows * cols], buffer[rows * cols:]
    if rows and cols:
        with native.on_device(x.device):
            native.call("gk_pack", native.ptr(x), stride, native.TYPES[x.dtype], rows, cols, native.ptr(codes),
                        native.ptr(scales), native.launch_stream(x.device, (x,)))
    return PackedActivation(codes, scales, shape, x.dtype, rows, cols)


def pack_activation(x: torch.Tensor) -> PackedActivation:
    """Pack a CUDA tensor of fp32, bf16 or fp16 values (any shape, none at all
    included). Blocks of 32 run through its values in row-major order; strided
    tensors are made contiguous first, and unpack as contiguous ones."""
    if not isinstance(x, torch.Tensor):
        raise TypeError("pack_activation packs a tensor")
    if x.device.type != "cuda" or x.dtype not in native.TYPES:
        raise ValueError("pack_activation packs CUDA tensors of float32, bfloat16 or float16")
    x = x.detach().contiguous()
    return pack_rows(x, 1, x.numel(), x.numel(), x.shape)


def _is_parameter(t: torch.Tensor) -> bool:
    """A leaf that is being trained, a view of one, or one cast to another type (autocast)."""
    base = t if t._base is None else t._base
    if base.is_leaf and base.requires_grad:
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
    parameters excepted (also their views and casts). Gradients are then those
    of the held values; the forward pass computes with the exact ones. A relu
    that keeps its output passes no gradient where the packed output is zero.
    ``linear`` and ``policy_loss`` keep their tensors as they are (``linear``
    has its own ``checkpoint``)."""
    if isinstance(min_elements, bool) or not isinstance(min_elements, int) or min_elements < 1:
        raise ValueError("min_elements must be a positive integer")

    def pack(t):
        if (t.device.type != "cuda" or t.dtype not in native.TYPES or t.numel() < min_elements
                or t.layout != torch.strided or _is_parameter(t)):
            return t
        return pack_activation(t)

    def unpack(kept):
        return kept.unpack() if isinstance(kept, PackedActivation) else kept

    depth = getattr(_active, "depth", 0)
    with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
        _active.depth = depth + 1
        try:
            yield
        finally:
            _active.depth = depth


def keep_saved_tensors():
    """A context in which saved tensors are kept as they are inside packed_activations."""
    if getattr(_active, "depth", 0) == 0:
        return contextlib.nullcontext()
    return torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t)


