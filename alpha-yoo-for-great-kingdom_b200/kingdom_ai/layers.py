"""The linear operator of a training step: product, bias, residual, activation.

``linear`` is ``activation(x @ weight.T + bias + residual)`` in one product
with a fused epilogue, its gradients, and its few-row form for serving. It
stands in for the ``nn.Linear`` layers and activations of the network's heads
(python/kingdom_ai/model.py:59-76) in training; bf16 and fp16 run on tcgen05
with fp32 accumulation, fp32 runs on the fp32 units.
"""

from __future__ import annotations

import torch

from . import _native as native
from .packing import keep_saved_tensors, packing_active

ACTIVATIONS = {None: 0, "relu": 1, "tanh": 2, "gelu": 3, "silu": 4}  # GK_ACT_*
_status: dict = {}  # device index -> the words that GK_ERR_TIMEOUT goes to
_operator = None


def _status_words(device) -> torch.Tensor:
    words = _status.get(device.index)
    if words is None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("call linear once on this device before capturing it in a CUDA graph")
        with torch.inference_mode(False):  # check_linear clears it in any mode
            words = torch.zeros(2, dtype=torch.int32, device=device)
        torch.cuda.current_stream(device).synchronize()
        words = _status.setdefault(device.index, words)
    return words


def check_linear(device="cuda") -> None:
    """Raise if a product on this device reported a bounded wait that gave up
    since the last check (waits for all of the device's streams)."""
    device = native.require_cuda(device)
    words = _status.get(device.index)
    if words is None:
        return
    torch.cuda.synchronize(device)
    code, where = (int(v) for v in words.tolist())
    if code:
        words.zero_()
        raise RuntimeError(f"linear reported error bits {code:#x} (wait at {where & 0x7fffffff:#x}, "
                           f"parity {(where >> 31) & 1})")


def linear(x, weight, bias=None, *, activation=None, residual=None, checkpoint=None) -> torch.Tensor:
    """``activation(x @ weight.T + bias + residual)``.

    ``x`` is [..., K], ``weight`` [N, K], ``bias`` [N], ``residual`` [..., N]
    (the output's shape; an expanded tensor is fine), all CUDA tensors of one
    dtype: fp32, bf16 or fp16; K and N are at least 1, the leading sizes may be
    0. ``activation`` is None, "relu", "tanh", "gelu" (the erf form) or "silu".
    Sums are fp32; the output is rounded once. Rows (the last dimension) are
    read in place where they are contiguous, other layouts are copied first.

    Every tensor argument gets its gradient. ``checkpoint="e4m3"`` keeps ``x``
    for the backward pass in 8 bits (``pack_activation``, blocks along its last
    dimension): the weight's gradient is then that of the packed input, every
    other gradient is unchanged. The gradient of the sum is rounded to the
    inputs' dtype before the products of the backward pass (not before narrow
    ones, of few outputs), and gelu and silu take their derivative from the
    rounded sum. For that they keep one more
    tensor of the output's size (tanh keeps one in fp32).

    Second derivatives and forward-mode ones (a tensor that carries a tangent)
    are refused. torch.compile cannot trace the call: keep it outside.

    Call it once on a device before capturing it in a CUDA graph. As with any
    operator, capture a backward pass only when no graph of the same leaves
    made outside the capture is alive (drop earlier outputs first): autograd
    would tie the captured pass to the stream of that graph.
    """
    global _operator
    if not isinstance(x, torch.Tensor) or not isinstance(weight, torch.Tensor):
        raise TypeError("x and weight must be tensors")
    if not (bias is None or isinstance(bias, torch.Tensor)):
        raise TypeError("bias must be a tensor")
    if not (residual is None or isinstance(residual, torch.Tensor)):
        raise TypeError("residual must be a tensor")
    if not x.is_cuda:
        raise ValueError("linear requires CUDA tensors")
    code = ACTIVATIONS.get(activation) if activation is None or isinstance(activation, str) else None
    if code is None:
        raise ValueError('activation must be None, "relu", "tanh", "gelu" or "silu"')
    if checkpoint is not None and checkpoint != "e4m3":
        raise ValueError('checkpoint must be None or "e4m3"')
    if _operator is None:
        _operator = native.operators().linear.default
    status = _status.get(x.device.index)
    if status is None:
        status = _status_words(x.device)
    if packing_active():
        with keep_saved_tensors():
            return _operator(x, weight, bias, residual, code, checkpoint is not None, status)
    return _operator(x, weight, bias, residual, code, checkpoint is not None, status)
