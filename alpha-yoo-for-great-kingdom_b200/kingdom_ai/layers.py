"""The linear operator of a training step: product, bias, residual, activation.

``linear`` is ``activation(x @ weight.T + bias + residual)`` in one product
with a fused epilogue, its gradients, and its few-row form for serving. It
stands in for the ``nn.Linear`` layers and activations of the network's heads
(python/kingdom_ai/model.py:59-76) in training; bf16 and fp16 run on tcgen05
with fp32 accumulation, fp32 runs on the fp32 units.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _native as native
from .packing import keep_saved_tensors, pack_rows

ACTIVATIONS = {None: 0, "relu": 1, "tanh": 2, "gelu": 3, "silu": 4}  # GK_ACT_*
_KEEPS_SUM = (3, 4)  # their derivative takes the sum before the activation; relu's and tanh's the output
_MOST = (1 << 31) - 1
_status: dict = {}


def _status_words(device) -> torch.Tensor:
    words = _status.get(device)
    if words is None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("call linear once on this device before capturing it in a CUDA graph")
        words = _status[device] = torch.zeros(2, dtype=torch.int32, device=device)
        torch.cuda.current_stream(device).synchronize()
    return words


def check_linear(device="cuda") -> None:
    """Raise if a product on this device reported a bounded wait that gave up
    since the last check (synchronises)."""
    device = native.require_cuda(device)
    words = _status.get(device)
    if words is None:
        return
    code, where = (int(v) for v in words.tolist())
    if code:
        words.zero_()
        raise RuntimeError(f"linear reported error bits {code:#x} (wait at {where & 0x7fffffff:#x}, "
                           f"parity {(where >> 31) & 1})")


def _rows(t: torch.Tensor, cols: int) -> torch.Tensor:
    """`t` as [rows, cols] with contiguous rows: a view where the layout allows, else a copy."""
    if t.ndim == 2:
        if t.stride(1) == 1 or cols == 1:
            return t if t.stride(0) >= 0 else t.contiguous()
        return t.contiguous()
    return t.contiguous().view(-1, cols)


def _stride(t: torch.Tensor) -> int:
    """Elements between rows; the row length where there is but one row."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _workspace(size: int, device):
    return None if size == 0 else torch.empty(size, dtype=torch.uint8, device=device)


def _forward(x, weight, bias, residual, activation, keep_sum):
    """(y, sum before the activation or None) of 2-D x."""
    m, k = x.shape
    n = weight.shape[0]
    y = torch.empty((m, n), dtype=x.dtype, device=x.device)
    pre = torch.empty_like(y) if keep_sum else None
    if m == 0:
        return y, pre
    p = native.LinearStruct(
        x.data_ptr(), weight.data_ptr(), None if bias is None else bias.data_ptr(),
        None if residual is None else residual.data_ptr(), y.data_ptr(), None if pre is None else pre.data_ptr(),
        m, n, k, _stride(x), _stride(weight), 0 if residual is None else _stride(residual), native.TYPES[x.dtype],
        activation)
    device = x.device
    with native.on_device(device):
        workspace = _workspace(native.library().gk_linear_workspace_bytes(p), device)
        used = [t for t in (x, weight, bias, residual) if t is not None]
        native.call("gk_linear_forward", p, native.ptr(workspace), native.ptr(_status_words(device)),
                    native.launch_stream(device, used))
    return y, pre


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation, packed):
        y, pre = _forward(x, weight, bias, residual, activation,
                          activation in _KEEPS_SUM)
        need_x, need_w = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        kept = None if activation == 0 else (pre if activation in _KEEPS_SUM else y)
        ctx.packed = None
        if need_w and packed:
            ctx.packed = pack_rows(x, x.shape[0], x.shape[1], _stride(x), x.shape)
        ctx.save_for_backward(x if need_w and not packed else None, weight if need_x else None, kept)
        ctx.sizes, ctx.activation = (x.shape[0], weight.shape[0], x.shape[1]), activation
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, kept = ctx.saved_tensors
        (m, n, k), activation, packed = ctx.sizes, ctx.activation, ctx.packed
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        dtype, device = dy.dtype, dy.device

        def new(wanted, *shape):
            return torch.empty(shape, dtype=dtype, device=device) if wanted else None

        dx, dw, db = new(need_x, m, k), new(need_w, n, k), new(need_b, n)
        if m == 0:
            for t in (dw, db):
                if t is not None:
                    t.zero_()
            return dx, dw, db, dy if need_r else None, None, None
        dy = _rows(dy, n)
        dz = new(need_r and activation != 0, m, n)
        if need_x or need_w or need_b or dz is not None:
            p = native.LinearGradStruct(
                dy.data_ptr(), None if kept is None else kept.data_ptr(), None if x is None else x.data_ptr(),
                None if packed is None else packed.codes.data_ptr(),
                None if packed is None else packed.scales.data_ptr(), None if weight is None else weight.data_ptr(),
                None if dx is None else dx.data_ptr(), None if dw is None else dw.data_ptr(),
                None if db is None else db.data_ptr(), None if dz is None else dz.data_ptr(), m, n, k, _stride(dy),
                0 if x is None else _stride(x), 0 if weight is None else _stride(weight), native.TYPES[dtype],
                activation)
            with native.on_device(device):
                workspace = _workspace(native.library().gk_linear_grad_workspace_bytes(p), device)
                native.call("gk_linear_backward", p, native.ptr(workspace), native.ptr(_status_words(device)),
                            native.launch_stream(device, (dy,)))
        return dx, dw, db, (dy if activation == 0 else dz) if need_r else None, None, None


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
    inputs' dtype before the products of the backward pass, and gelu and silu
    take their derivative from the rounded sum.

    Call it once on a device before capturing it in a CUDA graph. As with any
    operator, capture a backward pass only when no graph of the same leaves
    made outside the capture is alive (drop earlier outputs first): autograd
    would tie the captured pass to the stream of that graph.
    """
    tensors = (("x", x), ("weight", weight), ("bias", bias), ("residual", residual))
    for name, t in tensors:
        if t is None and name in ("bias", "residual"):
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a tensor")
    if x.device.type != "cuda":
        raise ValueError("linear requires CUDA tensors")
    if x.dtype not in native.TYPES:
        raise ValueError("linear takes float32, bfloat16 or float16")
    for name, t in tensors[1:]:
        if t is not None and (t.dtype != x.dtype or t.device != x.device):
            raise ValueError(f"{name} must have the dtype and device of x")
    if x.ndim < 1 or weight.ndim != 2 or weight.shape[1] != x.shape[-1] or 0 in weight.shape:
        raise ValueError("x must have shape [..., K] and weight [N, K], with N and K at least 1")
    n, k = weight.shape
    shape = (*x.shape[:-1], n)
    if bias is not None and bias.shape != (n,):
        raise ValueError(f"bias must have shape ({n},)")
    if residual is not None and residual.shape != shape:
        raise ValueError(f"residual must have the output's shape {shape}")
    if activation is not None and not isinstance(activation, str) or activation not in ACTIVATIONS:
        raise ValueError('activation must be None, "relu", "tanh", "gelu" or "silu"')
    if checkpoint not in (None, "e4m3"):
        raise ValueError('checkpoint must be None or "e4m3"')
    code = ACTIVATIONS[activation]
    rows = _rows(x, k)
    if max(rows.shape[0], n, k) > _MOST:
        raise ValueError("linear takes sizes below 2**31")
    weight = _rows(weight, k)
    if bias is not None:
        bias = bias.contiguous()
    if residual is not None:
        residual = _rows(residual, n)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for _, t in tensors):
        with keep_saved_tensors():
            y = _Linear.apply(rows, weight, bias, residual, code, checkpoint is not None)
    else:
        y = _forward(rows, weight, bias, residual, code, False)[0]
    return y if y.shape == shape else y.view(shape)
