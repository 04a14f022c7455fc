"""Refusals of the training-step operators that need no GPU: argument checks
in Python before any launch, and the C entry points' own checks."""

import ctypes
from pathlib import Path

import pytest
import torch

LIBRARY = (Path(__file__).resolve().parent.parent / "alpha-yoo-for-great-kingdom_b200" / "kingdom_ai" / "libgk.so")
EINVAL = -22


def test_cpu_tensors_are_refused():
    from kingdom_ai import linear, pack_activation, policy_loss
    x, w = torch.zeros(2, 3), torch.zeros(4, 3)
    with pytest.raises(ValueError):
        linear(x, w)
    with pytest.raises(ValueError):
        pack_activation(x)
    with pytest.raises(ValueError):
        policy_loss(x, target=x)


def test_wrong_kinds_are_refused():
    from kingdom_ai import linear, pack_activation, packed_activations, policy_loss, policy_value_loss
    for call in (lambda: linear([1.0], torch.zeros(1, 1)), lambda: linear(torch.zeros(1, 1), None),
                 lambda: pack_activation(3), lambda: policy_loss([0.0], target=None),
                 lambda: policy_value_loss(None, None)):
        with pytest.raises(TypeError):
            call()
    for bad in (0, -1, True, 1.5):
        with pytest.raises(ValueError):
            with packed_activations(min_elements=bad):
                pass


def test_packed_activations_leaves_cpu_tensors_alone():
    from kingdom_ai import packed_activations
    x = torch.randn(300, 300, requires_grad=True)
    with packed_activations(min_elements=1):
        y = (x * 1.5).exp()
    y.sum().backward()
    assert torch.equal(x.grad, 1.5 * (x * 1.5).exp().detach())


c_void_p, c_int64, c_int, c_float = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_float


class PolicyLossStruct(ctypes.Structure):
    _fields_ = [("logits", c_void_p), ("mask", c_void_p), ("target", c_void_p), ("actions", c_void_p),
                ("old_log_probs", c_void_p), ("advantages", c_void_p), ("reference_log_probs", c_void_p),
                ("denominator_ptr", c_void_p), ("rows", c_int64), ("cols", c_int64), ("logits_stride", c_int64),
                ("mask_stride", c_int64), ("target_stride", c_int64), ("clip_low", c_float), ("clip_high", c_float),
                ("kl_weight", c_float), ("target_weight", c_float), ("denominator", c_float), ("logits_type", c_int),
                ("target_type", c_int), ("loss", c_void_p), ("log_probs", c_void_p), ("stats", c_void_p),
                ("partials", c_void_p), ("grad", c_void_p)]


class LinearStruct(ctypes.Structure):
    _fields_ = [("x", c_void_p), ("w", c_void_p), ("bias", c_void_p), ("residual", c_void_p), ("y", c_void_p),
                ("pre", c_void_p), ("m", c_int64), ("n", c_int64), ("k", c_int64), ("x_stride", c_int64),
                ("w_stride", c_int64), ("residual_stride", c_int64),
                ("pre_stride", c_int64), ("dtype", c_int), ("activation", c_int)]


class LinearGradStruct(ctypes.Structure):
    _fields_ = [("dy", c_void_p), ("kept", c_void_p), ("x", c_void_p), ("x_codes", c_void_p), ("x_scales", c_void_p),
                ("w", c_void_p), ("dx", c_void_p), ("dw", c_void_p), ("db", c_void_p), ("dz", c_void_p),
                ("m", c_int64), ("n", c_int64), ("k", c_int64), ("dy_stride", c_int64), ("kept_stride", c_int64), ("x_stride", c_int64),
                ("w_stride", c_int64), ("dtype", c_int), ("activation", c_int)]


def library():
    if not LIBRARY.exists():
        pytest.skip("libgk.so not built")
    lib = ctypes.CDLL(str(LIBRARY))
    for name, result, arguments in (
            ("gk_linear_forward", c_int, [c_void_p] * 4), ("gk_linear_backward", c_int, [c_void_p] * 4),
            ("gk_linear_workspace_bytes", ctypes.c_size_t, [c_void_p]),
            ("gk_policy_loss_parts", c_int, [c_int64, c_int64]),
            ("gk_policy_loss_forward", c_int, [c_void_p] * 2),
            ("gk_policy_loss_backward", c_int, [c_void_p, c_void_p, c_int, c_void_p]),
            ("gk_pack", c_int, [c_void_p, c_int64, c_int, c_int64, c_int64, c_void_p, c_void_p, c_void_p]),
            ("gk_unpack", c_int, [c_void_p, c_void_p, c_int64, c_int64, c_void_p, c_int64, c_int, c_void_p])):
        fn = getattr(lib, name)
        fn.restype, fn.argtypes = result, arguments
    return lib


def linear_struct(**changes):
    p = LinearStruct()
    base = 1 << 20  # never read: the checks come first
    p.x, p.w, p.y = base, base, base
    p.m, p.n, p.k, p.x_stride, p.w_stride, p.dtype, p.activation = 4, 8, 16, 16, 16, 1, 0
    for k, v in changes.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("changes", [dict(n=0), dict(k=0), dict(m=-1), dict(dtype=3), dict(dtype=-1),
                                     dict(activation=5), dict(activation=-1), dict(x=None), dict(w=None),
                                     dict(y=None), dict(k=1 << 31), dict(x_stride=-16),
                                     dict(pre=1 << 20, pre_stride=7)])
def test_linear_entry_refuses(changes):
    lib = library()
    status = ctypes.c_void_p(1 << 20)
    assert lib.gk_linear_forward(ctypes.byref(linear_struct(**changes)), None, status, None) == EINVAL
    assert lib.gk_linear_workspace_bytes(ctypes.byref(linear_struct(**changes))) == 0


def test_linear_entry_refuses_missing_workspace_and_status():
    lib = library()
    status = ctypes.c_void_p(1 << 20)
    odd = linear_struct(m=64, k=17, x_stride=17, w_stride=17)  # rows that TMA cannot read: aligned copies
    assert lib.gk_linear_workspace_bytes(ctypes.byref(odd)) >= (64 + 8) * 24 * 2
    assert lib.gk_linear_forward(ctypes.byref(odd), None, status, None) == EINVAL
    assert lib.gk_linear_forward(ctypes.byref(linear_struct()), None, None, None) == EINVAL
    assert lib.gk_linear_forward(ctypes.byref(linear_struct(m=0)), None, status, None) == 0


def test_linear_backward_entry_refuses():
    lib = library()
    status = ctypes.c_void_p(1 << 20)

    def struct(**changes):
        p = LinearGradStruct()
        p.dy = p.kept = p.x = p.w = p.dx = p.dw = 1 << 20
        p.m, p.n, p.k, p.dy_stride, p.x_stride, p.w_stride, p.dtype, p.activation = 4, 8, 16, 8, 16, 16, 1, 1
        for k, v in changes.items():
            setattr(p, k, v)
        return ctypes.byref(p)

    for changes in (dict(m=0), dict(n=0), dict(k=0), dict(dy=None), dict(kept=None), dict(w=None), dict(x=None),
                    dict(x=None, x_codes=1 << 20), dict(activation=9), dict(dtype=7), dict(dy_stride=-1), dict(kept_stride=-1),
                    dict(activation=0, dz=1 << 20)):
        assert lib.gk_linear_backward(struct(**changes), None, status, None) == EINVAL, changes
    assert lib.gk_linear_backward(struct(), None, status, None) == EINVAL  # dz needs a workspace


def test_policy_loss_entry_refuses():
    lib = library()

    def struct(**changes):
        p = PolicyLossStruct()
        p.logits = p.target = p.loss = p.stats = p.partials = 1 << 20
        p.rows, p.cols, p.logits_stride, p.target_stride, p.denominator = 4, 82, 82, 82, 4.0
        for k, v in changes.items():
            setattr(p, k, v)
        return ctypes.byref(p)

    for changes in (dict(rows=-1), dict(cols=0), dict(cols=(1 << 30) + 1), dict(logits=None), dict(loss=None),
                    dict(stats=None), dict(partials=None), dict(logits_type=3), dict(target=None),
                    dict(logits_type=1, target_type=2), dict(actions=1 << 20), dict(reference_log_probs=1 << 20)):
        assert lib.gk_policy_loss_forward(struct(**changes), None) == EINVAL, changes
    assert lib.gk_policy_loss_backward(struct(), None, 0, None) == EINVAL
    assert lib.gk_policy_loss_backward(struct(), 1 << 20, 0, None) == EINVAL  # no gradient to write
    assert lib.gk_policy_loss_parts(0, 82) == 0 and lib.gk_policy_loss_parts(5, 0) == 0
    assert lib.gk_policy_loss_parts(5, 82) >= 1 and lib.gk_policy_loss_parts(5, 5000) >= 5


def test_pack_entries_refuse():
    lib = library()
    base = 1 << 20
    for args in ((None, 8, 0, 2, 8, base, base), (base, 8, 3, 2, 8, base, base), (base, 4, 0, 2, 8, base, base),
                 (base, 8, 0, -1, 8, base, base), (base, 8, 0, 1 << 30, 1 << 30, base, base),
                 (base, 8, 0, 2, 8, None, base), (base, 8, 0, 2, 8, base, None)):
        assert lib.gk_pack(*args, None) == EINVAL, args
    assert lib.gk_pack(None, 0, 0, 0, 8, None, None, None) == 0
    assert lib.gk_unpack(base, base, 2, 8, None, 8, 0, None) == EINVAL
    assert lib.gk_unpack(base, base, 2, 8, base, 8, 5, None) == EINVAL
