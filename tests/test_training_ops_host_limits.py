"""Numbers that policy_loss's kernels would not hold in fp32 are refused before any launch;
linear's workspaces are what its plans use."""

import ctypes

import pytest
import torch

from test_training_ops_host import LinearGradStruct, library


@pytest.mark.parametrize("name,bad", [("denominator", 1e39), ("denominator", 1e-39), ("denominator", 5e-324),
                                      ("denominator", 0.0), ("denominator", -1.0), ("denominator", float("inf")),
                                      ("kl_weight", 1e39), ("kl_weight", -1e39), ("target_weight", 1e300),
                                      ("target_weight", float("nan")), ("target_weight", 10 ** 39)])
def test_numbers_out_of_range(name, bad):
    from kingdom_ai import policy_loss
    x = torch.zeros(2, 3)
    with pytest.raises(ValueError, match=name):
        policy_loss(x, target=x, **{name: bad})


@pytest.mark.parametrize("name,good", [("denominator", 3e38), ("denominator", 2.0 ** -126), ("kl_weight", -3e38),
                                       ("target_weight", 0), ("clip", 1e39), ("denominator", 7)])
def test_numbers_in_range(name, good):
    from kingdom_ai import policy_loss
    x = torch.zeros(2, 3)
    with pytest.raises(ValueError, match="requires CUDA"):  # the next check
        policy_loss(x, target=x, **{name: good})


@pytest.mark.parametrize("activation", [2, 3, 4])
def test_workspace_of_narrow_gradients(activation):
    """Both gradients narrow: dz in fp32, in rows of whole 16 bytes, and none in the operands' type."""
    lib = library()
    lib.gk_linear_grad_workspace_bytes.restype = ctypes.c_size_t
    lib.gk_linear_grad_workspace_bytes.argtypes = [ctypes.c_void_p]
    p = LinearGradStruct()
    p.dy = p.kept = p.x = p.w = p.dx = p.dw = 1 << 20
    p.m, p.n, p.k, p.dtype, p.activation = 7, 17, 64, 1, activation
    p.dy_stride, p.kept_stride, p.x_stride, p.w_stride = 17, 24, 64, 64

    def whole(size):
        return -(-size // 256) * 256

    assert lib.gk_linear_grad_workspace_bytes(ctypes.byref(p)) == whole(7 * 24 * 4)
    p.dz = 1 << 20  # the residual's gradient is written where it goes
    assert lib.gk_linear_grad_workspace_bytes(ctypes.byref(p)) == whole(7 * 24 * 4)
    p.dz, p.m = None, 4000  # dx takes tcgen05 and an aligned dz, dw the fp32 one
    p.n, p.dy_stride, p.w_stride = 16, 16, 64
    assert lib.gk_linear_grad_workspace_bytes(ctypes.byref(p)) == whole(4000 * 16 * 4) + whole(4000 * 16 * 2)
