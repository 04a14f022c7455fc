"""pack_activation where single blocks take another path than their
neighbours: values that are not finite, anywhere."""

import pytest
import torch

from test_gpu_packing import TYPES, held, values

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("share", [0.002, 0.02, 0.5])
def test_blocks_that_are_not_finite_among_others(dtype, share):
    """Every mixture of the blocks that a warp holds, each with its own scale."""
    from kingdom_ai import pack_activation
    x = values((300, 1056), dtype, seed=3)
    g = torch.Generator(device="cuda").manual_seed(4)
    for bad in (float("nan"), float("inf"), float("-inf")):
        x[torch.rand(x.shape, generator=g, device="cuda") < share / 3] = bad
    x[7] = float("nan")  # whole blocks of nothing else
    packed = pack_activation(x)
    got, want = packed.unpack().cpu().double(), held(x)[0]
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))
    # The codes are the same bits as those of one block at a time.
    rows = [pack_activation(x[i]) for i in (0, 7, 299)]
    codes = packed.codes.view(300, 1056)
    assert all(torch.equal(codes[i], r.codes) for i, r in zip((0, 7, 299), rows))
    assert torch.equal(packed.unpack(torch.float32).isnan(), x.isnan() | x.isinf())
