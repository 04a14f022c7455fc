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


def test_packed_forms_that_do_not_fit_their_shape_are_refused():
    """Their fields are open: a form that was cut, moved or given another shape."""
    from kingdom_ai import PackedActivation, pack_activation
    p = pack_activation(values((10, 70), torch.float16))

    def form(codes=p.codes, scales=p.scales, shape=p.shape, dtype=p.dtype):
        return PackedActivation(codes, scales, shape, dtype)

    for bad in (form(shape=(11, 70)), form(shape=(10, 69)), form(codes=p.codes[:-1]), form(scales=p.scales[:-1]),
                form(codes=p.codes.cpu()), form(scales=p.scales.cpu()), form(codes=p.codes.short()),
                form(scales=p.scales.char()), form(codes=p.codes.repeat_interleave(2)[::2]),
                form(dtype=torch.float64), form(shape=(-10, -70)), form(shape=(1 << 40, 1 << 40, 700)),
                form(shape=(0, 1 << 62, 4))):
        with pytest.raises(ValueError):
            bad.unpack()
    assert torch.equal(form(shape=(700,)).unpack(), p.unpack().view(700))
    assert torch.equal(form(codes=p.codes.clone(), scales=p.scales.clone()).unpack(), p.unpack())
