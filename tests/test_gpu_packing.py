"""pack_activation: held values against the list of e4m3 numbers in 64 bits,
their error bounds, and packed_activations in a backward pass."""

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
GRID = torch.tensor([0.0] + [i * 2.0 ** -9 for i in range(1, 8)]
                    + [(1 + i / 8) * 2.0 ** e for e in range(-6, 9) for i in range(8) if (e, i) != (8, 7)],
                    dtype=torch.float64)


def held(x):
    """What a flat tensor's blocks of 32 hold, and each value's scale."""
    lowest = -15 if x.dtype == torch.float16 else -124
    flat = torch.nn.functional.pad(x.detach().reshape(-1).double().cpu(), (0, -x.numel() % 32)).reshape(-1, 32)
    finite = torch.where(flat.isfinite(), flat.abs(), 0.0)
    top = finite.amax(1, keepdim=True)
    power = torch.zeros_like(top)
    for i, t in enumerate(top.flatten().tolist()):
        if t > 0:
            s = -200
            while 448.0 * 2.0 ** s < t:
                s += 1
            power[i] = max(lowest, s)
    scale = torch.exp2(power)
    u = (finite / scale)
    above = torch.searchsorted(GRID, u.contiguous()).clamp_max(len(GRID) - 1)
    below = (above - 1).clamp_min(0)
    far, near = GRID[above] - u, u - GRID[below]
    value = torch.where((far < near) | ((far == near) & (above % 2 == 0)), GRID[above], GRID[below]) * scale
    most = torch.finfo(x.dtype).max
    value = torch.where(flat.isfinite(), (value * flat.sign()).clamp(-most, most), torch.full_like(flat, float("nan")))
    n = x.numel()
    return value.reshape(-1)[:n].reshape(x.shape), scale.expand_as(flat).reshape(-1)[:n].reshape(x.shape)


def values(shape, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(shape, generator=g, device="cuda") * torch.exp2(torch.randint(-12, 6, shape, generator=g,
                                                                                  device="cuda").float())
    return x.to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1,), (31,), (32,), (33,), (5, 7), (64, 81), (3, 64, 9, 9), (1000, 32), (4097, 24)])
def test_held_values(shape, dtype):
    from kingdom_ai import pack_activation
    x = values(shape, dtype)
    packed = pack_activation(x)
    assert packed.nbytes == x.numel() + -(-x.numel() // 32)
    got = packed.unpack()
    assert got.dtype == dtype and got.shape == x.shape
    want, scale = held(x)
    assert torch.equal(got.cpu().double(), want)
    assert torch.equal(packed.unpack(torch.float32).cpu().double(), want)
    error = (got.cpu().double() - x.cpu().double()).abs()
    # Half a step of three fraction bits, or half the smallest step of the block.
    assert bool((error <= torch.maximum(2.0 ** -4 * x.cpu().double().abs(), 2.0 ** -10 * scale)).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_extremes(dtype):
    from kingdom_ai import pack_activation
    info = torch.finfo(dtype)
    tiny = info.smallest_normal * info.eps
    x = torch.zeros(32 * 8, dtype=dtype, device="cuda")
    x[:32] = info.max
    x[32:64] = info.tiny
    x[64:96] = tiny                                  # the type's smallest subnormal
    x[96:128] = torch.linspace(-1, 1, 32) * info.max
    x[128], x[129], x[130], x[131] = float("nan"), float("inf"), float("-inf"), 3.0
    x[160:192] = -0.0
    x[192], x[193], x[194] = 448.0, 449.0, 1.0       # a maximum on and past the border of its scale
    x[224] = 448.0
    got, want = pack_activation(x).unpack().cpu().double(), held(x)[0]
    assert torch.equal(got.isnan(), want.isnan()) and int(got.isnan().sum()) == 3
    assert torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))
    assert bool(got[:128].isfinite().all()) and float(got[131]) == 3.0 and float(got[224]) == 448.0


def test_views_and_empty_tensors():
    from kingdom_ai import pack_activation
    x = values((40, 96), torch.bfloat16)
    for view in (x.t(), x[:, 1:50], x[::2], x[3:4].expand(7, 96), x[0, 0]):
        assert torch.equal(pack_activation(view).unpack().cpu().double(), held(view.contiguous())[0])
    none = pack_activation(torch.zeros(0, 5, device="cuda"))
    assert none.nbytes == 0 and none.unpack().shape == (0, 5)
    offset = torch.zeros(65, device="cuda")[1:]      # rows of whole blocks that do not start on 16 bytes
    offset.copy_(values((64,), torch.float32))
    assert torch.equal(pack_activation(offset).unpack().cpu().double(), held(offset)[0])


def test_large_tensor_both_ways():
    from kingdom_ai import pack_activation
    x = values((4096, 5184), torch.float32)
    packed = pack_activation(x)
    parts = [pack_activation(p).unpack() for p in x.reshape(8, -1)]
    assert torch.equal(packed.unpack().reshape(8, -1), torch.stack(parts))


def test_packed_activations_in_a_backward_pass():
    """Gradients are those of the held values, parameters are kept exact, the forward pass is unchanged."""
    from kingdom_ai import pack_activation, packed_activations
    x = values((64, 512), torch.float32).requires_grad_()
    w = torch.randn(512, 256, device="cuda", requires_grad=True)
    with packed_activations(min_elements=1024):
        y = x @ w
        z = y.square()
    assert torch.equal(z.detach(), (x @ w).square().detach())
    dz = torch.randn(64, 256, device="cuda")
    gx, gw = torch.autograd.grad(z, [x, w], dz)
    dy = dz * 2 * pack_activation(y).unpack()
    assert torch.equal(gx, dy @ w.t())               # x is a leaf that is trained: kept as it is
    assert torch.equal(gw, x.detach().t() @ dy)
    h = values((64, 512), torch.float32)             # an activation that is no leaf of the graph
    with packed_activations(min_elements=1024):
        y = h @ w
    gw, = torch.autograd.grad(y, w, dz)
    assert torch.equal(gw, pack_activation(h).unpack().t() @ dz)
    with packed_activations(min_elements=1 << 20):
        y = h @ w
    assert torch.equal(torch.autograd.grad(y, w, dz)[0], h.t() @ dz)


def test_packed_activations_saves_memory_and_keeps_cast_parameters():
    from kingdom_ai import packed_activations

    def kept(context):
        h = torch.randn(4096, 1024, device="cuda")
        w = torch.randn(1024, 1024, device="cuda", requires_grad=True)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        with context:
            y = h @ w
            for _ in range(4):
                y = torch.tanh(y)
        del h
        torch.cuda.synchronize()
        return torch.cuda.memory_allocated() - before, y

    import contextlib
    plain, y = kept(contextlib.nullcontext())
    del y
    packed, y = kept(packed_activations())
    assert packed < plain * 0.6
    y.sum().backward()
    w = torch.randn(512, 512, device="cuda", requires_grad=True)
    h = torch.randn(64, 512, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    with packed_activations(min_elements=1024):
        y = h @ w.to(torch.bfloat16)
    g, = torch.autograd.grad(y, h, torch.ones_like(y))
    assert torch.equal(g, torch.ones_like(y) @ w.detach().to(torch.bfloat16).t())


def test_frozen_parameters_are_kept():
    from kingdom_ai import packed_activations
    layer = torch.nn.Linear(512, 512, bias=False).cuda()
    layer.weight.requires_grad_(False)
    h = torch.randn(64, 512, device="cuda", requires_grad=True)
    with packed_activations(min_elements=1024):
        y = layer(h)
    g, = torch.autograd.grad(y, h, torch.ones_like(y))
    assert torch.equal(g, torch.ones_like(y) @ layer.weight)


def test_linear_and_policy_loss_keep_their_tensors_inside():
    from kingdom_ai import linear, packed_activations, policy_loss
    x = torch.randn(256, 512, device="cuda")
    w = (torch.randn(512, 512, device="cuda") * 0.05).requires_grad_()
    target = torch.softmax(torch.randn(256, 512, device="cuda"), 1)

    def grads():
        return torch.autograd.grad(policy_loss(linear(x, w, activation="gelu"), target=target).loss, w)[0]

    want = grads()
    with packed_activations(min_elements=1):
        assert torch.equal(grads(), want)


def test_refusals():
    from kingdom_ai import pack_activation
    with pytest.raises(TypeError):
        pack_activation([1.0])
    for bad in (torch.zeros(4), torch.zeros(4, device="cuda", dtype=torch.float64),
                torch.zeros(4, device="cuda", dtype=torch.int32)):
        with pytest.raises(ValueError):
            pack_activation(bad)
    with pytest.raises(ValueError):
        pack_activation(torch.zeros(4, device="cuda")).unpack(torch.float16)
