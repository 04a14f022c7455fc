"""The training-step operators among PyTorch's own machinery: forward-mode
derivatives, saved-tensor hooks, inference mode, layouts that a view can have."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_forward_mode_derivatives_are_refused():
    """An output without a tangent would stand for a derivative of zero."""
    import torch.autograd.forward_ad as forward_ad
    from kingdom_ai import linear, policy_loss
    x, w, b, r = (torch.randn(s, device="cuda") for s in ((12, 16), (8, 16), (8,), (12, 8)))
    target = torch.softmax(torch.randn(12, 16, device="cuda"), 1)
    want, loss = linear(x, w, b, residual=r), policy_loss(x, target=target).loss
    with forward_ad.dual_level():
        for i in range(4):
            args = [forward_ad.make_dual(t, torch.ones_like(t)) if i == j else t for j, t in enumerate((x, w, b, r))]
            for grad in (False, True):  # whether autograd records or not
                args[0 if i else 1] = args[0 if i else 1].detach().requires_grad_(grad)
                with pytest.raises(NotImplementedError):
                    linear(*args[:3], residual=args[3])
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(NotImplementedError):
            policy_loss(dual, target=target)
        with pytest.raises(NotImplementedError):
            policy_loss(x, target=forward_ad.make_dual(target, torch.ones_like(target)))
        # Without a tangent they run inside the level too.
        assert torch.equal(linear(x, w, b, residual=r), want) and torch.equal(policy_loss(x, target=target).loss, loss)
        assert torch.equal(linear(forward_ad.unpack_dual(dual).primal, w, b, residual=r), want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_packed_inputs_whose_rows_lie_over_one_another(dtype):
    """Expanded and unfolded inputs, as linear takes them without a checkpoint."""
    from kingdom_ai import linear
    g = torch.Generator(device="cuda").manual_seed(1)
    flat = torch.randn(400, generator=g, device="cuda").to(dtype)
    w = (torch.randn((24, 40), generator=g, device="cuda") * 0.2).to(dtype).requires_grad_()
    dy = torch.randn((64, 24), generator=g, device="cuda").to(dtype)
    for x in (flat[:40].expand(64, 40), flat.unfold(0, 40, 5)[:64], torch.as_strided(flat, (64, 40), (0, 1), 7)):
        y, z = linear(x, w, activation="gelu", checkpoint="e4m3"), linear(x.contiguous(), w, activation="gelu",
                                                                          checkpoint="e4m3")
        assert torch.equal(y, z)
        assert torch.equal(torch.autograd.grad(y, w, dy)[0], torch.autograd.grad(z, w, dy)[0])


@pytest.mark.parametrize("name", ["relu", "tanh", None])
def test_graphs_dropped_inside_packed_activations_are_freed(name):
    from kingdom_ai import linear, packed_activations, policy_loss
    x = torch.randn(64, 96, device="cuda")
    w = torch.randn(32, 96, device="cuda", requires_grad=True)
    target = torch.softmax(torch.randn(64, 32, device="cuda"), 1)

    def forward():  # an evaluation that never runs its backward pass
        with packed_activations():
            y = linear(x, w, activation=name)
            policy_loss(torch.relu(y), target=target)

    forward()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    for _ in range(5):
        forward()
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() == before


def test_changes_in_place_are_refused_inside_packed_activations():
    from kingdom_ai import linear, packed_activations, policy_loss
    x = torch.randn(20, 32, device="cuda")
    w = torch.randn(16, 32, device="cuda", requires_grad=True)
    target = torch.softmax(torch.randn(20, 16, device="cuda"), 1)
    with packed_activations():
        y = linear(x, w, activation="relu")
        y.neg_()  # its slope is taken from the kept output
        z = linear(x, w)
        loss = policy_loss(z, target=target).loss
        z.add_(1)
    for out in (y.sum(), loss):
        with pytest.raises(RuntimeError, match="inplace"):
            out.backward()


def test_training_after_a_first_call_in_inference_mode():
    from kingdom_ai import check_linear, layers, linear
    x = torch.randn(20, 32, device="cuda")
    w = torch.randn(16, 32, device="cuda", requires_grad=True)
    want, = torch.autograd.grad(linear(x, w, activation="tanh").sum(), w)
    kept = dict(layers._status)
    layers._status.clear()
    try:
        with torch.inference_mode():  # serving comes first
            linear(x, w, activation="tanh")
        got, = torch.autograd.grad(linear(x, w, activation="tanh").sum(), w)
        assert torch.equal(got, want)
        # An error of another call, reported and cleared between forward and backward pass.
        y = linear(x, w, activation="tanh")
        layers._status[0][0] = 4
        with pytest.raises(RuntimeError, match="linear reported error bits 0x4"):
            check_linear()
        assert torch.equal(torch.autograd.grad(y.sum(), w)[0], want)
        check_linear()
    finally:
        layers._status.clear()
        layers._status.update(kept)


def test_check_linear_waits_for_every_stream():
    from kingdom_ai import check_linear, layers, linear
    linear(torch.randn(4, 8, device="cuda"), torch.randn(8, 8, device="cuda"))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)  # a tenth of a second of work before a product that gives up
        layers._status[0][:1].fill_(4)  # which does not wait, as an assignment of a number would
    with pytest.raises(RuntimeError, match="linear reported error bits 0x4"):
        check_linear()
    check_linear()
