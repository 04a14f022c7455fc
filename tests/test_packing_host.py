"""packed_activations around tensors that it keeps as they are: lifetime,
derivatives, changes in place. Runs on CPU tensors, none of which is packed."""

import gc
import weakref

import pytest
import torch


def contexts():
    from kingdom_ai import packed_activations
    from kingdom_ai.packing import keep_saved_tensors
    return packed_activations, keep_saved_tensors


@pytest.mark.parametrize("which", [0, 1])
def test_a_dropped_graph_is_freed(which):
    """An operator that keeps its own output (tanh, relu) does not keep itself alive."""
    gc.collect()
    gc.disable()
    try:
        for f in (torch.tanh, torch.relu, torch.exp):
            x = torch.randn(500, requires_grad=True)
            with contexts()[which]():
                y = f(x * 2)
            gone = weakref.ref(y)
            del y
            assert gone() is None
    finally:
        gc.enable()


@pytest.mark.parametrize("which", [0, 1])
def test_kept_tensors_give_first_and_second_derivatives(which):
    x, w = torch.randn(6, 5, dtype=torch.float64), torch.randn(4, 5, dtype=torch.float64)
    x.requires_grad_(), w.requires_grad_()

    def f():
        return torch.tanh(torch.sigmoid(x @ w.t()).square() * torch.exp(w.sum()))

    def derivatives():
        y = f()
        first = torch.autograd.grad(y.sum(), (x, w), create_graph=True)
        return first + torch.autograd.grad(sum(g.square().sum() for g in first), (x, w))

    want = derivatives()
    with contexts()[which]():
        got = derivatives()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("which", [0, 1])
def test_kept_tensors_that_change_in_place_are_refused(which):
    x = torch.randn(40, requires_grad=True)
    for change in (lambda a, y: a.mul_(2), lambda a, y: y.add_(1), lambda a, y: a[:3].zero_(),
                   lambda a, y: y.detach().neg_()):
        a = x * 2
        with contexts()[which]():
            y = torch.tanh(a)
            z = a * y  # keeps both
        change(a, y)
        with pytest.raises(RuntimeError, match="inplace"):
            z.sum().backward()
    a = x * 2
    with contexts()[which]():
        z = a.exp().sum()
    a.mul_(2)  # exp keeps its output, not its input
    z.backward()


def test_operators_that_change_their_own_input_run_as_before():
    """Each keeps its tensors after the change, or a copy; norms update their statistics from pass to pass."""
    from kingdom_ai import packed_activations
    torch.manual_seed(0)
    net = torch.nn.Sequential(torch.nn.Conv2d(3, 8, 3), torch.nn.BatchNorm2d(8), torch.nn.ReLU(inplace=True),
                              torch.nn.Conv2d(8, 4, 3), torch.nn.GroupNorm(2, 4), torch.nn.SiLU(inplace=True),
                              torch.nn.Flatten(), torch.nn.Linear(100, 10), torch.nn.Dropout(0.0, inplace=True))
    data = torch.randn(2, 6, 3, 9, 9)

    def gradients(context):
        net.zero_grad(set_to_none=True)
        with context:
            outs = []
            for x in data:  # both forward passes before either backward pass
                outs.append(net(x).mul_(2).tanh_())
        sum(o.square().sum() for o in outs).backward()
        return [p.grad for p in net.parameters()]

    import contextlib
    for a, b in zip(gradients(contextlib.nullcontext()), gradients(packed_activations(1))):
        assert torch.equal(a, b)


def test_a_packed_form_that_is_not_on_a_device_is_refused():
    from kingdom_ai import PackedActivation
    codes, scales = torch.zeros(64, dtype=torch.uint8), torch.zeros(2, dtype=torch.uint8)
    with pytest.raises(ValueError):
        PackedActivation(codes, scales, torch.Size([64]), torch.float32).unpack()
