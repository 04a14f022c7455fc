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
