"""The operators together, as a training step uses them: a batch sampled from
the device replay buffer, the network's heads on linear, policy_loss, and the
activations in 8 bits."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def batch():
    from kingdom_ai import DeviceReplayBuffer
    from kingdom_ai.gpu_puct import GpuPUCTOptions
    from kingdom_ai.model import random_network
    from kingdom_ai.selfplay import SelfPlayEngine
    engine = SelfPlayEngine(random_network(64, 1, 5), 64, GpuPUCTOptions(simulations=8, seed=9),
                            replay_capacity=1 << 12)
    engine.step(60)
    n = min(engine.stats()["rows"], engine.replay.capacity)
    assert n >= 64
    buffer = DeviceReplayBuffer(1 << 12)
    buffer.ingest(engine.replay, 0, n)
    return buffer.sample(256, generator=torch.Generator().manual_seed(3))


def networks():
    from kingdom_ai.model import random_groupnorm_network, random_network
    yield random_network(64, 2, 1).cuda().train()
    yield random_groupnorm_network(32, 2, 2).cuda().train()


def exact(model, batch):
    """Loss terms and gradients of the module itself in 64 bits."""
    import copy
    model = copy.deepcopy(model).double()
    logits, values = model(batch.features.double())
    logits = logits.masked_fill(~batch.legal_mask, -torch.inf)
    t = batch.policy.double()
    logp = torch.where(t > 0, torch.log_softmax(logits, 1), 0.0)
    policy = (torch.special.xlogy(t, t) - t * logp).sum(1).mean()
    value = (values - batch.value.double()).square().mean()
    (policy + 0.5 * value).backward()
    return policy.detach(), value.detach(), {k: p.grad for k, p in model.named_parameters()}


def step(model, batch, **options):
    from kingdom_ai import check_linear, policy_value_loss
    model.zero_grad(set_to_none=True)
    out = policy_value_loss(model, batch, value_weight=0.5, **options)
    out.loss.backward()
    check_linear()
    return out, {k: p.grad.clone() for k, p in model.named_parameters()}


def norm_off(got, want):
    return float((got.double() - want).norm() / want.norm().clamp_min(1e-12))


def module_gradients(model, batch):
    """The same step on PyTorch's own heads and loss in fp32."""
    model.zero_grad(set_to_none=True)
    logits, values = model(batch.features)
    logp = torch.log_softmax(logits.masked_fill(~batch.legal_mask, -torch.inf), 1)
    policy = -torch.where(batch.policy > 0, batch.policy * logp, 0.0).sum(1).mean()
    (policy + 0.5 * (values - batch.value).square().mean()).backward()
    return {k: p.grad.clone() for k, p in model.named_parameters()}


def test_losses_and_gradients(batch):
    """The trunk is the same fp32 convolutions and norms on both sides, whose
    errors grow layer by layer; the operators add fp32 rounding of their own
    only, so no gradient is more than twice as far from the 64-bit one as
    PyTorch's own fp32 step is (1e-5 where that happens to be nearer)."""
    tf32 = torch.backends.cudnn.allow_tf32
    torch.backends.cudnn.allow_tf32 = False
    try:
        for model in networks():
            policy, value, want = exact(model, batch)
            theirs = module_gradients(model, batch)
            out, grads = step(model, batch)
            assert abs(float(out.policy - policy)) <= 1e-4 * (1 + float(policy))
            assert abs(float(out.value - value)) <= 1e-4 * (1 + float(value))
            assert abs(float(out.loss.detach()) - float(policy + 0.5 * value)) <= 2e-4 * (1 + float(policy + value))
            for name, g in want.items():
                assert norm_off(grads[name], g) <= 2 * norm_off(theirs[name], g) + 1e-5, name
    finally:
        torch.backends.cudnn.allow_tf32 = tf32


def test_eight_bit_checkpoints(batch):
    """The loss is the exact one bit for bit; a weight's gradient is off by
    what its packed input is off (each value by 2^-4 at most), and layer after
    layer by the packed values that activations and norms take their
    derivatives from: within 2^-4 a layer of the backward pass."""
    for model in networks():
        plain, exact_grads = step(model, batch)
        packed, grads = step(model, batch, checkpoint="e4m3")
        depth = sum(1 for _ in model.named_parameters())
        for name, g in exact_grads.items():
            assert norm_off(grads[name], g.double()) <= 2.0 ** -4 * depth, name
        # Only the heads' own input stands between these and the exact gradient.
        bias = "policy_fc.bias" if "policy_fc.bias" in grads else "policy_head.4.bias"
        assert norm_off(grads[bias], exact_grads[bias].double()) <= 1e-3
        assert abs(float(packed.policy - plain.policy)) <= 1e-4 * (1 + float(plain.policy))


def test_under_autocast(batch):
    """The heads take the trunk's bf16 (half step 2^-9 a value, at most eight roundings deep here)."""
    from kingdom_ai import policy_value_loss
    for model in networks():
        policy, value, _ = exact(model, batch)
        with torch.autocast("cuda", torch.bfloat16):
            out = policy_value_loss(model, batch, value_weight=0.5, checkpoint="e4m3")
        out.loss.backward()
        assert abs(float(out.loss.detach()) - float(policy + 0.5 * value)) <= 0.1 * (1 + float(policy + 0.5 * value))
        assert all(bool(p.grad.isfinite().all()) for p in model.parameters())


def test_forward_matches_the_module(batch):
    from kingdom_ai import training_forward
    for model in networks():
        model.eval()
        with torch.no_grad():
            want = model.double()(batch.features.double())
            got = training_forward(model.float(), batch.features)
        for g, w in zip(got, want):
            assert g.shape == w.shape and float((g.double() - w).abs().max()) <= 5e-3 * (1 + float(w.abs().max()))


def test_captured_step_updates_the_weights(batch):
    """A whole step (losses, gradients, update) replayed from a CUDA graph equals the eager one."""
    from kingdom_ai import policy_value_loss
    from kingdom_ai.model import random_groupnorm_network

    def make():
        model = random_groupnorm_network(32, 1, 4).cuda().train()
        return model, torch.optim.SGD(model.parameters(), lr=0.05)

    def one(model, optimiser):
        optimiser.zero_grad(set_to_none=True)
        out = policy_value_loss(model, batch, checkpoint="e4m3")
        out.loss.backward()
        optimiser.step()

    eager, optimiser = make()
    for _ in range(3):
        one(eager, optimiser)
    model, optimiser = make()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # warm up on another stream, as capture asks
        one(model, optimiser)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    optimiser.zero_grad(set_to_none=True)
    with torch.cuda.graph(graph):
        one(model, optimiser)
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(eager.parameters(), model.parameters()):
        # Three updates of at most 0.05 |g|; cuDNN may pick another algorithm under capture.
        assert float((a - b).abs().max().detach()) <= 1e-3 * (1 + float(a.abs().max().detach()))


def test_refusals(batch):
    from kingdom_ai import policy_value_loss, training_forward
    model = next(networks())
    for bad in (lambda: policy_value_loss(model, batch, value_weight=-1), lambda: policy_value_loss(
            model, batch, value_weight=float("nan")), lambda: policy_value_loss(model, batch, checkpoint="fp8"),
            lambda: training_forward(model, batch.features, checkpoint=1)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: policy_value_loss(torch.nn.Linear(1, 1), batch), lambda: policy_value_loss(
            model, batch, value_weight="1"), lambda: policy_value_loss(model, batch.features)):
        with pytest.raises(TypeError):
            bad()


def test_lazily_negated_views():
    """The imaginary part of a conjugate holds the negated values."""
    from kingdom_ai import linear, pack_activation, policy_loss
    g = torch.Generator(device="cuda").manual_seed(0)

    def negated(*shape):
        t = torch.randn(shape, generator=g, device="cuda")
        view = torch.complex(t, t).conj().imag
        assert view.is_neg()
        return view, torch.imag(torch.complex(t, t)).neg()

    (x, x1), (w, w1), (b, b1), (r, r1) = negated(40, 64), negated(24, 64), negated(24), negated(40, 24)
    assert torch.equal(linear(x, w, b, residual=r), linear(x1, w1, b1, residual=r1))
    w2 = w1.clone().requires_grad_()
    dy, dy1 = torch._neg_view(r), r1.neg()
    assert torch.equal(torch.autograd.grad(linear(x, w2), w2, dy)[0], torch.autograd.grad(linear(x1, w2), w2, dy1)[0])
    assert torch.equal(pack_activation(x).unpack(), pack_activation(x1).unpack())
    actions = torch.arange(40, device="cuda") % 64
    (old, old1), (adv, adv1) = negated(40), negated(40)
    assert torch.equal(policy_loss(x, actions=actions, old_log_probs=old, advantages=adv).loss,
                       policy_loss(x1, actions=actions, old_log_probs=old1, advantages=adv1).loss)
