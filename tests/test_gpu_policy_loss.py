"""policy_loss against its formula in 64 bits, loss, log-probabilities and gradient.

Tolerances are counted. With D the largest |z - M| that matters (40: beyond it
exp is below 1e-17) a term exp(z - M) is off by at most 2^-22 + D 2^-23 of
itself, and their sum of A terms by (A / 256 + 64) 2^-24 more (256 threads or
more, or 32 lanes of at most 8 terms, then trees): together `rel`. So log p is
off by rel and one fp32 rounding of it, a ratio by that times itself, and the
gradient by the terms' errors and one rounding to its type.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
ULP = 2.0 ** -23


def make(n, a, dtype, mask=False, clipped=True, target=None, reference=True, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + 1000 * n + a)
    logits = (torch.randn((n, a), generator=g, device="cuda") * 2).to(dtype)
    args = {}
    legal = torch.ones((n, a), dtype=torch.bool, device="cuda")
    if mask:
        legal = torch.rand((n, a), generator=g, device="cuda") < 0.4
        legal[:, -1] = True
        if n > 3:
            legal[1] = False       # nothing left
            legal[2] = False
            legal[2, a // 2] = True  # one entry left
        args["legal_mask"] = legal
    if target is not None:
        t = torch.rand((n, a), generator=g, device="cuda").pow(6) * legal
        t[:, ::3] = 0
        args["target"] = (t / t.sum(1, keepdim=True).clamp_min(1e-3)).to(target)
    if clipped:
        actions = (torch.rand((n, a), generator=g, device="cuda") * legal).argmax(1)
        if n > 3:
            actions[0] = -1
            actions[1 if mask else 0] = -7
        lp = torch.log_softmax(logits.double().masked_fill(~legal, -1e300), 1).gather(
            1, actions.clamp_min(0)[:, None])[:, 0]
        old = lp + torch.randn(n, generator=g, device="cuda").double() * 0.2
        for border in (0.8, 1.2):  # no ratio on a border
            old = torch.where(((lp - old).exp() - border).abs() < 1e-3, old + 0.01, old)
        args.update(actions=actions, old_log_probs=old.float().nan_to_num(0, 0, 0),
                    advantages=torch.randn(n, generator=g, device="cuda"))
        if reference:
            args.update(reference_log_probs=(lp.float() + torch.randn(n, generator=g, device="cuda") * 0.3
                                             ).nan_to_num(0, 0, 0), kl_weight=0.1)
    return logits, args


def formula(logits, legal_mask=None, actions=None, old_log_probs=None, advantages=None, reference_log_probs=None,
            target=None, clip=0.2, kl_weight=0.0, target_weight=1.0, denominator=None, upstream=1.0):
    """(loss, its error, log p, its error, gradient, its error)."""
    n, a = logits.shape
    z = logits.double()
    legal = torch.ones_like(z, dtype=torch.bool) if legal_mask is None else legal_mask
    z = torch.where(legal, z, torch.full_like(z, -math.inf))
    live = (z > -math.inf).any(1)
    if actions is not None:
        live = live & (actions >= 0)
    m = z.amax(1, keepdim=True)
    safe = torch.where(live[:, None], z - m, torch.zeros_like(z))
    p = torch.where(live[:, None], safe.exp(), 0.0)
    s = p.sum(1, keepdim=True).clamp_min(1e-300)
    p, logp_all = p / s, safe - s.log()
    rel = 2.0 ** -22 + 40 * ULP + (a / 256 + 64) * 2.0 ** -24
    scale = float(upstream) / (n if denominator is None else float(denominator))
    rows, erows = torch.zeros(n, dtype=torch.float64, device="cuda"), torch.zeros(n, dtype=torch.float64, device="cuda")
    c, ec = torch.zeros_like(rows), torch.zeros_like(rows)
    lp = torch.zeros_like(rows)
    if actions is not None:
        at = actions.clamp(0, a - 1)[:, None]
        lp = torch.where(live, logp_all.gather(1, at)[:, 0], 0.0)
        elp = rel + 2 * ULP * lp.abs()
        low, high = clip if isinstance(clip, tuple) else (clip, clip)
        q, adv = (lp - old_log_probs.double()).exp(), advantages.double()
        eq = q * (elp + 4 * ULP)
        held = q.clamp(1 - low, 1 + high)
        free = q * adv <= held * adv
        rows = -torch.minimum(q * adv, held * adv)
        erows = (eq + 4 * ULP) * adv.abs()
        c = torch.where(free, -q * adv, 0.0)
        ec = torch.where(free, erows, 0.0)
        if reference_log_probs is not None:
            d = reference_log_probs.double() - lp
            ed = elp + 4 * ULP * (1 + d.abs())
            rows = rows + kl_weight * (torch.expm1(d) - d)
            erows = erows + abs(kl_weight) * (d.exp() + 1) * ed
            c = c - kl_weight * torch.expm1(d)
            ec = ec + abs(kl_weight) * (d.exp() + 1) * ed
        rows, erows, c, ec = (torch.where(live, t, 0.0) for t in (rows, erows, c, ec))
    g = -c[:, None] * p
    eg = (ec + c.abs() * 2 * rel)[:, None] * p
    if actions is not None:
        g.scatter_add_(1, at, c[:, None])
        eg.scatter_add_(1, at, (ec + 2 * ULP * c.abs())[:, None])
    if target is not None:
        t = torch.where(legal & live[:, None], target.double(), 0.0)
        term = torch.where(t > 0, t * (t.clamp_min(1e-300).log() - logp_all), 0.0)
        rows = rows + target_weight * term.sum(1)
        erows = erows + target_weight * ((t * rel).sum(1) + (a / 256 + 80) * ULP * (
            t * (t.clamp_min(1e-300).log().abs() + safe.abs().nan_to_num(0, 0, 0) + 1 + s.log().abs())).sum(1))
        total = t.sum(1, keepdim=True)
        g = g + target_weight * (total * p - t)
        eg = eg + target_weight * ((2 * rel + (a / 256 + 64) * ULP) * total * p + 4 * ULP * (total * p + t))
    g, eg = g * scale, eg * abs(scale)
    info = torch.finfo(logits.dtype)
    eg = eg + info.eps / 2 * (g.abs() + eg) + info.smallest_normal * info.eps / 2
    div = n if denominator is None else float(denominator)
    loss = rows.sum() / div
    eloss = erows.sum() / abs(div) + 4 * ULP * loss.abs() + 1e-30
    elp = torch.where(live, rel + 2 * ULP * lp.abs(), 0.0)
    return loss, eloss, lp, elp, g, eg


def run(logits, args, upstream=None):
    from kingdom_ai import policy_loss
    z = logits.detach().requires_grad_()
    out = policy_loss(z, **args)
    grad, = torch.autograd.grad(out.loss, z, None if upstream is None else torch.full((), upstream, device="cuda"))
    return out, grad


def compare(logits, args, upstream=None):
    from kingdom_ai import policy_loss
    out, grad = run(logits, args, upstream)
    loss, eloss, lp, elp, g, eg = formula(logits, **args, upstream=1.0 if upstream is None else upstream)
    out = out._replace(loss=out.loss.detach())
    assert out.loss.dtype == torch.float32 and grad.dtype == logits.dtype
    assert abs(float(out.loss) - float(loss)) <= float(eloss), (float(out.loss), float(loss), float(eloss))
    if "actions" in args:
        assert bool(((out.log_probs.double() - lp).abs() <= elp).all())
    else:
        assert out.log_probs is None
    off = (grad.double() - g).abs()
    assert bool((off <= eg).all()), float((off / eg).max())
    with torch.no_grad():
        alone = policy_loss(logits, **args)
    assert torch.equal(alone.loss, out.loss)
    return out, grad


# Around a warp's row (256), vectors, the parts of clusters (4608 vectors of 16 bytes a CTA) and
# rows past a cluster's shared memory, odd lengths among them.
SHAPES = [(1, 1), (1, 2), (5, 82), (300, 82), (9, 97), (4, 255), (4, 256), (4, 257), (700, 300), (5, 1001), (3, 8193),
          (40, 20011), (2, 65536), (5, 131075), (1, 300007)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,a", SHAPES)
def test_shapes(n, a, dtype):
    compare(*make(n, a, dtype))
    compare(*make(n, a, dtype, mask=True, clipped=False, target=torch.float32))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("a", [82, 1003])
@pytest.mark.parametrize("mask", [False, True])
def test_terms(dtype, a, mask):
    for target in (None, torch.float32, dtype):
        for clipped, reference in ((True, False), (True, True), (False, False)):
            if clipped or target is not None:
                compare(*make(33, a, dtype, mask, clipped, target, reference))


def test_more_rows_than_the_grid():
    compare(*make(20000, 82, torch.float32, True, True, torch.float32))
    compare(*make(6000, 260, torch.bfloat16))


@pytest.mark.parametrize("upstream", [1024.0, -0.5, 0.0])
@pytest.mark.parametrize("dtype", TYPES)
def test_upstream_gradient(dtype, upstream):
    """The gradient that the forward pass made is for one; any other is formed anew, with one rounding."""
    for a in (82, 4099):
        compare(*make(21, a, dtype, True, True, torch.float32), upstream)


def test_second_backward_pass_over_one_graph():
    from kingdom_ai import policy_loss
    logits, args = make(50, 3001, torch.bfloat16)
    z = logits.requires_grad_()
    out = policy_loss(z, **args)
    first, = torch.autograd.grad(out.loss, z, retain_graph=True)
    kept = first.clone()
    second, = torch.autograd.grad(out.loss, z, torch.full((), 2.0, device="cuda"), retain_graph=True)
    third, = torch.autograd.grad(out.loss, z)
    assert torch.equal(first, kept) and torch.equal(second, 2 * first) and torch.equal(third, first)
    assert first.data_ptr() != second.data_ptr()


def test_options():
    logits, args = make(37, 82, torch.float32, True, True, torch.float32)
    for change in (dict(clip=(0.1, 0.4)), dict(clip=0.0), dict(denominator=5.5), dict(target_weight=0.25),
                   dict(kl_weight=-0.5), dict(target_weight=0.0, kl_weight=0.0)):
        got = {**args, **change}
        if change.get("clip") is not None:  # keep ratios off the moved borders
            low, high = change["clip"] if isinstance(change["clip"], tuple) else (change["clip"],) * 2
            lp = formula(logits, **got)[2]
            old = got["old_log_probs"]
            for border in (1 - low, 1 + high):
                near = ((lp - old.double()).exp() - border).abs() < 1e-3
                old = torch.where(near, old + 0.02, old)
            got["old_log_probs"] = old
        compare(logits, got)
    count = torch.full((1,), 29.0, device="cuda")
    a, ga = run(logits, {**args, "denominator": count})
    b, gb = run(logits, {**args, "denominator": 29.0})
    assert torch.equal(a.loss, b.loss) and torch.equal(ga, gb)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("a", [82, 500, 9001])
def test_masked_entries_may_hold_anything(dtype, a):
    logits, args = make(12, a, dtype, True, True, torch.float32)
    want, gw = run(logits, args)
    legal = args["legal_mask"]
    for junk in (float("nan"), float("inf"), float("-inf"), torch.finfo(dtype).min, torch.finfo(dtype).max):
        dirty = logits.masked_fill(~legal, junk)
        t = args["target"].masked_fill(~legal, junk if math.isnan(junk) else 7.0)
        got, gg = run(dirty, {**args, "target": t})
        assert torch.equal(got.loss, want.loss) and torch.equal(got.log_probs, want.log_probs)
        assert torch.equal(gg, gw) and not gg[~legal].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("a", [82, 700, 30001])
def test_infinities_and_lowest_values_as_masks(dtype, a):
    """Logits masked by -inf or by the type's lowest value; rows of nothing else."""
    logits, _ = make(6, a, dtype)
    logits[:, 1::2] = -math.inf
    logits[3] = -math.inf                      # nothing left
    logits[4] = torch.finfo(dtype).min         # uniform
    logits[5, 0::2] = torch.finfo(dtype).min   # -inf and the lowest value: uniform over the latter
    logits[2, 0] = 3e4                         # one entry far above the rest
    actions = torch.zeros(6, dtype=torch.int64, device="cuda")
    args = dict(actions=actions, old_log_probs=torch.full((6,), -1.0, device="cuda"),
                advantages=torch.ones(6, device="cuda"), clip=1e4)
    out, grad = run(logits, args)
    zero = torch.zeros(6, device="cuda")
    assert float(out.log_probs[3]) == 0.0 and not grad[3].any()
    # Its sum is one term, 2^r (1 +- 2^-22) undone by 2^-r (1 +- 2^-22).
    assert abs(float(out.log_probs[2])) <= 2.0 ** -21
    assert abs(float(out.log_probs[4]) + math.log(a)) <= 40 * ULP
    assert abs(float(out.log_probs[5]) + math.log((a + 1) // 2)) <= 40 * ULP
    assert bool(grad.isfinite().all()) and not grad[:4, 1::2].any() and not grad[5, 1::2].any()
    # Padding rows may hold NaN.
    logits[0] = float("nan")
    actions[0] = -1
    out, grad = run(logits, args)
    assert bool(out.loss.isfinite()) and not grad[0].any() and float(out.log_probs[0]) == float(zero[0])
    # A row that is not padding passes its NaN on, and only its own gradient has it.
    actions[0] = 0
    out, grad = run(logits, args)
    assert bool(out.loss.isnan()) and bool(grad[0].isnan().any()) and bool(grad[1:].isfinite().all())


@pytest.mark.parametrize("a", [82, 3000])
def test_actions_that_are_not_legal(a):
    logits, args = make(8, a, torch.float32, True)
    legal = args["legal_mask"]
    for action in (a, 1 << 40, int((~legal[5]).nonzero()[0])):
        bad = args["actions"].clone()
        bad[5] = action
        out, grad = run(logits, {**args, "actions": bad})
        assert bool(out.loss.isnan()) and bool(out.log_probs[5].isnan()) and bool(grad[5][legal[5]].isnan().all())
        others = [i for i in range(8) if i != 5]
        assert bool(grad[others].isfinite().all()) and bool(out.log_probs[others].isfinite().all())


@pytest.mark.parametrize("dtype", TYPES)
def test_strided_rows(dtype):
    for a in (82, 1500, 9003):
        logits, args = make(10, a, dtype, True, True, dtype)
        want, gw = run(logits, args)
        # Strides that keep the vectors in step, that do not, and transposed storage.
        for pad in (0, 8, 5):
            wide = torch.zeros(10, a + pad, dtype=dtype, device="cuda")
            wide[:, :a] = logits
            legal = torch.ones(10, a + 16, dtype=torch.bool, device="cuda")
            legal[:, 16:] = args["legal_mask"]
            got, gg = run(wide[:, :a], {**args, "legal_mask": legal[:, 16:]})
            # Other vectors add up in another order.
            assert abs(float((got.loss - want.loss).detach())) <= 2 * float(formula(logits, **args)[1])
            assert bool(((gg.double() - gw.double()).abs() <= 2 * formula(logits, **args)[5]).all())
        got, gg = run(logits.t().contiguous().t(), {**args, "target": args["target"].t().contiguous().t()})
        assert torch.equal(got.loss, want.loss) and torch.equal(gg, gw)


def test_gradient_against_differences():
    logits, args = make(6, 40, torch.float32, True, True, torch.float32)
    from kingdom_ai import policy_loss
    _, grad = run(logits, args)
    lp = formula(logits, **args)[2]
    live = args["actions"] >= 0
    q, e = (lp - args["old_log_probs"].double()).exp(), (args["reference_log_probs"].double() - lp).exp()
    for seed in range(3):
        direction = torch.randn(logits.shape, generator=torch.Generator().manual_seed(seed)).cuda()
        h = 2.0 ** -6
        with torch.no_grad():
            up = policy_loss(logits + h * direction, **args).loss.double()
            down = policy_loss(logits - h * direction, **args).loss.double()
        # Along d, whose entries spread by R in a row, log p has derivatives of at most R, R^2 / 4 and R^3 / 10;
        # q A and e^d so have third ones of at most (1 + 3 / 4 + 1 / 10) R^3 times themselves, a little more over
        # the step: 2 R^3. The target's term has R^3 / 10. The difference is off by h^2 / 6 of these, and by the
        # two losses' rounding over 2 h. Where the step (log q moves by h R at most) passes a clipping border, the
        # slope jumps by at most q A R, over at most half of the step.
        spread = (direction.amax(1) - direction.amin(1)).double()
        third = torch.where(live, spread ** 3 * (2 * q * args["advantages"].abs() + 0.1 * 2 * e + 0.1), 0.0).mean()
        passes = torch.minimum((q / 0.8).log().abs(), (q / 1.2).log().abs()) <= h * spread
        jump = torch.where(live & passes, q * args["advantages"].abs() * spread / 2, 0.0).mean()
        assert abs(float((up - down) / (2 * h) - (grad.double() * direction.double()).sum())) <= float(
            third * h * h / 6 + jump) + 64 * ULP / h


def test_empty_batch_streams_and_captured_graphs():
    from kingdom_ai import policy_loss
    z = torch.zeros(0, 82, device="cuda", requires_grad=True)
    out = policy_loss(z, target=torch.zeros(0, 82, device="cuda"))
    assert float(out.loss.detach()) == 0.0 and torch.autograd.grad(out.loss, z)[0].shape == (0, 82)
    pairs = [make(60, 5000, torch.bfloat16, seed=s) for s in (1, 2)]
    want = [run(*p) for p in pairs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out, grad = run(*pairs[0])
    torch.cuda.synchronize()
    assert torch.equal(out.loss, want[0][0].loss) and torch.equal(grad, want[0][1])
    want = [(o.loss.detach().clone(), g.clone()) for o, g in want]
    del out
    graphs = []
    for logits, args in pairs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, grad = run(logits, args)
        graphs.append((graph, out.loss.detach(), grad))
        del out
    for _ in range(2):
        for graph, loss, grad in graphs:
            loss.zero_()
            grad.zero_()
        for graph, _, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for (_, loss, grad), (l, g) in zip(graphs, want):
            assert torch.equal(loss, l) and torch.equal(grad, g)


def test_refusals():
    from kingdom_ai import policy_loss
    logits, args = make(4, 82, torch.float32, True, True, torch.float32)
    grad = torch.zeros(4, device="cuda", requires_grad=True)
    bad = [dict(), {**args, "actions": None}, {**args, "old_log_probs": None}, {**args, "advantages": None},
           {**args, "actions": args["actions"].int()}, {**args, "actions": args["actions"][:3]},
           {**args, "advantages": args["advantages"].double()}, {**args, "advantages": grad},
           {**args, "legal_mask": args["legal_mask"].byte()}, {**args, "legal_mask": args["legal_mask"][:, :81]},
           {**args, "target": args["target"].half()}, {**args, "target": args["target"].clone().requires_grad_()},
           {**args, "clip": -0.1}, {**args, "clip": float("nan")}, {**args, "denominator": 0},
           {**args, "denominator": -1.0}, {**args, "denominator": torch.ones(2, device="cuda")},
           {**args, "denominator": torch.ones(1)}, {**args, "kl_weight": float("inf")},
           {**args, "old_log_probs": args["old_log_probs"].cpu()}]
    for kw in bad:
        with pytest.raises(ValueError):
            policy_loss(logits, **kw)
    for kw in ({**args, "clip": "0.2"}, {**args, "kl_weight": None}, {**args, "target_weight": True},
               {**args, "legal_mask": [True]}, {**args, "advantages": 1.0}):
        with pytest.raises(TypeError):
            policy_loss(logits, **kw)
    for z in (logits.double(), logits[0], logits[:, :0]):
        with pytest.raises(ValueError):
            policy_loss(z, target=z)
    # A kept input that was changed in place is refused.
    z = logits.clone().requires_grad_()
    out = policy_loss(z, **args)
    args["advantages"].add_(1)
    with pytest.raises(RuntimeError):
        out.loss.backward()
