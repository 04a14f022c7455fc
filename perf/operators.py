"""The training-step operators and how they are measured.

Three operators of one training step on replay rows, and the same operators at
the sizes of a language model's layers and vocabularies:

- ``linear``: ``act(x @ W.T + bias + residual)``, forward, backward, and the
  few-row form of serving;
- the 8-bit activation checkpoint: ``pack_activation`` / ``unpack``, and
  ``linear(checkpoint="e4m3")``, whose weight gradient reads the packed input;
- ``policy_loss``: the clipped ratio loss with a KL term, and the KL of a
  target distribution (visit shares) to the masked softmax, with its gradient.

Where ``own`` is false, ``run`` computes them with elementary torch operations
in 32 bits (64 for the sums over rows), rounded once to the output's type.
"""

import functools
import math
import sys
from pathlib import Path

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
BLOCK = 32               # values that share a scale
CLIP = 0.2
KL_WEIGHT = 0.05
TARGET_WEIGHT = 1.0
LOSS_SCALE = 1024.0
MAX_PRODUCT = 8192 * 4096 * 8192
MAX_LOGITS = 4096 * 128000


@functools.lru_cache(maxsize=None)
def framework():
    package = str(Path(__file__).resolve().parent.parent / "alpha-yoo-for-great-kingdom_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    import kingdom_ai
    return kingdom_ai


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # A small minibatch of replay rows: 82 actions, the legal mask, visit shares as the target. Latency.
        {"name": "loss-game-256", "op": "loss", "rows": 256, "cols": 82, "dtype": "fp32", "mask": True,
         "clipped": False, "target": "fp32"},
        # A whole collection's rows at once, with the played action's clipped ratio and KL terms beside the target.
        {"name": "loss-game-65536", "op": "loss", "rows": 65536, "cols": 82, "dtype": "fp32", "mask": True,
         "clipped": True, "target": "fp32"},
        # Seven tokens of an odd vocabulary: one row is split over several SMs.
        {"name": "loss-vocab-7x100003", "op": "loss", "rows": 7, "cols": 100003, "dtype": "bf16", "mask": False,
         "clipped": True, "target": ""},
        # A distillation batch: a half-precision target distribution over an odd vocabulary.
        {"name": "loss-target-1024x32771", "op": "loss", "rows": 1024, "cols": 32771, "dtype": "fp16", "mask": False,
         "clipped": False, "target": "fp16"},
        # A policy-gradient batch of 4096 tokens over a large vocabulary: memory traffic.
        {"name": "loss-vocab-4096x128000", "op": "loss", "rows": 4096, "cols": 128000, "dtype": "bf16", "mask": False,
         "clipped": True, "target": ""},
        # The policy head of the 6x64 network at the self-play batch: 162 -> 82, fp32, rows not 16-byte aligned.
        {"name": "linear-head-4096", "op": "linear", "rows": 4096, "inner": 162, "cols": 82, "dtype": "fp32",
         "activation": "", "bias": True, "residual": False, "train": True, "packed": False},
        # One token through a wide layer: the weights are read once.
        {"name": "linear-serve-1", "op": "linear", "rows": 1, "inner": 4096, "cols": 12288, "dtype": "bf16",
         "activation": "gelu", "bias": True, "residual": False, "train": False, "packed": False},
        # A few tens of tokens in flight, down projection with the residual.
        {"name": "linear-serve-37", "op": "linear", "rows": 37, "inner": 8192, "cols": 4096, "dtype": "bf16",
         "activation": "", "bias": True, "residual": True, "train": False, "packed": False},
        # Odd sizes throughout: no row of any operand starts on a 16-byte boundary.
        {"name": "linear-odd-train", "op": "linear", "rows": 1037, "inner": 1531, "cols": 2051, "dtype": "fp16",
         "activation": "silu", "bias": True, "residual": False, "train": True, "packed": False},
        # A training step of a wide layer: three products, bias, residual and activation.
        {"name": "linear-train-8192", "op": "linear", "rows": 8192, "inner": 4096, "cols": 8192, "dtype": "bf16",
         "activation": "gelu", "bias": True, "residual": True, "train": True, "packed": False},
        # The same kind of step with the input kept in 8 bits for the backward pass.
        {"name": "packed-train-8192", "op": "linear", "rows": 8192, "inner": 4096, "cols": 4096, "dtype": "bf16",
         "activation": "relu", "bias": True, "residual": False, "train": True, "packed": True},
        # A convolution's saved input at 64 channels, fp32: packed in the forward pass, unpacked in the backward pass.
        {"name": "packed-conv-4096", "op": "pack", "rows": 4096, "cols": 64 * 81, "dtype": "fp32"},
    ]


def _size(rng, low, high):
    """A whole number spread over the logarithm of [low, high]."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["loss", "loss", "linear", "linear", "linear", "pack"])
    dtype = rng.choice(["bf16", "fp16", "fp32"])
    if op == "pack":
        rows = _size(rng, 1, 16384)
        return {"op": op, "rows": rows, "cols": _size(rng, 1, min(16384, 4096 * 64 * 81 // rows)), "dtype": dtype}
    if op == "loss":
        if rng.random() < 0.4:  # replay rows
            clipped = rng.random() < 0.5
            return {"op": op, "rows": _size(rng, 1, 65536), "cols": 82, "dtype": dtype, "mask": True,
                    "clipped": clipped, "target": "fp32"}
        rows = _size(rng, 1, 8192)
        cols = _size(rng, 2, min(131072, MAX_LOGITS // rows))
        target = rng.choice(["", "fp32", dtype])
        if target:
            rows = min(rows, max(1, MAX_LOGITS // 4 // cols))
        return {"op": op, "rows": rows, "cols": cols, "dtype": dtype, "mask": rng.random() < 0.25,
                "clipped": not target or rng.random() < 0.5, "target": target}
    train = rng.random() < 0.6
    rows = _size(rng, 1, 16384 if train else 512)
    inner = _size(rng, 1, 8192)
    most = MAX_PRODUCT if dtype != "fp32" else MAX_PRODUCT // 32
    cols = _size(rng, 1, max(1, min(16384, most // (rows * inner))))
    rows = max(1, min(rows, most // (inner * cols)))
    return {"op": op, "rows": rows, "inner": inner, "cols": cols, "dtype": dtype,
            "activation": rng.choice(["", "relu", "tanh", "gelu", "silu"]), "bias": rng.random() < 0.7,
            "residual": rng.random() < 0.4, "train": train, "packed": train and rng.random() < 0.3}


# ------------------------------------------------------------------ the inputs

def _logits(case, g):
    return (torch.randn((case["rows"], case["cols"]), generator=g, device="cuda") * 2.0).to(TYPES[case["dtype"]])


def _prepare_loss(case, g):
    n, a = case["rows"], case["cols"]
    state = {"op": "loss", "logits": _logits(case, g).requires_grad_(), "mask": None, "actions": None, "old": None,
             "advantages": None, "reference": None, "target": None,
             # Half-precision training scales its loss so that small gradients stay above the type's smallest values.
             "scale": torch.full((), LOSS_SCALE, device="cuda") if case["dtype"] == "fp16" else None}
    # About one row in 33 is padding: no action and, with a mask, nothing legal.
    padded = torch.rand(n, generator=g, device="cuda") < 0.03
    if n < 8:
        padded.zero_()
    legal = None
    if case["mask"]:
        share = torch.rand((n, 1), generator=g, device="cuda") * 0.9 + 0.05
        legal = torch.rand((n, a), generator=g, device="cuda") < share
        legal[:, -1] = True  # passing is always legal
        legal &= ~padded[:, None]
        state["mask"] = legal
    if case["target"]:
        # Visit shares: whole counts over a few of the actions, divided by their sum.
        kind = TYPES[case["target"]]
        target = torch.empty((n, a), dtype=kind, device="cuda")
        step = max(1, (1 << 26) // a)
        for i in range(0, n, step):
            r = torch.rand((min(step, n - i), a), generator=g, device="cuda")
            c = torch.floor(r.pow(8) * 400)
            c[:, -1] += 1
            if legal is not None:
                c *= legal[i:i + step]
            target[i:i + step] = (c / c.sum(1, keepdim=True).clamp_min(1)).to(kind)
        state["target"] = target
    if case["clipped"]:
        if legal is None:
            actions = torch.randint(a, (n,), generator=g, device="cuda")
        else:
            actions = (torch.rand((n, a), generator=g, device="cuda") * legal).argmax(1)
        logp = torch.empty(n, dtype=torch.float64, device="cuda")
        step = max(1, (1 << 26) // a)
        with torch.no_grad():
            for i in range(0, n, step):
                x = state["logits"][i:i + step].double()
                if legal is not None:
                    x = x.masked_fill(~legal[i:i + step], -math.inf)
                top = x.amax(1, keepdim=True).clamp_min(-1e30)
                lse = (x - top).exp().sum(1).log() + top[:, 0]
                logp[i:i + step] = x.gather(1, actions[i:i + step, None])[:, 0] - lse
        logp = torch.where(padded, torch.zeros_like(logp), logp)
        old = logp + torch.randn(n, generator=g, device="cuda").double() * 0.15
        # No ratio lies so near a clipping border that the last bit decides the gradient.
        ratio = (logp - old).exp()
        near = ((ratio - (1 - CLIP)).abs() < 1e-3) | ((ratio - (1 + CLIP)).abs() < 1e-3)
        state["old"] = torch.where(near, old + 0.01, old).float()
        state["reference"] = (logp + torch.randn(n, generator=g, device="cuda").double() * 0.2).float()
        state["advantages"] = torch.randn(n, generator=g, device="cuda")
        state["actions"] = torch.where(padded, torch.full_like(actions, -1), actions)
    return state


def _prepare_linear(case, g):
    m, k, n = case["rows"], case["inner"], case["cols"]
    kind = TYPES[case["dtype"]]

    def normal(shape, scale):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(kind)

    # Inputs come out of a normalisation or an activation, weights are scaled by their fan-in.
    x = normal((m, k), 1.0)
    if case["activation"] in ("relu", ""):
        x = x.clamp_min(0)
    w = normal((n, k), math.sqrt(1.0 / k))
    b = normal((n,), 0.1) if case["bias"] else None
    r = normal((m, n), 0.5) if case["residual"] else None
    state = {"op": "linear", "x": x, "w": w, "b": b, "r": r, "activation": case["activation"] or None,
             "train": case["train"], "packed": case["packed"], "dy": None}
    if case["train"]:
        dy = normal((m, n), 0.05)
        if case["activation"] == "relu" and case["dtype"] == "fp32":
            # No gradient where the sum is so near the corner of the relu that the last bit decides it.
            z = x.double() @ w.double().t()
            z = z if b is None else z + b.double()
            z = z if r is None else z + r.double()
            dy = dy.masked_fill(z.abs() < 1e-4, 0)
        state["dy"] = dy
        for t in (x, w, b, r):
            if t is not None:
                t.requires_grad_()
    return state


def _prepare_pack(case, g):
    # A convolution's input: half of it zero, a few far larger values, and blocks that are zero throughout.
    x = torch.randn((case["rows"], case["cols"]), generator=g, device="cuda").clamp_min(0)
    x *= torch.where(torch.rand(x.shape, generator=g, device="cuda") < 0.002, 20.0, 1.0)
    x *= torch.rand((case["rows"], 1), generator=g, device="cuda") > 0.02
    return {"op": "pack", "x": x.to(TYPES[case["dtype"]])}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {"loss": _prepare_loss, "linear": _prepare_linear, "pack": _prepare_pack}[case["op"]](case, g)


# ------------------------------------------------------------------ the plain forms

def _plain_loss(state):
    logits, mask, target, actions = state["logits"].detach(), state["mask"], state["target"], state["actions"]
    n = logits.shape[0]
    z = logits.float()
    if mask is not None:
        z = z.masked_fill(~mask, -math.inf)
    top = z.amax(1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    e = torch.exp(z - top)
    total = e.sum(1, keepdim=True)
    some = total[:, 0] > 0
    total = torch.where(total > 0, total, torch.ones_like(total))
    p = e / total
    lse = torch.log(total) + top
    rows = torch.zeros(n, dtype=torch.float32, device=z.device)
    grad = torch.zeros_like(p)
    counted = some if actions is None else some & (actions >= 0)
    logp = torch.zeros_like(rows)
    if actions is not None:
        at = actions.clamp_min(0)[:, None]
        logp = torch.where(counted, (z.gather(1, at) - lse)[:, 0], torch.zeros_like(rows))
        ratio = torch.exp(logp - state["old"])
        a = state["advantages"]
        free, held = ratio * a, ratio.clamp(1 - CLIP, 1 + CLIP) * a
        d = state["reference"] - logp
        rows = -torch.minimum(free, held) + KL_WEIGHT * (torch.expm1(d) - d)
        slope = torch.where(free <= held, -free, torch.zeros_like(free)) - KL_WEIGHT * torch.expm1(d)
        rows = torch.where(counted, rows, torch.zeros_like(rows))
        slope = torch.where(counted, slope, torch.zeros_like(slope))
        grad -= slope[:, None] * p
        grad.scatter_add_(1, at, slope[:, None])
    if target is not None:
        t = target.float()
        t = t * counted[:, None] if mask is None else torch.where(mask & counted[:, None], t, torch.zeros_like(t))
        log_t = torch.log(torch.where(t > 0, t, torch.ones_like(t)))
        log_p = torch.where(t > 0, z - lse, torch.zeros_like(z))
        rows = rows + TARGET_WEIGHT * (t * (log_t - log_p)).sum(1)
        grad += TARGET_WEIGHT * (t.sum(1, keepdim=True) * p - t)
    loss = (rows.double().sum() / n).float()
    step = 1.0 / n if state["scale"] is None else state["scale"] / n
    out = {"loss": loss, "grad": (grad * step).to(logits.dtype)}
    if actions is not None:
        out["log_probs"] = logp
    return out


def _plain_pack(x, cols):
    """The values that 8 bits hold: e4m3 with a power-of-two scale for every 32 values of a row of `cols`."""
    rows = x.reshape(-1, cols).float()
    short = -cols % BLOCK
    v = torch.nn.functional.pad(rows, (0, short)).reshape(rows.shape[0], -1, BLOCK)
    part, power = torch.frexp(v.abs().amax(2, keepdim=True))
    power = torch.where(part > 0.875, power - 8, power - 9)  # the largest e4m3 value is 448 = 0.875 * 2**9
    lowest = -15 if x.dtype == torch.float16 else -124
    power = torch.where(part > 0, power, torch.zeros_like(power)).clamp_min(lowest)
    scale = torch.exp2(power.double()).float()
    held = (v / scale).to(torch.float8_e4m3fn).float() * scale
    most = torch.finfo(x.dtype).max
    return held.clamp(-most, most).reshape(rows.shape[0], -1)[:, :cols].reshape(x.shape)


def _act(z, name):
    if name == "relu":
        return z.clamp_min(0)
    if name == "tanh":
        return torch.tanh(z)
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if name == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _slope(z, name):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "tanh":
        return 1 - torch.tanh(z).square()
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if name == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    return torch.ones_like(z)


def _plain_linear(state):
    x, w, b, r = (None if t is None else t.detach() for t in (state["x"], state["w"], state["b"], state["r"]))
    z = x.float() @ w.float().t()
    if b is not None:
        z = z + b.float()
    if r is not None:
        z = z + r.float()
    out = {"y": _act(z, state["activation"]).to(x.dtype)}
    if state["train"]:
        dz = state["dy"].float() * _slope(z, state["activation"])
        kept = _plain_pack(x, x.shape[1]) if state["packed"] else x.float()
        out["dx"] = (dz @ w.float()).to(x.dtype)
        out["dw"] = (dz.t() @ kept).to(w.dtype)
        if b is not None:
            out["db"] = dz.sum(0).to(b.dtype)
        if r is not None:
            out["dr"] = dz.to(r.dtype)
    return out


# ------------------------------------------------------------------ one pass

def _own_loss(state):
    out = framework().policy_loss(state["logits"], legal_mask=state["mask"], actions=state["actions"],
                                  old_log_probs=state["old"], advantages=state["advantages"],
                                  reference_log_probs=state["reference"], target=state["target"], clip=CLIP,
                                  kl_weight=KL_WEIGHT, target_weight=TARGET_WEIGHT)
    grad, = torch.autograd.grad(out.loss, [state["logits"]], state["scale"])
    got = {"loss": out.loss.detach(), "grad": grad}
    if state["actions"] is not None:
        got["log_probs"] = out.log_probs
    return got


def _own_linear(state):
    linear = framework().linear
    x, w, b, r = state["x"], state["w"], state["b"], state["r"]
    if not state["train"]:
        with torch.no_grad():
            return {"y": linear(x, w, b, activation=state["activation"], residual=r)}
    y = linear(x, w, b, activation=state["activation"], residual=r, checkpoint="e4m3" if state["packed"] else None)
    wanted = [(k, t) for k, t in (("dx", x), ("dw", w), ("db", b), ("dr", r)) if t is not None]
    grads = torch.autograd.grad(y, [t for _, t in wanted], state["dy"])
    return {"y": y.detach(), **{k: g for (k, _), g in zip(wanted, grads)}}


def run(state):
    if own:
        if state["op"] == "loss":
            return _own_loss(state)
        if state["op"] == "linear":
            return _own_linear(state)
        return {"x": framework().pack_activation(state["x"]).unpack(torch.float32)}
    if state["op"] == "loss":
        return _plain_loss(state)
    if state["op"] == "linear":
        return _plain_linear(state)
    return {"x": _plain_pack(state["x"], state["x"].numel())}


def work(case):
    """What a pass has to move and compute: inputs once, outputs once; the packed form is written and read."""
    s = BYTES[case["dtype"]]
    if case["op"] == "pack":
        return {"bytes": case["rows"] * case["cols"] * (2 * s + 2 * (1 + 1 / BLOCK)), "flops": 0}
    if case["op"] == "loss":
        entries = case["rows"] * case["cols"]
        a_row = 32 if case["clipped"] else 0
        each = 2 * s + (1 if case["mask"] else 0) + (BYTES[case["target"]] if case["target"] else 0)
        return {"bytes": entries * each + case["rows"] * a_row, "flops": 0}
    m, k, n = case["rows"], case["inner"], case["cols"]
    inputs = m * k + n * k + (n if case["bias"] else 0) + (m * n if case["residual"] else 0)
    if not case["train"]:
        return {"bytes": s * (inputs + m * n), "flops": 2 * m * n * k}
    packed = 2 * m * k * (1 + 1 / BLOCK) if case["packed"] else 0
    return {"bytes": s * (2 * inputs + 2 * m * n) + packed, "flops": 6 * m * n * k}


# ------------------------------------------------------------------ the definition in 64 bits

def _exact_loss(case, seed):
    s = prepare(case, seed)
    logits, n = s["logits"].detach(), case["rows"]
    total = torch.zeros((), dtype=torch.float64, device="cuda")
    grad = torch.zeros(logits.shape, dtype=torch.float64 if logits.numel() < 1 << 27 else torch.float32, device="cuda")
    logp = torch.zeros(n, dtype=torch.float64, device="cuda")
    step = max(1, (1 << 25) // case["cols"])
    for i in range(0, n, step):
        rows = slice(i, min(n, i + step))
        z = logits[rows].double()
        legal = torch.ones_like(z, dtype=torch.bool) if s["mask"] is None else s["mask"][rows]
        live = legal.any(1)
        if s["actions"] is not None:
            live = live & (s["actions"][rows] >= 0)
        legal = legal & live[:, None]
        z = torch.where(legal, z, torch.full_like(z, -math.inf))
        z[~live] = 0.0
        log_p = z - torch.logsumexp(z, 1, keepdim=True)
        p = log_p.exp() * legal
        g = torch.zeros_like(z)
        if s["actions"] is not None:
            index = torch.where(live, s["actions"][rows], torch.zeros_like(s["actions"][rows]))
            lp = log_p[torch.arange(len(index), device="cuda"), index]
            q, adv = (lp - s["old"][rows].double()).exp(), s["advantages"][rows].double()
            inside = torch.where(adv >= 0, q <= 1 + CLIP, q >= 1 - CLIP)
            held = torch.where(adv >= 0, 1 + CLIP, 1 - CLIP) * adv
            d = s["reference"][rows].double() - lp
            total += torch.where(live, -torch.where(inside, q * adv, held) + KL_WEIGHT * (d.exp() - 1 - d), 0.0).sum()
            c = torch.where(inside, -q * adv, 0.0) + KL_WEIGHT * (1 - d.exp())
            c = torch.where(live, c, 0.0)
            g -= p * c[:, None]
            g[torch.arange(len(index), device="cuda"), index] += c
            logp[rows] = torch.where(live, lp, 0.0)
        if s["target"] is not None:
            t = torch.where(legal, s["target"][rows].double(), 0.0)
            total += TARGET_WEIGHT * (torch.special.xlogy(t, t) - torch.where(t > 0, t * log_p, 0.0)).sum()
            g += TARGET_WEIGHT * (p * t.sum(1, keepdim=True) - t)
        grad[rows] = (g * (LOSS_SCALE if case["dtype"] == "fp16" else 1.0) / n).to(grad.dtype)
    out = {"loss": total / n, "grad": grad}
    if s["actions"] is not None:
        out["log_probs"] = logp
    return out


def _exact_kept(x):
    """The packed values of `x` as [rows, columns] in 64 bits, from the list of e4m3 numbers."""
    m, k = x.shape
    grid = torch.tensor([0.0] + [i * 2.0 ** -9 for i in range(1, 8)]
                        + [(1 + i / 8) * 2.0 ** e for e in range(-6, 9) for i in range(8) if (e, i) != (8, 7)],
                        dtype=torch.float64, device=x.device)
    out = torch.empty((m, k), dtype=torch.float64, device=x.device)
    rows_at_once = max(1, (1 << 25) // k)
    whole = k - k % BLOCK
    for i in range(0, m, rows_at_once):
        for j, width in ((0, whole), (whole, k % BLOCK)):
            if width == 0:
                continue
            v = x[i:i + rows_at_once, j:j + width].double()
            v = v.reshape(v.shape[0], -1, min(BLOCK, width))
            top = v.abs().amax(2, keepdim=True)
            power = torch.ceil(torch.log2(torch.where(top > 0, top, 1.0) / 448.0))
            power = power + (torch.exp2(power) * 448.0 < top).double()       # whatever log2 rounded
            power = power - (torch.exp2(power - 1) * 448.0 >= top).double()
            power = torch.where(top > 0, power, 0.0).clamp_min(-15.0 if x.dtype == torch.float16 else -124.0)
            u = (v / torch.exp2(power)).abs()
            above = torch.searchsorted(grid, u.contiguous()).clamp_max(len(grid) - 1)
            below = (above - 1).clamp_min(0)
            far, near = grid[above] - u, u - grid[below]
            up = (far < near) | ((far == near) & (above % 2 == 0))           # ties to the even code
            w = torch.where(up, grid[above], grid[below]) * torch.exp2(power) * v.sign()
            most = torch.finfo(x.dtype).max
            out[i:i + rows_at_once, j:j + width] = w.clamp(-most, most).reshape(w.shape[0], width)
    return out


def _exact_linear(case, seed):
    s = prepare(case, seed)
    if case["rows"] * case["inner"] * case["cols"] > 1 << 39:
        return None
    x, w, b, r = (None if t is None else t.detach().double() for t in (s["x"], s["w"], s["b"], s["r"]))
    z = torch.matmul(x, w.t())
    if b is not None:
        z += b
    if r is not None:
        z += r
    name = s["activation"]
    if name == "gelu":
        cdf = torch.special.ndtr(z)
        y, d = z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    elif name == "silu":
        sig = torch.sigmoid(z)
        y, d = z * sig, sig + z * sig * (1 - sig)
    elif name == "tanh":
        y = torch.tanh(z)
        d = 1 / torch.cosh(z) ** 2
    elif name == "relu":
        y, d = torch.where(z > 0, z, 0.0), torch.where(z > 0, 1.0, 0.0).double()
    else:
        y, d = z, torch.ones_like(z)
    out = {"y": y}
    if s["train"]:
        dz = s["dy"].double() * d
        out["dx"] = torch.matmul(dz, w)
        out["dw"] = torch.matmul(dz.t(), _exact_kept(s["x"].detach()) if s["packed"] else x)
        if b is not None:
            out["db"] = dz.sum(0)
        if r is not None:
            out["dr"] = dz
    return out


def exact(case, seed):
    if case["op"] == "loss":
        return _exact_loss(case, seed)
    if case["op"] == "linear":
        return _exact_linear(case, seed)
    x = prepare(case, seed)["x"]
    return {"x": _exact_kept(x.reshape(1, -1) if x.numel() < 1 << 25 or x.numel() % BLOCK
                             else x.reshape(-1, BLOCK)).reshape(x.shape)}
