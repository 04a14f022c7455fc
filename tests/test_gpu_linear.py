"""linear against its formula in 64 bits, forward and backward.

Tolerances are counted, not fitted. With u the half step of the type
(eps / 2) and S = |x| |W|^T + |b| + |r|:
- a sum of K products in fp32 is off by at most K steps of 2^-23 S (a
  tensor core may cut where the fp32 units round);
- activations have slopes of at most 1.2 and are evaluated to 2^-20;
- every stored 16-bit value is rounded once: u of itself, or half the
  smallest subnormal;
- dz takes the slope from the stored value (off by u of itself: gelu'' and
  silu'' are at most 0.8; tanh is kept in fp32, and its slope moves by twice
  what it is off) and is itself stored in the type.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
STEP = 2.0 ** -23


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def act(z, name):
    if name == "relu":
        return z.clamp_min(0), (z > 0).double()
    if name == "tanh":
        return torch.tanh(z), 1 - torch.tanh(z) ** 2
    if name == "gelu":
        cdf = torch.special.ndtr(z)
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    return z, torch.ones_like(z)


def stored(value, error, dtype):
    """The error once the value has been rounded to the type."""
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    return error + half_step(dtype) * (value.abs() + error) + tiny


def check(got, value, error):
    assert got.shape == value.shape
    off = (got.double() - value).abs()
    assert bool((off <= error).all()), float((off / error.clamp_min(1e-300)).max())


def reference(x, w, b, r, dy, name, kept_x=None):
    """Values and error bounds of y and the gradients."""
    dtype, (m, k), n = x.dtype, x.shape, w.shape[0]
    xd, wd = x.double(), w.double()
    z, size = xd @ wd.t(), xd.abs() @ wd.abs().t()
    for t in (b, r):
        if t is not None:
            z, size = z + t.double(), size + t.double().abs()
    ez = (k + 4) * STEP * size
    y, slope = act(z, name)
    out = {"y": (y, stored(y, 1.2 * ez + 2.0 ** -20 * y.abs(), dtype))}
    if dy is None:
        return out
    dyd, u = dy.double(), half_step(dtype)
    dz = dyd * slope
    bend = 0.0
    if name in ("gelu", "silu"):
        bend = 0.8 * (ez + u * (z.abs() + ez))
    elif name == "tanh":
        bend = 2 * (1.2 * ez + 2.0 ** -20)
    edz = dz * 0 if name is None else stored(dz, dyd.abs() * (bend + 2.0 ** -20), dtype)
    if name == "relu":
        # Where the sum's sign is not certain either slope is right.
        edz = edz + torch.where(z.abs() <= ez, dyd.abs(), 0.0)
    kept = xd if kept_x is None else kept_x.double()

    def product(a, ea, c, count):
        value, bound = a @ c, (ea + count * STEP * (a.abs() + ea)) @ c.abs()
        return value, stored(value, bound, dtype)

    out["x"] = product(dz, edz, wd, n + 4)
    out["w"] = product(dz.t(), edz.t(), kept, m + 4)
    out["b"] = (dz.sum(0), stored(dz.sum(0), (edz + (m + 4) * STEP * (dz.abs() + edz)).sum(0), dtype))
    out["r"] = (dz, edz)
    return out


def make(m, k, n, dtype, bias=True, residual=True, seed=0, grad=True):
    g = torch.Generator(device="cuda").manual_seed(seed + m * 7 + k * 3 + n)

    def t(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype).requires_grad_(grad)

    return (t(m, k), t(n, k, scale=k ** -0.5), t(n, scale=0.3) if bias else None,
            t(m, n, scale=0.5) if residual else None, t(m, n).detach())


def run(x, w, b, r, dy, name, checkpoint=None):
    from kingdom_ai import check_linear, linear
    y = linear(x, w, b, activation=name, residual=r, checkpoint=checkpoint)
    wanted = {k: t for k, t in (("x", x), ("w", w), ("b", b), ("r", r)) if t is not None and t.requires_grad}
    grads = dict(zip(wanted, torch.autograd.grad(y, list(wanted.values()), dy))) if wanted else {}
    check_linear()
    return {"y": y.detach(), **grads}


def compare(args, name, checkpoint=None):
    x, w, b, r, dy = args
    kept = None
    if checkpoint:
        from kingdom_ai import pack_activation
        pad = -x.shape[1] % 32  # rows are packed apart: pad each to whole blocks
        wide = torch.nn.functional.pad(x.detach(), (0, pad))
        kept = pack_activation(wide).unpack()[:, :x.shape[1]]
    got = run(x, w, b, r, dy, name, checkpoint)
    want = reference(*(None if t is None else t.detach() for t in args[:4]), dy, name, kept)
    for key, value in got.items():
        assert value.dtype == x.dtype
        check(value, *want[key])


# Sizes around the tiles (128 and 256 rows, 64, 128 and 256 columns, 64 k), the
# few-row form (8 and 9 rows), rows that are not 16-byte aligned, k split over
# a cluster, and the network's own heads.
SIZES = [(1, 1, 1), (1, 64, 8), (2, 81, 64), (8, 162, 82), (9, 162, 82), (7, 1000, 33), (127, 63, 65), (128, 64, 64),
         (129, 65, 129), (257, 72, 255), (64, 4096, 64), (40, 2048, 200), (5, 8, 3000), (1024, 1, 7), (300, 24, 1),
         (513, 200, 520)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n", SIZES)
def test_sizes(m, k, n, dtype):
    compare(make(m, k, n, dtype), "gelu" if (m + k + n) % 2 else None)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", [None, "relu", "tanh", "gelu", "silu"])
def test_activations(name, dtype):
    for bias, residual in ((True, True), (False, False)):
        compare(make(200, 136, 72, dtype, bias, residual), name)
        compare(make(3, 40, 24, dtype, bias, residual), name)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k,n", [(2560, 192, 2056), (2309, 328, 2305), (4096, 2048, 520), (1200, 1100, 2309)])
def test_tile_pairs(m, k, n, dtype):
    """Enough tiles for the persistent kernels, ragged at every edge."""
    compare(make(m, k, n, dtype), "silu")
    compare(make(m, k, n, dtype, bias=False), "tanh")


# Few rows against wide weights: dot products, and tiles that hold all rows and
# 128 weight rows, k shared by 1 to 8 CTAs in unequal parts; rows TMA cannot read.
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k,n", [(1, 8200, 24), (2, 4096, 160), (4, 4097, 1031), (8, 4104, 1100), (6, 4097, 4100),
                                   (9, 64, 8), (12, 1000, 392), (16, 2048, 5000), (33, 4104, 129), (48, 640, 2048),
                                   (47, 5000, 136), (49, 1024, 8192), (100, 1032, 8200), (128, 1025, 8193)])
def test_few_rows_against_wide_weights(m, k, n, dtype):
    compare(make(m, k, n, dtype), "gelu")
    compare(make(m, k, n, dtype, bias=False, residual=False), "tanh")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k,n", [(7, 4000, 17), (1000, 64, 82), (4096, 3, 5), (1, 700, 300), (33, 81, 64)])
def test_narrow_gradients_come_from_unrounded_dz(m, k, n, dtype):
    """Few outputs or few dz: the gradients bear one rounding, their own (tanh keeps its value in fp32)."""
    x, w, b, r, dy = make(m, k, n, dtype, residual=False)
    got = run(x, w, b, r, dy, "tanh")
    xd, wd, dyd = x.double(), w.double(), dy.double()
    z, size = xd @ wd.t() + b.double(), xd.abs() @ wd.abs().t() + b.double().abs()
    y, slope = act(z, "tanh")
    dz = dyd * slope
    # As in reference(), without the step that stores dz.
    edz = dyd.abs() * (2 * (1.2 * (k + 4) * STEP * size + 2.0 ** -20) + 2.0 ** -20)
    for key, a, ea, c, count in (("x", dz, edz, wd, n + 4), ("w", dz.t(), edz.t(), xd, m + 4)):
        if got[key].numel() > 1 << 14 and m * n > 1 << 12:  # runs on 16-bit operands
            continue
        value, bound = a @ c, (ea + count * STEP * (a.abs() + ea)) @ c.abs()
        check(got[key], value, stored(value, bound, dtype))


def test_rows_of_a_thin_product_do_not_touch_each_other():
    """A row that is not a number, beside the last row and in front of none."""
    x, w, b, _, _ = make(37, 512, 1000, torch.bfloat16, residual=False, grad=False)
    from kingdom_ai import linear
    want = linear(x, w, b)
    spoilt = x.clone()
    spoilt[36] = float("nan")
    got = linear(spoilt, w, b)
    assert torch.equal(got[:36], want[:36]) and bool(got[36].isnan().all())
    wide = torch.full((37, 640), float("nan"), dtype=x.dtype, device="cuda")
    wide[:, :512] = x
    assert torch.equal(linear(wide[:, :512], w, b), want)


@pytest.mark.parametrize("m,k,n", [(1025, 70, 1100), (3000, 48, 1300)])
def test_large_fp32_tiles(m, k, n):
    compare(make(m, k, n, torch.float32), "tanh")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n", [(300, 160, 72), (77, 81, 64), (2500, 256, 2304), (4, 33, 9)])
def test_packed_input(m, k, n, dtype):
    compare(make(m, k, n, dtype), "relu" if dtype is not torch.float32 else "gelu", checkpoint="e4m3")


def test_packed_input_changes_only_the_weight_gradient():
    args = make(384, 320, 136, torch.bfloat16)
    plain, packed = run(*args, "gelu"), run(*args, "gelu", "e4m3")
    for key in ("y", "x", "b", "r"):
        assert torch.equal(plain[key], packed[key])
    assert not torch.equal(plain["w"], packed["w"])


@pytest.mark.parametrize("dtype", TYPES)
def test_layouts(dtype):
    """Strided rows, transposed and expanded operands, offset storage, extra dimensions."""
    from kingdom_ai import linear
    x, w, b, r, dy = make(96, 80, 48, dtype, grad=False)
    want = linear(x, w, b, activation="relu", residual=r)
    wide = torch.zeros(96, 83, dtype=dtype, device="cuda")
    wide[:, 3:] = x
    assert torch.equal(linear(wide[:, 3:], w, b, activation="relu", residual=r), want)
    padded = torch.zeros(96, 96, dtype=dtype, device="cuda")
    padded[:, :80] = x
    assert torch.equal(linear(padded[:, :80], w, b, activation="relu", residual=r), want)
    assert torch.equal(linear(x.t().contiguous().t(), w.t().contiguous().t(), b, activation="relu", residual=r), want)
    assert torch.equal(linear(x.view(4, 24, 80), w, b, activation="relu", residual=r.view(4, 24, 48)),
                       want.view(4, 24, 48))
    assert torch.equal(linear(x[7], w, b, activation="relu", residual=r[7]).double(),
                       linear(x[7:8], w, b, activation="relu", residual=r[7:8])[0].double())
    one = x[:1].expand(96, 80)
    same = linear(one, w, b, residual=b.expand(96, 48))
    assert torch.equal(same, same[:1].expand(96, 48))
    assert torch.equal(same, linear(one.contiguous(), w, b, residual=b.expand(96, 48).contiguous()))
    flipped = torch.as_strided(torch.randn(8, 1, device="cuda").to(dtype), (8, 1), (1, 5))
    assert linear(flipped, w[:, :1].contiguous()).shape == (8, 48)


def test_gradients_of_broadcast_and_shared_operands():
    from kingdom_ai import linear
    x, w, b, _, _ = make(64, 40, 24, torch.float32, residual=False)
    row = torch.randn(24, device="cuda", requires_grad=True)
    y = linear(x, w, b, activation="tanh", residual=row.expand(64, 24))
    z = linear(y, w[:, :24].contiguous(), activation="silu")  # the weight a second time, cut
    loss = (z.sum() + linear(x, w).square().mean())          # and a third; an expanded gradient
    grads = torch.autograd.grad(loss, [x, w, b, row])
    xd, wd, bd, rd = (t.detach().double().requires_grad_() for t in (x, w, b, row))
    yd = torch.tanh(xd @ wd.t() + bd + rd)
    ld = torch.nn.functional.silu(yd @ wd[:, :24].t()).sum() + (xd @ wd.t()).square().mean()
    for got, want in zip(grads, torch.autograd.grad(ld, [xd, wd, bd, rd])):
        # At most 64 x 40 fp32 steps of the gradient's largest entry.
        assert float((got.double() - want).abs().max()) <= 2560 * STEP * float(want.abs().max())


def test_gradient_against_differences():
    from kingdom_ai import linear
    x, w, b, r, dy = make(12, 10, 6, torch.float32)
    for name in ("tanh", "gelu", "silu"):
        y = linear(x, w, b, activation=name, residual=r)
        grads = torch.autograd.grad(y, [x, w, b, r], dy)
        for t, g in zip((x, w, b, r), grads):
            direction = torch.randn(t.shape, generator=torch.Generator().manual_seed(5)).cuda()
            h = 2.0 ** -7

            def at(s):
                args = [v + s * direction if v is t else v for v in (x, w, b, r)]
                with torch.no_grad():
                    return (linear(args[0], args[1], args[2], activation=name, residual=args[3]).double()
                            * dy.double()).sum()

            slope = (at(h) - at(-h)) / (2 * h)
            # h^2 / 6 of the third derivative (at most 3 |direction|^3 terms of size one) and the sums' rounding / h.
            assert abs(float(slope - (g.double() * direction.double()).sum())) <= 72 * (h * h + 64 * STEP / h)


def test_only_wanted_gradients_and_empty_batches():
    from kingdom_ai import linear
    x, w, b, _, _ = make(20, 16, 12, torch.bfloat16, residual=False)
    for wanted in ([x], [w], [b], [x, b], [w, b]):
        y = linear(*(t if any(t is v for v in wanted) else t.detach() for t in (x, w, b)), activation="relu")
        full = torch.autograd.grad(linear(x, w, b, activation="relu").float().sum(), wanted)
        for g, f in zip(torch.autograd.grad(y.float().sum(), wanted), full):
            assert torch.equal(g, f)
    none = torch.zeros(0, 16, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    y = linear(none, w, b, activation="gelu")
    assert y.shape == (0, 12)
    gx, gw, gb = torch.autograd.grad(y.sum(), [none, w, b])
    assert gx.shape == (0, 16) and not gw.any() and not gb.any() and gw.shape == w.shape


@pytest.mark.parametrize("dtype", TYPES)
def test_not_a_number_and_infinities_pass_through(dtype):
    """A NaN or an infinity reaches its own row and no other, and no zero fill meets it."""
    from kingdom_ai import linear
    for m in (5, 130):
        x, w, b, _, _ = make(m, 70, 40, dtype, residual=False, grad=False)
        clean = linear(x, w, b, activation="relu")
        x[3, 69] = float("nan")
        got = linear(x, w, b, activation="relu")
        rows = [i for i in range(m) if i != 3]
        assert bool(got[3].isnan().all()) and torch.equal(got[rows], clean[rows])
        x[3, 69] = float("inf")
        y = linear(x, w, b)
        assert bool(y[3].isinf().all()) and bool(y[rows].isfinite().all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("name", ["relu", "tanh", "gelu", "silu"])
@pytest.mark.parametrize("cols", [64, 63])
def test_derivative_of_every_value(cols, name, dtype):
    """Every 16-bit value as the sum: in whole 16-byte groups, and one by one."""
    from kingdom_ai import check_linear, linear
    bits = torch.arange(-(1 << 15), 1 << 15, dtype=torch.int32).to(torch.int16).view(dtype).cuda()
    bits = torch.cat([bits, bits.new_zeros(-len(bits) % cols)]).view(-1, cols)
    r = bits.clone().requires_grad_()
    zero = torch.zeros(len(bits), 8, dtype=dtype, device="cuda"), torch.zeros(cols, 8, dtype=dtype, device="cuda")
    y = linear(*zero, activation=name, residual=r)
    got, = torch.autograd.grad(y, r, torch.ones_like(y))
    check_linear()
    assert torch.equal(got.isnan(), bits.isnan() & torch.tensor(name != "relu", device="cuda"))
    finite = bits.isfinite()
    value = act(bits.double(), name)[1]
    # 2^-20 of the derivative's terms, none above 1.2; tanh's own 2^-20 moves 1 - y^2 by twice that.
    error = stored(value, torch.full_like(value, 1.2 * 2.0 ** -20 * (2 if name == "tanh" else 1)), dtype)
    check(torch.where(finite, got, 0.0), torch.where(finite, value, 0.0), error.nan_to_num(0.0))
    if name in ("gelu", "silu", "tanh"):
        ends = got[bits == math.inf], got[bits == -math.inf]
        assert ends[0].tolist() == [0.0 if name == "tanh" else 1.0] and ends[1].tolist() == [0.0]


def test_another_stream_and_two_captured_graphs():
    from kingdom_ai import linear
    args = [make(300, 81, 64, torch.float16, residual=False, seed=s) for s in (1, 2)]
    args = [tuple(None if t is None else t.detach().requires_grad_(i < 3) for i, t in enumerate(a)) for a in args]

    def step(a):
        y = linear(a[0], a[1], a[2], activation="gelu", checkpoint="e4m3")
        return [y.detach(), *torch.autograd.grad(y, a[:3], a[4])]

    want = [[t.clone() for t in step(a)] for a in args]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for a, w in zip(args, want):
            for got, value in zip(step(a), w):
                assert torch.equal(got, value)
    torch.cuda.synchronize()
    graphs = []
    for a in args:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(a)
        graphs.append((graph, out))
    for _ in range(2):
        for graph, out in graphs:
            for t in out:
                t.zero_()
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for (_, out), w in zip(graphs, want):
            for got, value in zip(out, w):
                assert torch.equal(got, value)


def test_calls_on_two_streams_at_once():
    """Workspaces belong to their call: interleaved launches on two streams do not meet."""
    from kingdom_ai import linear
    args = [make(600, 1003, 517, torch.bfloat16, seed=s) for s in (1, 2)]
    want = [run(*a, "gelu", "e4m3") for a in args]
    streams = [torch.cuda.Stream() for _ in args]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(8):
        for i, (a, s) in enumerate(zip(args, streams)):
            with torch.cuda.stream(s):
                y = linear(a[0], a[1], a[2], activation="gelu", residual=a[3], checkpoint="e4m3")
                got[i].append((y.detach(), *torch.autograd.grad(y, a[:4], a[4])))
    torch.cuda.synchronize()
    for w, rows in zip(want, got):
        for row in rows:
            assert all(torch.equal(t, w[k]) for t, k in zip(row, ("y", "x", "w", "b", "r")))


def test_no_backward_memory_is_kept_or_lost():
    """Repeated steps leave the allocator where it was."""
    args = make(512, 333, 257, torch.float16)
    run(*args, "silu", "e4m3")
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    for _ in range(5):
        run(*args, "silu", "e4m3")
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() == before


def test_the_same_call_gives_the_same_bits():
    args = make(700, 2000, 130, torch.bfloat16)
    first = run(*args, "gelu", "e4m3")
    for _ in range(3):
        again = run(*args, "gelu", "e4m3")
        assert all(torch.equal(first[k], again[k]) for k in first)


def test_refusals():
    from kingdom_ai import linear
    x, w, b, r, _ = make(4, 8, 6, torch.float32, grad=False)
    for bad in (lambda: linear(x, w[:, :7].contiguous()), lambda: linear(x, w, b[:5]), lambda: linear(x, w, residual=r[:3]),
                lambda: linear(x.double(), w.double()), lambda: linear(x, w.half()), lambda: linear(x, w.cpu()),
                lambda: linear(x, w, activation="elu"), lambda: linear(x, w, activation=1),
                lambda: linear(x, w, checkpoint="e5m2"), lambda: linear(x[:, :0], w[:, :0]),
                lambda: linear(x, w[:0]), lambda: linear(x, w[0]), lambda: linear(x[0, 0], w),
                lambda: linear(x, w, residual=b)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: linear(x, 3), lambda: linear(None, w), lambda: linear(x, w, [0.0])):
        with pytest.raises(TypeError):
            bad()
    # Second derivatives are refused, not wrong.
    xg = x.clone().requires_grad_()
    y = linear(xg, w, activation="tanh")
    g, = torch.autograd.grad(y.sum(), xg, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), xg)
    # A kept output that was changed in place is refused.
    y = linear(xg, w, activation="relu")
    y.add_(1)
    with pytest.raises(RuntimeError):
        y.sum().backward()
