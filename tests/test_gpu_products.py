"""The gated linear layer and cross entropy over many items (hetuctr_amd.nn, hctr_gated_linear, hctr_linear_cross_entropy, ..) against
their definitions in 64 bits; tests/products_reference.py has these, and how far rounding may take a result from them."""
import numpy as np
import pytest
import torch

from hetuctr_amd import capi, nn
from tests import products_reference as ref

gpu = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ACTIVATIONS = ["silu", "gelu", "relu", "sigmoid"]


def values(shape, kind, seed, std=1.0, mean=0.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=gen) * std + mean).to(TYPES[kind]).cuda()


def wide(t):
    return None if t is None else t.detach().double()


def apart(t, by=3, at=1):
    """The same values as a slice of wider rows that hold NaN, at any address"""
    out = torch.full((*t.shape[:-1], t.shape[-1] + by), float("nan"), dtype=t.dtype, device="cuda")
    out[..., at:at + t.shape[-1]] = t
    return out[..., at:at + t.shape[-1]]


# ---- the gated linear layer -------------------------------------------------------------------------------------------------
# rows: those that go straight into registers (up to 64), and tiles of 128 and 256; width and hidden: whole vectors or not, less than a
# step of k, ends inside one, sums cut into parts (few tiles, long k)
GATED = [(1, 1, 1), (1, 128, 64), (1, 4096, 33), (2, 37, 5), (16, 32, 16), (17, 1000, 100), (33, 8, 200), (48, 72, 15), (64, 333, 48),
         (65, 64, 32), (70, 37, 41), (100, 2048, 24), (129, 200, 65), (300, 130, 300), (257, 1000, 520), (2000, 96, 136), (1111, 39, 1001)]


def gated_inputs(rows, width, hidden, kind, biased, seed=1):
    x, dh = values((rows, width), kind, seed), values((rows, hidden), kind, seed + 1, 0.1)
    gate_weight, up_weight = (values((hidden, width), kind, seed + 2 + i, 1.5 * width ** -0.5) for i in range(2))
    biases = [None, None] if biased == "none" else [values(hidden, "f32" if biased == "f32" else kind, seed + 4 + i, 0.3) for i in range(2)]
    return dh, x, gate_weight, up_weight, *biases


@gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows, width, hidden", GATED)
def test_gated_linear(rows, width, hidden, kind):
    for i, f in enumerate(ACTIVATIONS):
        _, x, gw, uw, gb, ub = gated_inputs(rows, width, hidden, kind, ("none", "f32", "act")[(i + rows) % 3])
        got = nn.gated_linear(x, gw, uw, gb, ub, f, saved=True)
        want = ref.gated(wide(x), wide(gw), wide(uw), wide(gb), wide(ub), f)
        for g, (value, slack), what in zip(got, want, ("h", "gate", "up")):
            assert g.dtype == x.dtype and g.shape == (rows, hidden) and g.is_contiguous()
            ref.check(g, value, slack, what + " " + f)
        assert torch.equal(nn.gated_linear(x, gw, uw, gb, ub, f), got[0])


@gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows, width, hidden", GATED)
def test_gated_linear_gradient(rows, width, hidden, kind):
    for i, f in enumerate(ACTIVATIONS):
        dh, x, gw, uw, gb, ub = gated_inputs(rows, width, hidden, kind, ("act", "none", "f32")[(i + rows) % 3])
        gate, up = values((rows, hidden), kind, 20, 2.0), values((rows, hidden), kind, 21)
        got = nn.gated_linear_backward(dh, x, gate, up, gw, uw, gb, ub, f)
        want = ref.gated_gradient(wide(dh), wide(x), wide(gate), wide(up), wide(gw), wide(uw), f, x.dtype)
        for g, like, (value, slack), what in zip(got, (x, gw, uw, gb, ub), want, ("dx", "dgate_weight", "dup_weight", "dgate_bias", "dup_bias")):
            if like is None:
                assert g is None
            else:
                assert g.dtype == like.dtype and g.shape == like.shape
                ref.check(g, value, slack, what + " " + f)


# Sizes for which the larger tiles are chosen (128, 256), whole and in parts, with ends inside a tile in every direction
MANY_GATED = [(4100, 2050, 1030), (5003, 300, 1001), (3000, 4100, 516), (9001, 130, 2050), (2500, 1030, 3070), (20000, 100, 300)]


@gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows, width, hidden", MANY_GATED)
def test_gated_linear_of_many_rows(rows, width, hidden, kind):
    f = ACTIVATIONS[rows % 4]
    dh, x, gw, uw, gb, ub = gated_inputs(rows, width, hidden, kind, "f32")
    got = nn.gated_linear(x, gw, uw, gb, ub, f, saved=True)
    for g, (value, slack), what in zip(got, ref.gated(wide(x), wide(gw), wide(uw), wide(gb), wide(ub), f), ("h", "gate", "up")):
        ref.check(g, value, slack, what)
    assert torch.equal(nn.gated_linear(x, gw, uw, gb, ub, f), got[0])
    _, gate, up = got
    back = nn.gated_linear_backward(dh, x, gate, up, gw, uw, gb, ub, f)
    want = ref.gated_gradient(wide(dh), wide(x), wide(gate), wide(up), wide(gw), wide(uw), f, x.dtype)
    for g, (value, slack), what in zip(back, want, ("dx", "dgate_weight", "dup_weight", "dgate_bias", "dup_bias")):
        ref.check(g, value, slack, what)


@gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows", [5, 90])
def test_gated_linear_of_any_layout(rows, kind):
    for width, hidden in ((64, 40), (37, 21)):
        dh, x, gw, uw, gb, ub = gated_inputs(rows, width, hidden, kind, "act", 7)
        gate, up = values((rows, hidden), kind, 20, 2.0), values((rows, hidden), kind, 21)
        want = nn.gated_linear(x, gw, uw, gb, ub, saved=True)
        back = nn.gated_linear_backward(dh, x, gate, up, gw, uw, gb, ub)
        turned = lambda t: t.t().contiguous().t()
        every = lambda t: torch.stack((t, t * float("nan")), 1)[:, 0]
        upside = lambda t: t
        for change in (apart, turned, every, upside, lambda t: apart(t, 8, 8), lambda t: apart(t, 16, 0)):
            a = [change(t) for t in (dh, x, gate, up, gw, uw)]
            cut = [torch.stack((b, b), 1)[:, 0] for b in (gb, ub)]
            for g, w in zip(nn.gated_linear(a[1], a[4], a[5], *cut, saved=True), want):
                assert torch.equal(g, w)
            for g, w in zip(nn.gated_linear_backward(*a, *cut), back):
                assert torch.equal(g, w)
            # one of the two weights as it was: the two lie differently
            for g, w in zip(nn.gated_linear(a[1], a[4], uw, gb, ub, saved=True), want):
                assert torch.equal(g, w)
            for g, w in zip(nn.gated_linear_backward(dh, x, gate, a[3], gw, a[5], gb, ub), back):
                assert torch.equal(g, w)
        # three dimensions, no rows, one matrix for both, rows read again and again
        assert torch.equal(nn.gated_linear(x.view(5, -1, width), gw, uw, gb, ub).view(rows, hidden), want[0])
        both = torch.cat((gw, uw))
        assert torch.equal(nn.gated_linear(x, both[:hidden], both[hidden:], gb, ub), want[0])
        one = nn.gated_linear(x[:1].expand(rows, width), gw, uw)
        assert (one == one[0]).all()
        none = nn.gated_linear(x[:0], gw, uw, gb, ub, saved=True)
        assert all(t.shape == (0, hidden) for t in none)
        zero = nn.gated_linear_backward(dh[:0], x[:0], gate[:0], up[:0], gw, uw, gb, ub)
        assert zero[0].shape == (0, width) and all((z == 0).all() for z in zero[1:])


@gpu
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_rows_of_a_product_do_not_touch_each_other(kind):
    # what is not finite stays in its row; and a row's result hangs on nothing but that row, though tiles end in the middle
    for rows in (20, 150):
        _, x, gw, uw, _, _ = gated_inputs(rows, 72, 40, kind, "none", 3)
        want = nn.gated_linear(x, gw, uw)
        for odd in (float("nan"), float("inf"), -float("inf")):
            bad = x.clone()
            bad[7, 3] = odd
            got = nn.gated_linear(bad, gw, uw)
            assert not got[7].isfinite().all()
            keep = torch.arange(rows, device="cuda") != 7
            assert torch.equal(got[keep], want[keep])
        assert torch.equal(nn.gated_linear(x[:rows - 3], gw, uw), want[:rows - 3])


@gpu
def test_steep_and_flat_ends_of_the_activations():
    # the products are the inputs themselves: x picks a row of the weight
    for kind in TYPES:
        v = torch.tensor([0.0, -0.0, 1e-6, -1e-6, 20.0, -20.0, 60.0, -60.0, 100.0, -100.0, 3e4, -3e4], dtype=TYPES[kind], device="cuda")
        x = torch.eye(12, dtype=TYPES[kind], device="cuda")
        one = torch.ones((12, 12), dtype=TYPES[kind], device="cuda")
        weight = v[None, :].expand(12, 12).contiguous()
        dh, gate, up = one, v[:, None].expand(12, 12).contiguous(), one
        for f in ACTIVATIONS:
            h = nn.gated_linear(x, weight, one, activation=f)
            value, slope = ref.activation(f, wide(v))
            least = 4 * 2.0 ** -149 * (1 + wide(v).abs())[:, None]         # an exponential among the smallest floats is off by steps of them
            assert h.isfinite().all()
            ref.check(h, value[:, None].expand(12, 12), ref.FUNCTION * value.abs()[:, None] + least, f)
            got = nn.gated_linear_backward(dh, x, gate, up, x, 0 * x, activation=f)      # dx = dgate
            assert got[0].isfinite().all()
            ref.check(got[0], slope[:, None].expand(12, 12), ref.rounding(slope, TYPES[kind])[:, None] + ref.FUNCTION * (slope.abs() + wide(v).abs().clamp_max(2))[:, None] + least, f + "'")


@gpu
@pytest.mark.parametrize("kind", list(TYPES))
def test_activations_between_their_ends(kind):
    # Values one by one from where the result is next to nothing, as products with one, which are exact.  Besides what FUNCTION counts the argument of an
    # exponential or of the normal distribution's integral is rounded twice and made with a rounded factor, three halves of a unit of itself: a
    # value of exp(-|v|) is off by 1.5 |v| units for it, one of exp(-v^2 / 2) or of the integral by 1.5 v^2 at most.
    x = torch.cat([torch.linspace(-12.5, 8, 1536), torch.linspace(-0.1, 0.1, 256)]).to(TYPES[kind]).cuda()[:, None].contiguous()
    one, flat = torch.ones((1, 1), dtype=TYPES[kind], device="cuda"), torch.zeros((1, 1), dtype=TYPES[kind], device="cuda")
    bias = torch.ones(1, device="cuda")                     # the second product is 0 x + 1
    v = wide(x)
    units = ref.FUNCTION + 1.5 * ref.U * torch.maximum(v * v, v.abs())
    # (torch.special.ndtr is 1 + erf over 2: nothing is left of it below -8)
    sigmoid, integral, density = torch.sigmoid(v), torch.special.erfc(v.cpu() * -0.5 ** 0.5).cuda() / 2, torch.exp(-v * v / 2) / (2 * np.pi) ** 0.5
    sizes = {"silu": sigmoid * (1 + v.abs() * (1 - sigmoid)), "gelu": integral + v.abs() * density, "relu": 0 * v, "sigmoid": sigmoid * (1 - sigmoid)}
    for f in ACTIVATIONS:
        value, slope = (v * integral, integral + v * density) if f == "gelu" else ref.activation(f, v)
        h, gate, up = nn.gated_linear(x, one, flat, None, bias, activation=f, saved=True)
        assert torch.equal(gate, x) and torch.equal(up, torch.ones_like(x))
        ref.check(h, value, units * value.abs(), f)
        dx = nn.gated_linear_backward(torch.ones_like(h), x, gate, up, one, flat, None, bias, activation=f)[0]       # dgate, rounded twice
        slack = 2 * units * sizes[f]                        # two factors
        ref.check(dx, slope, slack + ref.rounding(slope.abs() + slack, TYPES[kind]), f + "'")


@gpu
@pytest.mark.parametrize("rows", [3, 200])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_autograd_of_the_gated_layer(rows, kind):
    dh, *inputs = gated_inputs(rows, 24, 40, kind, "f32", 5)
    h, gate, up = nn.gated_linear(*inputs, "gelu", saved=True)
    want = nn.gated_linear_backward(dh, inputs[0], gate, up, *inputs[1:], "gelu")
    for wanted in ((0, 1, 2, 3, 4), (0,), (1,), (2,), (3,), (4,), (1, 2), (0, 4)):
        leaves = [t.clone().requires_grad_(i in wanted) for i, t in enumerate(inputs)]
        out, gate, up = nn.gated_linear(*leaves, "gelu", saved=True)
        assert torch.equal(out, h) and not gate.requires_grad and not up.requires_grad
        for i, g in zip(wanted, torch.autograd.grad(out, [leaves[i] for i in wanted], dh)):
            assert torch.equal(g, want[i])
    with torch.no_grad():
        assert not nn.gated_linear(*leaves).requires_grad
    # one tensor for both weights, and x with a gradient from elsewhere
    x, w = inputs[0].clone().requires_grad_(), inputs[1].clone().requires_grad_()
    got = torch.autograd.grad((nn.gated_linear(x, w, w), x), (x, w), (dh, inputs[0]))
    _, gate, up = nn.gated_linear(inputs[0], inputs[1], inputs[1], saved=True)
    parts = nn.gated_linear_backward(dh, inputs[0], gate, up, inputs[1], inputs[1])
    assert torch.equal(got[0], parts[0] + inputs[0]) and torch.equal(got[1], parts[1] + parts[2])


def test_reference_gradients_against_differences():
    # no GPU is needed: the formulas that the kernels are held against, in 64 bits, against central differences of the values
    torch.manual_seed(0)
    double = lambda *s: torch.randn(*s, dtype=torch.float64)
    step = 1e-5

    def slope(f, t):
        out = torch.zeros_like(t)
        for i in range(t.numel()):
            at = t.flatten().clone()
            at[i] += step
            high = f(at.view(t.shape))
            at[i] -= 2 * step
            out.view(-1)[i] = (high - f(at.view(t.shape))) / (2 * step)
        return out

    near = lambda a, b: torch.allclose(a, b, rtol=1e-6, atol=1e-8)
    x, gw, uw, gb, ub, dh = double(4, 3), double(5, 3), double(5, 3), double(5), double(5), double(4, 5)
    for f in ACTIVATIONS:
        args = [x, gw, uw, gb, ub]
        _, (gate, _), (up, _) = ref.gated(*args, f)
        want = ref.gated_gradient(dh, x, gate, up, gw, uw, f, torch.float32)
        for i in range(5):
            loss = lambda t: (ref.gated(*args[:i], t, *args[i + 1:], f)[0][0] * dh).sum()
            assert near(want[i][0], slope(loss, args[i])), (f, i)
    x, w, b, target, dloss = double(6, 3), double(7, 3), double(7), torch.tensor([0, 6, -100, 3, 3, 1]), double(6)
    _, (lse, _) = ref.cross_entropy(x, w, b, target, -100)
    want = ref.cross_entropy_gradient(dloss, x, w, b, target, lse, -100, torch.float32)
    for i, t in enumerate((x, w, b)):
        args = [x, w, b]
        loss = lambda t: (ref.cross_entropy(*args[:i], t, *args[i + 1:], target, -100)[0][0] * dloss).sum()
        assert near(want[i][0], slope(loss, t)), i


# ---- cross entropy over many items ------------------------------------------------------------------------------------------
ITEMS = [(1, 1, 1), (1, 16, 2), (1, 128, 1000), (3, 37, 5), (16, 32, 32), (17, 100, 100), (33, 8, 4097), (64, 333, 70), (65, 64, 129), (70, 37, 41),
         (130, 200, 65), (300, 16, 5000), (257, 1000, 520), (2049, 48, 300), (1111, 39, 1001), (35, 4100, 70), (100, 2056, 300)]
SHARES = [0.0, 0.3, 0.9]


def items_inputs(rows, width, items, kind, biased, share=0.0, seed=1):
    x, weight = values((rows, width), kind, seed), values((items, width), kind, seed + 1, 2 * width ** -0.5)
    bias = None if biased == "none" else values(items, "f32" if biased == "f32" else kind, seed + 2, 0.5)
    gen = torch.Generator().manual_seed(seed + 3)
    target = torch.randint(0, items, (rows,), generator=gen)
    target[torch.rand(rows, generator=gen) < share] = -100
    return x, weight, target.cuda(), bias


@gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows, width, items", ITEMS)
def test_linear_cross_entropy(rows, width, items, kind):
    for i, share in enumerate(SHARES):
        x, w, target, b = items_inputs(rows, width, items, kind, ("none", "f32", "act")[(i + rows) % 3], share)
        x[target == -100] = float("nan")
        got = nn.linear_cross_entropy(x, w, target, b, stats=True)
        want = ref.cross_entropy(wide(x).nan_to_num(0.0), wide(w), wide(b), target, -100)
        for g, (value, slack), what in zip(got, want, ("loss", "lse")):
            assert g.dtype == torch.float32 and g.shape == (rows,)
            ref.check(g, value, slack, what)
            assert (g[target == -100] == 0).all()
        assert torch.equal(nn.linear_cross_entropy(x, w, target, b), got[0])


@gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows, width, items", ITEMS)
def test_linear_cross_entropy_gradient(rows, width, items, kind):
    for i, share in enumerate(SHARES):
        x, w, target, b = items_inputs(rows, width, items, kind, ("act", "none", "f32")[(i + rows) % 3], share)
        clean = x.clone()
        x[target == -100] = float("inf")
        dloss = values(rows, "f32", 9, 1e-3)
        lse = ref.cross_entropy(wide(clean), wide(w), wide(b), target, -100)[1][0].float()
        got = nn.linear_cross_entropy_backward(dloss, x, w, target, lse, b)
        want = ref.cross_entropy_gradient(wide(dloss), wide(clean), wide(w), wide(b), target, wide(lse), -100, x.dtype)
        for g, like, (value, slack), what in zip(got, (x, w, b), want, ("dx", "dweight", "dbias")):
            if like is None:
                assert g is None
            else:
                assert g.dtype == like.dtype and g.shape == like.shape
                ref.check(g, value, slack, what)
        assert (got[0][target == -100] == 0).all()


@gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("share", [0.0, 0.4])
@pytest.mark.parametrize("rows, width, items", [(4100, 200, 3001), (3000, 1030, 5003), (9001, 136, 2050), (600, 520, 40000), (5000, 128, 7001), (9000, 100, 700)])
def test_cross_entropy_of_many_rows(rows, width, items, share, kind):
    x, w, target, b = items_inputs(rows, width, items, kind, "f32", share)
    clean = x.clone()
    x[target == -100] = float("nan")
    loss, lse = nn.linear_cross_entropy(x, w, target, b, stats=True)
    want = ref.cross_entropy(wide(clean), wide(w), wide(b), target, -100)
    ref.check(loss, *want[0], "loss")
    ref.check(lse, *want[1], "lse")
    dloss = values(rows, "f32", 9, 1e-3)
    got = nn.linear_cross_entropy_backward(dloss, x, w, target, lse, b)
    want = ref.cross_entropy_gradient(wide(dloss), wide(clean), wide(w), wide(b), target, wide(lse), -100, x.dtype)
    for g, (value, slack), what in zip(got, want, ("dx", "dweight", "dbias")):
        ref.check(g, value, slack, what)
    assert (got[0][target == -100] == 0).all()


@gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows", [4, 90])
def test_cross_entropy_of_any_layout(rows, kind):
    for width, items in ((64, 40), (37, 51)):
        x, w, target, b = items_inputs(rows, width, items, kind, "act", 0.3, 7)
        dloss = values(rows, "f32", 9, 1e-3)
        loss, lse = nn.linear_cross_entropy(x, w, target, b, stats=True)
        back = nn.linear_cross_entropy_backward(dloss, x, w, target, lse, b)
        every = lambda t: torch.stack((t, t), -1)[..., 0]
        for change in (apart, lambda t: t.t().contiguous().t(), lambda t: torch.stack((t, t * float("nan")), 1)[:, 0], lambda t: apart(t, 8, 8)):
            a, v = change(x), change(w)
            assert torch.equal(nn.linear_cross_entropy(a, v, every(target), every(b)), loss)
            assert torch.equal(nn.linear_cross_entropy(a, w, target, b), loss) and torch.equal(nn.linear_cross_entropy(x, v, target, b), loss)
            for g, want in zip(nn.linear_cross_entropy_backward(every(dloss), a, v, every(target), every(lse), every(b)), back):
                assert torch.equal(g, want)
        # other dimensions, another index for what is ignored, no rows
        got = nn.linear_cross_entropy(x.view(2, -1, width), w, torch.where(target == -100, items + 3, target).view(2, -1), b, ignore_index=items + 3)
        assert got.shape == (2, rows // 2) and torch.equal(got.flatten(), loss)
        assert nn.linear_cross_entropy(x[:0], w, target[:0], b).shape == (0,)
        zero = nn.linear_cross_entropy_backward(dloss[:0], x[:0], w, target[:0], lse[:0], b)
        assert zero[0].shape == (0, width) and (zero[1] == 0).all() and (zero[2] == 0).all()
        # one row, without a dimension for rows
        one = nn.linear_cross_entropy(x[0], w, target[1], b, stats=True)
        assert one[0].shape == () and nn.linear_cross_entropy_backward(dloss[0], x[0], w, target[1], one[1], b)[0].shape == (width,)
        # nothing takes part
        none = torch.full_like(target, -100)
        loss, lse = nn.linear_cross_entropy(x * float("nan"), w, none, b, stats=True)
        assert (loss == 0).all() and (lse == 0).all()
        for g in nn.linear_cross_entropy_backward(dloss * float("nan"), x * float("nan"), w, none, lse, b):
            assert (g == 0).all()
        # an index of an item may be ignored, too
        some = nn.linear_cross_entropy(x, w, torch.full_like(target, 3), b, ignore_index=3)
        assert (some == 0).all()


@gpu
@pytest.mark.parametrize("rows", [6, 100])
def test_targets_that_are_no_item(rows):
    x, w, target, b = items_inputs(rows, 24, 50, "f32", "f32", 0.0, 3)
    want = nn.linear_cross_entropy(x, w, target, b, stats=True)
    for odd in (-1, 50, 2 ** 32, 2 ** 62, -2 ** 63, 2 ** 32 - 1, -101):
        bad = target.clone()
        bad[3] = odd
        for g, v in zip(nn.linear_cross_entropy(x, w, bad, b, stats=True), want):
            assert g[3].isnan() and torch.equal(g[torch.arange(rows, device="cuda") != 3], v[torch.arange(rows, device="cuda") != 3])
    lse = nn.linear_cross_entropy(x, w, bad, b, stats=True)[1]
    dx, dweight, _ = nn.linear_cross_entropy_backward(torch.ones(rows, device="cuda"), x, w, bad, lse, b)
    assert dx[3].isnan().all() and dweight.isnan().all() and dx[:3].isfinite().all() and dx[4:].isfinite().all()


@gpu
@pytest.mark.parametrize("rows", [6, 100])
@pytest.mark.parametrize("kind", TYPES)
def test_items_that_do_not_count(rows, kind):
    # a bias of -infinity, and of the type's lowest value
    x, w, target, _ = items_inputs(rows, 24, 300, kind, "none", 0.0, 3)
    for low in (-float("inf"), torch.finfo(TYPES[kind]).min):
        b = torch.zeros(300, device="cuda", dtype=TYPES[kind])
        b[40:] = low
        aim = target % 40
        loss, lse = nn.linear_cross_entropy(x, w, aim, b, stats=True)
        want = nn.linear_cross_entropy(x, w[:40].contiguous(), aim, stats=True)
        torch.testing.assert_close(loss, want[0], rtol=2e-6, atol=2e-6)
        torch.testing.assert_close(lse, want[1], rtol=2e-6, atol=2e-6)
        dloss = torch.ones(rows, device="cuda")
        dx, dw, db = nn.linear_cross_entropy_backward(dloss, x, w, aim, lse, b)
        assert dx.isfinite().all() and (dw[40:] == 0).all() and (db[40:] == 0).all() and dw[:40].isfinite().all()
        # a target that does not count: never to be had, and a gradient that is finite
        loss, lse = nn.linear_cross_entropy(x, w, aim + 40, b, stats=True)
        assert (loss > 1e4).all() and lse.isfinite().all()
        assert all(g.isfinite().all() for g in nn.linear_cross_entropy_backward(dloss, x, w, aim + 40, lse, b)[:2])
    b[:] = -float("inf")
    loss, lse = nn.linear_cross_entropy(x, w, target, b, stats=True)
    assert loss.isnan().all() and (lse == -float("inf")).all()


@gpu
def test_logits_far_from_zero():
    # one item far above all others, in the first, a middle and the last tile; all logits equal and far from zero
    for rows, items in ((5, 1000), (200, 1000)):
        x, w, target, _ = items_inputs(rows, 16, items, "f32", "none", 0.0, 5)
        for at in (0, 500, items - 1):
            b = torch.zeros(items, device="cuda")
            b[at] = 3000.0
            got = nn.linear_cross_entropy(x, w, target, b, stats=True)
            want = ref.cross_entropy(wide(x), wide(w), wide(b), target, -100)
            for g, (value, slack) in zip(got, want):
                ref.check(g, value, slack + 16 * ref.U * 3000, "item %d" % at)
        for level in (-2000.0, 2000.0):
            b = torch.full((items,), level, device="cuda")
            loss, lse = nn.linear_cross_entropy(0 * x, w, target, b, stats=True)
            ref.check(loss, torch.full((rows,), np.log(items), dtype=torch.float64, device="cuda"), torch.full((), 16 * ref.U * 2010, device="cuda"), "loss")
            ref.check(lse, torch.full((rows,), np.log(items) + level, dtype=torch.float64, device="cuda"), torch.full((), 16 * ref.U * 2010, device="cuda"), "lse")


@gpu
@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
def test_gradient_in_several_pieces_of_the_items(kind):
    # more than is held at a time: 512 MiB of slopes
    rows, width, items = 4099, 24, 70001 if kind != "f32" else 35001
    x, w, target, b = items_inputs(rows, width, items, kind, "f32", 0.2, 3)
    dloss = values(rows, "f32", 9, 1e-3)
    loss, lse = nn.linear_cross_entropy(x, w, target, b, stats=True)
    want = ref.cross_entropy(wide(x), wide(w), wide(b), target, -100)
    ref.check(loss, *want[0], "loss")
    got = nn.linear_cross_entropy_backward(dloss, x, w, target, lse, b)
    want = ref.cross_entropy_gradient(wide(dloss), wide(x), wide(w), wide(b), target, wide(lse), -100, x.dtype)
    for g, (value, slack), what in zip(got, want, ("dx", "dweight", "dbias")):
        ref.check(g, value, slack, what)
    del want
    torch.cuda.empty_cache()


@gpu
@pytest.mark.parametrize("size", [1e-30, 1.0, 1e30])
def test_gradients_of_any_size_in_half_precision(size):
    # what is held of the slopes in half precision is scaled: neither a small nor a large gradient of the loss leaves its range
    x, w, target, _ = items_inputs(100, 32, 500, "f16", "none", 0.0, 3)
    b = values(500, "f32", 8)
    lse = nn.linear_cross_entropy(x, w, target, b, stats=True)[1]
    dloss = values(100, "f32", 9) * size
    got = nn.linear_cross_entropy_backward(dloss, x, w, target, lse, b)
    want = ref.cross_entropy_gradient(wide(dloss), wide(x), wide(w), wide(b), target, wide(lse), -100, x.dtype)
    ref.check(got[2], *want[2], "dbias")                # in 32 bits
    if size == 1.0:
        ref.check(got[0], *want[0], "dx")


@gpu
@pytest.mark.parametrize("rows", [3, 200])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_autograd_of_the_cross_entropy(rows, kind):
    x, w, target, b = items_inputs(rows, 24, 77, kind, "act", 0.2, 5)
    dloss = values(rows, "f32", 9)
    loss, lse = nn.linear_cross_entropy(x, w, target, b, stats=True)
    want = nn.linear_cross_entropy_backward(dloss, x, w, target, lse, b)
    for wanted in ((0, 1, 2), (0,), (1,), (2,), (0, 2)):
        leaves = [t.clone().requires_grad_(i in wanted) for i, t in enumerate((x, w, b))]
        out, other = nn.linear_cross_entropy(leaves[0], leaves[1], target, leaves[2], stats=True)
        assert torch.equal(out, loss) and torch.equal(other, lse) and not other.requires_grad
        for i, g in zip(wanted, torch.autograd.grad(out, [leaves[i] for i in wanted], dloss)):
            assert torch.equal(g, want[i])
    # of a mean: the gradient that comes in is one number, spread out
    leaf = x.clone().requires_grad_()
    nn.linear_cross_entropy(leaf, w, target, b).mean().backward()
    same = nn.linear_cross_entropy_backward(torch.full((rows,), 1.0, device="cuda") / rows, x, w, target, lse, b)[0]
    torch.testing.assert_close(leaf.grad, same)


# ---- far apart in memory ------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("rows", [3, 70])
def test_rows_further_apart_than_a_tile_can_count(rows):
    apart = 2 ** 22 + 8                                            # floats: 16 MiB and a bit
    space = torch.full((rows, apart), float("nan"), device="cuda")
    _, near, gw, uw, _, _ = gated_inputs(rows, 40, 24, "f32", "none", 3)
    x = space[:, 8:48]
    x.copy_(near)
    assert torch.equal(nn.gated_linear(x, gw, uw), nn.gated_linear(near, gw, uw))
    target = torch.arange(rows, device="cuda") % 24
    loss, lse = nn.linear_cross_entropy(near, gw, target, stats=True)
    assert torch.equal(nn.linear_cross_entropy(x, gw, target), loss)
    dloss = torch.ones(rows, device="cuda")
    for a, b in zip(nn.linear_cross_entropy_backward(dloss, x, gw, target, lse)[:2], nn.linear_cross_entropy_backward(dloss, near, gw, target, lse)):
        assert torch.equal(a, b)
    # rows of weights that far apart, and in the other direction
    weight = torch.full((24, apart), float("nan"), device="cuda")[:, 8:48]
    weight.copy_(gw)
    assert torch.equal(nn.gated_linear(near, weight, uw), nn.gated_linear(near, gw, uw))
    assert torch.equal(nn.linear_cross_entropy(near, weight, target), loss)
    del space, x, weight
    torch.cuda.empty_cache()


@gpu
@pytest.mark.parametrize("rows, width, items", [(5, 64, 40_000_003), (40, 256, 9_000_001), (5, 200, 12_000_001)])
def test_items_beyond_32_bits_of_bytes(rows, width, items):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    w = torch.empty((items, width), dtype=torch.bfloat16, device="cuda")
    for i in range(0, items, 1_000_000):
        w[i:i + 1_000_000].normal_(0.0, 2 * width ** -0.5, generator=gen)
    x = values((rows, width), "bf16", 2)
    target = torch.tensor([items - 1, 0, items // 2, 2 ** 31 // width + 1, items - 2], device="cuda").repeat(rows // 5 + 1)[:rows]
    loss, lse = nn.linear_cross_entropy(x, w, target, stats=True)
    # the halves' sums, joined; the targets' logits from their own rows
    half = items // 2
    first = torch.zeros(rows, dtype=torch.int64, device="cuda")
    parts = [nn.linear_cross_entropy(x, part, first, stats=True)[1].double() for part in (w[:half], w[half:])]
    want = torch.logaddexp(*parts)
    assert (lse.double() - want).abs().max() < 1e-5
    hit = (wide(x) * wide(w[target])).sum(1)
    assert (loss.double() - (want - hit)).abs().max() < 1e-5
    dloss = values(rows, "f32", 3)
    dx, dw, _ = nn.linear_cross_entropy_backward(dloss, x, w, target, lse)
    for at in (slice(0, 500), slice(items - 500, items), slice(2 ** 31 // width - 100, 2 ** 31 // width + 400)):
        d = torch.exp(wide(x) @ wide(w[at]).T - wide(lse)[:, None])
        for r in range(rows):
            if at.start <= target[r] < at.stop:
                d[r, target[r] - at.start] -= 1
        d *= wide(dloss)[:, None]
        got = wide(dw[at])
        want = d.T @ wide(x)
        # a rounding of d and one of the result, and what an exponential is off by (40 units), of the sizes
        assert ((got - want).abs() <= (2 * 2.0 ** -8 + 40 * ref.U) * (d.abs().T @ wide(x).abs()) + 1e-12).all()
    # dx: the pieces' slopes times the pieces, in 64 bits
    want, size = torch.zeros((rows, width), dtype=torch.float64, device="cuda"), torch.zeros((rows, width), dtype=torch.float64, device="cuda")
    for i in range(0, items, 1_000_000):
        part = wide(w[i:i + 1_000_000])
        d = torch.exp(wide(x) @ part.T - wide(lse)[:, None])
        here = (target >= i) & (target < i + part.shape[0])
        d[here, target[here] - i] -= 1
        d *= wide(dloss)[:, None]
        want += d @ part
        size += d.abs() @ part.abs()
    # the roundings of so many slopes do not add up all with one sign; that of the sum of n parts in 32 bits is some thousand units
    assert ((wide(dx) - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 4096 * ref.U) * size).all()
    del w, dw
    torch.cuda.empty_cache()


@gpu
def test_more_tiles_than_a_launch_has():
    rows, width, items = 300_000, 136, 8_000_000
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    w = torch.empty((items, width), dtype=torch.bfloat16, device="cuda")
    for i in range(0, items, 1_000_000):
        w[i:i + 1_000_000].normal_(0.0, 2 * width ** -0.5, generator=gen)
    x = torch.empty((rows, width), device="cuda").normal_(0.0, 1.0, generator=gen).bfloat16()
    target = torch.randint(0, items, (rows,), device="cuda", generator=gen)
    loss = nn.linear_cross_entropy(x, w, target)
    for at in (slice(0, 32), slice(rows // 2, rows // 2 + 32), slice(rows - 32, rows)):
        torch.testing.assert_close(loss[at], nn.linear_cross_entropy(x[at], w, target[at]), rtol=2e-6, atol=2e-5)
    assert loss.isfinite().all()
    del w, x
    torch.cuda.empty_cache()


@gpu
def test_a_gated_layer_beyond_32_bits_of_values():
    rows, width, hidden = 140_001, 16, 16_384
    x = values((rows, width), "bf16", 1)
    gw, uw = values((hidden, width), "bf16", 2, 0.3), values((hidden, width), "bf16", 3, 0.3)
    h, gate, up = nn.gated_linear(x, gw, uw, saved=True)
    for at in (slice(0, 70), slice(rows - 70, rows), slice(2 ** 31 // hidden - 30, 2 ** 31 // hidden + 40)):
        want = ref.gated(wide(x[at]), wide(gw), wide(uw), None, None, "silu")
        for g, (value, slack) in zip((h, gate, up), want):
            ref.check(g[at], value, slack, "rows from %d" % at.start)
    dx, dgw, duw, _, _ = nn.gated_linear_backward(h, x, gate, up, gw, uw)
    for at in (slice(0, 70), slice(rows - 70, rows)):
        want = ref.gated_gradient(wide(h[at]), wide(x[at]), wide(gate[at]), wide(up[at]), wide(gw), wide(uw), "silu", x.dtype)
        ref.check(dx[at], *want[0], "dx from %d" % at.start)
    del h, gate, up
    torch.cuda.empty_cache()


# ---- together -----------------------------------------------------------------------------------------------------------------
def small_step(x, weights, target, table):
    """Loss, gradients and their norm of one step: a gated layer and its way back, the next item among all, clipped"""
    leaves = [t.detach().requires_grad_() for t in (x, *weights, table)]
    h = nn.gated_linear(*leaves[:3])
    y, _ = nn.dropout_add_layer_norm(h @ leaves[3], leaves[0])
    loss = nn.linear_cross_entropy(y, leaves[4], target)
    grads = list(torch.autograd.grad(loss, leaves, torch.full_like(loss, 1 / 64)))
    norm = nn.clip_gradients(grads, 0.01)
    return (loss.detach(), norm, *grads)


def step_inputs(seed, rows=80, width=32):
    gen = torch.Generator().manual_seed(seed)
    make = lambda *s: (torch.randn(*s, generator=gen) / s[-1] ** 0.5).bfloat16().cuda()
    target = torch.randint(0, 500, (rows,), generator=gen)
    target[::7] = -100
    return make(rows, width) * 5, [make(64, width), make(64, width), make(64, width)], target.cuda(), make(500, width)


@gpu
@pytest.mark.parametrize("rows, width", [(40, 32), (300, 32), (20, 200), (300, 200), (40, 2048)])
def test_steps_in_graphs_and_on_streams(rows, width):
    x, weights, target, table = step_inputs(1, rows, width)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        small_step(x, weights, target, table)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = small_step(x, weights, target, table)
    for i in range(4):
        new = step_inputs(10 + i, rows, width)
        for to, t in zip((x, *weights, target, table), (new[0], *new[1], new[2], new[3])):
            to.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        for a, g in zip(small_step(x, weights, target, table), outs):
            assert torch.equal(a, g)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):                              # the same bits from another stream, beside the first
            other = small_step(x, weights, target, table)
        here = small_step(x, weights, target, table)
        torch.cuda.current_stream().wait_stream(side)
        for a, b, g in zip(other, here, outs):
            assert torch.equal(a, g) and torch.equal(b, g)


@gpu
@pytest.mark.parametrize("width", [32, 200])
def test_two_graphs_do_not_share_what_they_work_in(width):
    first, second = step_inputs(1, 300, width), step_inputs(2, 300, width)
    small_step(*first)
    graphs, outs = [], []
    for given in (first, second):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(small_step(*given))
    want = [small_step(*given) for given in (first, second)]
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for s, g in zip(streams, graphs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
        for got, w in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(got, w))


# ---- refusals -----------------------------------------------------------------------------------------------------------------
def test_the_c_entry_points_refuse_what_they_cannot_do():
    # refused before anything is launched: no GPU is needed
    m, none, space = (4096, 8), capi.NO_MATRIX, (4096, 1 << 40)
    f32, bf16, f16 = capi.F32, capi.BF16, capi.F16

    def gated(rows=100, width=8, hidden=8, x=m, gw=m, uw=m, h=m, gate=none, up=none, gb=0, ub=0, workspace=space, types=(f32, f32), f=0, **more):
        return capi.gated_linear(rows, width, hidden, x, gw, uw, h, gate, up, gb, ub, workspace, types, f, **more)

    def gated_back(rows=100, width=8, hidden=8, dh=m, x=m, gate=m, up=m, gw=m, uw=m, dx=m, dgw=m, duw=m, dgb=0, dub=0, workspace=space,
                   types=(f32, f32), f=0, **more):
        return capi.gated_linear_backward(rows, width, hidden, dh, x, gate, up, gw, uw, dx, dgw, duw, dgb, dub, workspace, types, f, **more)

    def items(rows=100, width=8, items=8, x=m, weight=m, bias=0, target=4096, loss=4096, lse=0, workspace=space, types=(f32, f32), **more):
        return capi.linear_cross_entropy(rows, width, items, x, weight, bias, target, -100, loss, lse, workspace, types, **more)

    def items_back(rows=100, width=8, items=8, x=m, weight=m, dx=m, dweight=m, bias=0, dbias=0, target=4096, dloss=4096, lse=4096, workspace=space,
                   types=(f32, f32), **more):
        return capi.linear_cross_entropy_backward(rows, width, items, x, weight, dx, dweight, bias, dbias, target, -100, dloss, lse, workspace,
                                                  types, **more)

    short = (4096, 7)
    for f, args, match in [
            (gated, dict(rows=2 ** 31), "rows"), (items, dict(rows=2 ** 26 + 1), "rows"), (gated, dict(width=0), "width"), (gated, dict(width=2 ** 20 + 1), "width"), (gated, dict(hidden=0), "hidden"),
            (gated, dict(hidden=2 ** 20 + 1), "hidden"), (gated, dict(types=(3, 0)), "type"), (gated, dict(f=4), "activation"), (gated, dict(f=-1), "activation"),
            (gated, dict(gb=4096, types=(bf16, f16)), "biases"), (gated, dict(x=none), "x: null"), (gated, dict(gw=none), "gate_weight: null"),
            (gated, dict(uw=none), "up_weight: null"), (gated, dict(h=none), "h: null"), (gated, dict(h=short), "h: .*overlap"), (gated, dict(gate=short), "gate: .*overlap"),
            (gated, dict(up=short), "up: .*overlap"),
            (gated_back, dict(rows=2 ** 31), "rows"), (gated_back, dict(width=0), "width"), (gated_back, dict(hidden=2 ** 21), "hidden"), (gated_back, dict(types=(7, 0)), "type"),
            (gated_back, dict(f=9), "activation"), (gated_back, dict(dub=4096, types=(f16, bf16)), "biases"), (gated_back, dict(dh=none), "dh: null"),
            (gated_back, dict(x=none), "x: null"), (gated_back, dict(gate=none), "gate: null"), (gated_back, dict(up=none), "up: null"),
            (gated_back, dict(gw=none), "gate_weight: null"), (gated_back, dict(uw=none), "up_weight: null"), (gated_back, dict(dx=short), "dx: .*overlap"),
            (gated_back, dict(dgw=short), "dgate_weight: .*overlap"), (gated_back, dict(duw=short), "dup_weight: .*overlap"), (gated_back, dict(workspace=(0, 0)), "workspace"),
            (items, dict(rows=2 ** 31), "rows"), (items, dict(width=0), "width"), (items, dict(items=0), "items"), (items, dict(items=2 ** 31), "items"),
            (items, dict(types=(5, 0)), "type"), (items, dict(bias=4096, types=(bf16, f16)), "bias"), (items, dict(x=none), "x: null"), (items, dict(weight=none), "weight: null"),
            (items, dict(target=0), "null"), (items, dict(loss=0), "null"), (items, dict(workspace=(0, 0)), "workspace"),
            (items_back, dict(rows=2 ** 31), "rows"), (items_back, dict(width=0), "width"), (items_back, dict(items=0), "items"), (items_back, dict(types=(5, 0)), "type"),
            (items_back, dict(dbias=4096, types=(bf16, f16)), "bias"), (items_back, dict(x=none), "x: null"), (items_back, dict(weight=none), "weight: null"),
            (items_back, dict(target=0), "null"), (items_back, dict(dloss=0), "null"), (items_back, dict(lse=0), "null"), (items_back, dict(dx=short), "dx: .*overlap"),
            (items_back, dict(dweight=short), "dweight: .*overlap")]:
        with pytest.raises(RuntimeError, match=match):
            f(**args)
    for f in (gated_back, items, items_back):
        need = f(space=True)
        assert need > 0
        for workspace in ((4096, need - 1), (4100, need), (0, need)):
            with pytest.raises(RuntimeError, match="workspace"):
                f(workspace=workspace)
    for f in (gated, gated_back, items, items_back):
        with pytest.raises(RuntimeError, match="width"):
            f(width=0, space=True)
    for name in ("gated_linear", "gated_linear_backward", "linear_cross_entropy", "linear_cross_entropy_backward"):
        with pytest.raises(RuntimeError, match="null argument"):
            capi._check(getattr(capi.lib(), "hctr_" + name)(None))
        assert getattr(capi.lib(), "hctr_%s_workspace" % name)(None) == 2 ** 64 - 1


def test_tensors_that_are_not_on_the_gpu_are_refused():
    x, w, t = torch.zeros((2, 8)), torch.zeros((4, 8)), torch.zeros(2, dtype=torch.int64)
    h = torch.zeros((2, 4))
    for f in (lambda: nn.gated_linear(x, w, w), lambda: nn.gated_linear_backward(h, x, h, h, w, w), lambda: nn.linear_cross_entropy(x, w, t),
              lambda: nn.linear_cross_entropy_backward(x[:, 0], x, w, t, x[:, 0])):
        with pytest.raises(RuntimeError, match="on the GPU"):
            f()


@gpu
def test_the_functions_refuse_what_does_not_fit():
    x, w, h, t = (torch.zeros(s, device="cuda") for s in ((2, 8), (4, 8), (2, 4), 2))
    b, target = torch.zeros(4, device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda")
    half = lambda v: v.half()
    for f, match in [
            (lambda: nn.gated_linear(x.double(), w.double(), w.double()), "float32, bfloat16 or float16"), (lambda: nn.gated_linear(x, half(w), w), "gate_weight"),
            (lambda: nn.gated_linear(x, w, half(w)), "up_weight"), (lambda: nn.gated_linear(x, w[:, :4], w), "gate_weight"), (lambda: nn.gated_linear(x, w, w[:3]), "up_weight"),
            (lambda: nn.gated_linear(x, w[0], w), "matrix"), (lambda: nn.gated_linear(x, w, w.cpu()), "up_weight"), (lambda: nn.gated_linear(x, w, w, b[:3]), "gate_bias"),
            (lambda: nn.gated_linear(x, w, w, None, half(b)), "up_bias"), (lambda: nn.gated_linear(half(x), half(w), half(w), b, half(b)), "one type"),
            (lambda: nn.gated_linear(x, w, w, activation="tanh"), "activation"), (lambda: nn.gated_linear(x[0, 0], w, w), "dimension"),
            (lambda: nn.gated_linear(x[:, :0], w[:, :0], w[:, :0]), "width"),
            (lambda: nn.gated_linear_backward(h[:, :3], x, h, h, w, w), "dh"), (lambda: nn.gated_linear_backward(h, x, half(h), h, w, w), "gate"),
            (lambda: nn.gated_linear_backward(h, x, h, h[:1], w, w), "up"), (lambda: nn.gated_linear_backward(h, x, h, h, w, w, b[:2]), "gate_bias"),
            (lambda: nn.gated_linear_backward(h, x, h, h, w, w, activation=""), "activation"),
            (lambda: nn.linear_cross_entropy(x, w, target.int()), "target"), (lambda: nn.linear_cross_entropy(x, w, target[:1]), "target"),
            (lambda: nn.linear_cross_entropy(x, w, target.cpu()), "target"), (lambda: nn.linear_cross_entropy(x, half(w), target), "weight"),
            (lambda: nn.linear_cross_entropy(x, w, target, b[:2]), "bias"), (lambda: nn.linear_cross_entropy(x, w[:0], target), "items"),
            (lambda: nn.linear_cross_entropy_backward(half(t), x, w, target, t), "dloss"), (lambda: nn.linear_cross_entropy_backward(t, x, w, target, t[:1]), "lse"),
            (lambda: nn.linear_cross_entropy_backward(t.cpu(), x, w, target, t), "GPU")]:
        with pytest.raises(RuntimeError, match=match):
            f()
    with pytest.raises(TypeError):
        nn.linear_cross_entropy(x, w, target, ignore_index="none")


# ---- with a table -------------------------------------------------------------------------------------------------------------
def the_example():
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples", "train_next_item.py")
    spec = importlib.util.spec_from_file_location("train_next_item", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    return example


@gpu
def test_the_example_runs():
    example = the_example()
    said = np.array(example.train(steps=6, samples=300))
    assert said.shape == (6, 2) and np.isfinite(said).all() and (said > 0).all()


@gpu
def test_gradients_of_the_example():
    # every gradient of its model against torch's own operators in 64 bits.  On the way to each there are about a dozen roundings to bfloat16, of
    # values and of their gradients, each at most 2^-8 of what it rounds; in the 2-norm they are allowed all at once
    example = the_example()
    torch.manual_seed(1)
    samples, model = 200, example.Model().cuda()
    rows = values((samples * example.HISTORY, example.WIDTH), "f32", 1, 0.1).requires_grad_()
    _, following = example.clicks(samples, np.random.default_rng(1))
    target = torch.from_numpy(following).cuda()
    names, leaves = zip(*model.named_parameters())
    got = torch.autograd.grad(model(rows, samples, target).sum(), (*leaves, rows))
    wide_leaves = {n: p.detach().double().requires_grad_() for n, p in zip(names, leaves)}
    r = rows.detach().double().requires_grad_()
    p = wide_leaves
    h = torch.nn.functional.layer_norm(r, (example.WIDTH,), p["scale"], p["shift"]).view(samples, -1)
    h = torch.nn.functional.silu(h @ p["gate"].T) * (h @ p["up"].T)
    logits = h @ p["down"].T @ p["items"].T + p["popular"]
    loss = torch.nn.functional.cross_entropy(logits, target, ignore_index=-100, reduction="sum")
    want = torch.autograd.grad(loss, (*[p[n] for n in names], r))
    for name, a, b in zip((*names, "rows"), got, want):
        assert (a.double() - b).norm() <= 12 * 2.0 ** -8 * b.norm(), name
