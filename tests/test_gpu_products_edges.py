"""Ends of the ranges of the gated linear layer and of cross entropy over many items, against their definitions in 64 bits
(tests/products_reference.py)."""
import math

import pytest
import torch

from hetuctr_amd import nn
from tests import products_reference as ref
from tests.test_gpu_products import ACTIVATIONS, TYPES, gated_inputs, values, wide

gpu = pytest.mark.gpu


# ---- slopes of half precision ---------------------------------------------------------------------------------------------
def gated_gradient_in_range(dh, x, gate, up, gate_weight, up_weight, f, many=None):
    """ref.gated_gradient for half precision, where dgate and dup are multiplied by a power of two before they are rounded.  Few: by none if the largest is in
    1 .. 2^15, else that which takes it to 2^13 at least.  Many: one that takes it to 2^8 at least.  As if dh were larger by half of that
    power, for which values become subnormal no later."""
    value, slope = ref.activation(f, wide(gate))
    d = torch.stack((wide(dh) * slope * wide(up), wide(dh) * value)).abs()
    most = d[d.isfinite()].max().item()
    many = dh.numel() >= 2 ** 22 if many is None else many
    by = 1.0 if 1 <= most < 2 ** 15 and not many else 2.0 ** ((7 if many else 12) - math.floor(math.log2(most)))
    want = ref.gated_gradient(wide(dh) * by, wide(x), wide(gate), wide(up), wide(gate_weight), wide(up_weight), f, torch.float16)
    return [(v / by, s / by) for v, s in want]


def check_half(got, value, slack, what):
    """As ref.check; a result that lies beyond the type's largest number is infinite"""
    inside, beyond = value.abs() + slack < 65504, value.abs() - slack > 65520
    ref.check(got[inside], value[inside], slack[inside], what)
    assert torch.equal(got[beyond].double(), value[beyond].sign() * math.inf)


# dh, up, x and weights: the slopes lie beyond 65504, or below the smallest half, and the results in between
SLOPES = {"beyond the largest half": (1e3, 100.0, 3e-4, 3e-4), "below the smallest half": (1e-6, 1e-2, 1e3, 1e3), "among the smallest halves": (1e-4, 1.0, 10.0, 10.0)}


@gpu
@pytest.mark.parametrize("sizes", SLOPES)
@pytest.mark.parametrize("rows, width, hidden", [(1, 40, 24), (5, 64, 40), (65, 37, 41), (300, 130, 300), (2000, 96, 136), (5003, 300, 1001)])
def test_slopes_of_any_size_in_half_precision(rows, width, hidden, sizes):
    dh_size, up_size, x_size, weight_size = SLOPES[sizes]
    dh, x, gw, uw, gb, ub = gated_inputs(rows, width, hidden, "f16", "f32", 9)
    dh, x = values((rows, hidden), "f16", 30, dh_size), values((rows, width), "f16", 31, x_size)
    gw, uw = (values((hidden, width), "f16", 32 + i, weight_size) for i in range(2))
    gate, up = values((rows, hidden), "f16", 34, 2.0), values((rows, hidden), "f16", 35, up_size)
    for f in ACTIVATIONS if rows < 5000 else ACTIVATIONS[:2]:
        got = nn.gated_linear_backward(dh, x, gate, up, gw, uw, gb, ub, f)
        assert all(g.isfinite().all() for g in got) and all(g.count_nonzero() > g.numel() // 8 for g in got)
        want = gated_gradient_in_range(dh, x, gate, up, gw, uw, f)
        for g, (value, slack), what in zip(got, want, ("dx", "dgate_weight", "dup_weight", "dgate_bias", "dup_bias")):
            ref.check(g, value, slack, what + " " + f)
        # some of the results, in the same call as another's scale
        only = nn.gated_linear_backward(dh[:1], x[:1], gate[:1], up[:1], gw, uw, None, None, f)
        want = gated_gradient_in_range(dh[:1], x[:1], gate[:1], up[:1], gw, uw, f)
        for g, (value, slack), what in zip(only, want, ("dx", "dgate_weight", "dup_weight")):
            ref.check(g, value, slack, what + " of one row " + f)


@gpu
def test_slopes_in_half_precision_beside_a_row_that_is_not_finite():
    rows, width, hidden = 150, 72, 40
    _, x, gw, uw, _, _ = gated_inputs(rows, width, hidden, "f16", "none", 3)
    gw, uw = gw * 1e-3, uw * 1e-3
    dh, gate, up = values((rows, hidden), "f16", 40, 1e3), values((rows, hidden), "f16", 41), values((rows, hidden), "f16", 42, 100.0)
    want = gated_gradient_in_range(dh, x, gate, up, gw, uw, "silu")[0]
    keep = torch.arange(rows, device="cuda") != 7
    for odd in (float("nan"), float("inf"), -float("inf")):
        bad = dh.clone()
        bad[7, 3] = odd
        dx = nn.gated_linear_backward(bad, x, gate, up, gw, uw)[0]
        assert not dx[7].isfinite().all()
        ref.check(dx[keep], want[0][keep], want[1][keep], "dx")


@gpu
@pytest.mark.parametrize("seen, others", [(1e-4, 1e3), (1e3, 1e-4), (0.0, 1e3), (0.0, 1e-6), (0.0, 0.0), (1.0, float("inf"))])
def test_many_slopes_in_half_precision_that_a_look_at_some_rows_misses(seen, others):
    # every 65th row, and the first, are of one size, the others of another: the scale that some rows suggest is far from what all need, or there is none
    rows, width, hidden = 64 * 65, 72, 1024
    _, x, gw, uw, _, _ = gated_inputs(rows, width, hidden, "f16", "none", 3)
    x, gw, uw = x * 1e-3, gw * 1e-3, uw * 1e-3
    gate, up = values((rows, hidden), "f16", 41), values((rows, hidden), "f16", 42, 100.0)
    some = torch.arange(rows, device="cuda") % 65 == 0
    dh = torch.where(some[:, None], seen, others) * values((rows, hidden), "f32", 40)
    dh = dh.nan_to_num(0.0, math.inf, -math.inf).half()
    got = nn.gated_linear_backward(dh, x, gate, up, gw, uw)
    if seen == others == 0:
        assert all((g == 0).all() for g in got[:3])
        return
    keep = some if others == math.inf else torch.ones_like(some)
    want = gated_gradient_in_range(dh[keep], x[keep], gate[keep], up[keep], gw, uw, "silu", True)
    for g, (value, slack), what in list(zip(got, want, ("dx", "dgate_weight", "dup_weight")))[:1 if others == math.inf else 3]:
        ref.check(g[keep] if what == "dx" else g, value, slack, what)


@gpu
def test_a_captured_gradient_finds_its_scale_again():
    # the largest slope is another one at each replay: beyond the range, within it, below it
    rows, width, hidden = 90, 64, 48
    _, x, gw, uw, _, _ = gated_inputs(rows, width, hidden, "f16", "none", 4)
    gw, uw = gw * 1e-2, uw * 1e-2
    dh, gate, up = (values((rows, hidden), "f16", 50 + i) for i in range(3))
    step = lambda: nn.gated_linear_backward(dh, x, gate, up, gw, uw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i, size in enumerate((1e3, 1.0, 1e-5, 300.0, 1e-3)):
        dh.copy_(values((rows, hidden), "f16", 60 + i, size))
        up.copy_(values((rows, hidden), "f16", 70 + i, 100.0))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out[:3]]
        for g, w in zip(got, step()):
            assert torch.equal(g, w)
        for g, (value, slack) in zip(got, gated_gradient_in_range(dh, x, gate, up, gw, uw, "silu")):
            check_half(g, value, slack, "size %g" % size)


# ---- losses next to nothing ------------------------------------------------------------------------------------------------
# rows, width, items: narrow rows of 16 bits, few rows, few but long ones, tiles of each size
CERTAIN = [(1, 24, 7), (20, 64, 900), (700, 128, 3000), (3000, 33, 5000), (3, 300, 2000), (32, 1000, 700), (40, 4096, 100), (90, 200, 700), (1500, 260, 1500),
           (6000, 520, 6000)]


@gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows, width, items", CERTAIN)
def test_a_loss_is_never_below_zero(rows, width, items, kind):
    # rows that are all but certain of their target: its logit is some hundreds, and the loss the little that the others add
    weight = values((items, width), kind, 80, width ** -0.5)
    target = torch.randint(0, items, (rows,), generator=torch.Generator().manual_seed(81)).cuda()
    x = (wide(weight)[target] * torch.linspace(1, 400, rows, device="cuda", dtype=torch.float64)[:, None]).to(TYPES[kind])
    for bias in (None, values(items, "f32", 82)):
        loss, lse = nn.linear_cross_entropy(x, weight, target, bias, stats=True)
        assert (loss >= 0).all()
        for got, (value, slack), what in zip((loss, lse), ref.cross_entropy(wide(x), wide(weight), wide(bias), target, -100), ("loss", "lse")):
            ref.check(got, value, slack, what)
        # of one item there is nothing to lose, whatever its logit
        one = nn.linear_cross_entropy(x, weight[:1], torch.zeros_like(target), None if bias is None else bias[:1])
        assert (one == 0).all()


# ---- more blocks than a launch has -------------------------------------------------------------------------------------------
@gpu
def test_few_rows_and_more_items_than_a_launch_has_blocks():
    # one row of one column, whose logits are 0 but for a few items, at both ends and where one launch ends and the next begins
    items = 2 ** 29 + 70
    weight = torch.zeros((items, 1), device="cuda")
    places = torch.tensor([0, 2 ** 29 - 512, 2 ** 29 - 1, 2 ** 29, 2 ** 29 + 69], device="cuda")
    logits = torch.tensor([15.0, 16.0, 14.0, 15.5, 16.5], device="cuda")
    weight[places, 0] = logits
    x = torch.ones((1, 1), device="cuda")
    total = items - len(places) + wide(logits).exp().sum().item()
    for place, logit in zip(places.tolist(), logits.tolist()):
        loss, lse = nn.linear_cross_entropy(x, weight, torch.tensor([place], device="cuda"), stats=True)
        # (sums of 2^29 terms, most of them 1: whole numbers below 2^24, then joined in pairs)
        assert abs(lse.item() - math.log(total)) < 128 * ref.U * math.log(total) and abs(loss.item() - (math.log(total) - logit)) < 128 * ref.U * math.log(total)
    dx, dweight, _ = nn.linear_cross_entropy_backward(torch.ones(1, device="cuda"), x, weight, torch.tensor([place], device="cuda"), lse)
    p = wide(logits).exp() / total
    p_slack = p * (16 + 4 * 20 + 128 * 20) * ref.U          # an exponential of up to 20, and lse as it was given
    assert abs(dx.item() - ((p * wide(logits)).sum().item() - logit)) < (p_slack * wide(logits)).sum().item() + 256 * ref.U * logit
    hit = torch.zeros_like(p)
    hit[-1] = 1
    ref.check(dweight[places, 0], p - hit, p_slack + 2 * ref.U, "dweight")
    rest = dweight[1:2 ** 29 - 512]
    assert rest.min() == rest.max() and dweight[-2] == rest[0] and abs(rest[0].item() * total - 1) < 2656 * ref.U


@gpu
@pytest.mark.parametrize("rows, width, hidden", [(2 ** 30 + 5, 8, 8), (2 ** 31 - 65536 - 50, 1, 1)])
def test_more_rows_of_a_gated_layer_than_large_tiles_are_in_a_launch(rows, width, hidden):
    # tiles of 64 rows, and of 128: with the threads that they have they are a launch, with the 512 that a tile of 256 has they would be 2^32 threads and
    # more.  A row's results hang on nothing but the row, so that a few at a time say what all have to be.
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("needs 80 GiB of free memory")
    x = torch.empty((rows, width), dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(5))
    gw, uw = values((hidden, width), "bf16", 6), values((hidden, width), "bf16", 7)
    h = nn.gated_linear(x, gw, uw)
    for first in (0, 2 ** 23, 2 ** 29 - 3000, 2 ** 30 - 777, rows // 2, 2 ** 31 - 2 ** 20, rows - 4000):
        assert torch.equal(h[first:first + 4000], nn.gated_linear(x[first:first + 4000], gw, uw))
    del h, x
    torch.cuda.empty_cache()


@gpu
def test_more_rows_of_a_gated_gradient_than_large_tiles_are_in_a_launch():
    # 2^23 tiles of 64 rows: 2^32 threads if each had 512
    rows = 2 ** 29 + 100
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 180 << 30:
        pytest.skip("needs 180 GiB of free memory")
    dh = torch.empty((rows, 1), dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(8))
    gw, uw, gate, up = (values((1, 1), "bf16", 9 + i) for i in range(4))
    every = lambda t, n: t.expand(n, 1)                     # one row again and again
    dx, dgate_weight, dup_weight, _, _ = nn.gated_linear_backward(dh, every(gw * 0, rows), every(gate, rows), every(up, rows), gw, uw)
    for first in (0, 2 ** 23 - 5, 2 ** 28, rows - 4000):
        want = nn.gated_linear_backward(dh[first:first + 4000], every(gw, 4000), every(gate, 4000), every(up, 4000), gw, uw)[0]
        assert torch.equal(dx[first:first + 4000], want) and want.count_nonzero() > 3000
    assert (dgate_weight == 0).all() and (dup_weight == 0).all()
    del dh, dx
    torch.cuda.empty_cache()


# ---- what autograd makes besides --------------------------------------------------------------------------------------------
def memory_of(f):
    """The most memory that f takes on top of what there was"""
    f()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    f()
    return torch.cuda.max_memory_allocated() - before


@gpu
def test_autograd_takes_no_more_memory_than_the_calls():
    # gate and up are of 16 MiB each, lse, mean and rstd of 4 MiB: none is the place for zeros that stand for a gradient that there is not
    dh, *inputs = gated_inputs(2048, 64, 4096, "bf16", "none")[:4]
    h, gate, up = nn.gated_linear(*inputs, saved=True)
    direct = memory_of(lambda: nn.gated_linear_backward(dh, inputs[0], gate, up, *inputs[1:]))
    leaves = [t.requires_grad_() for t in inputs]
    for saved in (False, True):
        out = nn.gated_linear(*leaves, saved=saved)
        out = out[0] if saved else out
        assert memory_of(lambda: torch.autograd.grad(out, leaves, dh, retain_graph=True)) < direct + (1 << 20)
    x, weight = values((1 << 20, 8), "bf16", 90), values((64, 8), "bf16", 91)
    target = torch.arange(1 << 20, device="cuda") % 64
    loss, lse = nn.linear_cross_entropy(x, weight, target, stats=True)
    dloss = torch.ones_like(loss)
    direct = memory_of(lambda: nn.linear_cross_entropy_backward(dloss, x, weight, target, lse))
    leaves = [x.requires_grad_(), weight.requires_grad_()]
    for stats in (False, True):
        out = nn.linear_cross_entropy(*leaves, target, stats=stats)
        out = out[0] if stats else out
        assert memory_of(lambda: torch.autograd.grad(out, leaves, dloss, retain_graph=True)) < direct + (1 << 20)
    x = values((1 << 20, 8), "f32", 92)
    y, mean, rstd = nn.layer_norm(x, stats=True)
    direct = memory_of(lambda: nn.layer_norm_backward(x, x, mean, rstd))
    leaf = x.clone().requires_grad_()
    out = nn.layer_norm(leaf)
    assert memory_of(lambda: torch.autograd.grad(out, leaf, x, retain_graph=True)) < direct + (1 << 20)


# ---- slopes of the cross entropy in half precision -----------------------------------------------------------------------------
# dloss, x and weights: slopes that would be below the smallest half, or beyond the largest, if they were not scaled, and of dx or dweight, or both, results in between
DLOSSES = {"small, for dx": (1e-7, 1e-3, 1e3), "small, for dweight": (1e-7, 1e3, 1e-3), "smaller": (1e-11, 300.0, 3e-3), "large, for dx": (1e6, 1.0, 1e-3), "large, for dweight": (1e6, 1e-3, 1.0),
           "larger": (1e9, 3e-5, 1e-4)}


@gpu
@pytest.mark.parametrize("sizes", DLOSSES)
@pytest.mark.parametrize("rows, width, items", [(20, 64, 900), (700, 128, 3000), (3000, 33, 500), (3, 300, 2000), (40, 4096, 100), (90, 200, 700), (1500, 260, 1500)])
def test_gradients_of_a_cross_entropy_of_any_size_in_half_precision(rows, width, items, sizes):
    dloss_size, x_size, weight_size = DLOSSES[sizes]
    x, weight = values((rows, width), "f16", 100, x_size), values((items, width), "f16", 101, weight_size)
    target = torch.randint(0, items, (rows,), generator=torch.Generator().manual_seed(102)).cuda()
    target[1::7] = -100
    dloss = values(rows, "f32", 103, dloss_size)
    _, lse = nn.linear_cross_entropy(x, weight, target, stats=True)
    dx, dweight, _ = nn.linear_cross_entropy_backward(dloss, x, weight, target, lse)
    want = ref.cross_entropy_gradient(wide(dloss), wide(x), wide(weight), None, target, wide(lse), -100, torch.float16)
    for got, (value, slack), what in zip((dx, dweight), want, ("dx", "dweight")):
        check_half(got, value, slack, what)
    # what the case is there for (results below half of the smallest half are zeros whatever the slopes)
    for got, (value, _), name in zip((dx, dweight), want, ("dx", "dweight")):
        if name in sizes:
            assert got.isfinite().all() and (got != 0).sum() >= (value.abs() > 2.0 ** -24).sum() > 50
