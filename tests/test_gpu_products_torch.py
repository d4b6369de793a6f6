"""The gated layer, cross entropy and clipping of hetuctr_amd.nn beside what torch does around its own operators."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from hetuctr_amd import nn
from tests.test_gpu_nn_torch import Watcher, Wrapper, differ, negative, values

gpu = pytest.mark.gpu


def inputs(seed, rows=5):
    gen = torch.Generator().manual_seed(seed)
    target = torch.randint(0, 12, (rows,), generator=gen)
    target[1] = -100
    return [values((rows, 16), seed), values((24, 16), seed + 1), values((24, 16), seed + 2), values(24, seed + 3), values((12, 24), seed + 4), values(12, seed + 5),
            target.cuda()]


def program(x, gw, uw, b, w, c, target):
    h, gate, up = nn.gated_linear(x, gw, uw, b, None, "gelu", saved=True)
    grads = nn.gated_linear_backward(h, x, gate, up, gw, uw, b, None, "gelu")
    assert grads[4] is None
    loss, lse = nn.linear_cross_entropy(h, w, target, c, stats=True)
    back = nn.linear_cross_entropy_backward(loss, h, w, target, lse, c)
    some = nn.linear_cross_entropy_backward(loss, h, w, target, lse)
    assert some[2] is None
    clipped = [torch.empty_like(g) for g in back]
    norm = nn.clip_gradients(back, 0.1, into=clipped)
    again = nn.clip_gradients(clipped, 0.05, norm=nn.gradient_norm(clipped))
    return (h, gate, up, *grads[:4], loss, lse, *back, *some[:2], norm, *clipped, again, nn.gated_linear(x, gw, uw), nn.linear_cross_entropy(h, w, target))


@gpu
@pytest.mark.parametrize("mode", ["real", "fake", "symbolic"])
def test_programs_recorded_as_graphs_compute_what_they_say(mode):
    graph = make_fx(program, tracing_mode=mode)(*inputs(1))
    for seed in (1, 50):
        assert differ(graph(*inputs(seed)), program(*inputs(seed))) == []


def loss_of(x, gw, uw, b, w, c, target):
    return nn.linear_cross_entropy(nn.gated_linear(x, gw, uw, b), w, target, c)


@gpu
@pytest.mark.parametrize("mode", ["real", "fake"])
def test_training_steps_recorded_as_graphs(mode):
    def step(*given):
        leaves = [t.detach().requires_grad_() for t in given[:-1]]
        loss = loss_of(*leaves, given[-1])
        return torch.autograd.grad(loss, leaves, torch.ones_like(loss))

    graph = make_fx(step, tracing_mode=mode)(*inputs(1))
    for seed in (1, 50):
        assert differ(graph(*inputs(seed)), step(*inputs(seed))) == []


@gpu
@pytest.mark.parametrize("needs", [False, True])
def test_traced_programs_compute_what_they_say(needs):
    given = [t.requires_grad_(needs and t.is_floating_point()) for t in inputs(1)]
    graph = torch.jit.trace(loss_of, given)
    for seed in (1, 50):
        assert differ([graph(*inputs(seed))], [loss_of(*inputs(seed))]) == []
    leaves = [t.requires_grad_(t.is_floating_point()) for t in inputs(3)]
    dloss = values(5, 9)
    assert differ(torch.autograd.grad(graph(*leaves), leaves[:-1], dloss), torch.autograd.grad(loss_of(*leaves), leaves[:-1], dloss)) == []


@gpu
def test_dispatch_modes_see_the_calls():
    want = program(*inputs(1))
    with Watcher() as outer, Watcher() as inner:
        got = program(*inputs(1))
    assert differ(got, want) == []
    for watcher in (outer, inner):
        own = [name for name in watcher.seen if name.startswith("hetuctr_amd.")]
        assert len(own) == 10
    given = [t.requires_grad_(t.is_floating_point()) for t in inputs(5)]
    dloss = values(5, 9)
    want = torch.autograd.grad(loss_of(*given), given[:-1], dloss)
    context = lambda: torch.utils.checkpoint.create_selective_checkpoint_contexts([torch.ops.aten.mm.default])
    out = torch.utils.checkpoint.checkpoint(loss_of, *given, use_reentrant=False, context_fn=context)
    assert differ(torch.autograd.grad(out, given[:-1], dloss), want) == []


def test_shapes_without_memory():
    # no GPU is needed: nothing is computed
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        make = lambda *s, dtype=torch.bfloat16: torch.empty(s, device="cuda", dtype=dtype)
        x, gw, b, w, target = make(3, 5, 16), make(24, 16), make(24, dtype=torch.float32), make(12, 24), make(3, 5, dtype=torch.int64)
        h, gate, up = nn.gated_linear(x, gw, gw, b, b, saved=True)
        assert h.shape == gate.shape == up.shape == (3, 5, 24) and h.dtype == torch.bfloat16
        grads = nn.gated_linear_backward(h, x, gate, up, gw, gw, b, None)
        assert [g.shape for g in grads[:4]] == [x.shape, gw.shape, gw.shape, b.shape] and grads[3].dtype == torch.float32 and grads[4] is None
        loss, lse = nn.linear_cross_entropy(h, w, target, stats=True)
        assert loss.shape == lse.shape == (3, 5) and loss.dtype == torch.float32
        dx, dw, db = nn.linear_cross_entropy_backward(loss, h, w, target, lse)
        assert dx.shape == h.shape and dw.shape == w.shape and db is None
        norm = nn.clip_gradients([dx, dw], 1.0)
        assert norm.shape == () and norm.dtype == torch.float32 and nn.gradient_norm([dx]).shape == ()


@gpu
def test_views_that_carry_a_sign():
    x, gw, uw, b, w, c, target = inputs(1)
    flip = lambda *ts: [negative(t) for t in ts]
    want = nn.gated_linear(x, gw, uw, b, b, saved=True)
    assert differ(nn.gated_linear(*flip(x, gw, uw, b, b), saved=True), want) == []
    h, gate, up = want
    assert differ(nn.gated_linear_backward(*flip(h, x, gate, up, gw, uw, b, b)), nn.gated_linear_backward(h, x, gate, up, gw, uw, b, b)) == []
    loss, lse = nn.linear_cross_entropy(h, w, target, c, stats=True)
    sign = torch._neg_view(-target)
    assert torch.equal(nn.linear_cross_entropy(*flip(h, w), sign, negative(c)), loss)
    got = nn.linear_cross_entropy_backward(*flip(loss, h, w), sign, *flip(lse, c))
    assert differ(got, nn.linear_cross_entropy_backward(loss, h, w, target, lse, c)) == []
    assert torch.equal(nn.gradient_norm(flip(x, b)), nn.gradient_norm([x, b]))


@gpu
def test_forward_mode_derivatives_are_refused_not_lost():
    x, gw, uw, b, w, c, target = inputs(1)
    h, gate, up = nn.gated_linear(x, gw, uw, b, b, saved=True)
    loss, lse = nn.linear_cross_entropy(h, w, target, c, stats=True)
    for f, args in ((nn.gated_linear, (x, gw, uw, b, b)), (nn.gated_linear_backward, (h, x, gate, up, gw, uw)),
                    (lambda h, w, c: nn.linear_cross_entropy(h, w, target, c), (h, w, c)),
                    (lambda d, h, w, l, c: nn.linear_cross_entropy_backward(d, h, w, target, l, c), (loss, h, w, lse, c)),
                    (lambda *g: nn.gradient_norm(g), (x, b)), (lambda *g: nn.clip_gradients(g, 1.0, into=[torch.empty_like(t) for t in (x, b)]), (x, b))):
        for i in range(len(args)):
            for needs in (False, True):
                with forward_ad.dual_level():
                    given = [a.clone().requires_grad_(needs) for a in args]
                    given[i] = forward_ad.make_dual(given[i], torch.ones_like(args[i]))
                    with pytest.raises(RuntimeError, match="forward-mode|jvp|not differentiable"):
                        f(*given)


@gpu
def test_tensors_without_memory_are_not_taken_for_missing_ones():
    x, gw, uw, b, w, c, target = inputs(1)
    h, gate, up = nn.gated_linear(x, gw, uw, b, b, saved=True)
    loss, lse = nn.linear_cross_entropy(h, w, target, c, stats=True)
    freed = b.clone()
    freed.untyped_storage().resize_(0)
    for t in (freed, Wrapper(b), torch._efficientzerotensor(24, device="cuda")):
        for f in (lambda: nn.gated_linear(x, gw, uw, t), lambda: nn.gated_linear(x, gw, uw, None, t), lambda: nn.gradient_norm([b, t]),
                  lambda: nn.clip_gradients([b.clone()], 1.0, into=[t]), lambda: nn.clip_gradients([t], 1.0, into=[b.clone()])):
            with pytest.raises((RuntimeError, NotImplementedError)):
                f()
    for t in (Wrapper(c), torch._efficientzerotensor(12, device="cuda")):
        for f in (lambda: nn.linear_cross_entropy(h, w, target, t), lambda: nn.linear_cross_entropy_backward(loss, h, w, target, lse, t)):
            with pytest.raises((RuntimeError, NotImplementedError)):
                f()
    for like, f in ((x, lambda t: nn.gated_linear(t, gw, uw)), (gw, lambda t: nn.gated_linear(x, t, uw)), (w, lambda t: nn.linear_cross_entropy(h, t, target)),
                    (h, lambda t: nn.gated_linear_backward(t, x, gate, up, gw, uw)), (h, lambda t: nn.gated_linear_backward(h, x, gate, t, gw, uw)),
                    (lse, lambda t: nn.linear_cross_entropy_backward(loss, h, w, target, t)), (lse, lambda t: nn.linear_cross_entropy_backward(t, h, w, target, lse))):
        for t in (Wrapper(like), torch._efficientzerotensor(like.shape, device="cuda")):
            with pytest.raises((RuntimeError, NotImplementedError)):
                f(t)
    # what a bias holds is not read by the gated layer's gradient
    want = nn.gated_linear_backward(h, x, gate, up, gw, uw, b, b)
    assert differ(nn.gated_linear_backward(h, x, gate, up, gw, uw, b, freed), want) == []


@gpu
def test_memory_that_runs_out():
    x = values((1, 1024), 1).expand(2 ** 30, 1024)             # its result would take 16 TiB
    w = values((4096, 1024), 2)
    with pytest.raises(torch.OutOfMemoryError):
        nn.gated_linear(x, w, w)
    target = torch.zeros(1, dtype=torch.int64, device="cuda")
    with pytest.raises(RuntimeError, match="too many rows"):
        nn.linear_cross_entropy(x, w, target.expand(2 ** 30))
    with pytest.raises(torch.OutOfMemoryError):
        nn.linear_cross_entropy(values((1, 8192), 3).expand(2 ** 26, 8192), values((16, 8192), 4), target.expand(2 ** 26))     # 2 TiB
    assert nn.gated_linear(x[:3], w, w).isfinite().all()
