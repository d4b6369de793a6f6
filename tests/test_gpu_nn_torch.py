"""hetuctr_amd.nn beside what torch does around its own operators."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

from hetuctr_amd import nn

gpu = pytest.mark.gpu


def values(shape, seed, dtype=torch.float32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


# ---- views that carry a sign ------------------------------------------------------------------------------------------------
def negative(t):
    """The values of t, as a view that holds them with the other sign"""
    view = torch.complex(torch.zeros_like(t), -t).conj().imag
    assert view.is_neg() and torch.equal(view, t)
    return view


@gpu
@pytest.mark.parametrize("width", [1, 37])
def test_views_that_carry_a_sign(width):
    x, r, dy, ds = (values((6, width), i) for i in range(4))
    w, b = values(width, 5), values(width, 6)
    drop = nn.Drop(0.3, 4, 4)
    assert torch.equal(nn.dropout(negative(x), drop), nn.dropout(x, drop))
    step = torch._neg_view(torch.tensor([-4], device="cuda"))
    assert step.item() == 4 and torch.equal(nn.dropout(x, nn.Drop(0.3, 4, 0, step)), nn.dropout(x, drop))
    y, mean, rstd = want = nn.layer_norm(x, w, b, stats=True)
    for a, g in zip(nn.layer_norm(negative(x), negative(w), negative(b), stats=True), want):
        assert torch.equal(a, g)
    want = nn.layer_norm_backward(dy, x, mean, rstd, w, b)
    for a, g in zip(nn.layer_norm_backward(negative(dy), negative(x), negative(mean), negative(rstd), negative(w), negative(b)), want):
        assert torch.equal(a, g)
    y, s, mean, rstd = want = nn.dropout_add_layer_norm(x, r, w, b, drop=drop, stats=True)
    for a, g in zip(nn.dropout_add_layer_norm(negative(x), negative(r), negative(w), negative(b), drop=drop, stats=True), want):
        assert torch.equal(a, g)
    want = nn.dropout_add_layer_norm_backward(dy, ds, s, mean, rstd, w, b, drop=drop)
    for a, g in zip(nn.dropout_add_layer_norm_backward(negative(dy), negative(ds), negative(s), mean, rstd, w, b, drop=drop), want):
        assert torch.equal(a, g)


# ---- forward-mode derivatives -----------------------------------------------------------------------------------------------
def calls(x, r, w, b, stat):
    drop = nn.Drop(0.3, 4, 4)
    yield "dropout", (x,), lambda x: nn.dropout(x, drop)
    yield "layer_norm", (x, w, b), lambda x, w, b: nn.layer_norm(x, w, b)
    yield "dropout_add_layer_norm", (x, r, w, b), lambda x, r, w, b: nn.dropout_add_layer_norm(x, r, w, b, drop=drop)
    yield "layer_norm_backward", (r, x, stat, stat, w), lambda dy, x, mean, rstd, w: nn.layer_norm_backward(dy, x, mean, rstd, w)
    yield ("dropout_add_layer_norm_backward", (r, r, x, stat, stat, w),
           lambda dy, ds, s, mean, rstd, w: nn.dropout_add_layer_norm_backward(dy, ds, s, mean, rstd, w))


@gpu
def test_forward_mode_derivatives_are_refused_not_lost():
    x, r, w, b, stat = values((4, 8), 1), values((4, 8), 2), values(8, 3), values(8, 4), values(4, 5).abs()
    for name, args, f in calls(x, r, w, b, stat):
        for i in range(len(args)):
            for needs in (False, True):
                with forward_ad.dual_level():
                    given = [a.clone().requires_grad_(needs) for a in args]
                    given[i] = forward_ad.make_dual(given[i], torch.ones_like(args[i]))
                    with pytest.raises(RuntimeError, match="forward-mode|jvp"):
                        f(*given)
        with forward_ad.dual_level(), torch.no_grad(), forward_ad._set_fwd_grad_enabled(False):
            f(forward_ad.make_dual(args[0], torch.ones_like(args[0])), *args[1:])      # nothing to lose


# ---- programs that are recorded ---------------------------------------------------------------------------------------------
def program(x, r, dy, w, b, step):
    drop = nn.Drop(0.3, -4, 2 ** 63 + 1)
    h, mean, rstd = nn.layer_norm(x, w, b, drop=drop, stats=True, dtype=torch.bfloat16)
    grads = nn.layer_norm_backward(dy.bfloat16(), x, mean, rstd, w, b, drop=drop)
    y, s, mean, rstd = nn.dropout_add_layer_norm(h, r, w, None, drop=drop, stats=True)
    back = nn.dropout_add_layer_norm_backward(dy.bfloat16(), r, s, mean, rstd, w, drop=drop)
    t, u = nn.dropout_add_layer_norm(r, x)
    same = nn.dropout_add_layer_norm_backward(dy, None, u, mean, rstd)
    assert same[0] is same[1] and back[3] is None
    return (h, *grads, y, s, *back[:3], t, u, same[0], nn.dropout(nn.layer_norm(x), nn.Drop(0.2, 1, 3, step)), nn.dropout(x, None))


def inputs(seed, rows=5):
    return [values(s, seed + i) for i, s in enumerate(((rows, 16), (rows, 16), (rows, 16), 16, 16))] + [torch.tensor([seed], device="cuda")]


def differ(got, want):
    return [i for i, (a, b) in enumerate(zip(got, want)) if a.dtype != b.dtype or not torch.equal(a, b)]


@gpu
@pytest.mark.parametrize("mode", ["real", "fake", "symbolic"])
def test_programs_recorded_as_graphs_compute_what_they_say(mode):
    graph = make_fx(program, tracing_mode=mode)(*inputs(1))
    for seed in (1, 50):
        assert differ(graph(*inputs(seed)), program(*inputs(seed))) == []
    if mode == "symbolic":
        assert differ(graph(*inputs(7, rows=9)), program(*inputs(7, rows=9))) == []


@gpu
@pytest.mark.parametrize("mode", ["real", "fake"])
def test_training_steps_recorded_as_graphs(mode):
    def step(x, r, dy, w, b, more):
        drop = nn.Drop(0.3, 4, 5, more)
        leaves = [t.detach().requires_grad_() for t in (x, r, w, b)]
        x, r, w, b = leaves
        y, s = nn.dropout_add_layer_norm(nn.dropout(x, drop), r, w, b, drop=drop)
        return torch.autograd.grad((nn.layer_norm(y, w, b, drop=drop), s), leaves, (dy, dy))

    graph = make_fx(step, tracing_mode=mode)(*inputs(1))
    for seed in (1, 50):
        assert differ(graph(*inputs(seed)), step(*inputs(seed))) == []


@gpu
@pytest.mark.parametrize("needs", [False, True])
def test_traced_programs_compute_what_they_say(needs):
    graph = torch.jit.trace(program, inputs(1) if not needs else [t.requires_grad_(t.is_floating_point()) for t in inputs(1)])
    for seed in (1, 50):
        assert differ(graph(*inputs(seed)), program(*inputs(seed))) == []
    # run with inputs that want gradients
    f = lambda x, w: nn.layer_norm(nn.dropout(x, nn.Drop(0.2, 1)), w)
    x, _, dy, w = inputs(3)[:4]
    if needs:
        x, w = x.requires_grad_(), w.requires_grad_()
    graph = torch.jit.trace(f, (x, w))
    x, w = (t.detach().clone().requires_grad_() for t in (x, w))
    assert differ(torch.autograd.grad(graph(x, w), (x, w), dy), torch.autograd.grad(f(x, w), (x, w), dy)) == []


class Watcher(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.seen = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.seen.append(str(func))
        return func(*args, **(kwargs or {}))


@gpu
def test_dispatch_modes_see_the_calls():
    want = program(*inputs(1))
    given = inputs(1)
    with Watcher() as outer, Watcher() as inner:
        got = program(*given)
    assert differ(got, want) == []
    for watcher in (outer, inner):
        own = [name for name in watcher.seen if name.startswith("hetuctr_amd.")]
        assert len(own) == 9 and not any(name.startswith("aten.empty") for name in watcher.seen)
    # a checkpointed layer is worked out again in its gradient's pass
    x, _, dy, w, b = (t.requires_grad_() for t in inputs(5)[:5])
    f = lambda x, w, b: nn.layer_norm(nn.dropout(x, nn.Drop(0.2, 1)), w, b)
    want = torch.autograd.grad(f(x, w, b), (x, w, b), dy)
    context = lambda: torch.utils.checkpoint.create_selective_checkpoint_contexts([torch.ops.aten.mm.default])
    out = torch.utils.checkpoint.checkpoint(f, x, w, b, use_reentrant=False, context_fn=context)
    assert differ(torch.autograd.grad(out, (x, w, b), dy), want) == []


def test_shapes_without_memory():
    # no GPU is needed: nothing is computed
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x = torch.empty((3, 5, 16), device="cuda")
        h = torch.empty((3, 5, 16), device="cuda", dtype=torch.bfloat16)
        w = torch.empty(16, device="cuda")
        drop = nn.Drop(0.1, 2 ** 64 - 1, -1)
        assert nn.dropout(h, drop).shape == (3, 5, 16)
        y, mean, rstd = nn.layer_norm(x, w, None, drop=drop, dtype=torch.bfloat16, stats=True)
        assert y.shape == x.shape and y.dtype == torch.bfloat16 and mean.shape == rstd.shape == (15,) and mean.dtype == torch.float32
        dx, dweight, dbias = nn.layer_norm_backward(h, x, mean, rstd, w)
        assert dx.shape == x.shape and dx.dtype == x.dtype and dweight.shape == (16,) and dbias is None
        y, s, mean, rstd = nn.dropout_add_layer_norm(h, x, w, w, drop=drop, stats=True)
        assert y.dtype == h.dtype and s.dtype == x.dtype and s.shape == x.shape and rstd.shape == (15,)
        dx, dresidual, dweight, dbias = nn.dropout_add_layer_norm_backward(h, x, s, mean, rstd, w, w, drop=drop)
        assert dx.dtype == h.dtype and dresidual.dtype == x.dtype and dweight.shape == dbias.shape == (16,)
        dx, dresidual, dweight, dbias = nn.dropout_add_layer_norm_backward(x, None, s, mean, rstd)
        assert dx is dresidual and dweight is None and dbias is None
        with pytest.raises(RuntimeError, match="on the GPU"):
            nn.dropout(torch.empty((2, 4)), drop)


# ---- tensors without memory -------------------------------------------------------------------------------------------------
class Wrapper(torch.Tensor):
    """A tensor whose values are elsewhere"""
    @staticmethod
    def __new__(cls, t):
        return torch.Tensor._make_wrapper_subclass(cls, t.size(), strides=t.stride(), dtype=t.dtype, device=t.device)

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise NotImplementedError("%s of a Wrapper" % func)


@gpu
def test_tensors_without_memory_are_not_taken_for_missing_ones():
    x, w, stat = values((4, 8), 1), values(8, 2), values(4, 3)
    step = torch.zeros(1, dtype=torch.int64, device="cuda")
    freed, hidden, nothing = w.clone(), Wrapper(w), torch._efficientzerotensor(8, device="cuda")
    freed.untyped_storage().resize_(0)
    for f in (lambda t: nn.layer_norm(x, t), lambda t: nn.layer_norm(x, None, t), lambda t: nn.layer_norm_backward(x, x, stat, stat, t),
              lambda t: nn.dropout_add_layer_norm(x, x, w, t)):
        for t in (freed, hidden, nothing):
            with pytest.raises(RuntimeError):
                f(t)
    for t in (Wrapper(x), torch._efficientzerotensor((4, 8), device="cuda")):
        with pytest.raises(RuntimeError):
            nn.dropout_add_layer_norm_backward(x, t, x, stat, stat)
    with pytest.raises(RuntimeError):
        nn.dropout(x, nn.Drop(0.5, 1, 0, Wrapper(step)))
    # what bias holds is not read by the gradient
    want = nn.layer_norm_backward(x, x, stat, stat, w, w)
    assert all(torch.equal(a, g) for a, g in zip(nn.layer_norm_backward(x, x, stat, stat, w, freed), want))


# ---- errors -----------------------------------------------------------------------------------------------------------------
@gpu
def test_errors_keep_their_type():
    x = values((1, 1024), 1).expand(2 ** 33, 1024)             # its result would take 32 TiB
    for f in (lambda: nn.dropout(x, nn.Drop(0.5, 1)), lambda: nn.layer_norm(x)):
        with pytest.raises(torch.OutOfMemoryError):
            f()
    x = values((2, 8), 1)
    with pytest.raises(RuntimeError) as e:
        nn.layer_norm(x, eps=-1.0)
    assert "eps" in str(e.value) and "frame #" not in str(e.value)
    with pytest.raises(TypeError):
        nn.layer_norm(x, eps="small")
    with pytest.raises(TypeError):
        nn.dropout(x, nn.Drop(0.5, "seed"))
    with pytest.raises(RuntimeError, match="Boolean value"):
        nn.layer_norm(x, stats=torch.ones(2))
    with pytest.raises(RuntimeError) as e:
        nn.layer_norm(x.to_sparse())
    assert "frame #" not in str(e.value)
