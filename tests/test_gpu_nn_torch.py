"""hetuctr_amd.nn beside what torch does around its own operators."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

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
