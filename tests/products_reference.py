"""The operators of tests/test_gpu_products.py in torch's float64, by their formulas, and how far rounding may take a result from them.

Every function returns (value, slack): the kernels' result may be off by `slack` before it is rounded to its type.

Units.  U = 2^-24: half a step of a float, relative.  A sum of n terms held in 32 bits, whatever its order, is off by at most n units of
the sum of their sizes; where a matrix core adds, 2 n, because it may cut off what it does not keep.  UNIT[t]: half a step of
type t, relative; TINY[t]: its smallest normal value, below which half a step is UNIT * TINY."""
import math

import torch

U = 2.0 ** -24
UNIT = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}
TINY = {t: torch.finfo(t).tiny for t in UNIT}


def rounding(value, dtype):
    return UNIT[dtype] * value.abs().clamp_min(TINY[dtype])


def check(got, want, slack, what):
    """Every value within `slack` and one rounding to got's type of what it should be"""
    dtype, got = got.dtype, got.detach().double().reshape(want.shape)
    allowed = slack + UNIT[dtype] * (want.abs() + slack).clamp_min(TINY[dtype])
    bad = ~((got - want).abs() <= allowed) & ~(got.isnan() & want.isnan()) & ~((got == want) & want.isinf())
    if bad.any():
        at = bad.nonzero()
        worst = ((got - want).abs() / allowed).nan_to_num(1e30, 1e30).max().item()
        raise AssertionError("%s: %d of %d values, first at %s (%g, not %g), last at %s, worst %.3g of what is allowed" % (
            what, len(at), bad.numel(), at[0].tolist(), got[tuple(at[0])], want[tuple(at[0])], at[-1].tolist(), worst))


def product(a, b, slack_a=None):
    """a @ b.T and its slack, where a itself may be off by slack_a"""
    size = a.abs() @ b.abs().T
    slack = 2 * (a.shape[1] + 64) * U * size
    return a @ b.T, slack if slack_a is None else slack + slack_a @ b.abs().T


def activation(f, v):
    """f(v), f'(v)"""
    if f == "relu":
        return v.clamp_min(0), (v > 0).double()
    if f == "gelu":
        whole = torch.special.ndtr(v)
        return v * whole, whole + v * torch.exp(-v * v / 2) / math.sqrt(2 * math.pi)
    s = torch.sigmoid(v)
    return (v * s, s + v * s * (1 - s)) if f == "silu" else (s, s * (1 - s))


# The steepest slope of any of them is that of gelu, 1.13, and its derivative's 0.8: what an error of the argument does to the value and to the
# slope.  A float exponential, quotient and integral of the normal distribution are within 16 units together, and an argument that is
# rounded on its way to the exponential counts as many units as it is large, at most 16 where the value matters (exp(-16) = 1e-7).
FUNCTION = 32 * U


def gated(x, gate_weight, up_weight, gate_bias, up_bias, f):
    gate, gate_slack = product(x, gate_weight)
    up, up_slack = product(x, up_weight)
    if gate_bias is not None:
        gate, gate_slack = gate + gate_bias, gate_slack + U * (gate.abs() + gate_bias.abs())
    if up_bias is not None:
        up, up_slack = up + up_bias, up_slack + U * (up.abs() + up_bias.abs())
    value, _ = activation(f, gate)
    value_slack = 1.13 * gate_slack + FUNCTION * (value.abs() + gate.abs().clamp_max(1))
    h_slack = value_slack * (up.abs() + up_slack) + value.abs() * up_slack + U * (value * up).abs()
    return (value * up, h_slack), (gate, gate_slack), (up, up_slack)


def gated_gradient(dh, x, gate, up, gate_weight, up_weight, f, dtype):
    """dx, dgate_weight, dup_weight, dgate_bias, dup_bias"""
    value, slope = activation(f, gate)
    ds = []
    for factor, more in ((slope, up), (value, None)):
        d = dh * factor if more is None else dh * factor * more
        slack = FUNCTION * (dh.abs() * (factor.abs() + gate.abs().clamp_max(2)) * (1 if more is None else more.abs()))
        ds.append((d, slack))
    (dg, sg), (du, su) = ds
    rows = dh.shape[0]
    # rounded to the type before the products
    rg, ru = sg + rounding(dg.abs() + sg, dtype), su + rounding(du.abs() + su, dtype)
    dx, slack = product(torch.cat((dg, du), 1), torch.cat((gate_weight, up_weight), 0).T, torch.cat((rg, ru), 1))
    out = [(dx, slack)]
    for d, r in ((dg, rg), (du, ru)):
        out.append(product(d.T, x.T, r.T))
    for d, s in ((dg, sg), (du, su)):
        out.append((d.sum(0), s.sum(0) + (rows + 16) * U * d.abs().sum(0)))
    return out


def logits(x, weight, bias):
    l, slack = product(x, weight)
    if bias is not None:
        l, slack = l + bias, slack + U * (l.abs() + torch.where(bias.isinf(), 0.0, bias.abs()))
    return l, slack


def cross_entropy(x, weight, bias, target, ignored):
    """loss, lse: an error of the logits is at most passed on; a difference of two floats is one more unit of them, and what an exponential is
    off by (16 units and as many as its argument is large) is averaged, weighted with itself"""
    l, slack = logits(x, weight, bias)
    there = target != ignored
    lse = torch.logsumexp(l, 1)
    p = torch.exp(l - lse[:, None])
    far = torch.where(p > 0, (l - lse[:, None]).abs(), 0.0)
    own = (p * (slack + (32 + 4 * far) * U)).sum(1) + (l.shape[1] + 64) * U + 4 * U * lse.abs()
    hit = l.gather(1, target.clamp(0, l.shape[1] - 1)[:, None])[:, 0]
    hit_slack = slack.gather(1, target.clamp(0, l.shape[1] - 1)[:, None])[:, 0]
    zero = torch.zeros((), dtype=torch.float64, device=x.device)
    loss = torch.where(there, lse - hit, zero)
    return (loss, torch.where(there, own + hit_slack + 4 * U * (lse.abs() + hit.abs()), zero)), (torch.where(there, lse, zero), torch.where(there, own, zero))


def cross_entropy_gradient(dloss, x, weight, bias, target, lse, ignored, dtype):
    """dx, dweight, dbias: lse and dloss as they are given"""
    l, slack = logits(x, weight, bias)
    there = target != ignored
    less = (l - lse[:, None])
    p = torch.exp(less)
    p_slack = p * (slack + (16 + 4 * torch.where(p > 0, less.abs(), 0.0)) * U)
    one = torch.zeros_like(p)
    one[there, target[there]] = 1
    scale = torch.where(there, dloss, 0.0)[:, None]
    keep = there[:, None]
    d = torch.where(keep, (p - one) * scale, 0.0)
    d_slack = torch.where(keep, (p_slack + 2 * U * (p + one)) * scale.abs(), 0.0)
    if dtype == torch.float16:
        # a power of two takes the largest |dloss| to 2^13 at least, so that what is smaller than 2^-14 of it there is 2^-27 of dloss
        step = UNIT[dtype] * (d.abs() + d_slack).clamp_min(2.0 ** -27 * scale.abs().max())
    else:
        step = rounding(d.abs() + d_slack, dtype)
    r = torch.where(keep, d_slack + step, 0.0)
    safe = torch.where(keep, x, 0.0)            # what an ignored row holds does not count
    dx, dx_slack = product(d, weight.T, r)
    dw, dw_slack = product(d.T, safe.T, r.T)
    # (the sums are multiplied by 1 / that power: exact)
    return (dx, dx_slack), (dw, dw_slack), (d.sum(0), d_slack.sum(0) + (d.shape[0] + 64) * U * d.abs().sum(0))
