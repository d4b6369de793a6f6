"""Operators between the table's rows and a dense model, on torch tensors: dropout from a counter-based generator, layer
normalisation, and both in one pass, with their gradients.  The reference has none of them: its table hands float rows to a model
that lives outside (tests/check.py:44), and takes the gradient of those rows back.

    table.preprocess(ids.data_ptr(), n); table.push_pull(grad_ptr, rows.data_ptr())
    rows.requires_grad_()
    h = nn.layer_norm(rows, weight, bias, drop=nn.Drop(0.1, seed=1, step=t), dtype=torch.bfloat16)
    ...                                                     # the dense model
    loss.backward()                                         # rows.grad: float32, what the next push_pull takes

A tensor's last dimension is a row; the others, if any, count rows.  Rows of float32, bfloat16 or float16 may lie any number of
elements apart; where the tensor's memory order does not allow that, a call copies it first.  Results are new contiguous
tensors.  Work goes to torch's current stream, nothing waits, and a call may be captured into a graph.  The functions without
`_backward` in their name can be differentiated (once, in reverse: a tensor with a tangent is refused); the others are the gradients
themselves, for programs that keep their own books.
"""
import importlib
import sys
from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from . import LIBDIR


def _load():
    if LIBDIR not in sys.path:
        sys.path.insert(0, LIBDIR)
    try:
        return importlib.import_module("hetuctr_nn")
    except ImportError as e:
        raise ImportError("the hetuctr_nn extension is not built: run `python -m hetuctr_amd.build` (%s)" % e)


_native = _load()
# (a twentieth of what torch.cuda.current_stream takes, 1.9 us of a call whose kernel may take 3)
_stream_of = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


class Drop(NamedTuple):
    """Which values are dropped: each with probability `p`, as a function of its row and column, `seed` and `step` alone
    (include/hetuctr_hip.h, hctr_drop).  Give every layer a seed and every training step a step; the gradient's call drops
    what the forward call dropped.  `step_tensor`, an int64 tensor of one element on the GPU, is added to the step: a
    captured graph draws new numbers as it changes."""
    p: float
    seed: int
    step: int = 0
    step_tensor: Optional[torch.Tensor] = None


def _run(f, x, *args):
    """f(*args, torch's current stream), on the device of x"""
    index = x.get_device()
    if index < 0:
        raise RuntimeError("hetuctr_amd.nn: the tensors must be on the GPU")
    if index == torch.cuda.current_device():
        return f(*args, _stream_of(index))
    with torch.cuda.device(index):
        return f(*args, _stream_of(index))


def _wants_gradient(*tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


# ---- dropout ----------------------------------------------------------------------------------------------------------
class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, drop, step_tensor):
        ctx.drop = drop
        ctx.save_for_backward(step_tensor)      # a step that changed before the gradient was drawn is an error
        return _run(_native.dropout, x, x, drop)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        ctx.saved_tensors
        return _run(_native.dropout, dy, dy, ctx.drop), None, None


def dropout(x, drop):
    """x with the values that `drop` (a Drop) names replaced by zero and the others multiplied by 1 / (1 - p); its own
    gradient: dropout(dy, drop)."""
    if _wants_gradient(x):
        return _Dropout.apply(x, drop, drop.step_tensor if drop else None)
    return _run(_native.dropout, x, x, drop)


# ---- layer normalisation ------------------------------------------------------------------------------------------------
class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, drop, dtype, step_tensor):
        y, mean, rstd = _run(_native.forward, x, x, None, weight, bias, eps, drop, dtype, True)
        ctx.drop = drop
        ctx.save_for_backward(x, weight, bias, mean, rstd, step_tensor)
        ctx.mark_non_differentiable(mean, rstd)
        return y, mean, rstd

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, _mean, _rstd):
        x, weight, bias, mean, rstd, _ = ctx.saved_tensors
        dx, dweight, dbias = _run(_native.backward, x, False, dy, None, x, mean, rstd, weight, bias, ctx.drop, True,
                                  *ctx.needs_input_grad[1:3])
        return dx, dweight, dbias, None, None, None, None


def layer_norm(x, weight=None, bias=None, eps=1e-5, *, drop=None, dtype=None, stats=False):
    """(x - mean) / sqrt(variance + eps) * weight + bias over the last dimension, values dropped as `drop` says.  The result has
    type `dtype`: that of x, or, where x is float32, any.  weight and bias are float32 or of the result's type.  With `stats`
    returns (result, mean, 1 / sqrt(variance + eps)), float32, one of each a row."""
    if _wants_gradient(x, weight, bias):
        out = _LayerNorm.apply(x, weight, bias, eps, drop, dtype, drop.step_tensor if drop else None)
    else:
        out = _run(_native.forward, x, x, None, weight, bias, eps, drop, dtype, stats)
    return out if stats else out[0]


def layer_norm_backward(dy, x, mean, rstd, weight=None, bias=None, *, drop=None):
    """(dx, dweight, dbias) of layer_norm, given the gradient of its result and what it was called with and returned.  dx has
    the type of x, dweight that of weight, dbias that of bias (None where there is none); what bias holds is not read."""
    return _run(_native.backward, x, False, dy, None, x, mean, rstd, weight, bias, drop, True, True, True)


# ---- residual + dropout, normalised -----------------------------------------------------------------------------------
class _DropoutAddLayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps, drop, step_tensor):
        y, s, mean, rstd = _run(_native.forward, x, x, residual, weight, bias, eps, drop, None, True)
        ctx.drop, ctx.act = drop, x.dtype
        ctx.save_for_backward(s, weight, bias, mean, rstd, step_tensor)
        ctx.mark_non_differentiable(mean, rstd)
        ctx.set_materialize_grads(False)
        return y, s, mean, rstd

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, ds, _mean, _rstd):
        s, weight, bias, mean, rstd, _ = ctx.saved_tensors
        if dy is None:                          # only the sum was used
            if ds is None:
                return (None,) * 7
            dx = _run(_native.dropout, ds, ds, ctx.drop) if ctx.drop else ds
            return dx.to(ctx.act), ds, None, None, None, None, None
        need_x, need_weight, need_bias = (ctx.needs_input_grad[i] for i in (0, 2, 3))
        dx, dresidual, dweight, dbias = _run(_native.backward, s, True, dy, ds, s, mean, rstd, weight, bias, ctx.drop, need_x,
                                             need_weight, need_bias)
        return dx, dresidual, dweight, dbias, None, None, None


def dropout_add_layer_norm(x, residual, weight=None, bias=None, eps=1e-5, *, drop=None, stats=False):
    """(y, s) with s = residual + dropout(x) and y = layer_norm(s): the step between two layers.  x and y are of one type, residual
    and s of that type or float32; weight and bias are float32 or of the type of x.  y is computed from s before it is
    rounded.  With `stats` returns (y, s, mean, 1 / sqrt(variance + eps)), as layer_norm does."""
    if _wants_gradient(x, residual, weight, bias):
        out = _DropoutAddLayerNorm.apply(x, residual, weight, bias, eps, drop, drop.step_tensor if drop else None)
    else:
        out = _run(_native.forward, x, x, residual, weight, bias, eps, drop, None, stats)
    return out if stats else out[:2]


def dropout_add_layer_norm_backward(dy, ds, s, mean, rstd, weight=None, bias=None, *, drop=None):
    """(dx, dresidual, dweight, dbias) of dropout_add_layer_norm, given the gradients of its two results (ds may be None), the sum
    s and the rows' statistics that it returned.  dx has the type of dy, dresidual that of s; without dropout and where these
    are one type, they are one tensor."""
    return _run(_native.backward, s, True, dy, ds, s, mean, rstd, weight, bias, drop, True, True, True)
