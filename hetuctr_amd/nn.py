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
import functools
import importlib
import sys
from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad
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
    """f(*args, torch's current stream), on the device of x; as one of torch's operators while something watches them"""
    index = _native.unseen_on(x)
    if index < 0:
        return _as_operator(f, x, args)
    if index == torch.cuda.current_device():
        return f(*args, _stream_of(index))
    with torch.cuda.device(index):
        return f(*args, _stream_of(index))


def _wants_gradient(*tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return not _native.traced()              # a traced operator asks again
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


# ---- the same as torch operators ----------------------------------------------------------------------------------------
# torch.jit.trace, make_fx, fake tensors and dispatch modes see what goes through torch's dispatcher: of a call into the extension only
# that memory was allocated, which a recorded program would then return unfilled.  While one of them is at work, a call
# goes to the extension through an operator of torch's (hetuctr_amd::..), which is what they see.  Otherwise it does not: a call of
# layer_norm on few rows takes 19 us through the operator, 5 without.
#
# The operators take a Drop as four arguments, and return the tensors that there are: what would be None is left out, and what
# would be one tensor twice is there once.
_DROP = "float p, int seed, int step, Tensor? step_tensor"
_SCHEMAS = {
    "dropout": "(Tensor x, %s) -> Tensor[]",
    "norm": "(Tensor x, Tensor? residual, Tensor? weight, Tensor? bias, float eps, %s, ScalarType? dtype, bool stats) -> Tensor[]",
    "norm_backward": "(bool add, Tensor dy, Tensor? ds, Tensor s, Tensor mean, Tensor rstd, Tensor? weight, Tensor? bias, %s, "
                     "bool need_x, bool need_weight, bool need_bias) -> Tensor[]",
}
_EXTENSION = {"dropout": _native.dropout, "norm": _native.forward, "norm_backward": _native.backward}
_DROP_AT = {"dropout": 1, "norm": 5, "norm_backward": 8}
_NAME_OF = {f: name for name, f in _EXTENSION.items()}
_library = torch.library.Library("hetuctr_amd", "DEF")


def _as_operator(f, x, args):
    if x.device.type != "cuda":
        raise RuntimeError("hetuctr_amd.nn: the tensors must be on the GPU")
    name = _NAME_OF[f]
    at = _DROP_AT[name]
    p, seed, step, step_tensor = args[at] or (0.0, 0, 0, None)
    signed = lambda v: (v + 2 ** 63) % 2 ** 64 - 2 ** 63       # the same modulo 2^64
    out = iter(getattr(torch.ops.hetuctr_amd, name)(*args[:at], p, signed(seed), signed(step), step_tensor, *args[at + 1:]))
    if f is _native.dropout:
        return next(out)
    if f is _native.forward:
        there = [True] * (1 if args[1] is None else 2) + [args[7]] * 2
    else:
        there = [True, args[6] is not None and args[10], args[7] is not None and args[11]]
        if args[0]:                                             # dx may be dresidual
            one = _one_gradient(args[1], args[3], p)
            there.insert(0, args[9] and not one)
    out = tuple(next(out) if t else None for t in there)
    if f is _native.backward and args[0] and args[9] and one:
        out = (out[1],) + out[1:]
    return out


def _one_gradient(dy, s, p):
    return dy.dtype == s.dtype and p == 0


def _with_drop(name, args):
    at = _DROP_AT[name]
    return args[:at] + (Drop(*args[at:at + 4]),) + args[at + 4:]


def _compute(name, *args):
    args = _with_drop(name, args)
    with torch.cuda.device(args[1 if name == "norm_backward" else 0].device):
        out = _EXTENSION[name](*args, torch.cuda.current_stream().cuda_stream)
    if name == "dropout":
        return [out]
    return [t for i, t in enumerate(out) if t is not None and not (i and t is out[i - 1])]


def _shapes(name, *args):
    args = _with_drop(name, args)
    per_row = lambda t: t.new_empty(t.numel() // t.shape[-1], dtype=torch.float32)
    if name == "dropout":
        return [args[0].new_empty(args[0].shape)]
    if name == "norm":
        x, residual, _, _, _, _, dtype, stats = args
        out = [x.new_empty(x.shape, dtype=dtype)] + ([] if residual is None else [residual.new_empty(x.shape)])
        return out + ([per_row(x), per_row(x)] if stats else [])
    add, dy, _, s, _, _, weight, bias, drop, need_x, need_weight, need_bias = args
    out = [s.new_empty(s.shape)]
    if add and need_x and not _one_gradient(dy, s, drop.p):
        out.insert(0, dy.new_empty(s.shape))
    return out + [t.new_empty(t.shape) for t, need in ((weight, need_weight), (bias, need_bias)) if t is not None and need]


def _differentiable(name, *args):
    """A recorded program may be run with tensors that want gradients."""
    tensors = [t for t in args if isinstance(t, torch.Tensor)]
    if not _wants_gradient(*tensors) and not any(forward_ad.unpack_dual(t, level=0).tangent is not None for t in tensors):
        with torch._C._AutoDispatchBelowAutograd():
            return getattr(torch.ops.hetuctr_amd, name)(*args)
    args = _with_drop(name, args)
    if name == "dropout":
        return [_Dropout.apply(*args, args[1].step_tensor)]
    x, residual, weight, bias, eps, drop, dtype, stats = args
    if residual is None:
        out = _LayerNorm.apply(x, weight, bias, eps, drop, dtype, drop.step_tensor)
    else:
        out = _DropoutAddLayerNorm.apply(x, residual, weight, bias, eps, drop, drop.step_tensor)
    return list(out if stats else out[:-2])


for _name, _schema in _SCHEMAS.items():
    _library.define(_name + _schema % _DROP)
    _library.impl(_name, functools.partial(_compute, _name), "CUDA")
    torch.library.register_fake("hetuctr_amd::" + _name, functools.partial(_shapes, _name), lib=_library)
    if _name != "norm_backward":
        _library.impl(_name, functools.partial(_differentiable, _name), "Autograd")
