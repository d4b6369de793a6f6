"""Operators between the table's rows and a dense model, and of the model's training step, on torch tensors: dropout from a
counter-based generator, layer normalisation, and both in one pass; a gated linear layer; softmax cross entropy over many items (the rows of a
table, say); with their gradients; the norm of all gradients and clipping by it.  The reference has none of them: its table hands
float rows to a model that lives outside (tests/check.py:44), and takes the gradient of those rows back.

    table.preprocess(ids.data_ptr(), n); table.push_pull(grad_ptr, rows.data_ptr())
    rows.requires_grad_()
    h = nn.layer_norm(rows, weight, bias, drop=nn.Drop(0.1, seed=1, step=t), dtype=torch.bfloat16)
    ...                                                     # the dense model
    h = nn.gated_linear(h, gate_weight, up_weight)
    loss = nn.linear_cross_entropy(h, item_vectors, target).mean()
    loss.backward()                                         # rows.grad: float32, what the next push_pull takes
    nn.clip_gradients([p.grad for p in parameters] + [rows.grad], 1.0)

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
    if x is None:
        raise RuntimeError("hetuctr_amd.nn: there are no gradients")
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
        ctx.set_materialize_grads(False)        # or zeros are made for mean and rstd
        return y, mean, rstd

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, _mean, _rstd):
        if dy is None:
            return (None,) * 7
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


# ---- a gated linear layer ---------------------------------------------------------------------------------------------
_ACTIVATIONS = {"silu": 0, "gelu": 1, "relu": 2, "sigmoid": 3}


class _GatedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate_weight, up_weight, gate_bias, up_bias, activation):
        h, gate, up = _run(_native.gated, x, x, gate_weight, up_weight, gate_bias, up_bias, activation, True)
        ctx.activation = activation
        ctx.save_for_backward(x, gate, up, gate_weight, up_weight, gate_bias, up_bias)
        ctx.mark_non_differentiable(gate, up)
        ctx.set_materialize_grads(False)        # or matrices of zeros are made for gate and up
        return h, gate, up

    @staticmethod
    @once_differentiable
    def backward(ctx, dh, _gate, _up):
        if dh is None:
            return (None,) * 6
        return (*_run(_native.gated_backward, dh, dh, *ctx.saved_tensors, ctx.activation, *ctx.needs_input_grad[:5]), None)


def gated_linear(x, gate_weight, up_weight, gate_bias=None, up_bias=None, activation="silu", *, saved=False):
    """f(x @ gate_weight.T + gate_bias) * (x @ up_weight.T + up_bias): both products, the activation f ("silu", "gelu", "relu" or
    "sigmoid") and their product in one pass.  The weights are [hidden, width], of the type of x; the biases are float32 or of
    that type.  With `saved` returns (result, gate product, up product), each rounded once, as the gradient needs them."""
    activation = _ACTIVATIONS.get(activation, -1)
    if _wants_gradient(x, gate_weight, up_weight, gate_bias, up_bias):
        out = _GatedLinear.apply(x, gate_weight, up_weight, gate_bias, up_bias, activation)
    else:
        out = _run(_native.gated, x, x, gate_weight, up_weight, gate_bias, up_bias, activation, saved)
    return out if saved else out[0]


def gated_linear_backward(dh, x, gate, up, gate_weight, up_weight, gate_bias=None, up_bias=None, activation="silu"):
    """(dx, dgate_weight, dup_weight, dgate_bias, dup_bias) of gated_linear, given the gradient of its result, what it was called with,
    and the products that it returned.  Each has the type of what it is the gradient of (None where that is); what the biases
    hold is not read."""
    return _run(_native.gated_backward, dh, dh, x, gate, up, gate_weight, up_weight, gate_bias, up_bias, _ACTIVATIONS.get(activation, -1),
                True, True, True, True, True)


# ---- cross entropy over many items ------------------------------------------------------------------------------------
class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, target, bias, ignore_index):
        loss, lse = _run(_native.items, x, x, weight, target, bias, ignore_index, True)
        ctx.ignore_index = ignore_index
        ctx.save_for_backward(x, weight, target, lse, bias)
        ctx.mark_non_differentiable(lse)
        ctx.set_materialize_grads(False)
        return loss, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss, _lse):
        if dloss is None:
            return (None,) * 5
        x, weight, target, lse, bias = ctx.saved_tensors
        dx, dweight, dbias = _run(_native.items_backward, dloss, dloss, x, weight, target, lse, bias, ctx.ignore_index,
                                  *(ctx.needs_input_grad[i] for i in (0, 1, 3)))
        return dx, dweight, None, dbias, None


def linear_cross_entropy(x, weight, target, bias=None, *, ignore_index=-100, stats=False):
    """The softmax cross entropy of x @ weight.T + bias with the items that `target` names, float32, one for each row, without a matrix of
    logits in memory.  weight is [items, width], of the type of x; bias is float32 or of that type; target is int64, of
    the shape of the result.  Rows whose target is `ignore_index` take no part, whatever x holds there: their loss is 0.  A
    target that is neither that nor an item gives NaN.  An item whose bias is below -1e30 does not count.  With `stats` returns (loss, log of the
    sum of exponentials)."""
    if _wants_gradient(x, weight, bias):
        out = _LinearCrossEntropy.apply(x, weight, target, bias, ignore_index)
    else:
        out = _run(_native.items, x, x, weight, target, bias, ignore_index, stats)
    return out if stats else out[0]


def linear_cross_entropy_backward(dloss, x, weight, target, lse, bias=None, *, ignore_index=-100):
    """(dx, dweight, dbias) of linear_cross_entropy, given the gradient of its result (float32, one for each row), what it was called
    with, and the log of the sum of exponentials that it returned.  Each has the type of what it is the gradient of."""
    return _run(_native.items_backward, dloss, dloss, x, weight, target, lse, bias, ignore_index, True, True, True)


# ---- many gradients ---------------------------------------------------------------------------------------------------
def gradient_norm(gradients):
    """The 2-norm of all the gradients together: a float32 on the GPU.  Squares and their sums are held in 64 bits.  Not differentiable."""
    gradients = list(gradients)
    if _wants_gradient(*gradients):
        raise RuntimeError("hetuctr_amd.nn: the norm of gradients is not differentiable: call this under torch.no_grad()")
    return _run(_native.gradient_norm, gradients[0] if gradients else None, gradients)


def clip_gradients(gradients, max_norm, *, norm=None, into=None):
    """Multiplies every gradient by min(1, max_norm / norm), in place or `into` tensors of the same types and shapes, and returns the norm: that
    of gradient_norm, or the one that is given (a float32 on the GPU: where several GPUs hold a part of the gradients
    each).  No result may lie where another gradient or result, or `norm`, does; each holds its values one behind the other.  Where the norm is
    not finite, what is multiplied is not either, or zero."""
    gradients = list(gradients)
    into = gradients if into is None else list(into)
    out = _run(_native.clip_gradients, gradients[0] if gradients else None, gradients, into, max_norm, norm, torch.is_grad_enabled())
    return out if norm is None else norm


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
    if f in _PLAIN_NAME_OF:
        return _as_plain_operator(f, args)
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


# Those without a Drop take the extension's arguments as they are, and return what there is of its results; `_there` says which of them
# that is.
_PLAIN_SCHEMAS = {
    "gated_linear": "(Tensor x, Tensor gate_weight, Tensor up_weight, Tensor? gate_bias, Tensor? up_bias, int activation, bool saved) "
                    "-> Tensor[]",
    "gated_linear_backward": "(Tensor dh, Tensor x, Tensor gate, Tensor up, Tensor gate_weight, Tensor up_weight, Tensor? gate_bias, "
                             "Tensor? up_bias, int activation, bool need_x, bool need_gate_weight, bool need_up_weight, "
                             "bool need_gate_bias, bool need_up_bias) -> Tensor[]",
    "linear_cross_entropy": "(Tensor x, Tensor weight, Tensor target, Tensor? bias, int ignore_index, bool stats) -> Tensor[]",
    "linear_cross_entropy_backward": "(Tensor dloss, Tensor x, Tensor weight, Tensor target, Tensor lse, Tensor? bias, int ignore_index, "
                                     "bool need_x, bool need_weight, bool need_bias) -> Tensor[]",
    "gradient_norm": "(Tensor[] gradients) -> Tensor",
    "clip_gradients": "(Tensor[] gradients, Tensor(a!)[] into, float max_norm, Tensor? norm, bool leaves) -> Tensor",
}
_PLAIN = {"gated_linear": _native.gated, "gated_linear_backward": _native.gated_backward, "linear_cross_entropy": _native.items,
          "linear_cross_entropy_backward": _native.items_backward, "gradient_norm": _native.gradient_norm,
          "clip_gradients": _native.clip_gradients}
_PLAIN_NAME_OF = {f: name for name, f in _PLAIN.items()}
_LISTS = ("gradient_norm", "clip_gradients")


def _there(name, args):
    if name == "gated_linear":
        return [True, args[6], args[6]]
    if name == "gated_linear_backward":
        return [*args[9:12], args[6] is not None and args[12], args[7] is not None and args[13]]
    if name == "linear_cross_entropy":
        return [True, args[5]]
    return [args[7], args[8], args[5] is not None and args[9]]


def _as_plain_operator(f, args):
    name = _PLAIN_NAME_OF[f]
    out = getattr(torch.ops.hetuctr_amd, name)(*args)
    if name in _LISTS:
        return out
    out = iter(out)
    return tuple(next(out) if there else None for there in _there(name, args))


def _plain_compute(name, *args):
    first = args[0][0] if name in _LISTS else args[0]
    with torch.cuda.device(first.device):
        out = _PLAIN[name](*args, torch.cuda.current_stream().cuda_stream)
    if name in _LISTS:
        return out if name == "gradient_norm" or args[3] is None else out.clone()      # an operator's result is a tensor of its own
    return [t for t in out if t is not None]


def _plain_shapes(name, *args):
    if name in _LISTS:
        return args[0][0].new_empty((), dtype=torch.float32)
    if name == "gated_linear":
        x, gate_weight = args[:2]
        return [x.new_empty((*x.shape[:-1], gate_weight.shape[0])) for there in _there(name, args) if there]
    if name == "linear_cross_entropy":
        return [args[0].new_empty(args[0].shape[:-1], dtype=torch.float32) for there in _there(name, args) if there]
    of = (args[1], *args[4:8]) if name == "gated_linear_backward" else (args[1], args[2], args[5])
    return [t.new_empty(t.shape) for t, there in zip(of, _there(name, args)) if there]


def _plain_differentiable(name, *args):
    tensors = [t for t in args if isinstance(t, torch.Tensor)]
    if not _wants_gradient(*tensors) and not any(forward_ad.unpack_dual(t, level=0).tangent is not None for t in tensors):
        with torch._C._AutoDispatchBelowAutograd():
            return getattr(torch.ops.hetuctr_amd, name)(*args)
    out = (_GatedLinear if name == "gated_linear" else _LinearCrossEntropy).apply(*args[:-1])
    return list(out if args[-1] else out[:1])


for _name, _schema in _PLAIN_SCHEMAS.items():
    _library.define(_name + _schema)
    _library.impl(_name, functools.partial(_plain_compute, _name), "CUDA")
    torch.library.register_fake("hetuctr_amd::" + _name, functools.partial(_plain_shapes, _name), lib=_library)
    if _name in ("gated_linear", "linear_cross_entropy"):
        _library.impl(_name, functools.partial(_plain_differentiable, _name), "Autograd")
