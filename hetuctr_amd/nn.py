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
`_backward` in their name can be differentiated (once); the others are the gradients themselves, for programs that keep
their own books.
"""
from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from . import capi

_DTYPES = {torch.float32: capi.F32, torch.bfloat16: capi.BF16, torch.float16: capi.F16}
_WORD = 0xFFFFFFFFFFFFFFFF


class Drop(NamedTuple):
    """Which values are dropped: each with probability `p`, as a function of its row and column, `seed` and `step` alone
    (include/hetuctr_hip.h, hctr_drop).  Give every layer a seed and every training step a step; the gradient's call drops
    what the forward call dropped.  `step_tensor`, an int64 tensor of one element on the GPU, is added to the step: a
    captured graph draws new numbers as it changes."""
    p: float
    seed: int
    step: int = 0
    step_tensor: Optional[torch.Tensor] = None


# The host's share of a call is several microseconds, more than a small kernel takes (1.9 of them torch.cuda.current_stream
# alone): what follows keeps to torch's cheaper calls.
_stream_of = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _drop(drop, device):
    if drop is None:
        return capi.NO_DROP
    p, seed, step, extra = drop
    if extra is None:
        return p, seed & _WORD, step & _WORD, 0
    if extra.device != device or extra.dtype != torch.int64 or extra.numel() != 1:
        raise RuntimeError("hetuctr_amd.nn: the step tensor must be one int64 on the device of the values")
    return p, seed & _WORD, step & _WORD, extra.data_ptr()


def _type(t, what):
    code = _DTYPES.get(t)
    if code is None:
        raise RuntimeError("hetuctr_amd.nn: %s must be float32, bfloat16 or float16, not %s" % (what, t))
    return code


def _matrix(t, what):
    """t as rows of its last dimension: a tensor that the caller keeps until the call is made, its (pointer, stride)."""
    if not t.is_cuda:
        raise RuntimeError("hetuctr_amd.nn: %s must be on the GPU" % what)
    if t.dim() != 2:
        if t.dim() == 0:
            raise RuntimeError("hetuctr_amd.nn: %s must have at least one dimension" % what)
        width = t.shape[-1]
        t = t.reshape(t.numel() // width if width else 0, width)
    row, column = t.stride()
    if column != 1 and t.shape[1] != 1:
        t = t.contiguous()
        row = t.stride(0)
    return t, (t.data_ptr(), row)


def _same(t, like, dtype, what):
    if t.shape != like.shape or t.dtype != dtype or t.device != like.device:
        raise RuntimeError("hetuctr_amd.nn: %s must be %s of shape %s on %s" % (what, dtype, tuple(like.shape), like.device))


def _per_column(t, width, act, device, what):
    """weight or bias, ready to be read"""
    if t is None:
        return None
    if t.shape != (width,) or t.device != device or (t.dtype != torch.float32 and t.dtype != act):
        raise RuntimeError("hetuctr_amd.nn: %s must hold %d values of float32 or %s on %s" % (what, width, act, device))
    return t if t.is_contiguous() else t.contiguous()


def _affine(weight, bias, width, act, device):
    """weight and bias (or None) ready to be read, and the code of their type"""
    weight, bias = _per_column(weight, width, act, device, "weight"), _per_column(bias, width, act, device, "bias")
    if weight is not None:
        if bias is not None and weight.dtype != bias.dtype:
            raise RuntimeError("hetuctr_amd.nn: weight and bias must be of one type")
        return weight, bias, _DTYPES[weight.dtype]
    return weight, bias, capi.F32 if bias is None else _DTYPES[bias.dtype]


def _pointer(t):
    return 0 if t is None else t.data_ptr()


def _result(like, dtype):
    return torch.empty_like(like, dtype=dtype, memory_format=torch.contiguous_format)


def _call(device, f, *args):
    """f on torch's current stream of `device`"""
    index = device.index
    if index == torch.cuda.current_device():
        f(*args, _stream_of(index))
    else:
        with torch.cuda.device(index):
            f(*args, _stream_of(index))


def _wants_gradient(*tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


# ---- dropout ----------------------------------------------------------------------------------------------------------
def _dropout(x, drop):
    m, at = _matrix(x, "x")
    y = _result(x, x.dtype)
    _call(x.device, capi.dropout, m.shape[0], m.shape[1], at, (y.data_ptr(), m.shape[1]), _drop(drop, x.device), _type(x.dtype, "x"))
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, drop, step_tensor):
        ctx.drop = drop
        ctx.save_for_backward(step_tensor)      # a step that changed before the gradient was drawn is an error
        return _dropout(x, drop)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        ctx.saved_tensors
        return _dropout(dy, ctx.drop), None, None


def dropout(x, drop):
    """x with the values that `drop` (a Drop) names replaced by zero and the others multiplied by 1 / (1 - p); its own
    gradient: dropout(dy, drop)."""
    if _wants_gradient(x):
        return _Dropout.apply(x, drop, drop.step_tensor if drop else None)
    return _dropout(x, drop)


# ---- layer normalisation ------------------------------------------------------------------------------------------------
def _statistics(rows, like):
    return like.new_empty(rows, dtype=torch.float32), like.new_empty(rows, dtype=torch.float32)


def _norm(x, weight, bias, eps, drop, dtype, stats):
    dtype = dtype or x.dtype
    m, at = _matrix(x, "x")
    rows, width = m.shape
    weight, bias, affine = _affine(weight, bias, width, dtype, x.device)
    y = _result(x, dtype)
    mean, rstd = _statistics(rows, x) if stats else (None, None)
    _call(x.device, capi.layer_norm, rows, width, at, (y.data_ptr(), width), _pointer(weight), _pointer(bias), _pointer(mean),
          _pointer(rstd), _drop(drop, x.device), eps, (_type(x.dtype, "x"), _type(dtype, "the result"), affine))
    return y, mean, rstd


def layer_norm_backward(dy, x, mean, rstd, weight=None, bias=None, *, drop=None):
    """(dx, dweight, dbias) of layer_norm, given the gradient of its result and what it was called with and returned.  dx has
    the type of x, dweight that of weight, dbias that of bias (None where there is none); what bias holds is not read."""
    return _norm_backward(dy, x, mean, rstd, weight, bias, drop, True, True)


def _columns(dy, rows, width, weight, bias, need_weight, need_bias):
    """dweight, dbias (or None) and the workspace their sums need"""
    dweight = torch.empty_like(weight) if weight is not None and need_weight else None
    dbias = torch.empty_like(bias) if bias is not None and need_bias else None
    need = capi.layer_norm_workspace(rows, width) if dweight is not None or dbias is not None else 0
    return dweight, dbias, dy.new_empty(need, dtype=torch.uint8) if need else None, need


def _statistic(t, rows, like, what):
    if t.numel() != rows or t.dtype != torch.float32 or t.device != like.device:
        raise RuntimeError("hetuctr_amd.nn: %s must hold a float32 for each of the %d rows on %s" % (what, rows, like.device))
    return t if t.is_contiguous() else t.contiguous()


def _norm_backward(dy, x, mean, rstd, weight, bias, drop, need_weight, need_bias):
    _same(dy, x, dy.dtype, "dy")
    m, at = _matrix(x, "x")
    g, g_at = _matrix(dy, "dy")
    rows, width = m.shape
    weight, bias, affine = _affine(weight, bias, width, dy.dtype, x.device)
    mean, rstd = _statistic(mean, rows, x, "mean"), _statistic(rstd, rows, x, "rstd")
    dx = _result(x, x.dtype)
    dweight, dbias, space, need = _columns(dy, rows, width, weight, bias, need_weight, need_bias)
    _call(x.device, capi.layer_norm_backward, rows, width, g_at, at, (dx.data_ptr(), width), _pointer(weight), _pointer(dweight),
          _pointer(dbias), mean.data_ptr(), rstd.data_ptr(), _pointer(space), need, _drop(drop, x.device),
          (_type(x.dtype, "x"), _type(dy.dtype, "dy"), affine))
    return dx, dweight, dbias


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, drop, dtype, step_tensor):
        y, mean, rstd = _norm(x, weight, bias, eps, drop, dtype, True)
        ctx.drop = drop
        ctx.save_for_backward(x, weight, bias, mean, rstd, step_tensor)
        ctx.mark_non_differentiable(mean, rstd)
        return y, mean, rstd

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, _mean, _rstd):
        x, weight, bias, mean, rstd, _ = ctx.saved_tensors
        dx, dweight, dbias = _norm_backward(dy, x, mean, rstd, weight, bias, ctx.drop, *ctx.needs_input_grad[1:3])
        return dx, dweight, dbias, None, None, None, None


def layer_norm(x, weight=None, bias=None, eps=1e-5, *, drop=None, dtype=None, stats=False):
    """(x - mean) / sqrt(variance + eps) * weight + bias over the last dimension, values dropped as `drop` says.  The result has
    type `dtype`: that of x, or, where x is float32, any.  weight and bias are float32 or of the result's type.  With `stats`
    returns (result, mean, 1 / sqrt(variance + eps)), float32, one of each a row."""
    if _wants_gradient(x, weight, bias):
        y, mean, rstd = _LayerNorm.apply(x, weight, bias, eps, drop, dtype, drop.step_tensor if drop else None)
    else:
        y, mean, rstd = _norm(x, weight, bias, eps, drop, dtype, stats)
    return (y, mean, rstd) if stats else y


# ---- residual + dropout, normalised -----------------------------------------------------------------------------------
def _add_norm(x, residual, weight, bias, eps, drop, stats):
    _same(residual, x, residual.dtype, "residual")
    m, at = _matrix(x, "x")
    r, r_at = _matrix(residual, "residual")
    rows, width = m.shape
    weight, bias, affine = _affine(weight, bias, width, x.dtype, x.device)
    y = _result(x, x.dtype)
    s = _result(x, residual.dtype)
    mean, rstd = _statistics(rows, x) if stats else (None, None)
    _call(x.device, capi.dropout_add_layer_norm, rows, width, at, r_at, (s.data_ptr(), width), (y.data_ptr(), width),
          _pointer(weight), _pointer(bias), _pointer(mean), _pointer(rstd), _drop(drop, x.device), eps,
          (_type(residual.dtype, "residual"), _type(x.dtype, "x"), affine))
    return y, s, mean, rstd


def dropout_add_layer_norm_backward(dy, ds, s, mean, rstd, weight=None, bias=None, *, drop=None):
    """(dx, dresidual, dweight, dbias) of dropout_add_layer_norm, given the gradients of its two results (ds may be None), the sum
    s and the rows' statistics that it returned.  dx has the type of dy, dresidual that of s; without dropout and where these
    are one type, they are one tensor."""
    return _add_norm_backward(dy, ds, s, mean, rstd, weight, bias, drop, True, True, True)


def _add_norm_backward(dy, ds, s, mean, rstd, weight, bias, drop, need_x, need_weight, need_bias):
    _same(dy, s, dy.dtype, "dy")
    m, at = _matrix(s, "s")
    g, g_at = _matrix(dy, "dy")
    d, d_at = None, capi.NO_MATRIX
    if ds is not None:
        _same(ds, s, s.dtype, "ds")
        d, d_at = _matrix(ds, "ds")
    rows, width = m.shape
    weight, bias, affine = _affine(weight, bias, width, dy.dtype, s.device)
    mean, rstd = _statistic(mean, rows, s, "mean"), _statistic(rstd, rows, s, "rstd")
    dresidual = _result(s, s.dtype)
    one = dy.dtype == s.dtype and (drop is None or drop.p == 0)
    dx = _result(s, dy.dtype) if need_x and not one else None
    dweight, dbias, space, need = _columns(dy, rows, width, weight, bias, need_weight, need_bias)
    _call(s.device, capi.dropout_add_layer_norm_backward, rows, width, g_at, at, d_at,
          capi.NO_MATRIX if dx is None else (dx.data_ptr(), width), (dresidual.data_ptr(), width), _pointer(weight),
          _pointer(dweight), _pointer(dbias), mean.data_ptr(), rstd.data_ptr(), _pointer(space), need, _drop(drop, s.device),
          (_type(s.dtype, "s"), _type(dy.dtype, "dy"), affine))
    return dresidual if one else dx, dresidual, dweight, dbias


class _DropoutAddLayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps, drop, step_tensor):
        y, s, mean, rstd = _add_norm(x, residual, weight, bias, eps, drop, True)
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
            dx = _dropout(ds, ctx.drop) if ctx.drop else ds
            return dx.to(ctx.act), ds, None, None, None, None, None
        dx, dresidual, dweight, dbias = _add_norm_backward(dy, ds, s, mean, rstd, weight, bias, ctx.drop, ctx.needs_input_grad[0],
                                                           *ctx.needs_input_grad[2:4])
        return dx, dresidual, dweight, dbias, None, None, None


def dropout_add_layer_norm(x, residual, weight=None, bias=None, eps=1e-5, *, drop=None, stats=False):
    """(y, s) with s = residual + dropout(x) and y = layer_norm(s): the step between two layers.  x and y are of one type, residual
    and s of that type or float32; weight and bias are float32 or of the type of x.  y is computed from s before it is
    rounded.  With `stats` returns (y, s, mean, 1 / sqrt(variance + eps)), as layer_norm does."""
    if _wants_gradient(x, residual, weight, bias):
        y, s, mean, rstd = _DropoutAddLayerNorm.apply(x, residual, weight, bias, eps, drop, drop.step_tensor if drop else None)
    else:
        y, s, mean, rstd = _add_norm(x, residual, weight, bias, eps, drop, stats)
    return (y, s, mean, rstd) if stats else (y, s)
