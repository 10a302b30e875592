"""Operators on CUDA tensors for networks that condition the point networks: embedding lookup, dropout and group norm
with an activation (channels last), each with its gradient.

Every function takes the :class:`cpde_b200.native.Engine` of the tensors' device, launches on torch's current stream of
that device and returns new contiguous tensors; nothing synchronises. The classes at the end are the same operators for
torch's autograd. Wrong arguments raise ``ValueError`` here or :class:`cpde_b200.native.EngineError` in the library. As
with any kernel launch, a tensor that another stream made has to be ordered before the current stream by the caller.

Equal inputs give equal bits: no result depends on the order in which blocks run.
"""
import ctypes
from functools import lru_cache

import torch

from .native import OK, load

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
ID_TYPES = {torch.int32: 0, torch.int64: 1}
ACTIVATIONS = {'sigmoid': 0, 'linear': 1, 'tanh': 2, 'silu': 3}

# The default stream's own handle: a null handle selects the engine's stream.
LEGACY_STREAM = 1
WORD = (1 << 64) - 1


def _stream(device):
    return torch._C._cuda_getCurrentRawStream(device) or LEGACY_STREAM


def _on(engine, *tensors):
    for t in tensors:
        if t is not None and (not t.is_cuda or t.device.index != engine.device):
            raise ValueError(f'every tensor must be on cuda:{engine.device}, the engine\'s device')


def _type(t, name):
    try:
        return TYPES[t.dtype]
    except KeyError:
        raise ValueError(f'{name} must be float32, bfloat16 or float16') from None


def _id_type(ids):
    try:
        return ID_TYPES[ids.dtype]
    except KeyError:
        raise ValueError('ids must be int32 or int64') from None


def _pointer(t):
    return None if t is None else t.data_ptr()


def _rows(t):
    """``t`` as a matrix with adjacent channels, and the stride of its rows; other layouts (transposed, broadcast) are
    copied first."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    if (t.shape[1] > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        t = t.contiguous()
    return t, t.stride(0) if t.shape[0] > 1 else t.shape[1]


@lru_cache(maxsize=256)
def _workspace_bytes(entry, *sizes):
    size = ctypes.c_size_t()
    if getattr(load(), entry)(*sizes, ctypes.byref(size)) != OK:
        raise ValueError(f'{entry.removesuffix("_workspace")}: invalid sizes {sizes}')
    return size.value


def embedding(engine, table, ids, scale=1.0, dtype=None):
    """``scale * table[ids]``; rows of ids outside the table are zeros. ``dtype`` (default: the table's) may be a 16-bit
    type for a float32 table."""
    if table.dim() != 2:
        raise ValueError('table must have shape (rows, channels)')
    _on(engine, table, ids)
    kind, id_kind = _type(table, 'table'), _id_type(ids)
    out = torch.empty((*ids.shape, table.shape[1]), dtype=dtype or table.dtype, device=table.device)
    ids = ids.contiguous()
    table, stride = _rows(table)
    engine._check(engine.lib.cpde_embedding(
        engine.handle, kind, table.data_ptr(), stride, table.shape[0], table.shape[1], id_kind, ids.data_ptr(),
        ids.numel(), scale, _type(out, 'dtype'), out.data_ptr(), _stream(engine.device)))
    return out


def embedding_gradient(engine, grad, ids, rows, scale=1.0, dtype=None):
    """Gradient of :func:`embedding`'s table of ``rows`` rows from the gradient of its output. ``dtype`` (default: the
    gradient's) may be float32 for a 16-bit gradient."""
    if grad.shape[:-1] != ids.shape:
        raise ValueError('grad must have the shape of ids and the channels')
    _on(engine, grad, ids)
    kind, id_kind = _type(grad, 'grad'), _id_type(ids)
    channels = grad.shape[-1]
    grad, stride = _rows(grad)
    ids = ids.contiguous()
    out = torch.empty((rows, channels), dtype=dtype or grad.dtype, device=grad.device)
    size = _workspace_bytes('cpde_embedding_gradient_workspace', ids.numel(), rows, channels)
    workspace = torch.empty(size, dtype=torch.uint8, device=grad.device)
    engine._check(engine.lib.cpde_embedding_gradient(
        engine.handle, kind, grad.data_ptr(), stride, id_kind, ids.data_ptr(), ids.numel(), rows, channels, scale,
        _type(out, 'dtype'), out.data_ptr(), workspace.data_ptr(), size, _stream(engine.device)))
    return out


def dropout(engine, x, rate, seed, offset=0, residual=None):
    """``residual + drop(x)``, with the mask of (``seed``, ``offset``, element index): a step that needs a new mask
    passes another offset. The rate counts in units of 1/65536."""
    _on(engine, x, residual)
    kind = _type(x, 'x')
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError('residual must have x\'s shape and type')
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if x.is_contiguous() and (residual is None or residual.is_contiguous()):
        rows, columns, stride, residual_stride = 1, x.numel(), x.numel(), x.numel()
    elif x.dim() == 0:
        rows = columns = stride = residual_stride = 1
    else:
        x, stride = _rows(x)
        rows, columns = x.shape
        residual, residual_stride = (None, columns) if residual is None else _rows(residual)
    engine._check(engine.lib.cpde_dropout(
        engine.handle, kind, x.data_ptr(), stride, _pointer(residual), residual_stride, rows, columns, rate,
        seed & WORD, offset & WORD, y.data_ptr(), _stream(engine.device)))
    return y


def dropout_gradient(engine, grad, rate, seed, offset=0):
    """Gradient of :func:`dropout`'s x; the residual's is ``grad`` itself."""
    return dropout(engine, grad, rate, seed, offset)


def _points(t, name):
    """``t`` with adjacent channels, and its point and instance strides; other layouts are copied first."""
    if t.dim() != 3:
        raise ValueError(f'{name} must have shape (instances, points, channels)')
    if (t.shape[2] > 1 and t.stride(2) != 1) or (t.shape[1] > 1 and t.stride(1) < t.shape[2]):
        t = t.contiguous()
    return t, max(t.stride(1), t.shape[2]), t.stride(0)


def _norm_arguments(engine, x, weight, bias, activation, lengths):
    kind = _type(x, 'x')
    if activation not in ACTIVATIONS:
        raise ValueError(f'activation must be one of {", ".join(ACTIVATIONS)}')
    parameter = torch.float32
    for p, name in ((weight, 'weight'), (bias, 'bias')):
        if p is not None:
            if p.shape != x.shape[2:] or not p.is_contiguous():
                raise ValueError(f'{name} must be a contiguous tensor with a value per channel')
            parameter = p.dtype
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError('weight and bias must have one type')
    if parameter != torch.float32 and parameter != x.dtype:
        raise ValueError('weight and bias must be float32 or of x\'s type')
    if lengths is not None and (lengths.dtype != torch.int32 or lengths.shape != x.shape[:1]
                                or not lengths.is_contiguous()):
        raise ValueError('lengths must be a contiguous int32 tensor with a value per instance')
    return kind, TYPES[parameter], ACTIVATIONS[activation]


def group_norm(engine, x, groups, weight=None, bias=None, eps=1e-5, activation='linear', lengths=None, rate=0.0,
               seed=0, offset=0):
    """``(y, mean, rstd)`` of group norm with an activation and dropout over x of shape (instances, points, channels).

    Statistics are over the points of an instance and the channels of a group; ``lengths`` limits each instance to its
    first points (y is zero behind them). ``rate``, ``seed`` and ``offset`` are those of :func:`dropout`, applied behind
    the activation. mean and rstd are float32 of shape (instances, groups)."""
    _on(engine, x, weight, bias, lengths)
    x, point, instance = _points(x, 'x')
    kind, parameter, code = _norm_arguments(engine, x, weight, bias, activation, lengths)
    n, p, c = x.shape
    size = _workspace_bytes('cpde_group_norm_workspace', n, p, c, groups)
    y = torch.empty((n, p, c), dtype=x.dtype, device=x.device)
    mean, rstd = torch.empty((2, n, groups), dtype=torch.float32, device=x.device).unbind()
    workspace = torch.empty(size, dtype=torch.uint8, device=x.device)
    engine._check(engine.lib.cpde_group_norm(
        engine.handle, kind, x.data_ptr(), point, instance, n, p, c, groups, parameter, _pointer(weight),
        _pointer(bias), eps, code, _pointer(lengths), rate, seed & WORD, offset & WORD, y.data_ptr(), mean.data_ptr(),
        rstd.data_ptr(), workspace.data_ptr(), size, _stream(engine.device)))
    return y, mean, rstd


def group_norm_gradient(engine, grad, x, mean, rstd, groups, weight=None, bias=None, activation='linear', lengths=None,
                        rate=0.0, seed=0, offset=0):
    """``(dx, dweight, dbias)`` of :func:`group_norm` from the gradient of y, its inputs, mean and rstd; dweight and
    dbias are None for parameters that are None."""
    _on(engine, grad, x, mean, rstd, weight, bias, lengths)
    if grad.shape != x.shape or grad.dtype != x.dtype:
        raise ValueError('grad must have x\'s shape and type')
    x, point, instance = _points(x, 'x')
    grad, grad_point, grad_instance = _points(grad, 'grad')
    kind, parameter, code = _norm_arguments(engine, x, weight, bias, activation, lengths)
    n, p, c = x.shape
    for t, name in ((mean, 'mean'), (rstd, 'rstd')):
        if t.dtype != torch.float32 or t.shape != (n, groups) or not t.is_contiguous():
            raise ValueError(f'{name} must be a contiguous float32 tensor of shape (instances, groups)')
    size = _workspace_bytes('cpde_group_norm_workspace', n, p, c, groups)
    dx = torch.empty((n, p, c), dtype=x.dtype, device=x.device)
    dweight, dbias = (None if v is None else torch.empty_like(v) for v in (weight, bias))
    workspace = torch.empty(size, dtype=torch.uint8, device=x.device)
    engine._check(engine.lib.cpde_group_norm_gradient(
        engine.handle, kind, grad.data_ptr(), grad_point, grad_instance, x.data_ptr(), point, instance,
        mean.data_ptr(), rstd.data_ptr(), n, p, c, groups, parameter, _pointer(weight), _pointer(bias), code,
        _pointer(lengths), rate, seed & WORD, offset & WORD, dx.data_ptr(), _pointer(dweight), _pointer(dbias),
        workspace.data_ptr(), size, _stream(engine.device)))
    return dx, dweight, dbias


# --- autograd --------------------------------------------------------------

class Embedding(torch.autograd.Function):
    """``Embedding.apply(engine, table, ids, scale)``: :func:`embedding` with its gradient for the table."""

    @staticmethod
    def forward(ctx, engine, table, ids, scale=1.0):
        ctx.save_for_backward(ids)
        ctx.engine, ctx.rows, ctx.scale = engine, table.shape[0], scale
        return embedding(engine, table, ids, scale)

    @staticmethod
    def backward(ctx, grad):
        ids, = ctx.saved_tensors
        return None, embedding_gradient(ctx.engine, grad, ids, ctx.rows, ctx.scale), None, None


class Dropout(torch.autograd.Function):
    """``Dropout.apply(engine, x, rate, seed, offset, residual)``: :func:`dropout` with its gradients."""

    @staticmethod
    def forward(ctx, engine, x, rate, seed, offset=0, residual=None):
        ctx.engine, ctx.rule, ctx.residual = engine, (rate, seed, offset), residual is not None
        return dropout(engine, x, rate, seed, offset, residual)

    @staticmethod
    def backward(ctx, grad):
        return (None, dropout_gradient(ctx.engine, grad, *ctx.rule), None, None, None,
                grad if ctx.residual else None)


class GroupNorm(torch.autograd.Function):
    """``GroupNorm.apply(engine, x, weight, bias, groups, eps, activation, lengths, rate, seed, offset)``:
    :func:`group_norm`'s y with its gradients."""

    @staticmethod
    def forward(ctx, engine, x, weight, bias, groups, eps=1e-5, activation='linear', lengths=None, rate=0.0, seed=0,
                offset=0):
        y, mean, rstd = group_norm(engine, x, groups, weight, bias, eps, activation, lengths, rate, seed, offset)
        ctx.save_for_backward(x, weight, bias, lengths, mean, rstd)
        ctx.engine, ctx.options = engine, (groups, activation, rate, seed, offset)
        return y

    @staticmethod
    def backward(ctx, grad):
        x, weight, bias, lengths, mean, rstd = ctx.saved_tensors
        groups, activation, rate, seed, offset = ctx.options
        dx, dweight, dbias = group_norm_gradient(ctx.engine, grad, x, mean, rstd, groups, weight, bias, activation,
                                                 lengths, rate, seed, offset)
        return None, dx, dweight, dbias, *(None,) * 7
