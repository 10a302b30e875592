"""Operators on CUDA tensors for torch networks beside the engine's, such as one that learns a family of its solutions:
embedding lookup, dropout and group norm with an activation (channels last), each with its gradient.

Every function takes the :class:`cpde_b200.native.Engine` of the tensors' device, launches on torch's current stream of
that device and returns new contiguous tensors; nothing synchronises. Wrong arguments raise ``ValueError`` here or
:class:`cpde_b200.native.EngineError` in the library. As with any kernel launch, a tensor that another stream made has to be
ordered before the current stream by the caller.

The functions compute values only, and refuse a tensor that requires gradients while torch records them. The classes at the
end are the same operators for torch's autograd, with first derivatives in reverse mode; forward mode, vmap, tracing and
higher derivatives are not supported.

Equal calls on equally laid out inputs give equal bits: no result depends on the order in which blocks run.
"""
import ctypes

import torch
from torch.autograd.function import once_differentiable

from . import native

try:
    from . import _operators
except ImportError as error:
    raise RuntimeError('the operators\' binding is not built; run python -m cpde_b200.build') from error

ACTIVATIONS = {'sigmoid': 0, 'linear': 1, 'tanh': 2, 'silu': 3}

_operators.bind(native.EngineError, {
    name: ctypes.cast(getattr(native.load(), name), ctypes.c_void_p).value
    for name in ('cpde_last_error', 'cpde_embedding', 'cpde_embedding_gradient_workspace', 'cpde_embedding_gradient',
                 'cpde_dropout', 'cpde_group_norm_forward_workspace', 'cpde_group_norm_workspace', 'cpde_group_norm',
                 'cpde_group_norm_gradient')})


def _handle(engine, tensor):
    if tensor.get_device() != engine.device:
        raise ValueError(f'every tensor must be on cuda:{engine.device}, the engine\'s device')
    if engine.handle is None:
        raise native.EngineError(native.REJECTED, 'the engine is closed')
    return engine.handle.value


def _activation(name):
    try:
        return ACTIVATIONS[name]
    except KeyError:
        raise ValueError(f'activation must be one of {", ".join(ACTIVATIONS)}') from None


def embedding(engine, table, ids, scale=1.0, dtype=None):
    """``scale * table[ids]``; rows of ids outside the table are zeros. ``dtype`` (default: the table's) may be a 16-bit
    type for a float32 table."""
    return _operators.embedding(_handle(engine, table), engine.device, table, ids, scale, dtype)


def embedding_gradient(engine, grad, ids, rows, scale=1.0, dtype=None):
    """Gradient of :func:`embedding`'s table of ``rows`` rows from the gradient of its output. ``dtype`` (default: the
    gradient's) may be float32 for a 16-bit gradient."""
    return _operators.embedding_gradient(_handle(engine, grad), engine.device, grad, ids, rows, scale, dtype)


def dropout(engine, x, rate, seed, offset=0, residual=None):
    """``residual + drop(x)``, with the mask of (``seed``, ``offset``, element index): a step that needs a new mask
    passes another offset. The rate counts in units of 1/65536."""
    return _operators.dropout(_handle(engine, x), engine.device, x, residual, rate, seed, offset)


def dropout_gradient(engine, grad, rate, seed, offset=0):
    """Gradient of :func:`dropout`'s x; the residual's is ``grad`` itself."""
    return dropout(engine, grad, rate, seed, offset)


def group_norm(engine, x, groups, weight=None, bias=None, eps=1e-5, activation='linear', lengths=None, rate=0.0,
               seed=0, offset=0):
    """``(y, mean, rstd)`` of group norm with an activation and dropout over x of shape (instances, points, channels).

    Statistics are over the points of an instance and the channels of a group; ``lengths`` limits each instance to its
    first points (y is zero behind them). ``rate``, ``seed`` and ``offset`` are those of :func:`dropout`, applied behind
    the activation. mean and rstd are float32 of shape (instances, groups)."""
    return _operators.group_norm(_handle(engine, x), engine.device, x, groups, eps, weight, bias, _activation(activation),
                                 lengths, rate, seed, offset)


def group_norm_gradient(engine, grad, x, mean, rstd, groups, weight=None, bias=None, activation='linear', lengths=None,
                        rate=0.0, seed=0, offset=0):
    """``(dx, dweight, dbias)`` of :func:`group_norm` from the gradient of y, its inputs, mean and rstd; dweight and
    dbias are None for parameters that are None."""
    return _operators.group_norm_gradient(_handle(engine, x), engine.device, grad, x, mean, rstd, groups, weight, bias,
                                          _activation(activation), lengths, rate, seed, offset)


# --- autograd --------------------------------------------------------------

class Embedding(torch.autograd.Function):
    """``Embedding.apply(engine, table, ids, scale)``: :func:`embedding` with its gradient for the table."""

    @staticmethod
    def forward(ctx, engine, table, ids, scale=1.0):
        ctx.save_for_backward(ids)
        ctx.engine, ctx.rows, ctx.scale = engine, table.shape[0], scale
        return embedding(engine, table, ids, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        ids, = ctx.saved_tensors
        if not ctx.needs_input_grad[1]:
            return (None,) * 4
        return None, embedding_gradient(ctx.engine, grad, ids, ctx.rows, ctx.scale), None, None


class Dropout(torch.autograd.Function):
    """``Dropout.apply(engine, x, rate, seed, offset, residual)``: :func:`dropout` with its gradients."""

    @staticmethod
    def forward(ctx, engine, x, rate, seed, offset=0, residual=None):
        ctx.engine, ctx.rule, ctx.residual = engine, (rate, seed, offset), residual is not None
        return dropout(engine, x, rate, seed, offset, residual)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        return (None, dropout_gradient(ctx.engine, grad, *ctx.rule) if ctx.needs_input_grad[1] else None, None, None, None,
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
    @once_differentiable
    def backward(ctx, grad):
        x, weight, bias, lengths, mean, rstd = ctx.saved_tensors
        groups, activation, rate, seed, offset = ctx.options
        dx, dweight, dbias = group_norm_gradient(ctx.engine, grad, x, mean, rstd, groups, weight, bias, activation,
                                                 lengths, rate, seed, offset)
        return None, dx, dweight, dbias, *(None,) * 7
