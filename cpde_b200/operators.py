"""Operators on CUDA tensors for torch networks beside the engine's, such as one that learns a family of its solutions:
embedding lookup, dropout, group norm with an activation (channels last) and linear layers, each with its gradient;
orthogonalised matrices and the optimiser step that takes them.

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
import numbers

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
                 'cpde_group_norm_gradient', 'cpde_linear_workspace', 'cpde_linear', 'cpde_linear_gradient_workspace',
                 'cpde_linear_gradient', 'cpde_orthogonalize_workspace', 'cpde_orthogonalize', 'cpde_muon_workspace',
                 'cpde_muon')})


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


def check(engine):
    """Raises :class:`cpde_b200.native.EngineError` if a kernel of an earlier call gave up waiting, so that its results are
    invalid. Every other function does so too, before it launches anything; nothing waits, so that a program which wants to
    know about its last calls synchronises first."""
    if engine.handle is None:
        raise native.EngineError(native.REJECTED, 'the engine is closed')
    engine._check(engine.lib.cpde_operator_check(engine.handle))


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


def linear(engine, x, weight, bias=None, activation='linear', residual=None, keep=False):
    """``(y, z)`` of ``y = residual + act(x @ weight.T + bias)`` over x of shape (..., inputs) and weight of shape
    (outputs, inputs). z, the sums before the activation that :func:`linear_gradient` takes, is None unless ``keep``.

    The products of 16-bit types are summed in FP32, to 1.2e-5 of the terms' absolute values; those of float32 have the
    error of FP32 products. A row of float32 x with an infinity gives infinities or NaNs."""
    return _operators.linear(_handle(engine, x), engine.device, x, weight, bias, _activation(activation), residual, keep)


def linear_gradient(engine, grad, x, weight, bias=None, activation='linear', z=None, need=(True, True), dtype=None):
    """``(dx, dweight, dbias)`` of :func:`linear` from the gradient of y, its inputs and z (not needed for a linear
    activation); the residual's gradient is ``grad`` itself. ``need`` says which of dx and dweight are computed, the others
    are None, and so is dbias without a bias. ``dtype`` of dweight and dbias (default: the parameters') may be float32 for
    a 16-bit weight.

    16-bit layers hold grad times the activation's slope in their type where they are large. With ``dtype=torch.float32``
    dweight sums what that rounding leaves too, in twice the time."""
    need_x, need_weight = need
    return _operators.linear_gradient(_handle(engine, x), engine.device, grad, x, weight, bias, _activation(activation), z,
                                      need_x, need_weight, dtype)


QUINTIC = (3.4445, -4.775, 2.0315)


def _coefficients(coefficients):
    """A triple, or a sequence of triples, as one tuple."""
    message = 'coefficients must be triples of numbers, one at least'
    try:
        items = list(coefficients)
        if items and not isinstance(items[0], numbers.Real):
            items = [v for a, b, c in items for v in (a, b, c)]
        flat = tuple(float(v) for v in items)
    except (TypeError, ValueError):
        raise ValueError(message) from None
    if not flat or len(flat) % 3:
        raise ValueError(message)
    return flat


def orthogonalize(engine, x, steps=5, coefficients=QUINTIC, eps=1e-7):
    """Each matrix of x, of shape (rows, columns) or (matrices, rows, columns), with its singular values taken near one:
    ``X = x / (|x| + eps)`` with the Frobenius norm, then ``steps`` times ``X = a X + b (X X') X + c (X X')^2 X``.
    ``coefficients`` is a triple (a, b, c), or one for each step (the last counts for the steps behind it).

    Values are held in 22 bits. Products take all of them for float32, whose result is good to about 2e-6 of its norm, for
    float16 and where a side is up to 256, and 11 for larger bfloat16 matrices, which leaves less than rounding to bfloat16
    adds."""
    return _operators.orthogonalize(_handle(engine, x), engine.device, x, steps, _coefficients(coefficients), eps)


def muon(engine, weight, grad, momentum, rate, beta=0.95, nesterov=True, decay=0.0, scale=None, steps=5,
         coefficients=QUINTIC, eps=1e-7, inplace=False):
    """``(weight, momentum)`` after an optimiser step of a weight matrix whose update is orthogonalised (Muon):
    ``m = beta momentum + (1 - beta) grad``, ``u = beta m + (1 - beta) grad`` (m itself without ``nesterov``) and
    ``(1 - rate decay) weight - rate scale O``, O being u as :func:`orthogonalize` gives it and the scale by default
    ``max(1, rows / columns) ** 0.5``. momentum is float32 or of the weight's type. With ``inplace`` the given tensors
    are written and returned."""
    if weight.dim() != 2 or not weight.numel():
        raise ValueError('weight must have shape (rows, columns), both positive')
    if scale is None:
        scale = max(1.0, weight.shape[0] / weight.shape[-1]) ** 0.5
    return _operators.muon(_handle(engine, weight), engine.device, weight, grad, momentum, rate, beta, nesterov, decay, scale,
                           steps, _coefficients(coefficients), eps, inplace)


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


class Linear(torch.autograd.Function):
    """``Linear.apply(engine, x, weight, bias, activation, residual)``: :func:`linear`'s y with its gradients."""

    @staticmethod
    def forward(ctx, engine, x, weight, bias=None, activation='linear', residual=None):
        keep = activation != 'linear' and any(ctx.needs_input_grad[1:4])
        y, z = linear(engine, x, weight, bias, activation, residual, keep)
        ctx.save_for_backward(x, weight, bias, z)
        ctx.engine, ctx.activation = engine, activation
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, weight, bias, z = ctx.saved_tensors
        # A flag for each argument that was passed: bias, activation and residual may be left out.
        _, need_x, need_weight, need_bias, _, need_residual = (*ctx.needs_input_grad, False, False, False)[:6]
        dx = dweight = dbias = None
        if need_x or need_weight or need_bias:
            dx, dweight, dbias = linear_gradient(ctx.engine, grad, x, weight, bias if need_bias else None, ctx.activation, z,
                                                 (need_x, need_weight))
        return None, dx, dweight, dbias, None, grad if need_residual else None


# --- optimiser -------------------------------------------------------------

class Muon(torch.optim.Optimizer):
    """Steps of :func:`muon`, in place, for the weight matrices of hidden layers; other parameters (biases, embeddings,
    heads) are for another optimiser. Momentum is float32 whatever the weights' type: a part 1 - beta of a gradient would be
    lost beside a 16-bit one. A state that was saved in another type is taken over in float32."""

    def __init__(self, engine, params, lr=0.02, beta=0.95, nesterov=True, weight_decay=0.0, steps=5, coefficients=QUINTIC,
                 eps=1e-7):
        self.engine = engine
        super().__init__(params, dict(lr=lr, beta=beta, nesterov=nesterov, weight_decay=weight_decay, steps=steps,
                                      coefficients=coefficients, eps=eps))

    def add_param_group(self, group):
        super().add_param_group(group)
        if any(p.dim() != 2 for p in self.param_groups[-1]['params']):
            self.param_groups.pop()
            raise ValueError('Muon takes matrices alone')

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)  # which gives the state the parameters' type
        ours = (p for group in self.param_groups for p in group['params'])
        for key, p in zip((key for group in state_dict['param_groups'] for key in group['params']), ours):
            if 'momentum' in state_dict['state'].get(key, {}):
                self.state[p]['momentum'] = state_dict['state'][key]['momentum'].to(p.device, torch.float32, copy=True).contiguous()

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            for p in group['params']:
                if p.grad is None:
                    continue
                state = self.state[p]
                if 'momentum' not in state:
                    state['momentum'] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.contiguous_format)
                muon(self.engine, p, p.grad, state['momentum'], group['lr'], group['beta'], group['nesterov'],
                     group['weight_decay'], None, group['steps'], group['coefficients'], group['eps'], inplace=True)
        return loss
