"""Workloads of the layer operators: linear layers with bias, activation and residual, their gradients, orthogonalised
matrices and the optimiser step that takes them.

Each case is one call that a training or evaluation step makes. ``run`` computes it either with the framework's operators
(``own``) or in a plain form: elementary torch operations in 32 bits, rounded once at the end. ``exact`` gives the same outputs
in 64 bits, from the definitions.
"""
import math

import torch

own = False

TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
BYTES = {'f32': 4, 'bf16': 2, 'f16': 2}

STEPS, COEFFICIENTS, TINY = 5, (3.4445, -4.775, 2.0315), 1e-7

_handle = None


def _engine():
    """The engine that a program creates once and keeps."""
    global _handle
    if _handle is None:
        from cpde_b200 import native
        _handle = native.Engine(0)
    return _handle


# --- cases ---------------------------------------------------------------

def listed():
    return [
        # First hidden layer of a small network at a few points: latency counts.
        dict(name='linear_points_small_f32', op='linear', points=257, inputs=48, outputs=128, type='f32', activation='tanh',
             bias=True, residual=False, keep=False, gap=0),
        # One query of a wide trunk: the weights are read once for a single row.
        dict(name='linear_row_bf16', op='linear', points=1, inputs=4096, outputs=4096, type='bf16', activation='silu',
             bias=True, residual=True, keep=False, gap=0),
        # A hidden layer of 128 neurons at 65,536 points, in FP32.
        dict(name='linear_points_f32', op='linear', points=65536, inputs=128, outputs=128, type='f32', activation='tanh',
             bias=True, residual=False, keep=False, gap=0),
        # A residual block of a trunk in training: the sum before the activation is kept for the gradient.
        dict(name='linear_trunk_bf16', op='linear', points=32768, inputs=2048, outputs=2048, type='bf16', activation='silu',
             bias=True, residual=True, keep=True, gap=0),
        # Odd sizes throughout, rows with a stride.
        dict(name='linear_ragged_f16', op='linear', points=4097, inputs=1001, outputs=515, type='f16', activation='sigmoid',
             bias=True, residual=False, keep=True, gap=3),
        # The gradients: a small odd layer, the 128 neurons at 65,536 points, the trunk's block.
        dict(name='linear_grad_small_f16', op='linear_gradient', points=300, inputs=100, outputs=77, type='f16',
             activation='silu', bias=True, gap=0),
        dict(name='linear_grad_points_f32', op='linear_gradient', points=65536, inputs=128, outputs=128, type='f32',
             activation='tanh', bias=True, gap=0),
        dict(name='linear_grad_trunk_bf16', op='linear_gradient', points=32768, inputs=2048, outputs=2048, type='bf16',
             activation='silu', bias=True, gap=0),
        # The updates of four hidden layers of 128 neurons at once.
        dict(name='orthogonalize_layers_f32', op='orthogonalize', matrices=4, rows=128, columns=128, type='f32'),
        # The update of a trunk's widest layer.
        dict(name='orthogonalize_wide_bf16', op='orthogonalize', matrices=1, rows=2048, columns=8192, type='bf16'),
        # Optimiser steps of a first layer and of a trunk's layer, weights in FP32.
        dict(name='muon_small_f32', op='muon', rows=128, columns=20, type='f32', nesterov=True, decay=0.01),
        dict(name='muon_trunk_f32', op='muon', rows=2048, columns=2048, type='f32', nesterov=True, decay=0.01),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _size(rng, high):
    """A width as layers have it: a multiple of 64 or 8 more often than not."""
    n = _log_int(rng, 1, high)
    unit = rng.choice([1, 8, 64])
    return min(high, (n + unit - 1) // unit * unit)


def draw(rng):
    op = rng.choice(['linear', 'linear', 'linear_gradient', 'linear_gradient', 'orthogonalize', 'muon'])
    kind = rng.choice(['f32', 'bf16', 'f16'])
    case = dict(op=op, type=kind)
    if op.startswith('linear'):
        inputs, outputs = _size(rng, 8192), _size(rng, 8192)
        points = _log_int(rng, 1, min(1 << 17, max(2, int(6.8e10 / (inputs * outputs)))))
        case.update(points=points, inputs=inputs, outputs=outputs, bias=rng.random() < 0.7,
                    activation=rng.choice(['linear', 'sigmoid', 'tanh', 'silu']), gap=rng.choice([0, 0, 0, 3, 8]))
        if op == 'linear':
            case.update(residual=rng.random() < 0.4, keep=rng.random() < 0.4)
    else:
        rows = _size(rng, 4096)
        columns = _size(rng, 4096 if rows > 1024 else 8192)
        if op == 'orthogonalize':
            most = int(2e11 / _newton_schulz_flops(rows, columns))
            case.update(matrices=_log_int(rng, 1, max(1, min(16, most))))
        else:
            case.update(nesterov=rng.random() < 0.7, decay=rng.choice([0.0, 0.01]))
        while _newton_schulz_flops(rows, columns) > 4e11:
            rows, columns = (rows + 1) // 2, (columns + 1) // 2
        case.update(rows=rows, columns=columns)
    return case


# --- inputs --------------------------------------------------------------

class Inputs:
    pass


def prepare(case, seed):
    g = torch.Generator(device='cuda')
    g.manual_seed(int(seed))
    s = Inputs()
    s.case, s.op = case, case['op']
    kind = TYPES[case['type']]

    def normal(*shape):
        return torch.randn(shape, generator=g, device='cuda')

    def rows(p, c, gap):
        """Rows of c values, `gap` further ones between them."""
        return normal(p, c + gap).to(kind)[:, :c]

    def update(*shape):
        """A gradient of a layer: a few strong directions over a weak rest."""
        m, n = shape[-2:]
        r = min(32, m, n)
        strong = normal(*shape[:-1], r) / torch.arange(1, r + 1, device='cuda') @ normal(*shape[:-2], r, n)
        return (1e-3 * (strong + 0.05 * normal(*shape))).to(kind)

    if s.op.startswith('linear'):
        p, c, o = case['points'], case['inputs'], case['outputs']
        s.activation = case['activation']
        s.x = rows(p, c, case['gap'])
        s.weight = (normal(o, c) / math.sqrt(c)).to(kind)
        s.bias = (0.2 * normal(o)).to(kind) if case['bias'] else None
        if s.op == 'linear':
            s.residual = rows(p, o, case['gap']) if case['residual'] else None
        else:
            s.grad = rows(p, o, case['gap'])
            s.z = None
            if s.activation != 'linear':
                s.z = _before(s.x.float(), s.weight.float(), None if s.bias is None else s.bias.float()).to(kind)
    elif s.op == 'orthogonalize':
        s.x = update(case['matrices'], case['rows'], case['columns'])
    else:
        m, n = case['rows'], case['columns']
        s.weight = (normal(m, n) / math.sqrt(n)).to(kind)
        s.grad, s.momentum = update(m, n), update(m, n)
        s.rate, s.beta, s.scale = 0.02, 0.95, math.sqrt(max(1.0, m / n))
        s.nesterov, s.decay = case['nesterov'], case['decay']
    return s


# --- one pass ------------------------------------------------------------

def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    from cpde_b200 import operators
    e = _engine()
    if s.op == 'linear':
        y, z = operators.linear(e, s.x, s.weight, s.bias, activation=s.activation, residual=s.residual, keep=s.case['keep'])
        return {'y': y, 'z': z} if s.case['keep'] else {'y': y}
    if s.op == 'linear_gradient':
        dx, dweight, dbias = operators.linear_gradient(e, s.grad, s.x, s.weight, s.bias, activation=s.activation, z=s.z)
        return {'dx': dx, 'dweight': dweight} if s.bias is None else {'dx': dx, 'dweight': dweight, 'dbias': dbias}
    if s.op == 'orthogonalize':
        return operators.orthogonalize(e, s.x, steps=STEPS, coefficients=COEFFICIENTS, eps=TINY)
    weight, momentum = operators.muon(e, s.weight, s.grad, s.momentum, s.rate, beta=s.beta, nesterov=s.nesterov,
                                      decay=s.decay, scale=s.scale, steps=STEPS, coefficients=COEFFICIENTS, eps=TINY)
    return {'weight': weight, 'momentum': momentum}


def _before(x, weight, bias):
    z = x @ weight.t()
    return z if bias is None else z + bias


def _activated(z, name):
    if name == 'linear':
        return z
    if name == 'tanh':
        return torch.tanh(z)
    f = 1 / (1 + torch.exp(-z))
    return f if name == 'sigmoid' else z * f


def _slope(z, name):
    if name == 'tanh':
        t = torch.tanh(z)
        return 1 - t * t
    f = 1 / (1 + torch.exp(-z))
    return f * (1 - f) if name == 'sigmoid' else f * (1 + z * (1 - f))


def _newton_schulz(x):
    """The odd polynomial of x's singular values, STEPS times, on matrices divided by their Frobenius norms."""
    a, b, c = COEFFICIENTS
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + TINY)
    tall = x.shape[-2] > x.shape[-1]
    for _ in range(STEPS):
        gram = x.transpose(-2, -1) @ x if tall else x @ x.transpose(-2, -1)
        q = b * gram + c * (gram @ gram)
        x = a * x + (x @ q if tall else q @ x)
    return x


def _plain(s):
    if s.op == 'linear':
        kind = s.x.dtype
        z = _before(s.x.float(), s.weight.float(), None if s.bias is None else s.bias.float())
        y = _activated(z, s.activation)
        if s.residual is not None:
            y = y + s.residual.float()
        return {'y': y.to(kind), 'z': z.to(kind)} if s.case['keep'] else {'y': y.to(kind)}
    if s.op == 'linear_gradient':
        kind = s.x.dtype
        dz = s.grad.float()
        if s.z is not None:
            dz = dz * _slope(s.z.float(), s.activation)
        out = {'dx': (dz @ s.weight.float()).to(kind), 'dweight': (dz.t() @ s.x.float()).to(kind)}
        if s.bias is not None:
            out['dbias'] = dz.sum(0).to(kind)
        return out
    if s.op == 'orthogonalize':
        return _newton_schulz(s.x.float()).to(s.x.dtype)
    kind = s.weight.dtype
    grad = s.grad.float()
    momentum = s.beta * s.momentum.float() + (1 - s.beta) * grad
    update = s.beta * momentum + (1 - s.beta) * grad if s.nesterov else momentum
    weight = (1 - s.rate * s.decay) * s.weight.float() - s.rate * s.scale * _newton_schulz(update)
    return {'weight': weight.to(kind), 'momentum': momentum.to(kind)}


# --- what a pass cannot do without ---------------------------------------

def _newton_schulz_flops(rows, columns):
    """Half of each of the two symmetric products, the third, and the sums."""
    m, n = min(rows, columns), max(rows, columns)
    return STEPS * (m * m * n + m ** 3 + 2 * m * m * n + 3 * m * m + 2 * m * n)


def work(case):
    e = BYTES[case['type']]
    if case['op'].startswith('linear'):
        p, c, o = case['points'], case['inputs'], case['outputs']
        bias = o if case['bias'] else 0
        if case['op'] == 'linear':
            arrays = 1 + case['residual'] + case['keep']
            return {'bytes': e * (p * c + o * c + bias + arrays * p * o), 'flops': 2 * p * c * o + 4 * p * o}
        arrays = 1 + (case['activation'] != 'linear')
        return {'bytes': e * (2 * p * c + 2 * o * c + bias + arrays * p * o), 'flops': 4 * p * c * o + 6 * p * o}
    m, n = case['rows'], case['columns']
    if case['op'] == 'orthogonalize':
        return {'bytes': 2 * e * case['matrices'] * m * n, 'flops': case['matrices'] * (_newton_schulz_flops(m, n) + 3 * m * n)}
    return {'bytes': 5 * e * m * n, 'flops': _newton_schulz_flops(m, n) + 10 * m * n}


# --- the same outputs in 64 bits -----------------------------------------

def _exact_newton_schulz(x):
    """From the definition: a X + b (X X') X + c (X X')^2 X, for each matrix, from whichever side is smaller."""
    out = []
    for v in x:
        flip = v.shape[0] > v.shape[1]
        v = v.mT if flip else v
        v = v / (torch.linalg.vector_norm(v) + TINY)
        for _ in range(STEPS):
            once = v @ (v.mT @ v) if v.shape[1] < 64 else (v @ v.mT) @ v
            twice = (v @ v.mT) @ once
            v = COEFFICIENTS[0] * v + COEFFICIENTS[1] * once + COEFFICIENTS[2] * twice
        out.append(v.mT if flip else v)
    return torch.stack(out)


def exact(case, seed):
    s = prepare(case, seed)
    d = torch.float64
    if s.op.startswith('linear'):
        act = {'linear': lambda v: v, 'sigmoid': torch.sigmoid, 'tanh': torch.tanh, 'silu': torch.nn.functional.silu}[s.activation]
        x, weight = s.x.to(d), s.weight.to(d)
        bias = None if s.bias is None else s.bias.to(d)
        if s.op == 'linear':
            z = torch.einsum('pc,oc->po', x, weight)
            if bias is not None:
                z = z + bias
            y = act(z) if s.residual is None else act(z) + s.residual.to(d)
            return {'y': y, 'z': z} if s.case['keep'] else {'y': y}
        # The activation's slope at the kept z, by autograd; the layer's gradients from the definition.
        dz = s.grad.to(d)
        if s.z is not None:
            z = s.z.to(d).requires_grad_()
            dz, = torch.autograd.grad(act(z), z, dz)
        out = {'dx': torch.einsum('po,oc->pc', dz, weight), 'dweight': torch.einsum('po,pc->oc', dz, x)}
        if bias is not None:
            out['dbias'] = torch.einsum('po->o', dz)
        return out
    if s.op == 'orthogonalize':
        return _exact_newton_schulz(s.x.to(d))
    grad = s.grad.to(d)
    momentum = s.momentum.to(d).lerp(grad, 1 - s.beta)
    update = grad.lerp(momentum, s.beta) if s.nesterov else momentum
    step = _exact_newton_schulz(update[None])[0]
    return {'weight': s.weight.to(d) * (1 - s.rate * s.decay) - step * (s.rate * s.scale), 'momentum': momentum}
