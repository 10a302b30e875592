"""The layer operators in 64 bits, with bounds for what a kernel in FP32 may differ by.

u is half a unit in the last place of the result's type, e = 2^-24 that of FP32. A tensor-core sum of K products cuts off
below 2^-23 of what it has reached, once for each 16 products and once inside; a sum of FP32 parts is taken out every 64
products, after at most 6 * 4 such steps, and added in FP32. With S the sum of the terms' absolute values both stay below
``chain(K) * S``."""
import torch

E = 2.0 ** -24
ROUNDING = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24}

ACTIVATIONS = {'linear': lambda z: z, 'sigmoid': torch.sigmoid, 'tanh': torch.tanh, 'silu': lambda z: z * torch.sigmoid(z)}


def slope(z, name):
    if name == 'linear':
        return torch.ones_like(z)
    if name == 'tanh':
        return 1 - torch.tanh(z) ** 2
    f = torch.sigmoid(z)
    return f * (1 - f) if name == 'sigmoid' else f + z * f * (1 - f)


def chain(terms, kind):
    """Rounding errors of a sum of ``terms`` products, relative to the sum of their absolute values. FP32 operands are
    three parts of 8 bits each: what is left out is below 4 e of a product. Splitting the sum and joining it adds less than
    the 64 e that cover both."""
    steps = 2 * (terms / 16 + 2) if kind != torch.float32 else 2 * 24 + terms / 64
    return (2 * steps + 64) * E


def linear(x, weight, bias, activation, residual):
    """(y, z, bound of y, bound of z) of flattened x."""
    kind, d = x.dtype, torch.float64
    u = ROUNDING[kind]
    X, W = x.to(d).reshape(-1, x.shape[-1]), weight.to(d)
    z, size = X @ W.mT, X.abs() @ W.abs().mT
    if bias is not None:
        z, size = z + bias.to(d), size + bias.to(d).abs()
    raw = chain(x.shape[-1], kind) * size  # of z before it is rounded
    act = ACTIVATIONS[activation](z)
    # Slopes are at most 1.1; an activation is good to some roundings of its argument and itself.
    off = 1.1 * raw + (0 if activation == 'linear' else 16 * E * (1 + z.abs()) * act.abs().clamp(min=E))
    y = act
    if residual is not None:
        r = residual.to(d).reshape(y.shape)
        y, off = act + r, off + E * (act.abs() + r.abs())
    return y, z, off + u * (y.abs() + off) + TINY[kind], raw + u * (z.abs() + raw) + TINY[kind]


def linear_gradient(grad, x, weight, activation, z, out=None):
    """((dx, bound), (dweight, bound), (dbias, bound)); ``out`` is the type of dweight and dbias."""
    kind, d = x.dtype, torch.float64
    u, v = ROUNDING[kind], ROUNDING[out or kind]
    X, W, G = x.to(d).reshape(-1, x.shape[-1]), weight.to(d), grad.to(d).reshape(-1, weight.shape[0])
    dz = G if activation == 'linear' else G * slope(z.to(d).reshape(G.shape), activation)
    # The slope by FP32 steps, off by some e of 1 + |z|; then dz in the type of the product's operands.
    off = torch.zeros_like(dz)
    if activation != 'linear':
        off = 16 * E * (1 + z.to(d).reshape(G.shape).abs()) * G.abs()
        raw = off
        off = off + (0 if kind == torch.float32 else u) * dz.abs() + TINY[kind]
    else:
        raw = off
    p, o = G.shape

    def product(a, a_off, b, terms):
        size = (a.abs() + a_off) @ b.abs()
        return a @ b, a_off @ b.abs() + chain(terms, kind) * size

    dx, dx_off = product(dz, off, W, o)
    dw, dw_off = product(dz.mT, off.mT, X, p)
    db, db_off = dz.sum(0), (raw + (p + 16) * E * dz.abs()).sum(0)
    return ((dx, dx_off + u * (dx.abs() + dx_off) + TINY[kind]), (dw, dw_off + v * (dw.abs() + dw_off) + TINY[out or kind]),
            (db, db_off + v * (db.abs() + db_off) + TINY[out or kind]))


QUINTIC = (3.4445, -4.775, 2.0315)


def _triples(steps, coefficients):
    flat = [coefficients] if isinstance(coefficients[0], (int, float)) else list(coefficients)
    return [flat[min(k, len(flat) - 1)] for k in range(steps)]


def orthogonalize(x, steps=5, coefficients=QUINTIC, eps=1e-7):
    """One matrix, from the definition."""
    x = x.to(torch.float64)
    x = x / (torch.linalg.vector_norm(x) + eps)
    for a, b, c in _triples(steps, coefficients):
        once = (x @ x.mT) @ x if x.shape[0] <= x.shape[1] else x @ (x.mT @ x)
        twice = (x @ x.mT) @ once if x.shape[0] <= x.shape[1] else once @ (x.mT @ x)
        x = a * x + b * once + c * twice
    return x


def _parts(v, count, shift):
    """``count`` FP16 parts of v 2^shift."""
    rest, out = v * 2.0 ** shift, 0
    for _ in range(count):
        h = rest.to(torch.float16).to(torch.float64)
        rest, out = rest - h, out + h
    return out / 2.0 ** shift


def orthogonalize_modelled(x, kind, steps=5, coefficients=QUINTIC, eps=1e-7, step=False):
    """The same with the roundings of the kernels: X in two FP16 parts, products of two parts (FP32, FP16 but for an optimiser's
    step, and small sides) or of the first ones, sums in FP32. How far it is from the exact result is the scale of a tolerance."""
    d = torch.float64
    count = 2 if kind == torch.float32 or (kind == torch.float16 and not step) or min(x.shape) <= 256 else 1

    def summed(v):
        return v.to(torch.float32).to(d)

    x = x.to(d)
    x = x / (torch.linalg.vector_norm(x) + eps)
    tall = x.shape[0] > x.shape[1]
    for a, b, c in _triples(steps, coefficients):
        x, first = _parts(summed(x), 2, 12), _parts(summed(x), count, 12)
        gram = _parts(summed(first.mT @ first if tall else first @ first.mT), count, 12)
        q = _parts(summed(b * gram + c * (gram @ gram)), count, 9)
        x = summed(a * x + (first @ q if tall else q @ first))
    return x
