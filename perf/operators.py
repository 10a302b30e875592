"""Workloads of the conditioning operators: embedding lookup and its gradient, dropout, group norm and its gradient.

Each case is one call that a training or evaluation step makes. ``run`` computes it either with the framework's operators
(``own``) or in a plain form: elementary torch operations in 32 bits, rounded once at the end. ``exact`` gives the same outputs
in 64 bits, from the definitions.
"""
import math

import numpy as np
import torch

own = False

TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
BYTES = {'f32': 4, 'bf16': 2, 'f16': 2}
IDS = {'i32': torch.int32, 'i64': torch.int64}

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
        # A latent code per instance for a small batch of points: latency counts.
        dict(name='embedding_codes_small', op='embedding', tokens=257, rows=1000, channels=20, type='f32', ids='i64',
             skew='uniform', absent=0.0),
        # Token features of a long batch, frequencies as in text, some padding.
        dict(name='embedding_tokens_bf16', op='embedding', tokens=32768, rows=128000, channels=2048, type='bf16',
             ids='i64', skew='log', absent=0.03),
        # Learned features of the cells that a million sample points fall into.
        dict(name='embedding_cells_f32', op='embedding', tokens=1048576, rows=65536, channels=8, type='f32', ids='i32',
             skew='uniform', absent=0.0),
        # The gradients of the three lookups above.
        dict(name='embedding_grad_codes_small', op='embedding_gradient', tokens=257, rows=1000, channels=20, type='f32',
             ids='i64', skew='uniform', absent=0.0),
        dict(name='embedding_grad_tokens_bf16', op='embedding_gradient', tokens=32768, rows=128000, channels=2048,
             type='bf16', ids='i64', skew='log', absent=0.03),
        dict(name='embedding_grad_cells_f32', op='embedding_gradient', tokens=1048576, rows=65536, channels=8,
             type='f32', ids='i32', skew='uniform', absent=0.0),
        # Dropout kept on in the evaluation of a few points (uncertainty), odd size.
        dict(name='dropout_small_f32', op='dropout', rows=7, columns=717, type='f32', rate=0.25, residual=False),
        # Dropout onto the residual stream of a training step.
        dict(name='dropout_residual_bf16', op='dropout', rows=65536, columns=1024, type='bf16', rate=0.1,
             residual=True),
        # Three small point sets.
        dict(name='group_norm_small_f32', op='group_norm', instances=3, points=67, channels=48, groups=6, type='f32',
             activation='tanh', ragged=False, rate=0.0),
        # A batch of instances of a wide trunk layer.
        dict(name='group_norm_batch_bf16', op='group_norm', instances=32, points=4096, channels=512, groups=32,
             type='bf16', activation='silu', ragged=False, rate=0.0),
        # Its gradient, with point counts from none to all and dropout behind the activation.
        dict(name='group_norm_grad_ragged_bf16', op='group_norm_gradient', instances=32, points=4096, channels=512,
             groups=32, type='bf16', activation='silu', ragged=True, rate=0.1),
        # One instance of a million points.
        dict(name='group_norm_grad_points_f32', op='group_norm_gradient', instances=1, points=1048576, channels=64,
             groups=8, type='f32', activation='sigmoid', ragged=False, rate=0.0),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(['embedding', 'embedding_gradient', 'dropout', 'group_norm', 'group_norm_gradient'])
    kind = rng.choice(['f32', 'bf16', 'bf16', 'f16'])
    case = dict(op=op, type=kind)
    if op.startswith('embedding'):
        channels = rng.choice([1, 2, 4, 8, 16, 20, 33, 64, 100, 128, 256, 512, 1000, 1024, 2048, 4096])
        tokens = _log_int(rng, 64, min(1 << 20, (1 << 26) // channels))
        rows = _log_int(rng, 16, min(1 << 20, (1 << 27) // channels))
        case.update(tokens=tokens, rows=rows, channels=channels, ids=rng.choice(['i32', 'i64']),
                    skew=rng.choice(['uniform', 'log']), absent=rng.choice([0.0, 0.03, 0.5]))
    elif op == 'dropout':
        columns = _log_int(rng, 1, 8192)
        rows = _log_int(rng, 1, (1 << 26) // columns)
        case.update(rows=rows, columns=columns, rate=rng.choice([0.0, 0.1, 0.25, 0.5, 1.0]),
                    residual=rng.random() < 0.5)
    else:
        groups = rng.choice([1, 2, 4, 6, 8, 16, 32])
        channels = groups * rng.choice([1, 2, 3, 4, 8, 8, 16, 16, 32, 64])
        instances = _log_int(rng, 1, 256)
        points = _log_int(rng, 1, max(2, (1 << 25) // (channels * instances)))
        case.update(instances=instances, points=points, channels=channels, groups=groups,
                    activation=rng.choice(['linear', 'sigmoid', 'tanh', 'silu']), ragged=rng.random() < 0.4,
                    rate=rng.choice([0.0, 0.0, 0.1]))
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

    if s.op.startswith('embedding'):
        t, v, c = case['tokens'], case['rows'], case['channels']
        u = torch.rand(t, generator=g, device='cuda', dtype=torch.float64)
        ids = torch.exp(u * math.log(v + 1)).long() - 1 if case['skew'] == 'log' else (u * v).long()
        ids = ids.clamp_(0, v - 1)
        if case['absent']:
            ids[torch.rand(t, generator=g, device='cuda') < case['absent']] = -1
        s.ids = ids.to(IDS[case['ids']])
        s.scale = math.sqrt(c)
        if s.op == 'embedding':
            s.table = (normal(v, c) / math.sqrt(c)).to(kind)
        else:
            s.grad = normal(t, c).to(kind)
            s.rows = v
    elif s.op == 'dropout':
        s.x = normal(case['rows'], case['columns']).to(kind)
        s.residual = normal(case['rows'], case['columns']).to(kind) if case['residual'] else None
        s.rate, s.seed, s.offset = case['rate'], int(seed) * 7919 + 5, (1 << 33) + int(seed)
    else:
        n, p, c = case['instances'], case['points'], case['channels']
        s.groups, s.activation, s.eps = case['groups'], case['activation'], 1e-5
        # Channels with levels and spreads of their own, as a linear layer gives them.
        s.x = torch.addcmul(0.5 * normal(c), normal(n, p, c), 0.5 + 0.25 * normal(c).abs()).to(kind)
        s.weight, s.bias = 1 + 0.2 * normal(c), 0.2 * normal(c)
        s.rate, s.seed, s.offset = case['rate'], int(seed) * 7919 + 5, (1 << 33) + int(seed)
        s.lengths = None
        if case['ragged']:
            order = torch.randperm(n, generator=g, device='cuda')
            s.lengths = _lengths(n, p)[order.cpu()].to('cuda', torch.int32)
        if s.op == 'group_norm_gradient':
            s.grad = normal(n, p, c).to(kind)
            s.mean, s.rstd = _statistics(s)
    return s


def _lengths(n, p):
    """Point counts from all to none, spread evenly."""
    return torch.tensor([p] if n == 1 else [round(p * (n - 1 - i) / (n - 1)) for i in range(n)])


def _statistics(s):
    x, mask, count = _grouped(s, s.x.float())
    mean = (x * mask).sum((1, 3)) / count
    off = (x - mean[:, None, :, None]) * mask
    rstd = torch.rsqrt((off * off).sum((1, 3)) / count + s.eps)
    if s.lengths is not None:
        some = (s.lengths > 0)[:, None]
        mean, rstd = mean * some, rstd * some
    return mean, rstd


# --- one pass ------------------------------------------------------------

def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    from cpde_b200 import operators
    e = _engine()
    if s.op == 'embedding':
        return operators.embedding(e, s.table, s.ids, scale=s.scale)
    if s.op == 'embedding_gradient':
        return operators.embedding_gradient(e, s.grad, s.ids, s.rows, scale=s.scale)
    if s.op == 'dropout':
        return operators.dropout(e, s.x, s.rate, s.seed, s.offset, residual=s.residual)
    if s.op == 'group_norm':
        y, mean, rstd = operators.group_norm(e, s.x, s.groups, s.weight, s.bias, eps=s.eps, activation=s.activation,
                                             lengths=s.lengths, rate=s.rate, seed=s.seed, offset=s.offset)
        return {'y': y, 'mean': mean, 'rstd': rstd}
    dx, dweight, dbias = operators.group_norm_gradient(e, s.grad, s.x, s.mean, s.rstd, s.groups, s.weight, s.bias,
                                                       activation=s.activation, lengths=s.lengths, rate=s.rate,
                                                       seed=s.seed, offset=s.offset)
    return {'dx': dx, 'dweight': dweight, 'dbias': dbias}


LOW = 0xFFFFFFFF


def _philox(index, seed, offset):
    """Philox4x32-10 (Salmon et al., 2011) of the counters (index, offset) as int64 tensors that hold 32 bits each."""
    c0, c1 = index & LOW, (index >> 32) & LOW
    c2, c3 = torch.full_like(c0, offset & LOW), torch.full_like(c0, (offset >> 32) & LOW)
    k0, k1 = seed & LOW, (seed >> 32) & LOW
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & LOW) ^ c1 ^ k0, b & LOW, ((a >> 32) & LOW) ^ c3 ^ k1, a & LOW
        k0, k1 = (k0 + 0x9E3779B9) & LOW, (k1 + 0xBB67AE85) & LOW
    return c0, c1, c2, c3


def _kept(count, rate, seed, offset, device):
    """Which of ``count`` elements are kept, and the factor of those: 16 random bits each, eight to a counter."""
    words = _philox(torch.arange((count + 7) // 8, device=device), seed, offset)
    bits = torch.stack([h for w in words for h in (w & 0xFFFF, w >> 16)], 1).reshape(-1)[:count]
    threshold = round(rate * 65536)
    return bits >= threshold, 65536 / (65536 - threshold) if threshold < 65536 else 0.0


def _dropped(x, s):
    """``x`` with the elements that are not kept at zero, the others scaled."""
    if not s.rate:
        return x
    kept, factor = _kept(x.numel(), s.rate, s.seed, s.offset, x.device)
    return torch.where(kept.view(x.shape), x * factor, 0.0)


def _grouped(s, x):
    """x as (instance, point, group, channel of the group), the points that count and the elements of a group."""
    n, p, c = x.shape
    if s.lengths is None:
        mask, count = torch.ones((1, 1, 1, 1), device=x.device, dtype=x.dtype), float(p * (c // s.groups))
    else:
        mask = (torch.arange(p, device=x.device)[None, :] < s.lengths[:, None]).to(x.dtype)[:, :, None, None]
        count = (s.lengths.clamp(min=1) * (c // s.groups)).to(x.dtype)[:, None]
    return x.view(n, p, s.groups, c // s.groups), mask, count


def _activated(z, name):
    if name == 'linear':
        return z
    if name == 'tanh':
        return torch.tanh(z)
    f = 1 / (1 + torch.exp(-z))
    return f if name == 'sigmoid' else z * f


def _slope(z, name):
    if name == 'linear':
        return torch.ones_like(z)
    if name == 'tanh':
        t = torch.tanh(z)
        return 1 - t * t
    f = 1 / (1 + torch.exp(-z))
    return f * (1 - f) if name == 'sigmoid' else f * (1 + z * (1 - f))


def _plain(s):
    if s.op == 'embedding':
        ids = s.ids.long()
        there = (ids >= 0) & (ids < s.table.shape[0])
        picked = s.table[torch.where(there, ids, 0)].float() * s.scale
        return torch.where(there[:, None], picked, 0.0).to(s.table.dtype)
    if s.op == 'embedding_gradient':
        ids = s.ids.long()
        there = (ids >= 0) & (ids < s.rows)
        total = torch.zeros((s.rows + 1, s.grad.shape[1]), device=ids.device)
        total.index_add_(0, torch.where(there, ids, s.rows), s.grad.float())
        return (total[:s.rows] * s.scale).to(s.grad.dtype)
    if s.op == 'dropout':
        y = _dropped(s.x.float(), s)
        return (y if s.residual is None else y + s.residual.float()).to(s.x.dtype)
    xs = s.x.float()
    shape = xs.shape
    x, mask, count = _grouped(s, xs)
    weight, bias = s.weight.view(s.groups, -1), s.bias.view(s.groups, -1)
    if s.op == 'group_norm':
        mean, rstd = _statistics(s)
        z = (x - mean[:, None, :, None]) * rstd[:, None, :, None] * weight + bias
        y = _dropped(_activated(z, s.activation).reshape(shape), s)
        return {'y': (y * mask[..., 0]).to(s.x.dtype), 'mean': mean, 'rstd': rstd}
    r = s.rstd[:, None, :, None]
    xhat = (x - s.mean[:, None, :, None]) * r
    h = _dropped(s.grad.float(), s).view(x.shape) * mask * _slope(xhat * weight + bias, s.activation)
    by_channel, by_xhat = h.sum(1), (h * xhat).sum(1)
    s1 = ((by_channel * weight).sum(2) / count)[:, None, :, None]
    s2 = ((by_xhat * weight).sum(2) / count)[:, None, :, None]
    dx = (h * weight - s1 - xhat * s2) * r * mask
    return {'dx': dx.reshape(shape).to(s.x.dtype), 'dweight': by_xhat.sum(0).reshape(-1),
            'dbias': by_channel.sum(0).reshape(-1)}


# --- what a pass cannot do without ---------------------------------------

def _distinct(case):
    """Expected number of table rows that the ids name."""
    t, v = case['tokens'] * (1 - case['absent']), case['rows']
    if case['skew'] == 'uniform':
        return -v * math.expm1(t * math.log1p(-1 / v)) if v > 1 else 1.0
    k = np.arange(v, dtype=np.float64)
    share = np.log1p(1 / (k + 1)) / math.log(v + 1)
    return float(-np.expm1(t * np.log1p(-np.minimum(share, 1 - 1e-12))).sum())


def work(case):
    e = BYTES[case['type']]
    if case['op'].startswith('embedding'):
        t, v, c = case['tokens'], case['rows'], case['channels']
        here = t * (1 - case['absent'])
        ids = t * (4 if case['ids'] == 'i32' else 8)
        if case['op'] == 'embedding':
            return {'bytes': ids + e * c * (_distinct(case) + t), 'flops': here * c}
        return {'bytes': ids + e * c * (here + v), 'flops': here * c + _distinct(case) * c}
    if case['op'] == 'dropout':
        n = case['rows'] * case['columns']
        return {'bytes': n * e * (3 if case['residual'] else 2), 'flops': n * (3 if case['residual'] else 2)}
    n, p, c, g = case['instances'], case['points'], case['channels'], case['groups']
    here = int(_lengths(n, p).sum()) if case['ragged'] else n * p
    if case['op'] == 'group_norm':
        return {'bytes': e * c * (here + n * p) + 8 * c + 8 * n * g, 'flops': 12 * here * c}
    return {'bytes': e * c * (2 * here + n * p) + 16 * c + 8 * n * g, 'flops': 24 * here * c}


# --- the same outputs in 64 bits -----------------------------------------

def _exact_kept(count, rate, seed, offset):
    """The kept elements' factors and zeros, from the generator's definition in numpy's unsigned integers."""
    at = np.arange((count + 7) // 8, dtype=np.uint64)
    low, half = np.uint64(LOW), np.uint64(32)
    x = [at & low, at >> half, np.full_like(at, offset & LOW), np.full_like(at, (offset >> 32) & LOW)]
    key = [seed & LOW, (seed >> 32) & LOW]
    for _ in range(10):
        p = x[0] * np.uint64(0xD2511F53)
        q = x[2] * np.uint64(0xCD9E8D57)
        x = [(q >> half) ^ x[1] ^ np.uint64(key[0]), q & low, (p >> half) ^ x[3] ^ np.uint64(key[1]), p & low]
        key = [(key[0] + 0x9E3779B9) & LOW, (key[1] + 0xBB67AE85) & LOW]
    halves = np.ascontiguousarray(np.stack(x, 1).astype('<u4')).view('<u2').reshape(-1)[:count]
    threshold = round(rate * 65536)
    factor = 65536 / (65536 - threshold) if threshold < 65536 else 0.0
    return torch.from_numpy(halves >= threshold).cuda(), factor


def exact(case, seed):
    s = prepare(case, seed)
    d = torch.float64
    if s.op == 'embedding':
        wide = torch.cat([s.table.to(d) * s.scale, torch.zeros((1, s.table.shape[1]), dtype=d, device='cuda')])
        ids = s.ids.long()
        return wide.index_select(0, torch.where((ids < 0) | (ids >= s.table.shape[0]), s.table.shape[0], ids))
    if s.op == 'embedding_gradient':
        ids = s.ids.long()
        at = torch.nonzero((ids >= 0) & (ids < s.rows))[:, 0]
        out = torch.zeros((s.rows, s.grad.shape[1]), dtype=d, device='cuda')
        out.index_put_((ids[at],), s.grad[at].to(d) * s.scale, accumulate=True)
        return out
    if s.op == 'dropout':
        y = s.x.to(d)
        if s.rate:
            kept, factor = _exact_kept(y.numel(), s.rate, s.seed, s.offset)
            y = (y * factor).masked_fill(~kept.view(y.shape), 0.0)
        return y if s.residual is None else y + s.residual.to(d)
    # The definition as a differentiable function of x, weight and bias; its gradients are autograd's.
    n, p, c = s.x.shape
    grad = s.op == 'group_norm_gradient'
    x, weight, bias = (v.to(d).requires_grad_(grad) for v in (s.x, s.weight, s.bias))
    lengths = torch.full((n,), p, device='cuda') if s.lengths is None else s.lengths.long()
    out = torch.arange(p, device='cuda')[None, :, None] >= lengths[:, None, None]
    count = (lengths.clamp(min=1) * (c // s.groups)).to(d)[:, None]
    split = x.masked_fill(out, 0.0).unflatten(2, (s.groups, c // s.groups))
    mean = split.sum((1, 3)) / count
    off = (split - mean[:, None, :, None]).masked_fill(out[..., None], 0.0)
    rstd = ((off ** 2).sum((1, 3)) / count + s.eps) ** -0.5
    z = (off * rstd[:, None, :, None]).flatten(2) * weight + bias
    y = {'linear': lambda v: v, 'sigmoid': torch.sigmoid, 'tanh': torch.tanh,
         'silu': lambda v: v * torch.sigmoid(v)}[s.activation](z)
    if s.rate:
        kept, factor = _exact_kept(y.numel(), s.rate, s.seed, s.offset)
        y = (y * factor).masked_fill(~kept.view(y.shape), 0.0)
    y = y.masked_fill(out, 0.0)
    if not grad:
        none = (lengths == 0)[:, None]
        return {'y': y, 'mean': mean.masked_fill(none, 0.0), 'rstd': rstd.masked_fill(none, 0.0)}
    dx, dweight, dbias = torch.autograd.grad(y, (x, weight, bias), s.grad.to(d))
    return {'dx': dx, 'dweight': dweight, 'dbias': dbias}
