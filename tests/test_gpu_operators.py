"""Embedding lookup, dropout and group norm with their gradients against 64-bit forms of the same formulas.

Tolerances come from the arithmetic: u is the output type's half unit in the last place, e = 2^-24 that of the FP32
operations in between. A product or a sum of two adds one e; a sum of k terms in any order at most k e of the terms'
absolute sum. Group norm: an error of a few e of |x| in a group's mean passes through (x - mean) rstd, so everything
behind it is good to 64 e (1 + max|mean| rstd + max|x - mean| rstd) and u of its norm (sums and activations are chains of
fewer than 64 roundings for these sizes); gradients have the same bound against the norm of their terms.
"""
import ctypes

import numpy as np
import pytest

torch = pytest.importorskip('torch')

import operator_oracle as oracle  # noqa: E402
from cpde_b200 import native, operators  # noqa: E402
from operator_oracle import EPS, ROUNDING, TINY, wide  # noqa: E402

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(scope='module')
def engine():
    torch.cuda.init()
    with native.Engine(0) as e:
        yield e


def made(seed, *shape, dtype=F32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).cuda()


def some_ids(seed, tokens, rows, kind=torch.int64, absent=False, skew=False):
    rng = np.random.default_rng(seed)
    ids = rng.integers(0, rows, tokens)
    if skew:
        ids = np.minimum((rows + 1.0) ** rng.random(tokens) - 1, rows - 1).astype(np.int64)
    if absent:
        ids[rng.random(tokens) < 0.2] = -1
        ids[rng.random(tokens) < 0.1] = rows
        ids[rng.random(tokens) < 0.1] = 2 ** 31 - 1
        if kind == torch.int64:
            ids[rng.random(tokens) < 0.1] = -2 ** 62
    return torch.from_numpy(ids).to(kind).cuda()


def lookup(table, ids, scale):
    t, i = wide(table), ids.cpu().numpy().astype(np.int64).reshape(-1)
    there = (i >= 0) & (i < len(t))
    return np.where(there[:, None], t[np.where(there, i, 0)] * float(np.float32(scale)), 0.0)


# --- embedding ---------------------------------------------------------------

@pytest.mark.parametrize('kind,out', [(F32, F32), (BF16, BF16), (F16, F16), (F32, BF16), (F32, F16)])
@pytest.mark.parametrize('tokens,rows,channels', [(1, 1, 1), (3, 5, 2), (300, 17, 20), (65, 1000, 33), (257, 9, 64),
                                                  (40, 100, 1000), (2, 3, 4096), (1000, 700, 6)])
def test_embedding(engine, kind, out, tokens, rows, channels):
    table = made(1, rows, channels, dtype=kind)
    for ids in (some_ids(2, tokens, rows), some_ids(3, tokens, rows, torch.int32, absent=True)):
        got = operators.embedding(engine, table, ids, scale=3.7, dtype=out)
        assert got.dtype == out and got.shape == (tokens, channels)
        want = lookup(table, ids, 3.7)
        bound = (EPS + (1 + EPS) * ROUNDING[out]) * abs(want) + TINY[out]
        assert (abs(wide(got) - want) <= bound).all()


def test_embedding_layouts(engine):
    whole = made(4, 50, 96)
    ids = some_ids(5, 60, 50).view(3, 20)
    for table in (whole[:, 8:40], whole[:, 3:36], whole[:, 1:2], whole[::2, 4:12], whole.t()[:50].t()):
        for i in (ids % table.shape[0], (ids % table.shape[0])[:, ::2], (ids % table.shape[0]).t()):
            got = operators.embedding(engine, table, i, scale=1.0)
            assert torch.equal(got, table[i])


def test_embedding_empty(engine):
    table = made(6, 4, 8)
    assert operators.embedding(engine, table, torch.zeros((0,), dtype=torch.int64, device='cuda')).shape == (0, 8)
    grad = operators.embedding_gradient(engine, made(7, 0, 8), torch.zeros((0,), dtype=torch.int64, device='cuda'), 4)
    assert torch.equal(grad, torch.zeros_like(grad))


def test_embedding_reads_nothing_of_other_rows(engine):
    table = torch.full((6, 8), float('nan'), device='cuda')
    table[2] = 1.0
    ids = torch.tensor([2, -1, 6, 2], device='cuda')
    got = operators.embedding(engine, table, ids)
    assert torch.equal(got[:, 0], torch.tensor([1.0, 0, 0, 1.0], device='cuda'))


def scattered(grad, ids, rows, scale):
    """(sums, sums of absolute terms, numbers of terms) by row."""
    g, i = wide(grad).reshape(-1, grad.shape[-1]), ids.cpu().numpy().astype(np.int64).reshape(-1)
    there = (i >= 0) & (i < rows)
    total, size, terms = np.zeros((rows, g.shape[1])), np.zeros((rows, g.shape[1])), np.zeros((rows, 1))
    np.add.at(total, i[there], g[there])
    np.add.at(size, i[there], abs(g[there]))
    np.add.at(terms, i[there], 1)
    s = float(np.float32(scale))
    return total * s, size * abs(s), terms


def check_gradient(engine, grad, ids, rows, scale=0.8, dtype=None):
    got = operators.embedding_gradient(engine, grad, ids, rows, scale=scale, dtype=dtype)
    again = operators.embedding_gradient(engine, grad, ids, rows, scale=scale, dtype=dtype)
    assert torch.equal(got.view(torch.uint8), again.view(torch.uint8))
    want, size, terms = scattered(grad, ids, rows, scale)
    u = ROUNDING[got.dtype]
    assert (abs(wide(got) - want) <= (terms + 1) * EPS * size * (1 + u) + u * abs(want) + TINY[got.dtype]).all()


@pytest.mark.parametrize('kind,out', [(F32, F32), (BF16, BF16), (F16, F16), (BF16, F32), (F16, F32)])
@pytest.mark.parametrize('tokens,rows,channels', [(1, 1, 1), (3, 5, 2), (300, 17, 20), (65, 1000, 33), (257, 9, 64),
                                                  (40, 100, 1000), (5, 3, 2048), (3000, 700, 6)])
def test_embedding_gradient(engine, kind, out, tokens, rows, channels):
    grad = made(8, tokens, channels, dtype=kind)
    for ids in (some_ids(9, tokens, rows), some_ids(10, tokens, rows, torch.int32, absent=True, skew=True)):
        check_gradient(engine, grad, ids, rows, dtype=out)


@pytest.mark.parametrize('tokens', [31, 32, 33, 2047, 2048, 2049, 8200, 33000, 70001, 300000])
@pytest.mark.parametrize('rows', [1, 2, 1023, 1024, 5000])
def test_embedding_gradient_sort_sizes(engine, tokens, rows):
    grad = made(11, tokens, 4)
    check_gradient(engine, grad, some_ids(12, tokens, rows, absent=True), rows)


@pytest.mark.parametrize('rows', [(1 << 20) - 1, 1 << 20, 3000000])
def test_embedding_gradient_many_rows(engine, rows):
    grad = made(13, 20000, 3, dtype=BF16)
    check_gradient(engine, grad, some_ids(14, 20000, rows, skew=True), rows, dtype=F32)


@pytest.mark.parametrize('tokens,channels', [(50000, 8), (4096, 1024), (9000, 1)])
def test_embedding_gradient_few_distinct_rows(engine, tokens, channels):
    grad = made(15, tokens, channels)
    check_gradient(engine, grad, torch.full((tokens,), 6, device='cuda'), 9)
    check_gradient(engine, grad, torch.full((tokens,), -1, device='cuda'), 9)
    check_gradient(engine, grad, (torch.arange(tokens, device='cuda') > tokens // 3).long() * 8, 9)


def test_embedding_gradient_layouts(engine):
    whole = made(16, 400, 96)
    ids = some_ids(17, 400, 30)
    for grad in (whole[:, 8:40], whole[:, 3:36], whole[:, 5:6], whole[:1].expand(400, 96), whole[:96].t()):
        check_gradient(engine, grad, ids[:len(grad)], 30)


# --- dropout -----------------------------------------------------------------

@pytest.mark.parametrize('kind', [F32, BF16, F16])
@pytest.mark.parametrize('shape', [(1,), (7,), (8,), (9,), (3, 5), (16, 64), (5, 717), (2, 3, 40)])
@pytest.mark.parametrize('rate,seed,offset', [(0.25, 1, 0), (0.1, (1 << 63) + 11, (1 << 40) + 3), (0.0, 5, 5),
                                              (1.0, 5, 5), (0.5, 0, 0)])
def test_dropout(engine, kind, shape, rate, seed, offset):
    x, residual = made(20, *shape, dtype=kind), made(21, *shape, dtype=kind)
    want = oracle.dropped(wide(x), rate, seed, offset)
    got = operators.dropout(engine, x, rate, seed, offset)
    assert ((wide(got) == 0) >= (want == 0)).all()
    assert (abs(wide(got) - want) <= (2 * EPS + (1 + EPS) * ROUNDING[kind]) * abs(want) + TINY[kind]).all()
    assert torch.equal(got, operators.dropout_gradient(engine, x, rate, seed, offset))
    both = operators.dropout(engine, x, rate, seed, offset, residual=residual)
    total = want + wide(residual)
    bound = 3 * EPS * (abs(want) + abs(total)) + (1 + EPS) * ROUNDING[kind] * abs(total) + TINY[kind]
    assert (abs(wide(both) - total) <= bound).all()


def test_dropout_layouts(engine):
    whole = made(22, 64, 96)
    for x in (whole[:, 8:40], whole[:, 3:36], whole[::2], whole.t(), whole[:, :1], whole[:1].expand(64, 96),
              whole.view(4, 16, 96)[:, :, 16:48], whole.view(4, 16, 96).transpose(0, 1), whole[3, 4]):
        want = operators.dropout(engine, x.contiguous(), 0.3, 7, 9)
        assert torch.equal(operators.dropout(engine, x, 0.3, 7, 9), want)
        r = torch.ones_like(x)
        assert torch.equal(operators.dropout(engine, x, 0.3, 7, 9, residual=r), want + 1)
    base = made(23, 1001)
    assert torch.equal(operators.dropout(engine, base[1:], 0.3, 7), operators.dropout(engine, base[1:].clone(), 0.3, 7))


def test_dropped_values_are_not_looked_at(engine):
    x = torch.full((64, 33), float('nan'), device='cuda')
    x[::2] = float('inf')
    keep, _ = oracle.kept(x.numel(), 0.5, 3, 4)
    got = operators.dropout(engine, x, 0.5, 3, 4).cpu().numpy().reshape(-1)
    assert (got[~keep] == 0).all() and not np.isfinite(got[keep]).any()


def test_dropout_empty(engine):
    assert operators.dropout(engine, made(24, 0, 5), 0.5, 1).shape == (0, 5)


# --- group norm ---------------------------------------------------------------

SHAPES = [(1, 1, 1, 1), (2, 1, 8, 2), (3, 67, 48, 6), (2, 5, 6, 3), (1, 300, 33, 11), (2, 33, 20, 1), (4, 9, 512, 32),
          (1, 4100, 16, 4), (2, 130, 640, 5), (1, 20, 1100, 10), (1, 7, 4096, 2), (5, 64, 64, 64), (2, 700, 24, 2)]


def norm_inputs(n, p, c, kind, seed=30, level=0.5):
    x = (made(seed, n, p, c) * (0.5 + made(seed + 1, c).abs()) + level * made(seed + 2, c)).to(kind)
    return x, 1 + 0.3 * made(seed + 3, c), 0.3 * made(seed + 4, c)


def check_norm(engine, x, groups, weight, bias, activation='linear', lengths=None, rate=0.0, seed=3, offset=8,
               eps=1e-5, grad_seed=35):
    kind = x.dtype
    options = dict(activation=activation, lengths=lengths, rate=rate, seed=seed, offset=offset)
    grad = made(grad_seed, *x.shape, dtype=kind)
    y, mean, rstd = operators.group_norm(engine, x, groups, weight, bias, eps=eps, **options)
    dx, dweight, dbias = operators.group_norm_gradient(engine, grad, x, mean, rstd, groups, weight, bias, **options)
    wx, wg = wide(x), wide(grad)
    if lengths is not None:  # what is masked is not part of the definition
        for i, m in enumerate(lengths.tolist()):
            wx[i, max(m, 0):] = 0
            wg[i, max(m, 0):] = 0
    w, b = (None if v is None else wide(v) for v in (weight, bias))
    want = oracle.group_norm(wx, groups, w, b, eps, activation, None if lengths is None else lengths.tolist(), rate,
                             seed, offset, wg)
    width = x.shape[2] // groups
    scale = np.repeat(want[2], width, 1)[:, None]
    spread = abs(wx - np.repeat(want[1], width, 1)[:, None]) * scale
    condition = 1 + (abs(want[1]) * want[2]).max() + (spread.max() if spread.size else 0)
    e = 64 * EPS * condition
    u = ROUNDING[kind]
    big = 1.0 if w is None else max(1.0, abs(w).max())
    shift = 1.0 if b is None else 1.0 + abs(b).max()
    factor = 65536 / (65536 - round(rate * 65536))

    def near(got, expected, size, rounding):
        assert np.isfinite(wide(got)).all()
        root = np.sqrt(expected.size)
        assert np.linalg.norm(wide(got) - expected) <= e * size * root + rounding * np.linalg.norm(expected) + root * TINY[F16]

    assert (abs(wide(mean) - want[1]) <= 64 * EPS * abs(wx).max() + 1e-30).all()
    assert (abs(wide(rstd) - want[2]) <= e * want[2]).all()
    near(y, want[0], big * shift * factor, u)
    terms = abs(wg).max() * factor * big * shift
    near(dx, want[3], terms * scale.max() * condition, u)
    counts = x.shape[0] * x.shape[1]
    for got, expected, parameter in ((dweight, want[4], weight), (dbias, want[5], bias)):
        assert (got is None) == (parameter is None)
        if got is not None:
            assert got.dtype == parameter.dtype
            near(got, expected, terms * condition * np.sqrt(counts), ROUNDING[got.dtype])
    again = operators.group_norm(engine, x, groups, weight, bias, eps=eps, **options)
    assert all(torch.equal(a, b) for a, b in zip((y, mean, rstd), again))
    again = operators.group_norm_gradient(engine, grad, x, mean, rstd, groups, weight, bias, **options)
    assert all(a is None or torch.equal(a, b) for a, b in zip((dx, dweight, dbias), again))
    return y, dx


@pytest.mark.parametrize('kind', [F32, BF16, F16])
@pytest.mark.parametrize('n,p,c,groups', SHAPES)
def test_group_norm(engine, kind, n, p, c, groups):
    x, weight, bias = norm_inputs(n, p, c, kind)
    check_norm(engine, x, groups, weight, bias)


@pytest.mark.parametrize('kind', [F32, BF16])
@pytest.mark.parametrize('activation', ['sigmoid', 'tanh', 'silu'])
@pytest.mark.parametrize('rate', [0.0, 0.2])
@pytest.mark.parametrize('n,p,c,groups', [(3, 67, 48, 6), (2, 5, 6, 3), (1, 300, 33, 11), (2, 130, 640, 5)])
def test_group_norm_activations(engine, kind, activation, rate, n, p, c, groups):
    x, weight, bias = norm_inputs(n, p, c, kind)
    check_norm(engine, x, groups, weight, bias, activation, rate=rate)


@pytest.mark.parametrize('n,p,c,groups', [(6, 67, 48, 6), (6, 5, 6, 3), (6, 300, 128, 4), (6, 1, 16, 2)])
@pytest.mark.parametrize('rate', [0.0, 0.2])
def test_group_norm_lengths(engine, n, p, c, groups, rate):
    x, weight, bias = norm_inputs(n, p, c, BF16)
    lengths = torch.tensor([p, 0, 1, p // 2, -3, p + 9], dtype=torch.int32, device='cuda')
    for i, m in enumerate(lengths.clamp(0, p).tolist()):
        x[i, m:] = float('nan') if i % 2 else float('inf')
    y, dx = check_norm(engine, x, groups, weight, bias, 'silu', lengths, rate)
    for i, m in enumerate(lengths.clamp(0, p).tolist()):
        assert not y[i, m:].any() and not dx[i, m:].any()


def test_group_norm_all_instances_empty(engine):
    x, weight, bias = norm_inputs(2, 40, 16, F32)
    lengths = torch.zeros(2, dtype=torch.int32, device='cuda')
    y, mean, rstd = operators.group_norm(engine, x, 4, weight, bias, lengths=lengths)
    parts = operators.group_norm_gradient(engine, x, x, mean, rstd, 4, weight, bias, lengths=lengths)
    for t in (y, mean, rstd, *parts):
        assert not t.any()


@pytest.mark.parametrize('n,p', [(0, 5), (2, 0)])
def test_group_norm_no_points(engine, n, p):
    x = made(36, n, p, 8)
    weight = made(37, 8)
    y, mean, rstd = operators.group_norm(engine, x, 2, weight, weight)
    assert y.shape == (n, p, 8) and mean.shape == (n, 2) and not mean.any() and not rstd.any()
    dx, dweight, dbias = operators.group_norm_gradient(engine, x, x, mean, rstd, 2, weight, weight)
    assert dx.shape == (n, p, 8) and not dweight.any() and not dbias.any()


@pytest.mark.parametrize('weight,bias', [(True, False), (False, True), (False, False)])
@pytest.mark.parametrize('kind', [F32, F16])
def test_group_norm_parameters(engine, weight, bias, kind):
    x, w, b = norm_inputs(2, 70, 24, kind)
    check_norm(engine, x, 3, w if weight else None, b if bias else None, 'silu')
    if kind != F32:
        check_norm(engine, x, 3, w.to(kind) if weight else None, b.to(kind) if bias else None, 'silu')


@pytest.mark.parametrize('p', [50, 3000, 40000])
def test_group_norm_level_far_above_the_spread(engine, p):
    x = 1000 + made(38, 2, p, 16)
    check_norm(engine, x, 2, None, None)
    x[:, 0] += 3000  # a first point that is not like the others
    check_norm(engine, x, 2, None, None)


def test_group_norm_constant_groups(engine):
    x = torch.full((2, 60, 8), 2.5, device='cuda')
    y, mean, rstd = operators.group_norm(engine, x, 2)
    assert not y.any() and torch.equal(mean, torch.full_like(mean, 2.5))
    assert torch.allclose(rstd, torch.full_like(rstd, 1e-5 ** -0.5), rtol=1e-6)


def test_group_norm_layouts(engine):
    whole = made(39, 4, 50, 96)
    for x in (whole[:, :, 8:40], whole[:, :, 3:35], whole[:, ::2], whole[::2], whole.transpose(0, 1),
              whole.transpose(1, 2), whole[:1].expand(4, 50, 96), whole[:, :1].expand(4, 50, 96)):
        weight, bias = made(40, x.shape[2]), made(41, x.shape[2])
        check_norm(engine, x, 2, weight, bias, 'tanh')


@pytest.mark.parametrize('n,p,c,groups', [(1, 70000, 32, 4), (3, 9000, 128, 8), (40, 600, 256, 16)])
@pytest.mark.parametrize('kind', [F32, BF16])
def test_group_norm_large(engine, n, p, c, groups, kind):
    x, weight, bias = norm_inputs(n, p, c, kind)
    lengths = torch.full((n,), p - 3, dtype=torch.int32, device='cuda')
    lengths[0] = p // 3
    check_norm(engine, x, groups, weight, bias, 'sigmoid', lengths if n > 1 else None)


@pytest.mark.parametrize('activation', ['linear', 'sigmoid', 'tanh', 'silu'])
def test_group_norm_gradient_against_differences(engine, activation):
    """Central differences of the forward along random directions: truncation O(h^2) = 1e-4 and FP32 noise
    2 e sqrt(size) / h, both well under 2e-3 of the directional derivative's scale."""
    x, weight, bias = norm_inputs(2, 40, 24, F32)
    grad = made(42, *x.shape)
    options = dict(activation=activation, rate=0.2, seed=5, offset=6)

    def loss(x, weight, bias):
        return float((wide(operators.group_norm(engine, x, 3, weight, bias, **options)[0]) * wide(grad)).sum())

    y, mean, rstd = operators.group_norm(engine, x, 3, weight, bias, **options)
    parts = operators.group_norm_gradient(engine, grad, x, mean, rstd, 3, weight, bias, **options)
    h = 1e-2
    for at in range(3):
        v = [torch.zeros_like(t) for t in (x, weight, bias)]
        v[at] = made(43 + at, *v[at].shape)
        up, down = (loss(*(a + s * h * b for a, b in zip((x, weight, bias), v))) for s in (1, -1))
        slope = float((wide(parts[at]) * wide(v[at])).sum())
        assert abs((up - down) / (2 * h) - slope) <= 2e-3 * np.linalg.norm(wide(grad)) * np.sqrt(v[at].numel())


# --- together -----------------------------------------------------------------

def test_autograd(engine):
    table, weight, bias = made(50, 30, 16).requires_grad_(), made(51, 16).requires_grad_(), made(52, 16).requires_grad_()
    ids = some_ids(53, 120, 30, absent=True).view(4, 30)
    x = operators.Embedding.apply(engine, table, ids, 1.5)
    h = operators.GroupNorm.apply(engine, x, weight, bias, 4, 1e-5, 'silu', None, 0.1, 3, 4)
    y = operators.Dropout.apply(engine, h, 0.2, 3, 5, x)
    y.sum().backward()  # an expanded gradient
    d = torch.float64
    t64, w64, b64 = (v.detach().cpu().to(d).requires_grad_() for v in (table, weight, bias))
    i = ids.cpu()
    there = (i >= 0) & (i < 30)
    e = t64[torch.where(there, i, 0)] * 1.5 * there[..., None]
    z = e.view(4, 30, 4, 4)
    z = (z - z.mean((1, 3), keepdim=True)) / (z.var((1, 3), unbiased=False, keepdim=True) + 1e-5).sqrt()
    z = torch.nn.functional.silu(z.reshape(4, 30, 16) * w64 + b64)
    for rate, offset, add in ((0.1, 4, None), (0.2, 5, e)):
        keep, factor = oracle.kept(z.numel(), rate, 3, offset)
        z = z * torch.from_numpy(keep.reshape(z.shape) * factor)
        z = z if add is None else z + add
    z.sum().backward()
    assert np.linalg.norm(wide(y) - z.detach().numpy()) <= 1e-5 * np.linalg.norm(z.detach().numpy())
    for got, want in ((table, t64), (weight, w64), (bias, b64)):
        want = want.grad.numpy()
        assert np.linalg.norm(wide(got.grad) - want) <= 2e-5 * np.linalg.norm(want)


def one_step(engine, table, ids, weight, bias, grad):
    x = operators.embedding(engine, table, ids)
    y, mean, rstd = operators.group_norm(engine, x, 4, weight, bias, activation='silu', rate=0.1, seed=1)
    out = operators.dropout(engine, y, 0.1, 1, 2, residual=x)
    dx, dweight, dbias = operators.group_norm_gradient(engine, grad, x, mean, rstd, 4, weight, bias,
                                                       activation='silu', rate=0.1, seed=1)
    return out, dx, dweight, dbias, operators.embedding_gradient(engine, dx, ids, len(table))


def step_inputs():
    return (made(60, 500, 64), some_ids(61, 1200, 500).view(3, 400), made(62, 64), made(63, 64), made(64, 3, 400, 64))


def test_other_streams(engine):
    inputs = step_inputs()
    want = one_step(engine, *inputs)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(one_step(engine, *inputs))
    torch.cuda.synchronize()
    for outs in got:
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_graph_capture(engine):
    inputs = step_inputs()
    want = one_step(engine, *inputs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = one_step(engine, *inputs)
    inputs[0].mul_(2.0)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(operators.embedding(engine, inputs[0], inputs[1]),
                       2 * operators.embedding(engine, inputs[0] / 2, inputs[1]))
    assert all(torch.equal(a, b) for a, b in zip(got, one_step(engine, *inputs)))
    assert not torch.equal(got[0], want[0])
    del graph


# --- refusals -----------------------------------------------------------------

def test_wrong_arguments_are_refused(engine):
    x, ids = made(70, 2, 6, 8), torch.zeros(6, dtype=torch.int64, device='cuda')
    table = x[0]
    weight = made(71, 8)
    mean = torch.zeros((2, 2), device='cuda')
    bad = [
        lambda: operators.embedding(engine, table.cpu(), ids),
        lambda: operators.embedding(engine, table.double(), ids),
        lambda: operators.embedding(engine, table, ids.float()),
        lambda: operators.embedding(engine, x, ids),
        lambda: operators.embedding(engine, table, ids, dtype=torch.float64),
        lambda: operators.embedding_gradient(engine, x[0], ids[:5], 4),
        lambda: operators.embedding_gradient(engine, x[0], ids, 0),
        lambda: operators.dropout(engine, x.long(), 0.1, 1),
        lambda: operators.dropout(engine, x, 0.1, 1, residual=x[:1]),
        lambda: operators.group_norm(engine, x, 3),
        lambda: operators.group_norm(engine, x, 0),
        lambda: operators.group_norm(engine, x[0], 2),
        lambda: operators.group_norm(engine, x, 2, weight[:4]),
        lambda: operators.group_norm(engine, x, 2, weight.half(), weight),
        lambda: operators.group_norm(engine, x, 2, weight.half()),
        lambda: operators.group_norm(engine, x, 2, activation='relu'),
        lambda: operators.group_norm(engine, x, 2, lengths=torch.zeros(2, device='cuda')),
        lambda: operators.group_norm_gradient(engine, x.half(), x, mean, mean, 2),
        lambda: operators.group_norm_gradient(engine, x, x, mean[:1], mean, 2),
    ]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    refused = [
        lambda: operators.embedding(engine, table.half(), ids, dtype=F32),
        lambda: operators.embedding_gradient(engine, table, ids, 4, dtype=BF16),
        lambda: operators.dropout(engine, x, -0.1, 1),
        lambda: operators.dropout(engine, x, 1.5, 1),
        lambda: operators.dropout(engine, x, float('nan'), 1),
        lambda: operators.group_norm(engine, x, 2, eps=0.0),
        lambda: operators.group_norm(engine, x, 2, eps=float('nan')),
        lambda: operators.group_norm(engine, x, 2, rate=2.0),
    ]
    for call in refused:
        with pytest.raises(native.EngineError) as error:
            call()
        assert error.value.status == native.REJECTED and str(error.value)


def test_c_entries_refuse_bad_pointers_and_sizes(engine):
    """Refused on the host, before any launch: nothing here reaches the device."""
    lib, h = engine.lib, engine.handle
    a = made(72, 64, 8)
    p = a.data_ptr()
    size = ctypes.c_size_t()
    assert lib.cpde_embedding(h, 0, None, 8, 8, 8, 1, p, 4, 1.0, 0, p, None) == native.REJECTED
    assert lib.cpde_embedding(h, 0, p + 2, 8, 8, 8, 1, p, 4, 1.0, 0, p, None) == native.REJECTED
    assert lib.cpde_embedding(h, 3, p, 8, 8, 8, 1, p, 4, 1.0, 3, p, None) == native.REJECTED
    assert lib.cpde_embedding(h, 0, p, 8, 8, 8, 2, p, 4, 1.0, 0, p, None) == native.REJECTED
    assert lib.cpde_embedding(h, 0, p, 7, 8, 8, 1, p, 4, 1.0, 0, p, None) == native.REJECTED
    assert lib.cpde_embedding(h, 0, p, 8, 8, 8, 1, p, -1, 1.0, 0, p, None) == native.REJECTED
    assert lib.cpde_embedding(h, 0, p, 8, 1 << 31, 8, 1, p, 4, 1.0, 0, p, None) == native.REJECTED
    assert lib.cpde_embedding(h, 0, p, 8, 8, 0, 1, p, 4, 1.0, 0, p, None) == native.REJECTED
    assert lib.cpde_embedding_gradient(h, 0, p, 8, 1, p, 4, 8, 8, 1.0, 0, p, None, 1 << 20, None) == native.REJECTED
    assert lib.cpde_embedding_gradient(h, 0, p, 8, 1, p, 4, 8, 8, 1.0, 0, p, p, 16, None) == native.REJECTED
    assert 'workspace' in lib.cpde_last_error(h).decode()
    assert lib.cpde_embedding_gradient_workspace(4, 0, 8, ctypes.byref(size)) == native.REJECTED
    assert lib.cpde_dropout(h, 0, p, 8, None, 0, 1 << 40, 1 << 40, 0.5, 1, 1, p, None) == native.REJECTED
    assert lib.cpde_dropout(h, 0, p, 4, None, 0, 8, 8, 0.5, 1, 1, p, None) == native.REJECTED
    assert lib.cpde_dropout(h, 0, p, 8, None, 0, 8, 8, 0.5, 1, 1, None, None) == native.REJECTED
    assert lib.cpde_group_norm_workspace(1, 1, 8, 3, ctypes.byref(size)) == native.REJECTED
    norm = lambda **k: lib.cpde_group_norm(*{**dict(h=h, type=0, x=p, xp=8, xi=64, n=1, p=8, c=8, g=2, pt=0, w=None,
                                                    b=None, eps=1e-5, act=1, len=None, rate=0.0, seed=0, off=0, y=p,
                                                    mean=p, rstd=p, ws=p, size=1 << 20, stream=None), **k}.values())
    for wrong in (dict(x=None), dict(y=None), dict(mean=None), dict(rstd=p + 1), dict(act=4), dict(act=-1), dict(pt=1),
                  dict(g=3), dict(xp=7), dict(xi=-1), dict(size=8), dict(ws=None), dict(ws=p + 16), dict(n=-1),
                  dict(c=1 << 25, g=1), dict(eps=-1.0), dict(w=p + 2), dict(len=p + 1), dict(rate=-1.0)):
        assert norm(**wrong) == native.REJECTED, wrong
