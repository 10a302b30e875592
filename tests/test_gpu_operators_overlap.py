"""Calls that run back to back on inputs of their own, whose launches overlap: a kernel holds the stream while they are
queued, so that no result is there by luck of an idle GPU, and the workspace that a call gets holds what the last one left.
Tolerances: norm_bounds.py, test_gpu_operators.py."""
import ctypes
import random

import numpy as np
import pytest

torch = pytest.importorskip('torch')

import norm_bounds  # noqa: E402
from cpde_b200 import native, operators  # noqa: E402
from operator_oracle import EPS, ROUNDING, TINY, wide  # noqa: E402
from test_gpu_operators import made, scattered, some_ids  # noqa: E402

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
LEGACY = 1  # the default stream's handle


@pytest.fixture(scope='module')
def engine():
    torch.cuda.init()
    with native.Engine(0) as e:
        yield e


def queued(*calls):
    """The last call's result, all of them queued before the first one starts."""
    torch.cuda.synchronize()
    torch.cuda._sleep(2000000)  # about a millisecond
    for call in calls:
        result = call()
    torch.cuda.synchronize()
    return result


# --- lookup gradient --------------------------------------------------------

@pytest.mark.parametrize('tokens,rows,channels', [
    (2000, 3000, 24), (30000, 5000, 8), (65536, 40, 16),  # one cluster's sort
    (70001, 500, 8), (70001, 5000, 8), (150000, 300, 4),  # launches of one pass and of two
    (70001, (1 << 18) - 1, 2), (70001, 1 << 18, 2), (90000, 400000, 4)])  # of two and of three
def test_lookup_gradients(engine, tokens, rows, channels):
    for skew in (False, True):
        inputs = [(made(80 + i, tokens, channels), some_ids(90 + i, tokens, rows, absent=True, skew=skew)) for i in range(3)]
        got = queued(*[lambda g=g, i=i: operators.embedding_gradient(engine, g, i, rows) for g, i in inputs])
        want, size, terms = scattered(*inputs[-1], rows, 1.0)
        assert (abs(wide(got) - want) <= (terms + 2) * EPS * size).all()


def test_lookup_gradients_with_undefined_workspace(engine):
    tokens, rows, channels = 70001, 300000, 4
    grad, ids = made(100, tokens, channels), some_ids(101, tokens, rows, absent=True)
    size = ctypes.c_size_t()
    assert engine.lib.cpde_embedding_gradient_workspace(tokens, rows, channels, ctypes.byref(size)) == native.OK
    workspace = torch.full((size.value,), 0xFF, dtype=torch.uint8, device='cuda')
    out = torch.full((rows, channels), float('nan'), device='cuda')
    torch.cuda.synchronize()
    assert engine.lib.cpde_embedding_gradient(engine.handle, 0, grad.data_ptr(), channels, 1, ids.data_ptr(), tokens, rows,
                                              channels, 1.0, 0, out.data_ptr(), workspace.data_ptr(), size.value,
                                              LEGACY) == native.OK
    torch.cuda.synchronize()
    want, total, terms = scattered(grad, ids, rows, 1.0)
    assert (abs(wide(out) - want) <= (terms + 2) * EPS * total).all()


# --- group norm ---------------------------------------------------------------

class Case:
    def __init__(self, rng):
        self.groups = rng.choice([1, 2, 3, 4, 6, 8, 16, 32])
        self.width = rng.choice([1, 1, 2, 3, 4, 5, 6, 8, 8, 12, 16, 16, 24, 32, 33, 64])
        most = 60000 // (self.groups * self.width)
        self.n = max(1, min(64, int(np.exp(rng.uniform(0, np.log(max(2, most)))) ** 0.6)))
        self.p = max(1, int(np.exp(rng.uniform(0, np.log(max(2, most // self.n))))))
        self.kind = rng.choice([F32, BF16, F16])
        self.parameters = rng.choice([F32, self.kind])
        self.activation = rng.choice(['linear', 'sigmoid', 'tanh', 'silu'])
        self.rate = rng.choice([0.0, 0.1, 0.5])
        self.lengths = None
        if rng.random() < 0.5:
            self.lengths = [rng.choice([0, self.p, rng.randint(0, self.p), 1, -2, self.p + 3]) for _ in range(self.n)]
        self.seed, self.offset = rng.getrandbits(64), rng.getrandbits(64)
        self.with_weight, self.with_bias = rng.random() < 0.9, rng.random() < 0.9

    def inputs(self, seed):
        c = self.groups * self.width
        x = (made(seed, self.n, self.p, c) * (0.5 + made(seed + 1, c).abs()) + 0.5 * made(seed + 2, c)).to(self.kind)
        if self.lengths is not None:
            for i, m in enumerate(self.lengths):
                x[i, max(m, 0):] = float('nan')
        weight = (1 + 0.3 * made(seed + 3, c)).to(self.parameters) if self.with_weight else None
        bias = (0.3 * made(seed + 4, c)).to(self.parameters) if self.with_bias else None
        return x, made(seed + 5, self.n, self.p, c, dtype=self.kind), weight, bias

    def options(self):
        lengths = None if self.lengths is None else torch.tensor(self.lengths, dtype=torch.int32, device='cuda')
        return dict(activation=self.activation, lengths=lengths, rate=self.rate, seed=self.seed, offset=self.offset)

    def exact(self, x, weight, bias):
        return norm_bounds.Norm(wide(x), self.groups, None if weight is None else wide(weight),
                                None if bias is None else wide(bias), 1e-5, self.activation, self.lengths, self.rate, self.seed,
                                self.offset)


def within(got, want, bound):
    got = wide(got)
    assert np.isfinite(got).all()
    assert (abs(got - want) <= bound).all(), float((abs(got - want) / np.maximum(bound, 1e-300)).max())


def check(case, x, grad, weight, bias, y, mean, rstd, dx, dweight, dbias):
    norm = case.exact(x, weight, bias)
    m, r, off_m, off_r = norm.statistics()
    within(mean, m, off_m)
    within(rstd, r, off_r)
    u, tiny = ROUNDING[case.kind], TINY[case.kind]
    m, r = wide(mean), wide(rstd)
    within(y, *norm.forward(m, r, u, tiny))
    parts = norm.gradient(wide(grad), m, r, u, tiny)
    within(dx, *parts[0])
    for got, (want, bound), parameter in ((dweight, parts[1], weight), (dbias, parts[2], bias)):
        if parameter is not None:
            within(got, want, bound + ROUNDING[got.dtype] * abs(want) + TINY[got.dtype])


def run(engine, case, x, grad, weight, bias):
    options = case.options()
    y, mean, rstd = operators.group_norm(engine, x, case.groups, weight, bias, **options)
    parts = operators.group_norm_gradient(engine, grad, x, mean, rstd, case.groups, weight, bias, **options)
    return y, mean, rstd, *parts


@pytest.mark.parametrize('n,p,c,groups', [(1, 30000, 6, 3), (5, 9000, 30, 10), (1, 70000, 16, 8), (40, 600, 96, 32)])
@pytest.mark.parametrize('kind', [F32, BF16])
def test_group_norms_in_two_passes(engine, n, p, c, groups, kind):
    """Point sets that take many blocks a launch: the second of each pair waits for all of the first."""
    case = Case(random.Random(3))
    case.n, case.p, case.groups, case.width, case.kind, case.parameters = n, p, groups, c // groups, kind, F32
    case.activation, case.rate, case.lengths = 'silu', 0.1, [p - 7 * i for i in range(n)]
    case.with_weight = case.with_bias = True
    first, other = case.inputs(230), case.inputs(240)
    check(case, *first, *queued(lambda: run(engine, case, *other), lambda: run(engine, case, *first)))


def test_streams_with_inputs_of_their_own(engine):
    """Three streams at once, each with its own inputs: workspaces, counters and statistics stay apart."""
    case = Case(random.Random(7))
    case.n, case.p, case.groups, case.width, case.kind, case.parameters = 20, 900, 8, 8, BF16, F32
    case.activation, case.rate, case.lengths = 'silu', 0.1, [900 - 40 * i for i in range(20)]
    case.with_weight = case.with_bias = True
    inputs = [case.inputs(400 + 10 * i) for i in range(3)]
    lookups = [(made(440 + i, 70001, 8), some_ids(450 + i, 70001, 30000, absent=True)) for i in range(3)]

    def step(i):
        return (*run(engine, case, *inputs[i]), operators.embedding_gradient(engine, *lookups[i], 30000))

    want = [step(i) for i in range(3)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(3)], [[] for _ in range(3)]
    for s in streams:
        with torch.cuda.stream(s):
            torch.cuda._sleep(2000000)
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(step(i))
    torch.cuda.synchronize()
    for i in range(3):
        for outs in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(outs, want[i]))
