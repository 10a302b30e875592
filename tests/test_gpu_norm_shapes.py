"""Group norm and its gradient over random shapes: types, activations, dropout, lengths, widths and parameters together.
Tolerances: norm_bounds.py."""
import ctypes
import random

import pytest

torch = pytest.importorskip('torch')

from cpde_b200 import native, operators  # noqa: E402
from test_gpu_operators_overlap import LEGACY, Case, check, engine, queued, run  # noqa: E402,F401

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.mark.parametrize('number', range(96))
def test_group_norms_of_random_shapes(engine, number):
    """Types, activations, dropout, lengths and widths together: three steps, the middle one on other inputs."""
    case = Case(random.Random(1000 + number))
    first, other = case.inputs(200), case.inputs(210)
    got = queued(lambda: run(engine, case, *first), lambda: run(engine, case, *other), lambda: run(engine, case, *first))
    check(case, *first, *got)
    x, grad, weight, bias = first
    mean, rstd = got[1:3]
    options = case.options()
    gradient = queued(*[lambda v=v, g=g: operators.group_norm_gradient(engine, g, v, mean, rstd, case.groups, weight, bias,
                                                                       **options)
                        for v, g in ((x, grad), other[:2], (x, grad))])
    for a, b in zip(gradient, got[3:]):
        assert (a is None and b is None) or torch.equal(a, b)


@pytest.mark.parametrize('number', range(48))
def test_group_norms_with_undefined_workspace(engine, number):
    """The C entries with NaN in the workspace and in every output."""
    case = Case(random.Random(2000 + number))
    x, grad, weight, bias = case.inputs(220)
    n, p, c = x.shape
    size = ctypes.c_size_t()
    assert engine.lib.cpde_group_norm_workspace(n, p, c, case.groups, ctypes.byref(size)) == native.OK

    def undefined(shape, dtype):
        return torch.full(shape, float('nan'), dtype=dtype, device='cuda')

    def at(t):
        return None if t is None else t.data_ptr()

    code, parameter = {F32: 0, BF16: 1, F16: 2}[case.kind], {F32: 0, BF16: 1, F16: 2}[case.parameters]
    if weight is None and bias is None:
        parameter = 0
    lengths = case.options()['lengths']
    y, dx = undefined(x.shape, case.kind), undefined(x.shape, case.kind)
    mean, rstd = undefined((n, case.groups), F32), undefined((n, case.groups), F32)
    dweight, dbias = (None if t is None else undefined(t.shape, t.dtype) for t in (weight, bias))
    workspace = torch.empty(size.value, dtype=torch.uint8, device='cuda')
    activation = operators.ACTIVATIONS[case.activation]

    def step():
        workspace.fill_(0xFF)
        assert engine.lib.cpde_group_norm(engine.handle, code, at(x), c, p * c, n, p, c, case.groups, parameter, at(weight),
                                          at(bias), 1e-5, activation, at(lengths), case.rate, case.seed, case.offset, at(y),
                                          at(mean), at(rstd), at(workspace), size.value, LEGACY) == native.OK
        workspace.fill_(0xFF)
        assert engine.lib.cpde_group_norm_gradient(engine.handle, code, at(grad), c, p * c, at(x), c, p * c, at(mean), at(rstd),
                                                   n, p, c, case.groups, parameter, at(weight), at(bias), activation,
                                                   at(lengths), case.rate, case.seed, case.offset, at(dx), at(dweight),
                                                   at(dbias), at(workspace), size.value, LEGACY) == native.OK

    queued(step)
    check(case, x, grad, weight, bias, y, mean, rstd, dx, dweight, dbias)


@pytest.mark.parametrize('kind', [F32, BF16, F16])
@pytest.mark.parametrize('activation', ['linear', 'sigmoid', 'tanh', 'silu'])
@pytest.mark.parametrize('n,p,width,groups', [(2, 40, 16, 2), (3, 33, 24, 1), (2, 50, 4, 4), (3, 20, 2, 8), (2, 30, 3, 32),
                                              (1, 9000, 8, 2), (1, 9000, 2, 8)])
def test_every_type_with_dropout_and_lengths(engine, kind, activation, n, p, width, groups):
    """Vectors of eight and four channels, of one group and of several, in one pass over memory and in two."""
    case = Case(random.Random(4))
    case.n, case.p, case.width, case.groups, case.kind, case.parameters = n, p, width, groups, kind, F32
    case.activation, case.rate, case.lengths = activation, 0.5, [p - 3 * i for i in range(n)]
    case.with_weight = case.with_bias = True
    inputs = case.inputs(250)
    check(case, *inputs, *run(engine, case, *inputs))


@pytest.mark.parametrize('kind', [F32, BF16, F16])
@pytest.mark.parametrize('activation', ['linear', 'sigmoid', 'tanh', 'silu'])
@pytest.mark.parametrize('p,channels', [(1, 16), (1, 7), (9, 16), (9, 5), (3000, 8)])
def test_a_group_of_one_value_does_not_depend_on_it(engine, kind, activation, p, channels):
    """One channel a group and one point: xhat is 0, dx and dweight are exactly 0, and dbias is the gradient's sum."""
    case = Case(random.Random(5))
    case.n, case.p, case.width, case.groups, case.kind, case.parameters = 40, p, 1, channels, kind, F32
    case.activation, case.rate, case.lengths = activation, 0.1, None if p == 1 else [1] * 40
    case.with_weight = case.with_bias = True
    inputs = case.inputs(260)
    y, mean, rstd, dx, dweight, dbias = run(engine, case, *inputs)
    check(case, *inputs, y, mean, rstd, dx, dweight, dbias)
    assert torch.equal(mean, inputs[0][:, 0].float())
    assert not dx.any() and not dweight.any() and dbias.any()


@pytest.mark.parametrize('kind,parameters', [(F32, F32), (BF16, F32), (BF16, BF16)])
@pytest.mark.parametrize('n,p,c,groups', [(1, 30000, 64, 8), (1, 3000, 512, 8), (300, 33, 64, 16), (3, 5000, 96, 4), (70, 90, 192, 12),
                                          (2, 2000, 1024, 2), (1, 60000, 24, 8), (9, 700, 21, 7), (600, 3, 64, 64), (1, 1, 8, 2)])
def test_nothing_is_written_behind_the_workspace(engine, kind, parameters, n, p, c, groups):
    """The queried sizes, forward and gradient, and 64 KB behind them that stay as they were."""
    case = Case(random.Random(6))
    case.n, case.p, case.width, case.groups, case.kind, case.parameters = n, p, c // groups, groups, kind, parameters
    x, grad, weight, bias = case.inputs(270)
    code, parameter = {F32: 0, BF16: 1}[kind], {F32: 0, BF16: 1}[parameters]
    y, dx = torch.empty_like(x), torch.empty_like(x)
    mean, rstd = torch.empty((n, groups), device='cuda'), torch.empty((n, groups), device='cuda')
    dweight, dbias = torch.empty_like(weight), torch.empty_like(bias)
    size = ctypes.c_size_t()
    for query, entry, arguments in (
            (engine.lib.cpde_group_norm_forward_workspace, engine.lib.cpde_group_norm,
             lambda: (code, x.data_ptr(), c, p * c, n, p, c, groups, parameter, weight.data_ptr(), bias.data_ptr(), 1e-5, 3, None,
                      0.1, 1, 2, y.data_ptr(), mean.data_ptr(), rstd.data_ptr())),
            (engine.lib.cpde_group_norm_workspace, engine.lib.cpde_group_norm_gradient,
             lambda: (code, grad.data_ptr(), c, p * c, x.data_ptr(), c, p * c, mean.data_ptr(), rstd.data_ptr(), n, p, c, groups,
                      parameter, weight.data_ptr(), bias.data_ptr(), 3, None, 0.1, 1, 2, dx.data_ptr(), dweight.data_ptr(),
                      dbias.data_ptr()))):
        assert query(n, p, c, groups, ctypes.byref(size)) == native.OK
        workspace = torch.full((size.value + 65536,), 0xA5, dtype=torch.uint8, device='cuda')
        assert entry(engine.handle, *arguments(), workspace.data_ptr(), size.value, LEGACY) == native.OK
        assert bool((workspace[size.value:] == 0xA5).all())
    options = dict(activation='silu', rate=0.1, seed=1, offset=2)
    want, m, r = operators.group_norm(engine, x, groups, weight, bias, **options)
    assert torch.equal(y, want) and torch.equal(mean, m) and torch.equal(rstd, r)
    for got, want in zip((dx, dweight, dbias), operators.group_norm_gradient(engine, grad, x, m, r, groups, weight, bias, **options)):
        assert torch.equal(got, want)
