"""Group norm where a value that counts is not finite, or so large that sums of squares leave FP32: the statistics say so."""
import numpy as np
import pytest

torch = pytest.importorskip('torch')

import norm_bounds  # noqa: E402
from cpde_b200 import native, operators  # noqa: E402
from operator_oracle import wide  # noqa: E402
from test_gpu_operators import made  # noqa: E402

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
# One pass over memory in one CTA and in several, two passes in vectors and value by value.
SHAPES = [(2, 40, 64, 8), (2, 3000, 64, 8), (1, 40, 512, 2), (2, 40, 24, 8), (2, 40, 21, 7), (1, 9000, 24, 8), (1, 300000, 8, 2)]


@pytest.fixture(scope='module')
def engine():
    torch.cuda.init()
    with native.Engine(0) as e:
        yield e


def step(engine, x, grad, groups, weight, bias, lengths=None):
    y, mean, rstd = operators.group_norm(engine, x, groups, weight, bias, activation='silu', lengths=lengths)
    return y, mean, rstd, *operators.group_norm_gradient(engine, grad, x, mean, rstd, groups, weight, bias, activation='silu',
                                                         lengths=lengths)


@pytest.mark.parametrize('n,p,c,groups', SHAPES)
@pytest.mark.parametrize('kind', [F32, BF16, F16])
@pytest.mark.parametrize('value', [float('nan'), float('inf'), -float('inf')])
@pytest.mark.parametrize('place', ['first', 'second', 'middle', 'last'])
def test_a_value_that_is_not_finite(engine, n, p, c, groups, kind, value, place):
    """Its group's statistics and outputs are the definition's (an infinite mean, else NaN), all others what they were."""
    x, grad, weight, bias = made(300, n, p, c, dtype=kind), made(301, n, p, c, dtype=kind), made(302, c), made(303, c)
    before = step(engine, x, grad, groups, weight, bias)
    width, group = c // groups, groups - 1
    point, channel = {'first': (0, 0), 'second': (0, 1), 'middle': (p // 2, width // 2), 'last': (p - 1, width - 1)}[place]
    x[n - 1, point, group * width + channel] = value
    y, mean, rstd, dx, dweight, dbias = after = step(engine, x, grad, groups, weight, bias)
    hit = torch.zeros((n, groups), dtype=torch.bool, device='cuda')
    hit[n - 1, group] = True
    assert torch.equal(torch.isnan(rstd), hit)
    if np.isnan(value):
        assert torch.equal(torch.isnan(mean), hit)
    else:
        assert float(mean[n - 1, group]) == value and int(torch.isfinite(mean).sum()) == n * groups - 1
    values = hit[:, None, :, None].expand(n, p, groups, width).reshape(n, p, c)
    for t in (y, dx):
        assert torch.equal(torch.isnan(t), values)
    channels = hit.any(0)[:, None].expand(groups, width).reshape(c)
    for t in (dweight, dbias):
        assert torch.equal(torch.isnan(t), channels)
    for t, was, where in zip(after, before, (values, hit, hit, values, channels, channels)):
        assert torch.equal(t[~where], was[~where])


@pytest.mark.parametrize('n,p,c,groups', SHAPES)
def test_infinities_of_both_signs(engine, n, p, c, groups):
    x = made(304, n, p, c)
    x[0, 0, 0], x[0, p - 1, 0] = float('inf'), -float('inf')
    _, mean, rstd = operators.group_norm(engine, x, groups)
    assert torch.isnan(mean[0, 0]) and torch.isnan(rstd[0, 0])
    assert torch.isfinite(mean.reshape(-1)[1:]).all() and torch.isfinite(rstd.reshape(-1)[1:]).all()


@pytest.mark.parametrize('n,p,c,groups', SHAPES)
@pytest.mark.parametrize('scale', [1e15, 1e17, 5e17, 1e18, 2e18, 5e18, 1e19, 1e20, 3e37])
@pytest.mark.parametrize('kind', [F32, BF16])
def test_values_whose_squares_overflow(engine, n, p, c, groups, scale, kind):
    """Right as far as the squares' sum stays within FP32 with room to spare; beyond, rstd is right, zero or NaN. It is never
    the 1 / sqrt(eps) of a group without variance."""
    x = (made(305, n, p, c) * scale).to(kind)
    y, mean, rstd = operators.group_norm(engine, x, groups)
    norm = norm_bounds.Norm(wide(x), groups, None, None, 1e-5, 'linear', None, 0.0, 0, 0)
    want_mean, want, off_mean, off = norm.statistics()
    got = wide(rstd)
    # Deviations are from a value of the group: no more than twice the largest.
    far = 2 * abs(norm.x).max((1, 3))
    safe = norm.values * far ** 2 < 3e38
    assert (abs(got - want) <= off)[safe].all()
    assert (abs(wide(mean) - want_mean) <= off_mean)[safe].all()
    assert ((abs(got - want) <= off) | (got == 0) | np.isnan(got)).all()
    if scale <= 1e15:
        assert safe.all()


@pytest.mark.parametrize('value', [float('nan'), float('inf')])
def test_behind_the_length_it_does_not_count(engine, value):
    lengths = torch.tensor([30, 0], dtype=torch.int32, device='cuda')
    x, grad = made(306, 2, 40, 64), made(307, 2, 40, 64)
    before = step(engine, x, grad, 8, None, None, lengths)
    x[0, 30:], x[1] = value, value
    for a, b in zip(step(engine, x, grad, 8, None, None, lengths), before):
        assert (a is None and b is None) or torch.equal(a, b)


@pytest.mark.parametrize('n,p,c,groups', [(2, 50, 16, 2), (2, 3000, 16, 2), (2, 40000, 16, 2), (3, 700, 21, 7), (1, 9000, 24, 8)])
@pytest.mark.parametrize('level,outlier', [(1000.0, 0.0), (1000.0, 3000.0), (-300.0, 0.0)])
@pytest.mark.parametrize('activation', ['linear', 'silu'])
def test_level_far_above_the_spread(engine, n, p, c, groups, level, outlier, activation):
    """The gradient against the formula with the kernel's own statistics, so that their error does not widen its bound; a first
    point that is not like the others is what the deviations are taken from."""
    x, grad = level + made(310, n, p, c), 1 + made(311, n, p, c)
    x[:, 0] += outlier
    weight, bias = 1 + 0.3 * made(312, c), 0.3 * made(313, c)
    y, mean, rstd = operators.group_norm(engine, x, groups, weight, bias, activation=activation)
    parts = operators.group_norm_gradient(engine, grad, x, mean, rstd, groups, weight, bias, activation=activation)
    norm = norm_bounds.Norm(wide(x), groups, wide(weight), wide(bias), 1e-5, activation, None, 0.0, 0, 0)
    want, want_rstd, off, off_rstd = norm.statistics()
    assert (abs(wide(mean) - want) <= off).all() and (abs(wide(rstd) - want_rstd) <= off_rstd).all()
    u = 2.0 ** -24
    want, bound = norm.forward(wide(mean), wide(rstd), u, 2.0 ** -150)
    assert (abs(wide(y) - want) <= bound).all()
    for got, (want, bound) in zip(parts, norm.gradient(wide(grad), wide(mean), wide(rstd), u, 2.0 ** -150)):
        assert np.linalg.norm(bound) < 0.05 * np.linalg.norm(want)  # the bound can fail
        assert (abs(wide(got) - want) <= bound + u * abs(want)).all()


def test_eps_is_positive_in_fp32(engine):
    """1e-60 is zero in FP32, in which the kernels add it: groups without variance would be NaN."""
    x = torch.full((2, 40, 64), 2.5, device='cuda')
    for eps in (1e-60, 1e-46, 0.0, -1.0):
        with pytest.raises(native.EngineError, match='eps') as error:
            operators.group_norm(engine, x, 8, eps=eps)
        assert error.value.status == native.REJECTED
    for shape in (x, x[:, :, :21]):
        y, _, rstd = operators.group_norm(engine, shape, 1, eps=1e-40)
        assert not y.any() and torch.allclose(rstd.double(), torch.full_like(rstd, 1e20).double(), rtol=1e-4)
