"""Group norm of as many points as a call may have."""
import pytest

torch = pytest.importorskip('torch')

from cpde_b200 import native, operators  # noqa: E402
from operator_oracle import EPS, ROUNDING  # noqa: E402

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
MOST = 2 ** 31 - 2
CHUNK = 1 << 26


@pytest.fixture(scope='module')
def engine():
    torch.cuda.init()
    with native.Engine(0) as e:
        yield e
    torch.cuda.empty_cache()


def filled(seed, points):
    g = torch.Generator(device='cuda').manual_seed(seed)
    t = torch.empty(points, dtype=BF16, device='cuda')
    for part in t.split(CHUNK):
        part.copy_(0.5 + torch.randn(len(part), generator=g, device='cuda'))
    return t


def chunks(*arrays):
    return zip(*(a.split(CHUNK) for a in arrays))


@pytest.mark.parametrize('length', [None, MOST - 16384, MOST - 300])
def test_most_points(engine, length):
    """One channel of 2^31 - 2 points. The longest chain of additions has 512 points of a thread, 256 threads and 512 joined
    blocks: 1280 e of the terms."""
    x, grad = filled(1, MOST), filled(2, MOST)
    count = length or MOST
    lengths = None if length is None else torch.tensor([length], dtype=torch.int32, device='cuda')
    weight, bias = torch.full((1,), 1.5, device='cuda'), torch.full((1,), -0.25, device='cuda')
    y, mean, rstd = operators.group_norm(engine, x.view(1, -1, 1), 1, weight, bias, lengths=lengths)
    dx, dweight, dbias = operators.group_norm_gradient(engine, grad.view(1, -1, 1), x.view(1, -1, 1), mean, rstd, 1, weight,
                                                       bias, lengths=lengths)
    y, dx = y.view(-1), dx.view(-1)
    m = sum(p.double().sum() for p in x[:count].split(CHUNK)) / count
    v = sum((p.double() - m).square().sum() for p in x[:count].split(CHUNK)) / count
    chain, far = 1280 * EPS, 16.0
    assert abs(mean.double() - m).item() <= chain * far
    assert abs(rstd.double() * (v + 1e-5).sqrt() - 1).item() <= chain * far
    m, r = mean.double().view(()), rstd.double().view(())
    sums = [0.0, 0.0, 0.0]
    for px, pg in chunks(x[:count], grad[:count]):
        g, xhat = pg.double(), (px.double() - m) * r
        for i, t in enumerate((g, g * xhat, (g * xhat).abs())):
            sums[i] = sums[i] + t.sum()
    assert abs(dbias.double() - sums[0]).item() <= chain * 2 * count
    assert abs(dweight.double() - sums[1]).item() <= chain * 2 * float(sums[2])
    m1, m2 = 1.5 * sums[0] / count, 1.5 * sums[1] / count
    u = ROUNDING[BF16]
    for px, pg, py, pd in chunks(x[:count], grad[:count], y[:count], dx[:count]):
        xhat = (px.double() - m) * r
        want = 1.5 * xhat - 0.25
        assert bool(((py.double() - want).abs() <= u * want.abs() + 16 * EPS * (1 + xhat.abs())).all())
        want = r * (1.5 * pg.double() - m1 - xhat * m2)
        assert bool(((pd.double() - want).abs() <= u * want.abs() + 4 * chain * (1 + xhat.abs())).all())
    assert not y[count:].any() and not dx[count:].any()
