"""Linear layers whose arrays pass 2^31 elements, and calls queued back to back."""
import pytest

torch = pytest.importorskip('torch')

import layer_oracle as oracle  # noqa: E402
from cpde_b200 import native, operators  # noqa: E402
from test_gpu_layers import BF16, F16, F32, made, same_bits, update, within  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def engine():
    torch.cuda.init()
    with native.Engine(0) as e:
        yield e


def ends(points):
    """Some rows at the start, around the 2^31st element and at the end."""
    return torch.cat([torch.arange(3), torch.arange(points // 2 - 2, points // 2 + 2), torch.arange(points - 3, points)])


@pytest.mark.parametrize('kind,inputs,outputs', [(BF16, 1024, 24), (BF16, 16, 1040), (F16, 1023, 3), (F32, 1000, 72)])
def test_offsets_beyond_31_bits(engine, kind, inputs, outputs):
    points = (1 << 31) // max(inputs, outputs) + 1000
    x = torch.empty((points, inputs), dtype=kind, device='cuda')
    block = made(1, 4096, inputs, dtype=kind)
    for at in range(0, points, 4096):
        x[at:at + 4096] = block[:points - at]
    x[-1] = made(2, inputs, dtype=kind)
    weight, bias = made(3, outputs, inputs, dtype=kind, scale=inputs ** -0.5), made(4, outputs, dtype=kind)
    y, _ = operators.linear(engine, x, weight, bias, 'tanh')
    at = ends(points).cuda()
    want, _, bound, _ = oracle.linear(x[at], weight, bias, 'tanh', None)
    within(y[at], want, bound)
    assert same_bits(y[4096:8192], y[:4096]) and same_bits(y[points // 4096 * 4096:-1], y[:points % 4096 - 1])
    del want, bound
    if kind == BF16:
        dx, dweight, _ = operators.linear_gradient(engine, y, x, weight)
        want = oracle.linear_gradient(y[at], x[at], weight, 'linear', None)[0]
        within(dx[at], *want)
        # The weight's gradient by blocks of points in 64 bits; a sum of so many terms is off by chain(points) at most.
        total, size = (torch.zeros((outputs, inputs), dtype=torch.float64, device='cuda') for _ in range(2))
        for a in range(0, points, 1 << 18):
            g, v = y[a:a + (1 << 18)].double(), x[a:a + (1 << 18)].double()
            total += g.mT @ v
            size += g.abs().mT @ v.abs()
        bound = oracle.chain(points, kind) * size
        within(dweight, total, bound + oracle.ROUNDING[kind] * (total.abs() + bound))


def test_queued_calls(engine):
    """Kernels begin beside the ones ahead of them: calls that follow each other without a wait give what they give alone."""
    sizes = [(3000, 512, 512), (1, 2048, 2048), (257, 48, 128), (65536, 128, 128), (500, 75, 33), (9000, 256, 8)]
    cases = [(kind, made(10 + i, p, c, dtype=kind), made(30 + i, o, c, dtype=kind, scale=c ** -0.5), made(50 + i, p, o, dtype=kind),
              update(70 + i, 20 + 40 * i, 300 - 40 * i, dtype=kind)) for i, (p, c, o) in enumerate(sizes) for kind in (F32, BF16)]

    def call(kind, x, weight, grad, matrix):
        y, z = operators.linear(engine, x, weight, None, 'silu', grad, True)
        return (y, z, *operators.linear_gradient(engine, y, x, weight, None, 'silu', z)[:2], operators.orthogonalize(engine, matrix))

    want = []
    for case in cases:
        want.append([t.clone() for t in call(*case)])
        torch.cuda.synchronize()
    for _ in range(3):
        got = [call(*case) for case in cases]
        for a, b in zip(got, want):
            assert all(same_bits(p, q) for p, q in zip(a, b))
