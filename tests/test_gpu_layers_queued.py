"""Kernels that hold tensor memory, queued behind each other so that each may begin before the one ahead has ended."""
import pytest

torch = pytest.importorskip('torch')

from cpde_b200 import native, operators  # noqa: E402
from test_gpu_layers import BF16, F16, F32, made, same_bits, update  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def engine():
    torch.cuda.init()
    with native.Engine(0) as e:
        yield e


@pytest.mark.parametrize('streams', [1, 3])
def test_small_matrices_between_products(engine, streams):
    """Matrices of one launch, fewer and more than the GPU's multiprocessors, with the tiles of products between them."""
    matrices = [update(1 + i, n, r, c, dtype=kind) for i, (n, r, c, kind) in enumerate(
        ((700, 24, 40, F32), (1, 5, 3, BF16), (150, 128, 250, F16), (300, 16, 16, BF16), (40, 128, 128, F32)))]
    layers = [(made(20 + i, p, c, dtype=kind), made(30 + i, o, c, dtype=kind, scale=c ** -0.5)) for i, (p, c, o, kind) in enumerate(
        ((3000, 512, 512, BF16), (20001, 100, 77, F32), (1500, 264, 600, F32), (9000, 1000, 64, F16), (300, 64, 2000, BF16)))]

    def call():
        out = []
        for x, (a, w) in zip(matrices, layers):
            out += [operators.orthogonalize(engine, x), operators.orthogonalize(engine, x, steps=2),
                    operators.linear(engine, a, w)[0], operators.orthogonalize(engine, x[:1])]
        return out

    want = []
    for x, (a, w) in zip(matrices, layers):
        for one in (lambda: operators.orthogonalize(engine, x), lambda: operators.orthogonalize(engine, x, steps=2),
                    lambda: operators.linear(engine, a, w)[0], lambda: operators.orthogonalize(engine, x[:1])):
            want.append(one())
            torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for _ in range(streams):
            with torch.cuda.stream(torch.cuda.Stream()):
                got.append(call())
        torch.cuda.synchronize()
        for outputs in got:
            assert all(same_bits(a, b) for a, b in zip(outputs, want))
