"""Layers large enough for the tensor cores' tiles: arrays that TMA reads, arrays that become parts, and rows that are gathered,
each at odd sizes, layouts, types of parameters and values, against 64-bit forms (layer_oracle)."""
import pytest

torch = pytest.importorskip('torch')

from cpde_b200 import native  # noqa: E402
from test_gpu_layers import ACTIVATIONS, KINDS, check_gradient, check_linear, made  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def engine():
    torch.cuda.init()
    with native.Engine(0) as e:
        yield e


@pytest.mark.parametrize('kind', KINDS)
@pytest.mark.parametrize('activation', ACTIVATIONS)
@pytest.mark.parametrize('points,inputs,outputs', [(1500, 200, 600), (1501, 264, 603), (1029, 1030, 130)])
def test_ragged_tiles(engine, kind, activation, points, inputs, outputs):
    """Tiles whose warps have lanes behind the last row and columns behind the last one, and functions with branches."""
    x, weight = made(1, points, inputs, dtype=kind), made(2, outputs, inputs, dtype=kind, scale=2 * inputs ** -0.5)
    bias, residual = made(3, outputs, dtype=kind), made(4, points, outputs, dtype=kind)
    _, z = check_linear(engine, x, weight, bias, activation, residual)
    check_gradient(engine, made(5, points, outputs, dtype=kind), x, weight, bias, activation, None if activation == 'linear' else z)
