"""The bound in norm of FP32 products (NORM in test_gpu_layers_routes) against emulated products of BF16 parts, without a GPU: three
parts stay below it and two do not."""
import pytest

torch = pytest.importorskip('torch')

from test_gpu_layers_routes import NORM  # noqa: E402


def parts(v, count):
    out = []
    for _ in range(count):
        out.append(v.to(torch.bfloat16).to(torch.float32))
        v = v - out[-1]
    return out


def product(x, w, count):
    """The products of parts that are not below the last part's own rounding, in FP32 sums of 64 terms that are added in FP32."""
    xs, ws = parts(x, count), parts(w, count)
    total = torch.zeros(x.shape[0], w.shape[0])
    for k in range(0, x.shape[1], 64):
        for i in reversed(range(count)):
            for j in range(count - i):
                total = total + xs[i][:, k:k + 64] @ ws[j][:, k:k + 64].t()
    return total


@pytest.mark.parametrize('points,inputs,outputs', [(129, 65, 257), (300, 2000, 100), (200, 128, 128), (40, 4096, 64), (100, 16, 8)])
def test_two_parts_are_seen_in_norm(points, inputs, outputs):
    torch.manual_seed(0)
    x, w = torch.randn(points, inputs), torch.randn(outputs, inputs) * inputs ** -0.5
    want = x.double() @ w.double().t()
    off = [float((product(x, w, count) - want).norm() / want.norm()) for count in (2, 3)]
    assert off[1] <= 0.5 * NORM and off[0] >= 2 * NORM, off
