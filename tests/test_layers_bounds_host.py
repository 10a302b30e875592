"""The bound in norm of FP32 products (NORM in test_gpu_layers_routes) against emulated products of BF16 parts, without a GPU: three
parts stay below it and two do not."""
import pytest

torch = pytest.importorskip('torch')

from test_gpu_layers_routes import NORM  # noqa: E402


def test_gradient_workspace_is_enough_for_both_types():
    """Without a word about the type of dweight the query covers both."""
    import ctypes

    from cpde_b200 import native
    lib, size = native.load(), ctypes.c_size_t()
    sizes = {}
    for want in (2, 2 + 8, 7, 7 + 8):
        assert lib.cpde_linear_gradient_workspace(1, 1 << 20, 2048, 3, 1 << 30, 2048, 30000, 2048, 2048, 1 << 35, 2048, want,
                                                  ctypes.byref(size)) == native.OK
        sizes[want] = size.value
    assert sizes[2] >= sizes[2 + 8] + 30000 * 2048 * 2 and sizes[7] >= sizes[7 + 8] + 30000 * 2048 * 2


def test_gradient_workspace_of_any_size_is_enough_for_both_types():
    """Contractions of different lengths are split differently, so that either type may need more for its partial sums."""
    import ctypes
    import random

    from cpde_b200 import native
    lib, size, rng = native.load(), ctypes.c_size_t(), random.Random(0)

    def query(points, inputs, outputs, kind, activation, want):
        assert lib.cpde_linear_gradient_workspace(kind, 1 << 20, outputs, activation, 1 << 30, inputs, points, inputs, outputs, 1 << 35,
                                                  inputs, want, ctypes.byref(size)) == native.OK
        return size.value

    for _ in range(20000):
        shape = [int(2 ** rng.uniform(0, top)) for top in (20, 13, 13)]
        kind, activation, want = rng.choice((0, 1, 2)), rng.choice((1, 3)), rng.choice((2, 3, 6, 7))
        assert query(*shape, kind, activation, want) >= query(*shape, kind, activation, want + 8), (shape, kind, activation, want)


def test_blocks_of_small_layers_go_through_few_slabs():
    """Layers whose blocks would go through many slabs in turn, or come in many waves, take the tensor cores' tiles, which need a
    workspace for FP32 arrays; small ones take blocks, which need none."""
    import ctypes

    from cpde_b200 import native
    lib, size = native.load(), ctypes.c_size_t()

    def forward(points, inputs, outputs):
        assert lib.cpde_linear_workspace(0, 1 << 20, inputs, points, inputs, outputs, 1 << 35, inputs, ctypes.byref(size)) == native.OK
        return size.value

    def gradient(points, inputs, outputs, kind=0):
        assert lib.cpde_linear_gradient_workspace(kind, 1 << 20, outputs, 3, 1 << 30, inputs, points, inputs, outputs, 1 << 35, inputs, 7,
                                                  ctypes.byref(size)) == native.OK
        return size.value

    assert not any(forward(*s) for s in ((257, 48, 128), (1000, 64, 64), (256, 256, 256), (40, 10, 10)))
    assert all(forward(*s) for s in ((1440, 64, 1440), (1000, 128, 1024), (352, 1024, 352), (700, 256, 256)))
    for kind in (0, 1, 2):
        assert not any(gradient(*s, kind) for s in ((300, 100, 77), (60, 64, 64), (256, 256, 256)))
        assert all(gradient(*s, kind) for s in ((1000, 100, 77), (1024, 40, 16), (1025, 40, 16), (512, 256, 256)))


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
