"""The layer operators without a GPU: workspace sizes, refusals, and the oracle's own formulas."""
import ctypes

import pytest

from cpde_b200 import native

torch = pytest.importorskip('torch')

import layer_oracle as oracle  # noqa: E402


def test_workspace_sizes():
    lib, size = native.load(), ctypes.c_size_t()
    x, w = 1 << 20, 1 << 30  # addresses that nothing reads
    for kind in (0, 1, 2):
        assert lib.cpde_linear_workspace(kind, x, 64, 1000, 64, 32, w, 64, ctypes.byref(size)) == native.OK
        assert lib.cpde_linear_workspace(kind, x, 64, 0, 64, 32, w, 64, ctypes.byref(size)) == native.OK and size.value == 0
    # Wide layers: three BF16 parts of FP32; 16-bit rows in whole 16 bytes need nothing, others a copy. Narrow ones are
    # gathered from the arrays.
    assert lib.cpde_linear_workspace(0, x, 2048, 30000, 2048, 2048, w, 2048, ctypes.byref(size)) == native.OK
    assert size.value >= 30000 * 2048 * 6
    assert lib.cpde_linear_workspace(1, x, 2048, 30000, 2048, 2048, w, 2048, ctypes.byref(size)) == native.OK
    assert size.value == 0
    assert lib.cpde_linear_workspace(1, x + 2, 2048, 30000, 2048, 2048, w, 2048, ctypes.byref(size)) == native.OK
    assert size.value >= 30000 * 2048 * 2
    assert lib.cpde_linear_workspace(0, x, 128, 100000, 128, 128, w, 128, ctypes.byref(size)) == native.OK
    assert size.value == 0
    for bad in ((3, 10, 8, 8), (0, -1, 8, 8), (0, 1 << 31, 8, 8), (0, 10, 0, 8), (0, 10, 8, 0), (0, 10, (1 << 20) + 1, 8),
                (0, (1 << 31) - 511, 8, 8), (0, 10, 8, (1 << 20) + 1)):
        kind, points, inputs, outputs = bad
        assert lib.cpde_linear_workspace(kind, x, 8, points, inputs, outputs, w, 8, ctypes.byref(size)) == native.REJECTED
        assert lib.cpde_linear_gradient_workspace(kind, x, 8, 1, x, 8, points, inputs, outputs, w, 8, 7,
                                                  ctypes.byref(size)) == native.REJECTED
    assert lib.cpde_linear_gradient_workspace(1, x, 64, 4, x, 64, 10, 64, 64, w, 64, 7, ctypes.byref(size)) == native.REJECTED
    # X twice in two parts, and a step's update in FP32; a matrix that one CTA holds needs nothing.
    assert lib.cpde_orthogonalize_workspace(0, 3, 300, 400, ctypes.byref(size)) == native.OK and size.value > 3 * 300 * 400 * 8
    assert lib.cpde_muon_workspace(0, 300, 400, ctypes.byref(size)) == native.OK and size.value > 300 * 400 * 12
    assert lib.cpde_orthogonalize_workspace(0, 3, 100, 50, ctypes.byref(size)) == native.OK and size.value == 0
    for bad in ((3, 1, 5, 5), (0, -1, 5, 5), (0, 65536, 5, 5), (0, 1, 0, 5), (0, 1, 5, 0), (0, 1, 5, (1 << 20) + 1)):
        assert lib.cpde_orthogonalize_workspace(*bad, ctypes.byref(size)) == native.REJECTED
    for bad in ((3, 5, 5), (0, 0, 5), (0, 5, -1)):
        assert lib.cpde_muon_workspace(*bad, ctypes.byref(size)) == native.REJECTED
    assert lib.cpde_muon_workspace(0, 5, 5, None) == native.REJECTED


def test_no_engine_is_refused():
    lib = native.load()
    assert lib.cpde_linear(None, 0, None, 1, 1, 1, 1, None, 1, 0, None, 1, None, 0, None, None, None, 0, None) == native.REJECTED
    assert lib.cpde_muon(None, 0, None, None, 0, None, 1, 1, 0.1, 0.9, 1, 0.0, 1.0, 5, None, 1, 1e-7, None, None, None, 0,
                         None) == native.REJECTED


def test_tensors_off_the_engines_device_are_refused():
    from cpde_b200 import operators

    class Device:
        device = 0

    x = torch.zeros(3, 4)
    for call in (lambda: operators.linear(Device, x, x), lambda: operators.linear_gradient(Device, x[:, :3], x, x),
                 lambda: operators.orthogonalize(Device, x), lambda: operators.muon(Device, x, x, x, 0.1)):
        with pytest.raises(ValueError, match='device'):
            call()


def test_optimiser_takes_matrices():
    from cpde_b200 import operators
    with pytest.raises(ValueError, match='matrices'):
        operators.Muon(None, [torch.nn.Parameter(torch.zeros(5))])


def test_oracle_gradient_is_autograds():
    torch.manual_seed(0)
    x, weight, bias, grad = (torch.randn(s, dtype=torch.float64) for s in ((9, 5), (7, 5), (7,), (9, 7)))
    for activation in oracle.ACTIVATIONS:
        leaves = [t.clone().requires_grad_() for t in (x, weight, bias)]
        z = leaves[0] @ leaves[1].t() + leaves[2]
        want = torch.autograd.grad(oracle.ACTIVATIONS[activation](z), leaves, grad)
        oracle.ROUNDING[torch.float64] = oracle.TINY[torch.float64] = 0.0
        got = oracle.linear_gradient(grad, x, weight, activation, z.detach())
        for (value, _), part in zip(got, want):
            assert torch.allclose(value, part, rtol=1e-12, atol=1e-12)


def test_oracle_orthogonalizes():
    """Singular vectors stay, singular values go through the polynomial; steps of a convergent one end at an orthogonal
    matrix."""
    torch.manual_seed(1)
    for shape in ((6, 9), (9, 6)):
        x = torch.randn(shape, dtype=torch.float64)
        u, s, v = torch.linalg.svd(x, full_matrices=False)
        t = s / s.norm()
        for _ in range(5):
            a, b, c = oracle.QUINTIC
            t = a * t + b * t ** 3 + c * t ** 5
        assert torch.allclose(oracle.orthogonalize(x, eps=0.0), u @ torch.diag(t) @ v, atol=1e-10)
        whole = oracle.orthogonalize(x, steps=40, coefficients=(1.5, -0.5, 0.0))
        assert torch.allclose(whole, u @ v, atol=1e-8)
