"""The autograd function of linear layers with the operators' functions replaced by torch forms, without a GPU."""
import pytest

torch = pytest.importorskip('torch')

import layer_oracle as oracle  # noqa: E402
from cpde_b200 import operators  # noqa: E402


@pytest.fixture
def plain(monkeypatch):
    """The two functions in 64 bits, by the formulas."""
    def linear(engine, x, weight, bias=None, activation='linear', residual=None, keep=False):
        z = x @ weight.t() if bias is None else x @ weight.t() + bias
        y = oracle.ACTIVATIONS[activation](z)
        return (y if residual is None else y + residual), z if keep else None

    def linear_gradient(engine, grad, x, weight, bias=None, activation='linear', z=None, need=(True, True), dtype=None):
        assert activation == 'linear' or z is not None
        dz = grad if activation == 'linear' else grad * oracle.slope(z, activation)
        flat = dz.reshape(-1, dz.shape[-1])
        return (dz @ weight if need[0] else None, flat.t() @ x.reshape(-1, x.shape[-1]) if need[1] else None,
                flat.sum(0) if bias is not None else None)

    monkeypatch.setattr(operators, 'linear', linear)
    monkeypatch.setattr(operators, 'linear_gradient', linear_gradient)


@pytest.mark.parametrize('count', [2, 3, 4, 5])
@pytest.mark.parametrize('bias', [True, False])
def test_arguments_may_be_left_out(plain, count, bias):
    """Backward after a forward of x and the weight alone, and with each further argument."""
    torch.manual_seed(0)
    d = torch.float64
    x, weight, b, r, grad = (torch.randn(s, dtype=d) for s in ((2, 5, 3), (4, 3), (4,), (2, 5, 4), (2, 5, 4)))
    arguments = [x, weight, b if bias else None, 'tanh', r][:count]
    for wanted in range(count):
        if not isinstance(arguments[wanted], torch.Tensor):
            continue
        leaves = [t.clone().requires_grad_(wanted in (i, 0)) if isinstance(t, torch.Tensor) else t for i, t in enumerate(arguments)]
        twins = [t.detach().clone().requires_grad_(t.requires_grad) if isinstance(t, torch.Tensor) else t for t in leaves]
        operators.Linear.apply(None, *leaves).backward(grad)
        tx, tw, tb, ta, tr = twins + [None, 'linear', None][count - 2:]
        z = tx @ tw.t() if tb is None else tx @ tw.t() + tb
        y = oracle.ACTIVATIONS[ta](z)
        (y if tr is None else y + tr).backward(grad)
        for a, t in zip(leaves, twins):
            if isinstance(a, torch.Tensor):
                assert (a.grad is None) == (t.grad is None)
                assert a.grad is None or torch.allclose(a.grad, t.grad, rtol=1e-12, atol=1e-12)
