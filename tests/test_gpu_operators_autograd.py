"""The operators' functions beside torch's autograd, and which gradients the autograd functions return."""
import pytest

torch = pytest.importorskip('torch')

from cpde_b200 import native, operators  # noqa: E402
from test_gpu_operators import made  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def engine():
    torch.cuda.init()
    with native.Engine(0) as e:
        yield e


def calls(engine, requires):
    x, table, weight = made(1, 2, 6, 8), made(2, 5, 8), made(3, 8)
    ids = torch.tensor([0, 4, 2], device='cuda')
    mean, rstd = torch.zeros((2, 2), device='cuda'), torch.ones((2, 2), device='cuda')

    def g(t):
        return t.clone().requires_grad_(requires)

    return [lambda: operators.embedding(engine, g(table), ids),
            lambda: operators.embedding_gradient(engine, g(made(4, 3, 8)), ids, 5),
            lambda: operators.dropout(engine, g(x), 0.1, 1),
            lambda: operators.dropout(engine, x, 0.1, 1, residual=g(x)),
            lambda: operators.group_norm(engine, g(x), 2)[0],
            lambda: operators.group_norm(engine, x, 2, g(weight), weight)[0],
            lambda: operators.group_norm(engine, x, 2, weight, g(weight))[0],
            lambda: operators.group_norm_gradient(engine, g(x), x, mean, rstd, 2)[0]]


def test_functions_refuse_what_they_would_detach(engine):
    for call in calls(engine, True):
        with pytest.raises(ValueError, match='requires gradients'):
            call()


def test_functions_compute_values_without_recording(engine):
    want = [call() for call in calls(engine, False)]
    for record in (torch.no_grad, torch.inference_mode):
        with record():
            got = [call() for call in calls(engine, True)]
        for a, b in zip(got, want):
            assert torch.equal(a, b) and not a.requires_grad


def test_only_wanted_gradients(engine):
    x, residual = made(5, 4, 16), made(6, 4, 16).requires_grad_()
    operators.Dropout.apply(engine, x, 0.5, 1, 0, residual).sum().backward()
    assert x.grad is None and torch.equal(residual.grad, torch.ones_like(residual))
    x, residual = x.requires_grad_(), residual.detach()
    operators.Dropout.apply(engine, x, 0.5, 1, 0, residual).sum().backward()
    assert residual.grad is None
    assert torch.equal(x.grad, operators.dropout(engine, torch.ones_like(x.detach()), 0.5, 1))
    weight, bias = made(7, 16).requires_grad_(), made(8, 16)
    v = made(9, 2, 5, 16)
    operators.GroupNorm.apply(engine, v, weight, bias, 4).sum().backward()
    assert v.grad is None and bias.grad is None and weight.grad is not None
