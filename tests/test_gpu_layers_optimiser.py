"""The optimiser class on weights of every type over dozens of steps."""
import copy

import pytest

torch = pytest.importorskip('torch')

import layer_oracle as oracle  # noqa: E402
from cpde_b200 import native, operators  # noqa: E402
from test_gpu_layers import F32, KINDS, made, same_bits, update, within  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def engine():
    torch.cuda.init()
    with native.Engine(0) as e:
        yield e


@pytest.mark.parametrize('kind', KINDS)
@pytest.mark.parametrize('shape', [(24, 40), (300, 515)])
@pytest.mark.parametrize('size', [1.0, 1e-6])
def test_momentum_of_many_steps(engine, kind, shape, size):
    """Against the running mean in 64 bits: each step rounds it by some 2^-24 of what it adds up. The gradients of a step differ from
    the mean by little, and at 1e-6 a twentieth of one is below the smallest number of float16."""
    p = torch.nn.Parameter(made(1, *shape, dtype=kind))
    optimiser = operators.Muon(engine, [p], lr=0.02)
    base, m, most = update(2, *shape, scale=size), torch.zeros(shape, dtype=torch.float64, device='cuda'), 0.0
    for step in range(40):
        p.grad = (base * (1 + 0.01 * step) + update(5 + step, *shape, scale=0.01 * size)).to(kind)
        before = p.detach().clone()
        optimiser.step()
        m = 0.95 * m + 0.05 * p.grad.double()
        most = max(most, float(p.grad.abs().max()))
        state = optimiser.state[p]['momentum']
        assert state.dtype == F32
        within(state, m, torch.full_like(m, 8 * (step + 1) * oracle.E * most))
        if step in (0, 39):
            u = 0.95 * m + 0.05 * p.grad.double()
            want = oracle.orthogonalize(u)
            off = (oracle.orthogonalize_modelled(u, kind, step=True) - want).norm()
            rate = 0.02 * max(1.0, shape[0] / shape[1]) ** 0.5
            # Two roundings of 2^-24 a step leave 40 of them in the running mean. A step's polynomial multiplies an error of X, whose
            # norm is one, by its first coefficient at most.
            amplified = 40 * oracle.E * oracle.QUINTIC[0] ** 5
            bound = rate * (8 * off + amplified + 2.0 ** -20 * want.norm()) + (oracle.ROUNDING[kind] + 4 * oracle.E) * before.double().norm()
            assert (p.detach().double() - (before.double() - rate * want)).norm() <= bound


@pytest.mark.parametrize('kind', KINDS)
def test_a_loaded_state_goes_on_as_the_saved_one(engine, kind):
    def made_with(weight):
        p = torch.nn.Parameter(weight.clone())
        return p, operators.Muon(engine, [p], lr=0.1)

    p, a = made_with(made(60, 30, 20, dtype=kind))
    for step in range(3):
        p.grad = update(61 + step, 30, 20, dtype=kind)
        a.step()
    q, b = made_with(p.detach())
    b.load_state_dict(copy.deepcopy(a.state_dict()))
    for step in range(3):
        p.grad = q.grad = update(70 + step, 30, 20, dtype=kind)
        a.step(), b.step()
        assert same_bits(p.detach(), q.detach()) and same_bits(a.state[p]['momentum'], b.state[q]['momentum'])


def test_steps_are_not_cut_to_32_bits(engine):
    x = made(80, 8, 8)
    for steps in ((1 << 32) + 5, -(1 << 32) + 5, 65, 0):
        for call in (lambda: operators.orthogonalize(engine, x, steps=steps), lambda: operators.muon(engine, x, x, x, 0.1, steps=steps)):
            with pytest.raises((ValueError, native.EngineError), match='steps'):
                call()
