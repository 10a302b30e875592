"""Arguments that the layer operators' Python functions refuse or take in several forms, without a GPU."""
import pytest

torch = pytest.importorskip('torch')

from cpde_b200 import operators  # noqa: E402


class Device:
    device = 0


@pytest.mark.parametrize('shape', [(), (5,), (5, 0), (0, 5), (2, 3, 4)])
def test_muon_refuses_what_is_no_matrix(shape):
    x = torch.zeros(shape)
    with pytest.raises(ValueError, match='shape'):
        operators.muon(Device, x, x, x, 0.1)


@pytest.mark.parametrize('bad', [(), [], [()], None, 1.0, (1.0, 2.0), (1.0, 2.0, 3.0, 4.0), [(1.0, 2.0)] * 3, [(1.0, 2.0), (1.0, 2.0, 3.0, 4.0)],
                                 [1.0, (1.0, 2.0, 3.0)], [(1.0, 2.0, 3.0), 1.0], ('a', 'b', 'c'), [('a', 'b', 'c')], (None, None, None)])
def test_coefficients_are_triples(bad):
    with pytest.raises(ValueError, match='triples'):
        operators._coefficients(bad)


def test_coefficients_of_any_sequence():
    numpy = pytest.importorskip('numpy')
    one, two = (1.5, -0.5, 0.0), (2, -1, 0.5)
    assert operators._coefficients(one) == one and operators._coefficients(list(one)) == one
    assert operators._coefficients([one, two]) == one + two == operators._coefficients(one + two)
    assert operators._coefficients(numpy.array(one)) == one == operators._coefficients(numpy.float32(one))
    assert operators._coefficients(numpy.array([one, two])) == one + two
