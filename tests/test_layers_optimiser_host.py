"""The optimiser's state without a GPU."""
import copy

import pytest

torch = pytest.importorskip('torch')

from cpde_b200 import operators  # noqa: E402


@pytest.mark.parametrize('kind', [torch.float32, torch.bfloat16, torch.float16])
def test_momentum_is_loaded_as_it_was_saved(kind):
    """In float32, as memory of its own, for the parameters that had one."""
    shapes = [(3, 4), (5, 2), (4, 4)]

    def made():
        ps = [torch.nn.Parameter(torch.zeros(s, dtype=kind)) for s in shapes]
        return operators.Muon(None, [{'params': ps[:2]}, {'params': ps[2:], 'lr': 0.5}]), ps

    a, ps = made()
    for i in (0, 2):
        a.state[ps[i]]['momentum'] = torch.randn(shapes[i]) * 1e-9
    saved = copy.deepcopy(a.state_dict())
    b, qs = made()
    b.load_state_dict(saved)
    assert b.param_groups[1]['lr'] == 0.5
    for i in (0, 2):
        got = b.state[qs[i]]['momentum']
        assert got.dtype == torch.float32 and torch.equal(got, a.state[ps[i]]['momentum'])
        assert got.data_ptr() != saved['state'][i]['momentum'].data_ptr()
    assert 'momentum' not in b.state[qs[1]]
    # A state in the parameters' type.
    saved['state'][0]['momentum'] = saved['state'][0]['momentum'].to(torch.bfloat16)
    b.load_state_dict(saved)
    assert b.state[qs[0]]['momentum'].dtype == torch.float32
    assert torch.equal(b.state[qs[0]]['momentum'], saved['state'][0]['momentum'].float())
