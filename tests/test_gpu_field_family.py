"""The operators and the engine together, as examples/field_family.py uses them."""
import sys
from pathlib import Path

import pytest

torch = pytest.importorskip('torch')

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / 'examples'))

pytestmark = pytest.mark.gpu


def test_family_is_learned_and_has_a_spread():
    import field_family
    losses, spread = field_family.main(['--points', '96', '--epochs', '60', '--steps', '120', '--masks', '8'])
    assert losses[-1] < 0.2 * losses[0]
    assert torch.isfinite(spread).all() and (spread > 0).any()
    again, _ = field_family.main(['--points', '96', '--epochs', '60', '--steps', '3', '--masks', '2'])
    assert again[0] == losses[0]  # same seeds, same masks, same bits
