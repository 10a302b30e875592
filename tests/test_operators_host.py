"""Device-tensor operators without a GPU: the oracle's generator, workspace sizes, refusals."""
import ctypes

import numpy as np
import pytest

import operator_oracle as oracle
from cpde_b200 import native

torch = pytest.importorskip('torch')


def test_oracle_generator_known_answers():
    """Published test vectors of Philox4x32-10 (Salmon et al., 2011)."""
    ones = (1 << 64) - 1
    assert [f'{w:08x}' for w in oracle.philox([0], 0, 0)[0]] == ['6627e8d5', 'e169c58d', 'bc57ac4c', '9b00dbd8']
    assert [f'{w:08x}' for w in oracle.philox([ones], ones, ones)[0]] == ['408f276d', '41c83b0e', 'a20bc7c6',
                                                                          '6d5451fd']


def test_oracle_mask_has_the_rate():
    keep, factor = oracle.kept(200000, 0.1, 12, 13)
    assert abs(keep.mean() * factor - 1) < 5 * np.sqrt(0.1 / 0.9 / keep.size)


def test_oracle_gradient_against_differences():
    """Central differences in 64 bits: truncation 1e-8 of the scale."""
    rng = np.random.default_rng(3)
    x, w, b, grad = rng.normal(size=(3, 7, 12)), rng.normal(size=12), rng.normal(size=12), rng.normal(size=(3, 7, 12))
    for activation in ('linear', 'sigmoid', 'tanh', 'silu'):
        def loss(x, w, b):
            return (oracle.group_norm(x, 3, w, b, 1e-5, activation, [7, 0, 4], 0.2, 1, 2)[0] * grad).sum()
        parts = oracle.group_norm(x, 3, w, b, 1e-5, activation, [7, 0, 4], 0.2, 1, 2, grad)[3:]
        for at, part in enumerate(parts):
            v = rng.normal(size=part.shape)
            args = [[a + (s * 1e-5 * v if i == at else 0) for i, a in enumerate((x, w, b))] for s in (1, -1)]
            slope = (loss(*args[0]) - loss(*args[1])) / 2e-5
            assert abs(slope - (part * v).sum()) < 1e-7 * np.linalg.norm(grad) * np.linalg.norm(v)


def test_workspace_sizes():
    lib = native.load()
    size = ctypes.c_size_t()
    assert lib.cpde_embedding_gradient_workspace(1000, 50, 8, ctypes.byref(size)) == native.OK
    assert size.value >= 1000 * 16
    assert lib.cpde_group_norm_workspace(4, 1000, 64, 8, ctypes.byref(size)) == native.OK
    assert size.value > 0
    for bad in ((-1, 50, 8), (10, 0, 8), (10, 1 << 31, 8), (1 << 31, 5, 8), (10, 5, 0), (10, 5, (1 << 24) + 1)):
        assert lib.cpde_embedding_gradient_workspace(*bad, ctypes.byref(size)) == native.REJECTED
    for bad in ((1, 10, 8, 3), (1, 10, 8, 0), (-1, 10, 8, 2), (1, -1, 8, 2), (1, 10, 0, 1), ((1 << 20) + 1, 1, 8, 2)):
        assert lib.cpde_group_norm_workspace(*bad, ctypes.byref(size)) == native.REJECTED


def test_tensors_off_the_engines_device_are_refused():
    from cpde_b200 import operators

    class Device:
        device = 0

    x = torch.zeros(2, 3, 4)
    for call in (lambda: operators.embedding(Device, x[0], torch.zeros(2, dtype=torch.int64)),
                 lambda: operators.embedding_gradient(Device, x[0], torch.zeros(3, dtype=torch.int64), 5),
                 lambda: operators.dropout(Device, x, 0.1, 1),
                 lambda: operators.group_norm(Device, x, 2),
                 lambda: operators.group_norm_gradient(Device, x, x, x[0, :2, :2], x[0, :2, :2], 2)):
        with pytest.raises(ValueError, match='device'):
            call()
