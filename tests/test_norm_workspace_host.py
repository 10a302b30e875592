"""Workspace sizes of group norm: what the sums take, not what the largest cluster could."""
import ctypes

import pytest

from cpde_b200 import native

MANY = [(1 << 20, 1, 64, 8), (1 << 20, 4, 512, 32), (65536, 16, 512, 32), (65536, 1, 512, 32), (4096, 100, 64, 4), (1000, 7, 21, 7)]


def sizes(*shape):
    lib, size = native.load(), ctypes.c_size_t()
    got = []
    for query in (lib.cpde_group_norm_forward_workspace, lib.cpde_group_norm_workspace):
        assert query(*shape, ctypes.byref(size)) == native.OK
        got.append(size.value)
    return got


@pytest.mark.parametrize('n,p,c,groups', MANY)
def test_many_instances_of_few_points(n, p, c, groups):
    """Two FP32 sums a channel and instance and two or three a group and tile (at most the channels) for the gradient, three a
    group and tile for the forward."""
    forward, both = sizes(n, p, c, groups)
    tiles = -(-c // 64)
    pieces = 12 * n * (groups + tiles * 2)
    assert forward <= pieces + 512
    assert both <= max(8 * n * c, pieces) + pieces + 512


@pytest.mark.parametrize('n,p,c,groups', MANY + [(1, 1 << 20, 64, 8), (32, 4096, 512, 32), (1, 1, 1, 1), (3, 67, 48, 6)])
def test_the_forward_needs_no_more_than_both(n, p, c, groups):
    forward, both = sizes(n, p, c, groups)
    assert 0 < forward <= both


def test_no_points_need_none():
    assert sizes(0, 5, 8, 2) == [0, 0] and sizes(5, 0, 8, 2) == [0, 0]


def test_wrong_sizes_are_refused():
    lib, size = native.load(), ctypes.c_size_t()
    for bad in ((1, 10, 8, 3), (1, 10, 8, 0), (-1, 10, 8, 2), (1, -1, 8, 2), (1, 10, 0, 1), ((1 << 20) + 1, 1, 8, 2)):
        assert lib.cpde_group_norm_forward_workspace(*bad, ctypes.byref(size)) == native.REJECTED
    assert lib.cpde_group_norm_forward_workspace(1, 10, 8, 2, None) == native.REJECTED


def test_more_items_than_a_launch_counts_take_two_passes():
    """2^20 instances of 2^18 groups: 2^38 items of the one-pass kernel, whose sums of eight CTAs would be asked for."""
    n, p, c, groups = 1 << 20, 3000, 1 << 20, 1 << 18
    _, both = sizes(n, p, c, groups)
    assert both < 4 * 8 * n * c
