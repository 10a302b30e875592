"""The ranges of points that the blocks of the two-pass group norm take, up to the largest point count."""
import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / 'cpde_b200' / 'csrc'
HARNESS = r'''
#include "point_range.hpp"
// Whether the splits' ranges cover [0, length) once and in order; 0, or the split at fault + 1.
extern "C" int check(int32_t length, int32_t splits) {
    int32_t at = 0;
    for (int32_t i = 0; i < splits; ++i) {
        int32_t lo, hi;
        cpde::ops::split_range(length, i, splits, lo, hi);
        if (lo != at || hi < lo || hi > length) return i + 1;
        at = hi;
    }
    return at == length ? 0 : splits + 1;
}
extern "C" int32_t longest(int32_t length, int32_t splits) {
    int32_t lo, hi;
    cpde::ops::split_range(length, 0, splits, lo, hi);
    return hi - lo;
}
'''
MOST = 2 ** 31 - 2  # points of a call


@pytest.fixture(scope='module')
def ranges(tmp_path_factory):
    gxx = shutil.which('g++')
    if not gxx:
        pytest.skip('g++ not available')
    d = tmp_path_factory.mktemp('ranges')
    (d / 'harness.cpp').write_text(HARNESS)
    subprocess.run([gxx, '-std=c++17', '-O1', '-fsanitize=undefined', '-fno-sanitize-recover=all', '-shared', '-fPIC',
                    f'-I{CSRC}', str(d / 'harness.cpp'), '-o', str(d / 'libranges.so')], check=True)
    return ctypes.CDLL(str(d / 'libranges.so'))


@pytest.mark.parametrize('length', [0, 1, 2, 591, 592, 593, 2 ** 24 + 1, 2 ** 30, MOST - 16384, MOST - 256, MOST - 1, MOST])
@pytest.mark.parametrize('splits', [1, 2, 148, 592, 16384, 1 << 20])
def test_ranges_cover_every_point_once(ranges, length, splits):
    assert ranges.check(length, splits) == 0
    assert ranges.longest(length, splits) == (length + splits - 1) // splits


def test_steps_of_a_block_stay_in_32_bits(ranges):
    """A thread counts its points from its range's begin, in steps of at most 256 from at most 255; a call has at least a split
    for 512 points of each of a block's 256 threads, or of the few that wide rows leave."""
    for ys in (4, 256):
        splits = -(-MOST // (ys * 512))
        assert ranges.longest(MOST, splits) <= ys * 512
        assert ys * 512 + 255 + 256 < 2 ** 31
