"""Limits of the norm and join kernels' launches and of their argument checks, which need no GPU."""
import ctypes as C

import pytest

from geeps_b200.ops import _lib as L

TYPES = ((0, 0), (1, 0), (1, 1))
SIZES = [(70000, 2, 4), (100000, 2, 3), (75776, 2, 1), (75775, 3, 7), (65532, 5, 8), (56832, 2, 8), (400000, 2, 2), (1 << 20, 8, 1), (1, 60000, 8),
         (9000, 40, 40), (40000, 3, 129), (30, 900, 9000), (1 << 22, 2, 16), (7, 1, 8), (3, 5, 16384)]


def sums_shape(rows, images, c, mode, vec, types):
    out = (C.c_int * 4)()
    assert L.lib().geeps_norm_sums_shape(C.c_longlong(rows), C.c_longlong(images), c, mode, int(vec), *types, out) == 0
    return list(out)


@pytest.mark.parametrize("images,pixels,c", SIZES)
@pytest.mark.parametrize("mode", [2, 3])
def test_the_launch_that_joins_the_sums_fits_a_grid(images, pixels, c, mode):
    """A grid has at most 65535 blocks along y, and an image's shares are few where there are many images."""
    for types in TYPES:
        for vec in ((True, False) if c % 8 == 0 else (False,)):
            x, y, parts, merged = sums_shape(images * pixels, images, c, mode, vec, types)
            assert 0 <= x <= 512 and 0 <= y <= 65535, (x, y, parts, merged)
            assert parts in (1, 2, 4, 8, 16, 32) and merged in (1, 2, 4, 8, 16, 32)
