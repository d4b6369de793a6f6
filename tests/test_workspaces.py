"""How much memory cross entropy over many items works in (include/hetuctr_hip.h): no GPU is needed to ask."""
import os

import pytest

from hetuctr_amd import build, capi

pytestmark = pytest.mark.skipif(not os.path.exists(build.LIB), reason="needs the built library")
MIB = 1 << 20


def up(n, to):
    return (n + to - 1) // to * to


def around(rows, width, items, size):
    """The copy of x, what is known of the rows and of the items; whole pieces of 256"""
    return up(rows * up(width * size, 16), 256) + 256 + 16 * up(rows, 256) + up(8 * up(rows, 1024) // 1024, 256) + 4 * up(items, 256)


@pytest.mark.parametrize("dtype, size", [(capi.F32, 4), (capi.BF16, 2), (capi.F16, 2)])
@pytest.mark.parametrize("rows, width, items", [(4096, 256, 1_000_000), (65536, 256, 50_000), (131072, 512, 50_000), (1 << 20, 256, 100_000), (1 << 20, 160, 100), (1 << 26, 136, 5000),
                                                (33, 4096, 131072), (5000, 129, 20)])
def test_slopes_that_a_gradient_holds(rows, width, items, dtype, size):
    m, none = (4096, up(width, 64)), capi.NO_MATRIX
    need = capi.linear_cross_entropy_backward(rows, width, items, m, m, none, none, 0, 0, 4096, -100, 4096, 4096, (0, 0), (dtype, capi.F32), space=True)
    slopes = min(rows * up(items, 64) * size, max(512 * MIB, 2048 * rows * size))
    copied = up(items * up(width * size, 16), 256) if width * size % 16 else 0             # weights whose rows are not whole pieces of 16 bytes
    assert need <= around(rows, width, items, size) + slopes + copied + 256
    if rows * items * size > slopes:                # and not much less
        assert need > slopes - 256 * rows * size


@pytest.mark.parametrize("rows, width, items", [(4096, 128, 1_000_000), (1, 32, 10_000_000), (65536, 64, 20_000), (1 << 20, 128, 100)])
def test_narrow_rows_hold_none(rows, width, items):
    m, none = (4096, 128), capi.NO_MATRIX
    for dx in (none, (4096, 128)):
        need = capi.linear_cross_entropy_backward(rows, width, items, m, m, dx, none, 0, 0, 4096, -100, 4096, 4096, (0, 0), (capi.BF16, capi.F32), space=True)
        assert need <= around(rows, width, items, 2) + (max(rows * width * 4, 512 * 256 * width * 4) + 256 if dx[0] else 0)
    need = capi.linear_cross_entropy(rows, width, items, m, m, 0, 4096, -100, 4096, 0, (0, 0), (capi.BF16, capi.F32), space=True)
    assert need <= around(rows, width, items, 2) + 8 * 768 * rows + 256


@pytest.mark.parametrize("dtype, size", [(capi.F32, 4), (capi.F16, 2)])
@pytest.mark.parametrize("rows, width, items", [(1, 4096, 131072), (32, 4096, 131072), (33, 1000, 100_000), (8192, 4096, 65537), (1 << 20, 256, 1000), (300, 9000, 100)])
def test_what_the_losses_hold(rows, width, items, dtype, size):
    m = (4096, up(width, 64))
    need = capi.linear_cross_entropy(rows, width, items, m, m, 0, 4096, -100, 4096, 0, (0, 0), (dtype, capi.F32), space=True)
    assert need <= around(rows, width, items, size) + 8 * rows * ((items + 31) // 32) + 256
