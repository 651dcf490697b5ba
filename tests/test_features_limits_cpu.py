"""CPU: sizes that the gated unit refuses, and the scratch memory of those that it takes."""
import ctypes as C

import pytest

pytest.importorskip('torch')

from bayesian_optimization_amd import _lib as L  # noqa: E402

P = C.c_void_p(4096)      # stands for a device pointer: a refused call never looks at it
MOST = 1 << 28


@pytest.mark.parametrize('rows,cols,hidden', [(4, MOST + 1, 8), (4, 8, MOST + 1), (0, MOST + 1, 8), (0, 8, MOST + 1)])
def test_columns_and_hidden_units_beyond_the_most(rows, cols, hidden):
    lib = L.load()
    for dtype in (L.TYPE_F32, L.TYPE_BF16, L.TYPE_F16):
        assert lib.gpbo_gated_workspace(dtype, rows, cols, hidden) == -1
        assert lib.gpbo_gated_backward_workspace(dtype, rows, cols, hidden) == -1
        assert lib.gpbo_gated(0, None, dtype, 0, P, cols, rows, cols, P, P, cols, hidden, P, hidden, None, None, P, 1 << 50) == L.ERR_BAD_ARG
        assert lib.gpbo_gated_backward(0, None, dtype, 0, P, hidden, P, cols, rows, cols, P, P, cols, hidden, P, P, P, cols, P, P, cols, P, 1 << 50) == L.ERR_BAD_ARG
    assert lib.gpbo_gated_workspace(L.TYPE_BF16, 0, MOST, 8) == lib.gpbo_gated_workspace(L.TYPE_BF16, 0, 8, MOST) == 0


def test_packed_rows_take_8_gigabytes_at_most():
    lib = L.load()
    weights = 2 * 64 * 64 * 2
    for rows, cols in ((1 << 30, 1), (1 << 28, 3), ((1 << 31) - 1, 60), (100000000, 64)):
        assert weights <= lib.gpbo_gated_workspace(L.TYPE_BF16, rows, cols, 64) <= (1 << 33) + weights
    assert lib.gpbo_gated_workspace(L.TYPE_BF16, 1 << 20, 64, 64) == (1 << 27) + weights
