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


@pytest.mark.parametrize('dtype,step', [(L.TYPE_F32, 32), (L.TYPE_BF16, 64), (L.TYPE_F16, 64)])
def test_operands_read_in_place_need_no_workspace(dtype, step):
    lib = L.load()
    rows, hidden = 1 << 16, 512
    whole, wide, odd = 4 * step, 4 * step + 8, 4 * step + 1
    most = lib.gpbo_gated_workspace(dtype, rows, whole, hidden)
    assert most > 0

    def need(x=4096, xs=whole, cols=whole, wg=4096, wu=8192, ws=whole):
        return lib.gpbo_gated_workspace_for(dtype, x, xs, rows, cols, wg, wu, ws, hidden)
    assert need() == need(xs=wide) == need(xs=wide, ws=wide) == 0
    for kw in (dict(x=4100), dict(wg=4100), dict(wu=4100), dict(xs=odd), dict(ws=odd)):
        assert need(**kw) == most, kw
    assert need(cols=whole - 1) == lib.gpbo_gated_workspace(dtype, rows, whole - 1, hidden) > 0
    for kw in (dict(xs=whole - 1), dict(ws=whole - 1), dict(cols=0)):
        assert need(**kw) == -1
    assert lib.gpbo_gated(0, None, dtype, 0, 4100, whole, rows, whole, 4096, 4096, whole, hidden, 4096, hidden, None, None, None, 0) == L.ERR_BAD_ARG
