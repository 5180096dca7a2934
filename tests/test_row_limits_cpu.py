"""CPU: sizes at which the row operators' launches and sums change their form (no GPU call is made)."""
import ctypes as C

import pytest

OVERFLOW = 10
F32, S64 = 6, 9


def _rows(pkg, dtype=F32, cols=8, count=4, stride=None, base=4096):
    r = pkg.rows._Rows(base, dtype, cols)
    r.count[:], r.stride[:] = (count, 1, 1), (cols * 4 if stride is None else stride, 0, 0)
    return r


@pytest.mark.parametrize("accumulate", [0, 1])
def test_a_gradient_that_is_too_large_is_refused_before_anything_happens(pkg, accumulate):
    """The workspace query and the call give the same answer; the call would have to launch 8e14 jobs."""
    L, need = pkg.rows._lib(), C.c_size_t(0)
    count, cols = (1 << 31) - 1, (1 << 31) - (1 << 16)
    g, i, t = _rows(pkg, cols=cols, count=count, stride=0), _rows(pkg, S64, 1, count, 8), _rows(pkg, cols=cols)
    assert L.b200ppEmbeddingBackwardWorkspace(C.byref(g), C.byref(t), C.byref(need)) == OVERFLOW
    op = pkg.rows._EmbeddingGradOp(1.0, accumulate, -1)
    assert L.b200ppEmbeddingBackward(C.byref(g), C.byref(i), C.byref(t), C.byref(op), 65536, 1 << 62, None) == OVERFLOW
    assert b"too large" in L.b200ppGetLastErrorMessage()
    # wide tables and few indices are not too large
    g, t = _rows(pkg, cols=1 << 30, count=70), _rows(pkg, cols=1 << 30)
    assert L.b200ppEmbeddingBackwardWorkspace(C.byref(g), C.byref(t), C.byref(need)) == 0 and need.value > 0


@pytest.mark.parametrize("rows,cols,chains", [(300_000, 65_537, 8), (300_000, 40_000, 1), (300_000, 20_000, 1), (10_000_000, 65_537, 8)])
def test_sums_over_many_long_rows_have_parts(pkg, rows, cols, chains):
    """Room for as many parts as leave each of their chains of additions 1024 rows."""
    need = C.c_size_t(0)
    assert pkg.rows._lib().b200ppLayerNormBackwardWorkspace(C.byref(_rows(pkg, cols=cols, count=rows)), C.byref(need)) == 0
    assert need.value // (2 * 4 * cols) * chains * 1024 >= rows
