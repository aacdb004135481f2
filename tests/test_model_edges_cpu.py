"""CPU checks of the edges of what stands around the losses: which elements of a matrix the norm reads in whole packs."""
import ctypes

import pytest

from test_capi_cpu import _lib


def reads(C, rows, cols, stride, base, size):
    low, high = ctypes.c_int64(), ctypes.c_int64()
    assert C.lib.ctb_debug_norm_reads(rows, cols, stride, base, size, ctypes.byref(low), ctypes.byref(high)) == C.OK
    return low.value, high.value


@pytest.mark.parametrize("size", [4, 2])
def test_norm_reads_stay_inside_the_matrix(size):
    """Rows that start anywhere are read in packs of 16 bytes of memory, which must not reach out of the matrix on either side: of
    rows narrower than a pack one would reach over several rows."""
    C, vec = _lib(), 16 // size
    for rows in (1, 2, 3, 4, 5, 9, 17):
        for cols in (1, 2, 3, 5, 6, 7, 8, 9, 15, 16, 17, 33):
            for stride in (cols, cols + 1, cols + 2, cols + 5, cols + vec):
                for base in range(vec):
                    low, high = reads(C, rows, cols, stride, base, size)
                    assert low >= 0 and high <= (rows - 1) * stride + cols - 1, (rows, cols, stride, base)


def test_norm_reads_whole_packs_where_it_can():
    C = _lib()
    assert reads(C, 3, 2, 2, 0, 2) == (0, 0)  # rows narrower than a pack are read element by element
    assert reads(C, 9, 7, 7, 0, 2) == (0, 55)
    assert reads(C, 4, 16, 17, 0, 2) == (0, 63)  # a gap between rows belongs to the matrix, what follows the last row does not
    assert reads(C, 4, 16, 17, 3, 2) == (0, 60)


def test_norm_reads_refuses_what_is_no_matrix():
    C = _lib()
    a, b = ctypes.c_int64(), ctypes.c_int64()
    for rows, cols, stride, base, size in ((0, 4, 4, 0, 4), (2, 0, 4, 0, 4), (2, 4, 3, 0, 4), (2, 4, 4, -1, 4), (2, 4, 4, 0, 8)):
        assert C.lib.ctb_debug_norm_reads(rows, cols, stride, base, size, ctypes.byref(a), ctypes.byref(b)) != C.OK
