"""CPU checks of the edges of what stands around the losses: which elements of a matrix the norm reads in whole packs, and what
scratch the projection asks for."""
import ctypes

import pytest

from test_capi_cpu import _lib, view
from test_model_cpu import BF16, F32, P, head, head_base


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


def test_a_projection_without_gradients_holds_no_logits():
    """In bfloat16: the statistics of every 128 columns, 8 bytes each, 256 MiB of them at a time, and numbers a row."""
    C = _lib()
    need, both = C.lib.ctb_linear_loss_forward_scratch_bytes, C.lib.ctb_linear_loss_scratch_bytes
    for rows, dim, vocab in ((1, 64, 500), (8192, 4096, 131072), (1 << 20, 4096, 131072), (100_000, 64, 256_000), (1 << 20, 8, 500), (3, 8, 1 << 24)):
        x, w = view(C, [rows, dim], dtype=BF16), view(C, [vocab, dim], dtype=BF16)
        tiles = -(-vocab // 128)
        most = max(256 << 20, 256 * tiles * 8) + rows * 40 + (1 << 14)
        for weighted in (0, 1):
            # rows that count are packed
            packed = rows * dim * 2 if weighted else 0
            assert need(P(x), P(w), weighted) <= most + packed
            assert need(P(x), P(w), weighted) <= both(P(x), P(w), weighted, 0) <= both(P(x), P(w), weighted, 1)
    assert need(P(view(C, [8192, 4096], dtype=BF16)), P(view(C, [131072, 4096], dtype=BF16)), 0) < 0.04 * 8192 * 131072 * 2
    f = view(C, [900, 64]), view(C, [5000, 64])  # float32 keeps its logits
    assert 900 * 5000 * 4 <= need(P(f[0]), P(f[1]), 0) == both(P(f[0]), P(f[1]), 0, 0)
    assert need(P(x), P(view(C, [500, 4], dtype=BF16)), 0) == 0 and need(None, P(w), 0) == 0


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_projection_without_gradients_refuses_less_scratch(dtype):
    C = _lib()
    d = head_base(C)
    d.update(h=view(C, [2, 3, 8], dtype=dtype), w=view(C, [11, 8], dtype=dtype), gh=None, gw=None)
    d["nbytes"] = C.lib.ctb_linear_loss_forward_scratch_bytes(P(d["h"]), P(d["w"]), 0) - 1
    assert head(C, d) == C.ERR_SCRATCH


def test_views_of_too_many_dims_are_refused():
    """By the error that other operands of that rank get."""
    import torch

    import ctorch_b200 as cb
    from ctorch_b200 import losses, model

    for f, dtype in ((losses._view, torch.float32), (model._view8, torch.float8_e4m3fn)):
        f(torch.empty([1] * 16, dtype=dtype))
        with pytest.raises(cb.ShapeError, match="rank"):
            f(torch.empty([1] * 17, dtype=dtype))
