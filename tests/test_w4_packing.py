"""The host packing of 4-bit weights refuses what the product would not take."""
import os

import pytest
import torch

INVALID = 1


@pytest.fixture(scope="module")
def L():
    from hpcdeepneuralnetworks_amd import _lib

    if not os.path.exists(_lib.LIB_PATH):
        _lib.build()
    return _lib.lib()


def test_more_columns_than_the_product_takes(L):
    """2^24 are the most (and a count near 2^31 would pass the range of the loops' counters)."""
    from hpcdeepneuralnetworks_amd import blas

    N = 1 << 24
    W = torch.zeros(1, N + 1)
    q, s = torch.zeros(1, N // 2 + 1, dtype=torch.uint8), torch.zeros(1, N // 128 + 1)
    with pytest.raises(blas.HpcdnnError, match="invalid"):
        blas.w4_quantize(1, N + 1, 128, W, q, s)
    W[0, N - 1] = 7.0
    blas.w4_quantize(1, N, 128, W, q, s)
    assert int(q[0, N // 2 - 1]) == 0xF8 and float(s[0, N // 128 - 1]) == 1.0
    # nothing is read or written: the sizes alone are refused
    assert L.hpcdnn_w4_quantize(0, (1 << 30) + 1, 1, 32, W.data_ptr(), 1, q.data_ptr(), 1, s.data_ptr(), None, 1) == INVALID


def test_pointers_between_elements(L):
    W, q, s = torch.zeros(2, 33), torch.zeros(2, 17, dtype=torch.uint8), torch.zeros(4, 4)
    go = lambda type_, w, sc: L.hpcdnn_w4_quantize(type_, 1, 32, 32, w, 32, q.data_ptr(), 17, sc, None, 1)  # noqa: E731
    for off in (1, 2, 3):
        assert go(0, W.data_ptr() + off, s.data_ptr()) == INVALID
        assert go(0, W.data_ptr(), s.data_ptr() + off) == INVALID
    assert go(1, W.data_ptr(), s.data_ptr() + 1) == INVALID and go(2, W.data_ptr(), s.data_ptr() + 3) == INVALID
    assert go(1, W.data_ptr(), s.data_ptr() + 2) == 0 and go(0, W.data_ptr() + 4, s.data_ptr() + 4) == 0
