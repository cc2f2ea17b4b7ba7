"""Checking batches of a sliding window on the host: pages in front of every
row's window may be gone, as the kernels do not look at them."""
import ctypes as C

import numpy as np
import pytest

from eos_amd import _lib
from eos_amd._lib import EosHipError
from eos_amd.kvcache import check_batch

CACHE = ("bf16", 2, 64, 16, 10)


def test_pages_in_front_of_the_window_may_be_gone():
    # 100 tokens: the row at 99 sees 60 .. 99 of a window of 40, from page 3 on
    table = [[-1, -1, -1, 3, 4, 5, 6]]
    with pytest.raises(EosHipError, match="page 0 of its table row is -1"):
        check_batch(*CACHE, table, [100])
    check_batch(*CACHE, table, [100], window=40, writes=True)
    check_batch(*CACHE, table, [100], window=52)                       # 48 .. 99
    with pytest.raises(EosHipError, match="page 2 of its table row is -1"):
        check_batch(*CACHE, table, [100], window=53)                   # 47 .. 99
    # several rows: the first one's window counts (rows at 90 .. 99)
    check_batch(*CACHE, table, [100], [0, 10], window=43, writes=True)  # 48 .. 99
    with pytest.raises(EosHipError, match="page 2"):
        check_batch(*CACHE, table, [100], [0, 10], window=44)


def test_windows_beside_padding_and_empty_sequences():
    # rows in front of position 0, a sequence without rows, one without tokens
    check_batch(*CACHE, [[1], [-1], [-1]], [5, 16, 0], [0, 9, 9, 12], window=3)
    check_batch(*CACHE, [[1], [2]], [5, 16], [0, 9, 9], window=2 ** 31 - 1)
    with pytest.raises(EosHipError, match="sequence 1"):
        check_batch(*CACHE, [[1], [-1]], [5, 16], [0, 9, 9])
    with pytest.raises(EosHipError, match="sequence 0: page 0"):
        check_batch(*CACHE, [[-1]], [5], [0, 9], window=1)


@pytest.mark.parametrize("bad,what", [([[-1, 10]], "page 1 of its table row is 10"),
                                      ([[-1, -1]], "page 1 of its table row is -1")])
def test_what_the_rows_need_is_still_asked_for(bad, what):
    with pytest.raises(EosHipError, match=what):
        check_batch(*CACHE, bad, [32], window=1)
    with pytest.raises(EosHipError, match="length 33"):
        check_batch(*CACHE, [[-1, 2]], [33], window=1)
    with pytest.raises(EosHipError, match="page 4 is written twice"):
        check_batch(*CACHE, [[-1, 4], [-1, 4]], [20, 20], window=1, writes=True)


def test_window_refusals():
    with pytest.raises(EosHipError, match="window must not be negative"):
        check_batch(*CACHE, [[1]], [4], window=-1)
    # the entry without a window as before
    d = _lib.EosHipKVDesc(format=1, kv_heads=2, head_dim=64, page_tokens=16, pages=10)
    t, n = np.array([[-1, 2]], np.int32), np.array([20], np.int32)
    with pytest.raises(EosHipError, match="page 0"):
        _lib.call("eoship_kv_check_batch", C.byref(d), t.ctypes.data_as(C.c_void_p), 2, 1,
                  n.ctypes.data_as(C.c_void_p), None, 1, 0)
