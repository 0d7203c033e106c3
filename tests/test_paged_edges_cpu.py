"""What the paged cache's entries refuse at the ends of their ranges, without a GPU."""
import ctypes

import numpy as np
import pytest

import tinygiant_b200 as tg

BUF = np.zeros(1 << 14, np.float32)
P = BUF.ctypes.data


def gather(lib, total):
    return lib.tg_paged_gather(0, 16, P, P, P, P, P, P, P, P, total, 2, 3, 16, 2, 2, 64, (ctypes.c_int64 * 17)(*[64] * 17), None)


@pytest.mark.parametrize("total", [1 << 30, 2147483647, 2147483647 - 30])
def test_rows_beyond_the_index_arithmetic_are_refused(lib, total):
    assert gather(lib, total) == 3 and "2^30" in tg.last_error(lib)[1]
