"""Sizes that a Q4_0 layer refuses before it reads a block."""
import ctypes

import pytest

from trit_b200 import lm


@pytest.mark.parametrize("n, k", [(2**31 - 16383, 32), (2**31 - 1, 32), (1, 2**31 - 32), (1, 2**31 - 8192), (2**31, 32),
                                  (1, 2**40)])
def test_sizes_past_32_bits(n, k):
    lib = lm.library()
    block = (ctypes.c_uint8 * 18)()
    assert lib.trit_dense_q4_0(block, n, k, 0, 0) is None
    assert "at most 2^31 - 16384" in lib.trit_cuda_last_error().decode()
