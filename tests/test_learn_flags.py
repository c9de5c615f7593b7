"""Flags that a great many columns share (CPU): the C struct counts them in 32 bits, which ctypes
cuts without a word, and the kernel would then read beyond the flags."""

import math

import pytest

from swarp_b200 import _lib
from swarp_b200.learn.advantage import _flag_dims


@pytest.mark.parametrize("shape,dims,want", [
    ((8, 4, 2), 1, 1), ((8, 4, 2), 3, 3), ((8,), 1, 1), ((0, 4), 1, 1),
    ((1, 2 ** 31 - 1), 1, 1), ((1, 2 ** 31), 1, 2), ((1, 2 ** 32 + 4), 1, 2),
    ((2, 2 ** 20, 2 ** 12), 1, 2), ((2, 3, 2 ** 20, 2 ** 12), 1, 3), ((2, 3, 2 ** 31), 2, 3),
])
def test_columns_that_share_a_flag_fit_the_struct(shape, dims, want):
    assert _flag_dims(shape, dims) == want
    per_flag = math.prod(shape[want:])
    assert _lib.Gae(0, per_flag).columns_per_flag == per_flag
    if want > dims:  # without it the struct would hold another number
        per_flag = math.prod(shape[dims:])
        assert _lib.Gae(0, per_flag).columns_per_flag != per_flag
