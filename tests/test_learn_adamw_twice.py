"""A parameter that is given twice is refused before anything is launched: the two updates of its
memory would race (CPU: the check of the addresses)."""

import pytest

from swarp_b200.learn.adamw import _once


def test_the_same_address_twice():
    with pytest.raises(ValueError, match=r"params\[3\] and params\[1\] are the same memory"):
        _once([256, 512, 768, 512], [1, 2, 3, 4])


def test_empty_tensors_share_an_address():
    _once([0, 512, 0, 768, 512], [0, 2, 0, 4, 0])
