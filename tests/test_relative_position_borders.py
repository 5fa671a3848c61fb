"""CPU: numbers for the bucket borders that are not Python's whole numbers, and borders that the kernels' 32 bits do not hold."""
import numpy as np
import pytest
import torch

from aotriton_b200 import autograd


def test_other_whole_numbers():
    far = 12345      # (looked up here first: a number that equals it must not leave its own answer for others)
    got = autograd.relative_position_borders(np.int32(16), np.int64(far))
    assert got == autograd.relative_position_borders(16, far)
    assert all(type(b) is int for b in got)
    # (far / 8) ** 1 at bucket 16 - 1: the smallest r with r ** 8 >= 8 * far ** 7
    assert got[-1] ** 8 >= 8 * far ** 7 > (got[-1] - 1) ** 8


@pytest.mark.parametrize("buckets,far", [(16, 777.0), (16.0, 777), (16, "777"), (16, None)])
def test_not_whole_numbers(buckets, far):
    with pytest.raises(ValueError):
        autograd.relative_position_borders(buckets, far)
    assert all(type(b) is int for b in autograd.relative_position_borders(16, 777))


def test_borders_beyond_32_bits():
    class Table:      # (what the checks look at)
        shape, dtype, is_cuda = torch.Size((6, 4)), torch.float32, True

        def dim(self):
            return 2

    far = (2 ** 32 + 5) ** 2      # three buckets: the last from the square root on, whose low 32 bits are 5
    assert autograd.relative_position_borders(3, far) == (1, 2 ** 32 + 5)
    for edge in (far, (2 ** 31) ** 2):
        with pytest.raises(ValueError, match="32 bits"):
            autograd.relative_position_bias(Table(), 5, 6, max_distance=edge)
