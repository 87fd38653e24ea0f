"""Host numbers of the serving calls: what a list of Python numbers is refused for, an array is refused for too (a cast to
C ints would wrap 2^32 + 5 round to 5 and cut 1.5 down to 1, and the call would run on another slot or row)."""
import ctypes

import numpy as np
import pytest

from conftest import pkg  # noqa: F401


@pytest.fixture(scope="module")
def sa():
    from smol_genius_amd import smol_attn
    return smol_attn


@pytest.mark.parametrize("a", [np.array([3, 1, 2], t) for t in (np.int8, np.uint8, np.int16, np.int32, np.uint32, np.int64, np.uint64)]
                         + [np.array([[3, 9], [1, 9], [2, 9]])[:, 0], np.array([3, 1, 2], ">i4")], ids=lambda a: str(a.dtype))
def test_whole_numbers(sa, a):
    keep, at = sa._host_ints(a, 3, "slots")
    assert list((ctypes.c_int * 3).from_address(at)) == [3, 1, 2]


def test_the_ends_of_the_range(sa):
    lo, hi = -2 ** 31, 2 ** 31 - 1
    for a in ([lo, hi], np.array([lo, hi]), np.array([lo, hi], np.int32)):
        keep, at = sa._host_ints(a, 2, "pos")
        assert list((ctypes.c_int * 2).from_address(at)) == [lo, hi]
    for none in (np.zeros(0, np.int64), np.array([]), []):
        sa._host_ints(none, 0, "pos")


@pytest.mark.parametrize("a", [np.array([2 ** 32 + 5, 1, 2]), np.array([-2 ** 31 - 1, 1, 2]), np.array([2 ** 31, 1, 2], np.uint32),
                               np.array([2 ** 63, 1, 2], np.uint64)], ids=lambda a: str(a.dtype))
def test_beyond_an_int(sa, a):
    with pytest.raises(OverflowError):
        sa._host_ints(a, 3, "slots")


@pytest.mark.parametrize("a", [np.array([1.5, 2, 3]), np.array([1.0, 2, 3], np.float32), np.array([1 + 0j, 2, 3]),
                               np.array(["1", "2", "3"])], ids=lambda a: str(a.dtype))
def test_no_whole_numbers(sa, a):
    with pytest.raises(TypeError):
        sa._host_ints(a, 3, "slots")
