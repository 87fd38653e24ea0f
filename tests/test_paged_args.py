"""What the calls on a paged cache refuse before any device work. Runs where there is no GPU (a call that got past its checks
there would have no context to run on)."""
import ctypes

import numpy as np
import pytest

from conftest import pkg  # noqa: F401


@pytest.fixture(scope="module")
def sa():
    from smol_genius_amd import smol_attn
    smol_attn.load()
    return smol_attn


def message(sa):
    return sa.load().smol_attn_last_error().decode()


def test_without_handles(sa):
    L = sa.load()
    one = np.zeros(4, np.int32).ctypes.data
    h = ctypes.c_void_p(1)
    assert L.smol_kv_pages_create(None, 1, 1, 1, 64, 1, ctypes.byref(h)) == -1
    assert L.smol_kv_pages_destroy(None) == 0
    p = [ctypes.c_void_p() for _ in range(4)]
    assert L.smol_kv_pages_pointers(None, 0, *(ctypes.byref(x) for x in p)) == -1
    assert L.smol_kv_pages_append(None, 0, None, 1, one, 1, one, one, 1, one, one, 0, None, 1e-6) == -1
    assert "pool is NULL" in message(sa)
    assert L.smol_kv_pages_read(None, 0, 1, one, 1, one, one, 1, one, one, 0) == -1
    assert "pool is NULL" in message(sa)
    assert L.smol_attn_decode_paged(None, None, 0, None, 1, one, 1, one, None, None, None, 0, 1, 1.0, 0, 0.0, None, None, 1e-6,
                                    None) == -1
    assert "pool is NULL" in message(sa)
    assert L.smol_attn_decode_paged_top(None, None, 0, None, 1, one, 1, one, 4, 1, 1, None, None, None, 0, 1, 1.0, 0.0, None,
                                        None, 1e-6, None, None) == -1
    assert "pool is NULL" in message(sa)


@pytest.mark.parametrize("top,first,recent", [(0, 0, 1), (-1, 0, 1), (4, -1, 1), (4, 0, 0), (4, 2, 3), (4, 4, 1), (2 ** 31 - 1, 0, 1),
                                              (4, 0, 2 ** 31 - 1), (4, 2 ** 31 - 1, 1), (1, 0, -2 ** 31)])
def test_pages_to_choose(sa, top, first, recent):
    L = sa.load()
    one = np.zeros(4, np.int32).ctypes.data
    assert L.smol_attn_decode_paged_top(None, None, 0, None, 1, one, 1, one, top, first, recent, None, None, None, 0, 1, 1.0, 0.0,
                                        None, None, 1e-6, None, None) == -1
    assert "pages" in message(sa)


def test_dtype_and_norm_of_rows(sa):
    L = sa.load()
    one = np.zeros(4, np.int32).ctypes.data
    assert L.smol_kv_pages_append(ctypes.c_void_p(0), 0, None, 1, one, 1, one, one, 1, one, one, 0, ctypes.c_void_p(one + 2), 1e-6) == -1
    assert "norm weights" in message(sa)
    assert L.smol_kv_pages_append(ctypes.c_void_p(0), 0, None, 1, one, 1, one, one, 1, one, one, 0, one, -1.0) == -1
    assert "eps" in message(sa)
