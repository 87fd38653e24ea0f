"""What the serving operators refuse before any device work: no handle, no arrays, sizes that cannot be. Runs where there
is no GPU (a call that got past its checks there would have no context to run on)."""
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


def test_decode_steps_without_handles(sa):
    L = sa.load()
    one = np.zeros(1, np.int32).ctypes.data
    assert L.smol_attn_decode_shared(None, None, 0, 0, None, 0, None, 1, one, one, None, None, None, 0, 1, 1.0, 0, 0.0, None,
                                     None, 1e-6, None) == -1
    assert "cache is NULL" in message(sa)
    assert L.smol_attn_decode_scored(None, None, 0, None, 1, one, one, one, None, None, None, 0, 1, 1.0, 0.0, None, None, 1e-6,
                                     None, None, 1, 1.0, None) == -1
    assert "cache is NULL" in message(sa)


def test_eviction_and_pointers_without_a_cache(sa):
    L = sa.load()
    one = np.zeros(1, np.int32).ctypes.data
    assert L.smol_kv_cache_evict(None, 0, 1, one, one, one, None, None, None, None, 1, 1, 0, 0) == -1
    assert "cache is NULL" in message(sa)
    k, v = ctypes.c_void_p(), ctypes.c_void_p()
    assert L.smol_kv_cache_pointers(None, 0, ctypes.byref(k), ctypes.byref(v)) == -1
    assert "NULL argument" in message(sa)


def test_adapters_without_a_context(sa):
    L = sa.load()
    h = ctypes.c_void_p(1)
    assert L.smol_adapters_create(None, 1, 8, 8, None, None, None, None, ctypes.byref(h)) == -1
    assert "null context" in message(sa)
    assert L.smol_adapters_destroy(None) == 0
    assert L.smol_linear_adapters_dev(None, None, 0, None, 0, None, None, 1, 8, 8, None, None) == -1
    assert "null context" in message(sa)


def test_host_numbers(sa):
    """lists, tuples and arrays become C ints; the wrong number of them, and what is no whole number, is refused"""
    for a in ([3, 1, 2], (3, 1, 2), np.array([3, 1, 2]), np.array([3, 1, 2], np.int32), [np.int64(3), 1, 2]):
        keep, at = sa._host_ints(a, 3, "slots")
        assert list((ctypes.c_int * 3).from_address(at)) == [3, 1, 2]
    for a in ([1, 2], np.zeros((3, 1), np.int32)):
        with pytest.raises(sa.SmolAttnError):
            sa._host_ints(a, 3, "slots")
    with pytest.raises(TypeError):
        sa._host_ints([1.5, 2, 3], 3, "slots")
    with pytest.raises(OverflowError):
        sa._host_ints([2 ** 31, 2, 3], 3, "slots")


def test_tensors_off_the_device(sa):
    """a CPU tensor, a transposed one, another dtype or shape is refused by name"""
    torch = pytest.importorskip("torch")

    class Ctx:
        device = 0
    t = torch.zeros(4, 8)
    for x, dtype, shape in ((t, torch.float32, (4, 8)), (t.double(), torch.float32, (4, 8)), (t, torch.float32, (8, 4)),
                            (t.t(), torch.float32, (8, 4))):
        with pytest.raises(sa.SmolAttnError, match="mass must be"):
            sa._on(Ctx, x, dtype, shape, "mass")
