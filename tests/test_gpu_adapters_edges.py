"""Calls of the adapters at the edge: a batch without rows, sizes past the range."""
import ctypes

import pytest

from conftest import pkg  # noqa: F401

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_adapters import Case, ctx, sa  # noqa: E402,F401


@pytest.mark.parametrize("ids", [[], (), torch.zeros(0, dtype=torch.int32).numpy()], ids=["list", "tuple", "array"])
def test_no_rows(sa, ctx, ids):
    """as smol_linear_dev: nothing to do, whatever holds the empty ids"""
    t = Case(2, 64, 48, [8])
    t.call(sa, ctx)
    x, w, bias = t.dev
    y = sa.linear_adapters(ctx, x[:0], w, t.set, ids, bias=bias)
    assert y.shape == (0, 48) and sa.linear(ctx, x[:0], w, bias).shape == (0, 48)


@pytest.mark.parametrize("k,n", [(2 ** 31 - 1, 2 ** 30), (2 ** 31 - 1, 8), (8, 2 ** 31 - 1), (2 ** 29, 8), (2 ** 21, 2 ** 20)])
def test_sizes_past_the_range(sa, ctx, k, n):
    """refused by their numbers, before a weight is read (an in_dim of 2^31 - 1 rounds up past 31 bits)"""
    a, b = (ctypes.c_void_p * 1)(16), (ctypes.c_void_p * 1)(16)
    h = ctypes.c_void_p(1)
    assert sa.load().smol_adapters_create(ctx.h, 1, k, n, a, b, (ctypes.c_int * 1)(8), (ctypes.c_float * 1)(1.0),
                                          ctypes.byref(h)) == -4
    assert not h.value and "range" in sa.load().smol_attn_last_error().decode()
