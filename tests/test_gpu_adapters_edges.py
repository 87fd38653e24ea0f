"""Calls of the adapters that a server makes at the edge: a batch without rows."""
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
