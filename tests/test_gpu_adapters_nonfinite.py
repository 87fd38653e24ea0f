"""Infinities in x, and fp32 values at the end of the range, through the projection with an adapter a row: what the formula's
products and sums give, elementwise: an infinity where all terms agree, NaN where they do not or where a zero meets one.
The ranks that pad an adapter take no part in it, and the other rows keep their bits."""
import pytest

from conftest import pkg  # noqa: F401

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_adapters import Case, ctx, sa  # noqa: E402,F401


def product(m, v):
    """m [r, k] times v [k] as a sum of products"""
    return (m.double() * v.double()).sum(-1)


def formula(t, s):
    y = product(t.w, t.x[s])
    if t.ids[s] >= 0:
        a, b, scale = t.ab[t.ids[s]]
        y = y + product(b, scale * product(a, t.x[s]))
    return y + t.bias.double()


# one launch, two launches with 16, 32 and 64 rows, more rows beside the library's product; ranks of whole tiles and not
@pytest.mark.parametrize("n,ranks", [(3, [1, 8, 16]), (9, [1, 8, 17]), (20, [1, 33, 16]), (50, [1, 100, 7]), (130, [1, 3, 64])])
@pytest.mark.parametrize("bf16", [False, True], ids=["x_f32", "x_bf16"])
@pytest.mark.parametrize("out_bf16", [False, True], ids=["f32", "y_bf16"])
def test_infinite_elements(sa, ctx, n, ranks, bf16, out_bf16):
    t = Case(n, 96, 80, ranks, bf16=bf16, ids=[(i + 1) % 4 - 1 for i in range(n)])
    d, row = 41, 2
    for i, (a, b, _) in enumerate(t.ab):
        # the terms of B t agree in sign for all but every fifth output
        b.copy_(b.abs() * a[:, d].sign())
        b[::5] = b[::5] * torch.where(torch.arange(b.shape[1]) % 2 == 0, 1, -1).to(torch.bfloat16)
        b[7] = 0.0
    clean = t.call(sa, ctx, out_bf16).clone()
    t.check(clean, out_bf16)
    rest = [s for s in range(n) if s != row]
    seen = set()
    for turn in range(4):
        t.ids = [(i + 1 + turn) % 4 - 1 for i in range(n)]
        t.x[row] = t.x[row].clamp(-4, 4)
        t.dev = (t.x.cuda(),) + t.dev[1:]
        clean = t.call(sa, ctx, out_bf16).clone()
        for bad in (float("inf"), -float("inf")):
            keep = t.x[row, d].clone()
            t.x[row, d] = bad
            t.dev = (t.x.cuda(),) + t.dev[1:]
            y = t.call(sa, ctx, out_bf16)
            assert torch.equal(y[rest], clean[rest])
            got = (y.view(torch.bfloat16) if out_bf16 else y)[row].cpu().double()
            want = formula(t, row)
            assert not torch.isfinite(want).any()
            assert torch.equal(torch.nan_to_num(got, 7.0, 1.0, -1.0), torch.nan_to_num(want, 7.0, 1.0, -1.0)), (turn, bad)
            seen |= set(torch.nan_to_num(want, 7.0, 1.0, -1.0).tolist())
            t.x[row, d] = keep
    assert seen == {7.0, 1.0, -1.0}


@pytest.mark.parametrize("n", [3, 9, 50])
def test_the_end_of_the_range(sa, ctx, n):
    """finite fp32 values that would round to an infinite bf16 value (those of more than 64 rows are the library's product)"""
    t = Case(n, 96, 80, [1, 8, 17], bias=False, ids=[i % 4 - 1 for i in range(n)])
    t.x[:] = 0.0
    t.x[:, 3], t.x[:, 50] = 3.4e38, -3.402e38
    t.w.copy_(t.w * 2.0 ** -6)
    for a, b, _ in t.ab:
        a.copy_(a * 2.0 ** -6)
        b.copy_(b * 2.0 ** -6)
    t.check(t.call(sa, ctx))
