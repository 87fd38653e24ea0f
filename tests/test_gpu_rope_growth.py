"""A RoPE table that grows, as a wide page table makes it do: its rows, and what the host holds meanwhile."""
import os
import threading

import numpy as np
import pytest

from conftest import pkg  # noqa: F401

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_paged import ctx, sa  # noqa: E402,F401


@pytest.mark.parametrize("inter", [0, 1])
@pytest.mark.parametrize("hd", [64, 80])
def test_rows_after_growth(sa, ctx, hd, inter):
    """a table grown in several steps has the rows of the formula: those it had, across its pieces, the last"""
    table = sa.RopeTable(ctx, hd, 1e4, inter)
    pos = [0, 1, 1023, 1024, 2047, 2048, 16383, 16384, 17407, 17408, 17409, 33791, 33792, 39999, 65535]
    for grow in (1024, 1025, 40000, 65536):
        table.ensure(grow)
        seen = [p for p in pos if p < grow]
        x = torch.randn(len(seen), hd, generator=torch.Generator().manual_seed(grow))
        y = x.cuda()
        sa.apply_rope(ctx, table, y, seen, 1)
        ctx.synchronize()
        c, s = (torch.from_numpy(np.concatenate(a)).double() for a in zip(*(sa.rope_fill_host(p, 1, hd, 1e4, inter) for p in seen)))
        x = x.double()
        if inter:
            other = torch.stack([-x[:, 1::2], x[:, 0::2]], -1).flatten(-2)
        else:
            a, b = x.chunk(2, -1)
            other = torch.cat([-b, a], -1)
        # two products and a sum in fp32
        assert ((y.cpu().double() - (x * c + other * s)).abs() <= 2.0 ** -22 * (x.abs() + other.abs())).all(), grow


def test_growth_needs_little_host_memory(sa, ctx):
    """a million positions, 512 MB of a table: the host holds a piece of it at a time"""
    pages, peak, done = os.sysconf("SC_PAGE_SIZE"), [0], threading.Event()

    def rss():
        with open("/proc/self/statm") as f:
            return int(f.read().split()[1]) * pages

    def watch():
        while not done.wait(0.002):
            peak[0] = max(peak[0], rss())

    table = sa.RopeTable(ctx, 64, 1e4)
    table.ensure(4096)
    before, t = rss(), threading.Thread(target=watch)
    t.start()
    try:
        table.ensure(1 << 20)
    finally:
        done.set()
        t.join()
    assert table.capacity == 1 << 20
    assert peak[0] - before < 200 << 20, (before, peak[0])
