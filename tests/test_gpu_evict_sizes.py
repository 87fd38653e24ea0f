"""Cache eviction on both sides of every size that k_evict_select is built for: the rows that its LDS holds, 8192 and
32768, and any number; a few moves made by the same workgroup (at most 128), and lists of them; in place and apart."""
import os
import re

import pytest

from conftest import ROOT, pkg  # noqa: F401

torch = pytest.importorskip("torch")

from test_gpu_shared import Evict, ctx, sa  # noqa: E402,F401

SMALL, LARGE, FUSED = 8192, 32768, 128


def test_sizes_are_the_sources():
    """the sizes below are those that the launch chooses by"""
    text = open(os.path.join(ROOT, "smol-genius_amd", "csrc", "attn_evict.hip")).read()
    sizes = re.findall(r"k_evict_select<(\d+)>", text)
    assert sizes == [str(SMALL), str(LARGE), "0"]
    assert re.findall(r"max_rows <= (\d+)", text) == [str(SMALL), str(LARGE)]
    assert "EV_FUSED = %d;" % FUSED in text


@pytest.mark.gpu
@pytest.mark.parametrize("apart", [False, True], ids=["in_place", "apart"])
@pytest.mark.parametrize("few", [True, False], ids=["few_moves", "lists"])
@pytest.mark.parametrize("rows", [SMALL, SMALL + 1, 20000, LARGE, LARGE + 1])
def test_evict_sizes(sa, ctx, rows, few, apart):
    keep = rows - FUSED if few else rows // 5
    e = Evict(sa, ctx, 2, 64, [rows, rows - 1], keep, first=3, recent=17, kind="all" if few else "ties", extra=2)
    e.check(*e.call(apart), apart)
