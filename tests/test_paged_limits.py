"""The largest batches of rows that a paged cache's calls take: their grids' threads stay below 2^32. Runs where there is no GPU."""
import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest

from conftest import ROOT

SRC = r"""
#include "paged_plan.h"
extern "C" {
long long blocks(int threads) { return pg_max_blocks(threads); }
int threads(int append) { return append ? PG_APPEND_TPB : PG_TPB; }
}
"""


def test_a_grid_has_fewer_threads_than_32_bits_count(tmp_path):
    if not shutil.which("g++"):
        pytest.skip("no g++")
    src, so = tmp_path / "limits.cpp", tmp_path / "limits.so"
    src.write_text(SRC)
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC",
                    "-I" + os.path.join(ROOT, "smol-genius_amd", "csrc"), str(src), "-o", str(so)], check=True)
    lib = ctypes.CDLL(str(so))
    lib.blocks.restype = ctypes.c_longlong
    for append in (0, 1):
        t = lib.threads(append)
        assert lib.blocks(t) * t < 2 ** 32 <= (lib.blocks(t) + 1) * t
    with open(os.path.join(ROOT, "smol-genius_amd", "csrc", "paged.hip")) as f:
        text = f.read()
    assert "PA_TPB = PG_APPEND_TPB" in text  # what k_pg_append is launched with


@pytest.mark.parametrize("rows,write,read", [(64 * (2 ** 23 - 3), "not refused", "not refused"), (64 * (2 ** 23 - 2), "rows", "not refused"),
                                             (64 * (2 ** 24 - 2), "rows", "rows"), (2 ** 31 - 1, "rows", "rows")])
def test_rows_of_a_call(rows, write, read):
    """the sizes are looked at before the pool is: zeros in its place, so what is not refused for its rows is for its layer"""
    from smol_genius_amd import smol_attn as sa
    L = sa.load()
    pool = ctypes.create_string_buffer(4096)
    at = np.zeros(64, np.float32)
    p = at.ctypes.data + -at.ctypes.data % 16
    for call, what in ((L.smol_kv_pages_append(pool, 0, None, 1, p, 1, p, p, rows, p, p, 1, None, 1e-6), write),
                       (L.smol_kv_pages_read(pool, 0, 1, p, 1, p, p, rows, p, p, 1), read)):
        assert call == (-4 if what == "rows" else -1)
    assert L.smol_kv_pages_append(pool, 0, None, 1, p, 1, p, p, rows, p, p, 1, None, 1e-6) == (-4 if write == "rows" else -1)
    assert ("%d rows" % rows in L.smol_attn_last_error().decode()) == (write == "rows")
