"""What the kernels of a paged cache touch, decided by smol-genius_amd/csrc/paged_plan.h, with every kind of length, table and
range (also such as are none): compiled for the host and driven here, so nothing out of range has to reach a GPU to be seen."""
import ctypes
import os
import random
import shutil
import subprocess

import numpy as np
import pytest

from conftest import ROOT

SRC = r"""
#include "paged_plan.h"
extern "C" {
int units(int len, int stride, int positions, int window, int top, int unit, int *first) {
    PgUnits u = pg_units(len, stride, positions, window, top, unit);
    *first = u.first;
    return u.n;
}
int len_ok(int len, int stride, int positions) { return pg_len_ok(len, stride, positions); }
int first_row(int len, int window) { return pg_first_row(len, window); }
int chunk(long long sum, int slots) { return pg_chunk(sum, slots); }
int chunks(int len, int units, int c) { return pg_chunks(len, units, c); }
long long max_chunks(int n, int slots) { return pg_max_chunks(n, slots); }
int bad_page(int page, int n) { return pg_bad_page(page, n); }
int order(int r, int codes) { return pg_order(r, codes != 0); }
int run_ok(int a, int b, int rows, int pos, int stride, int positions) { return pg_run_ok(a, b, rows, pos, stride, positions); }
int run_pages(int a, int b, int rows, int pos, int stride, int positions) { return pg_run_pages(a, b, rows, pos, stride, positions); }
long long max_run_pages(int n, int rows) { return pg_max_run_pages(n, rows); }
unsigned digits(int n) { return pg_digits(n); }
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    if not shutil.which("g++"):
        pytest.skip("no g++")
    d = tmp_path_factory.mktemp("plan")
    src, so = d / "plan.cpp", d / "plan.so"
    src.write_text(SRC)
    inc = os.path.join(ROOT, "smol-genius_amd", "csrc")
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-shared",
                    "-fPIC", "-I" + inc, str(src), "-o", str(so)], check=True)
    lib = ctypes.CDLL(str(so))
    for f in ("max_chunks", "max_run_pages"):
        getattr(lib, f).restype = ctypes.c_longlong
    lib.chunk.argtypes = [ctypes.c_longlong, ctypes.c_int]
    lib.digits.restype = ctypes.c_uint
    return lib


INT_MAX = 2 ** 31 - 1
WILD = [-2 ** 31, -1, 0, 1, 31, 32, 33, 63, 64, 65, 127, 128, 1000, 4095, 4096, 4097, INT_MAX - 64, INT_MAX - 1, INT_MAX]


def test_lengths(plan):
    """a length counts when its row has a page and a position; none of the rest names a unit"""
    first = ctypes.c_int()
    for len_ in WILD:
        for stride in (1, 2, 64, 65, INT_MAX // 128):
            for positions in (1, 64, 4096, INT_MAX):
                ok = len_ >= 0 and len_ // 64 < stride and len_ < positions
                assert plan.len_ok(len_, stride, positions) == ok
                for window in (0, 1, 2, 33, 5000, INT_MAX):
                    for unit in (32, 64):
                        n = plan.units(len_, stride, positions, window, 0, unit, ctypes.byref(first))
                        if not ok:
                            assert n == 0
                            continue
                        lo = max(0, len_ - window + 1) if window else 0
                        if lo >= len_:
                            assert n == 0
                            continue
                        f = first.value
                        # the units hold each visible row, every one of them at least one, and the last page is the table's
                        assert f * unit <= lo < (f + 1) * unit and (f + n - 1) * unit < len_ <= (f + n) * unit
                        assert ((f + n - 1) * unit) // 64 < stride
                for top in (1, 3, 4096):
                    for unit in (32, 64):
                        n = plan.units(len_, stride, positions, 0, top, unit, ctypes.byref(first))
                        assert n == (min(top, -(-len_ // 64)) * (64 // unit) if ok else 0)


@pytest.mark.parametrize("seed", range(6))
def test_chunks_cover_every_unit_once(plan, seed):
    """the workgroups that the host starts are enough, and their chunks share every sequence's units out"""
    r = random.Random(seed)
    first = ctypes.c_int()
    for _ in range(300):
        n, stride = r.choice([1, 2, 5, 64, 65, 200]), r.choice([1, 4, 64, 300])
        unit, window, slots = r.choice([32, 64]), r.choice([0, 0, 1, 100]), r.choice([1, 2, 7, 64, 512])
        top = r.choice([0, 0, 3, 40]) if not window else 0
        lens = [r.choice(WILD + [r.randrange(stride * 64) for _ in range(20)]) for _ in range(n)]
        counts = [plan.units(l, stride, INT_MAX, window, top, unit, ctypes.byref(first)) for l in lens]
        c = plan.chunk(sum(counts), slots)
        assert c >= 4 and c % 4 == 0
        each = [plan.chunks(l, k, c) for l, k in zip(lens, counts)]
        assert sum(each) <= plan.max_chunks(n, slots)
        for l, k, e in zip(lens, counts, each):
            if l < 0:
                assert e == 0  # no sequence: no workgroup, nothing read, nothing written
                continue
            got = [u for w in range(e) for u in range(w * c, min(k, (w + 1) * c))]
            assert e >= 1 and got == list(range(k))
            assert e == 1 or all(w * c < k for w in range(e))


def test_page_numbers(plan):
    for n in (1, 2, 1000, INT_MAX):
        for page in WILD + [n - 1, n - 2]:
            assert plan.bad_page(page, n) == (not 0 <= page < n)


def test_runs(plan):
    """row ranges of a batch: what is none has no page, and the pages of the others fit the grid"""
    r = random.Random(3)
    for _ in range(20000):
        rows, stride = r.choice([0, 1, 63, 64, 65, 5000]), r.choice([1, 2, 80])
        a, b, pos = (r.choice(WILD + [r.randrange(rows + 1), r.randrange(200)]) for _ in range(3))
        positions = r.choice([64, 1024, INT_MAX])
        ok = 0 <= a <= b <= rows and (a == b or (pos >= 0 and pos + (b - a) <= stride * 64 and pos + (b - a) <= positions))
        assert plan.run_ok(a, b, rows, pos, stride, positions) == ok
        pages = plan.run_pages(a, b, rows, pos, stride, positions)
        if not ok or a == b:
            assert pages == 0
        else:
            assert pages == (pos + b - a - 1) // 64 - pos // 64 + 1 and pos // 64 + pages <= stride
            assert pages <= plan.max_run_pages(1, b - a)
    for _ in range(500):
        n = r.randrange(1, 70)
        lens = [r.choice([0, 1, 2, 63, 64, 65, 130, r.randrange(500)]) for _ in range(n)]
        rows, at, pages = sum(lens), 0, 0
        for l in lens:
            pages += plan.run_pages(at, at + l, rows, r.randrange(1000), INT_MAX // 128, INT_MAX)
            at += l
        assert pages <= plan.max_run_pages(n, rows)


def test_order_and_digits(plan):
    """V's order is a permutation of a page's rows (of each half for bf16); three balanced digits give a number back"""
    assert sorted(plan.order(r, 1) for r in range(64)) == list(range(64))
    assert sorted(plan.order(r, 0) for r in range(32)) == list(range(32))
    assert [plan.order(32 + r, 0) for r in range(32)] == [32 + plan.order(r, 0) for r in range(32)]
    n = np.concatenate([np.arange(-127 * 65536, -127 * 65536 + 70000), np.arange(-70000, 70000),
                        np.arange(127 * 65536 - 70000, 127 * 65536 + 2)])
    for x in n[::37]:
        d = plan.digits(int(x))
        a, b, c = (np.uint8(d >> s & 0xFF).view(np.int8).astype(int) for s in (16, 8, 0))
        assert a * 65536 + b * 256 + c == x
