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
int piece(long long sum, int slots) { return pg_piece(sum, slots); }
int places(int len, int units) { return pg_places(len, units); }
void cut(int off, int units, int piece, int w, int *out) {
    PgCut c = pg_cut(off, units, piece, w);
    out[0] = c.mine, out[1] = c.u0, out[2] = c.u1, out[3] = c.nth, out[4] = c.chunks;
}
int slot(int off, int piece, int nth) { return pg_slot(off, piece, nth); }
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
    lib.max_run_pages.restype = ctypes.c_longlong
    lib.piece.argtypes = [ctypes.c_longlong, ctypes.c_int]
    lib.digits.restype = ctypes.c_uint
    return lib


INT_MAX = 2 ** 31 - 1
EXTRA = 12  # PG_EXTRA
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
def test_pieces_cover_every_unit_once(plan, seed):
    """the workgroups that the host starts share every sequence's units out, each live sequence has one last chunk, no sequence none,
    and no two chunks leave their state in one place"""
    r = random.Random(seed)
    first, out = ctypes.c_int(), (ctypes.c_int * 5)()
    for _ in range(120):
        n, stride = r.choice([1, 2, 5, 64, 65, 130]), r.choice([1, 4, 64, 300])
        unit, window, slots = r.choice([32, 64]), r.choice([0, 0, 1, 100]), r.choice([1, 2, 7, 64, 256])
        top = r.choice([0, 0, 3, 40]) if not window else 0
        lens = [r.choice(WILD + [r.randrange(stride * 64) for _ in range(20)]) for _ in range(n)]
        counts = [plan.units(l, stride, INT_MAX, window, top, unit, ctypes.byref(first)) for l in lens]
        places = [plan.places(l, k) for l, k in zip(lens, counts)]
        assert all(p == (0 if l < 0 else EXTRA + k) for p, l, k in zip(places, lens, counts))
        c = plan.piece(sum(places), slots)
        assert c >= 4 and c % 4 == 0 and c * slots >= sum(places)
        used, off = set(), 0
        for l, k, p in zip(lens, counts, places):
            if l < 0:
                continue  # the kernel asks no piece about it
            got, chunks = [], None
            for w in range(max(0, off // c - 1), min(slots, (off + p) // c + 2)):
                plan.cut(off, k, c, w, out)
                mine, u0, u1, nth, chunks = out[:]
                if not mine:
                    continue
                assert nth == len(got) and off // c <= w <= (off + p) // c
                got.append((u0, u1))
                if chunks > 1:
                    s = plan.slot(off, c, nth)
                    assert s // 2 == w and s < 2 * slots and s not in used
                    assert s >= 2 * ((off + EXTRA) // c)  # where the sequence's places begin
                    used.add(s)
            assert len(got) == chunks
            if k == 0:
                assert got == [(0, 0)]
            else:
                assert got[0][0] == 0 and got[-1][1] == k and all(a < b for a, b in got)
                assert all(a[1] == b[0] for a, b in zip(got, got[1:]))
            off += p


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
