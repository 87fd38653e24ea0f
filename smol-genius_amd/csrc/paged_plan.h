/*
 * paged_plan.h - which rows of a paged cache a workgroup takes: the part of
 * the kernels of paged.hip that decides what they touch. Plain C++ for host
 * and device, so that a CPU test covers it with every length and page number.
 *
 * A sequence of `len` cached rows and a table of `stride` pages: rows
 * [lo, len) are visible, cut into units (64 rows of codes, or 32 bf16 rows: what
 * one round of matrix products takes). The sequences' units lie on one line,
 * each sequence behind PG_EXTRA places that stand for its start-up, and every
 * workgroup takes a piece of that line of the same length: all of them end
 * together, whatever the lengths, and their number is fixed by the machine.
 * The lengths are on the device, so each workgroup forms the line for itself.
 */
#ifndef SMOL_PAGED_PLAN_H
#define SMOL_PAGED_PLAN_H

#if defined(__HIPCC__)
#define PG_FN __host__ __device__ __forceinline__
#else
#define PG_FN inline
#endif

#define PG_ROWS 64  /* rows of a page (SMOL_PAGE_ROWS) */
#define PG_WAVES 4  /* waves of a decode workgroup: units of a chunk go to them in turn */

/* rows of a unit */
PG_FN int pg_unit(bool codes) { return codes ? 64 : 32; }

/* A sequence's length is used when its new row has a place in the table (and a position in the RoPE table of `positions`
 * rows); a negative one is no sequence. */
PG_FN bool pg_len_ok(int len, int stride, int positions) { return len >= 0 && len / PG_ROWS < stride && len < positions; }

/* the first visible row: window > 0 leaves the rows past len - window */
PG_FN int pg_first_row(int len, int window) { return window > 0 && len >= window ? len - window + 1 : 0; }

/* units of the rows [lo, len): the first and how many; top > 0: of min(top, pages) listed pages */
struct PgUnits {
    int first, n;
};
PG_FN PgUnits pg_units(int len, int stride, int positions, int window, int top, int unit) {
    PgUnits u = {0, 0};
    if (!pg_len_ok(len, stride, positions)) return u;
    if (top > 0) {
        const int pages = (len + PG_ROWS - 1) / PG_ROWS;
        u.n = (pages < top ? pages : top) * (PG_ROWS / unit);
        return u;
    }
    const int lo = pg_first_row(len, window);
    if (lo >= len) return u; /* a window of one row: the new token's alone */
    u.first = lo / unit;
    u.n = (len + unit - 1) / unit - u.first;
    return u;
}

/* What the start of a sequence costs a workgroup, in units: its rows of Q, and no unit under way before them. Measured with 0, 4, 12 and 24,
 * us: 16 sequences of 3000 to 4160 rows of codes 42.5, 40.2, 36.4 and 39.2; 24 of 500 to 8191 bf16 rows of head_dim 256 46.7, 44.0, 38.0
 * and 37.8; 64 of 4000 to 16384 rows of codes 256, 252, 251 and 255. */
#define PG_EXTRA 12

/* places of a sequence on the line */
PG_FN int pg_places(int len, int units) { return len < 0 ? 0 : PG_EXTRA + units; }

/* places of a piece, for `sum` of them in all: at most `slots` pieces */
PG_FN int pg_piece(long long sum, int slots) {
    long long c = (sum + slots - 1) / slots;
    c = (c + PG_WAVES - 1) / PG_WAVES * PG_WAVES;
    return c < PG_WAVES ? PG_WAVES : (int)c;
}

/* What piece w holds of a sequence whose places begin at `off`: units [u0, u1), of which it is number `nth` of `chunks` pieces; a sequence
 * without units belongs to the piece with its first place. A chunk of several leaves its state in place `slot`: 2 w when it is the
 * first of its piece, 2 w + 1 when it begins behind others; no piece has two of either. */
struct PgCut {
    bool mine;
    int u0, u1, nth, chunks;
};
PG_FN PgCut pg_cut(int off, int units, int piece, int w) {
    PgCut c = {false, 0, 0, 0, 1};
    const int at = off + PG_EXTRA, lo = w * piece, hi = lo + piece;
    if (units == 0) {
        c.mine = off >= lo && off < hi;
        return c;
    }
    c.u0 = lo > at ? lo - at : 0;
    c.u1 = hi < at + units ? hi - at : units;
    c.mine = c.u0 < c.u1;
    const int first = at / piece;
    c.nth = w - first;
    c.chunks = (at + units - 1) / piece - first + 1;
    return c;
}
PG_FN int pg_slot(int off, int piece, int nth) {
    const int at = off + PG_EXTRA, first = at / piece;
    return nth == 0 && at % piece ? 2 * first + 1 : 2 * (first + nth);
}

/* a page number that is none of the pool's */
PG_FN bool pg_bad_page(int page, int n_pages) { return page < 0 || page >= n_pages; }

/* Where row r of a page lies along V's line. The products of a page leave lane (c, g) with the weights of rows
 * 16 t + 4 g + i; in this order they are the operand of the product with V without a move between lanes. */
PG_FN int pg_order(int r, bool codes) {
    const int t = r >> 4, g = (r >> 2) & 3, i = r & 3;
    return codes ? g * 16 + t * 4 + i : (t >> 1) * 32 + g * 8 + (t & 1) * 4 + i;
}

/* ---- rows of a ragged batch, as smol_kv_pages_append and _read take them ---- */

/* sequence of input rows [start, end) of `rows`, at positions pos ..: its pages, 0 where it is empty or not to be used */
PG_FN bool pg_run_ok(int start, int end, int rows, int pos, int stride, int positions) {
    if (start < 0 || end < start || end > rows) return false;
    if (end == start) return true;
    return pos >= 0 && (long long)pos + (end - start) <= (long long)stride * PG_ROWS &&
           (long long)pos + (end - start) <= positions;
}
PG_FN int pg_run_pages(int start, int end, int rows, int pos, int stride, int positions) {
    if (!pg_run_ok(start, end, rows, pos, stride, positions) || end == start) return 0;
    return (pos + (end - start) - 1) / PG_ROWS - pos / PG_ROWS + 1;
}
/* workgroups along one axis of a grid: its threads are counted in 32 bits */
#define PG_TPB (64 * PG_WAVES) /* threads of a workgroup */
#define PG_APPEND_TPB 512      /* of one that writes rows */
PG_FN long long pg_max_blocks(int threads) { return 0xFFFFFFFFLL / threads; }
/* pages of all runs at most: each row opens one, and a run's first and last may be parts */
PG_FN long long pg_max_run_pages(int n, int rows) { return (long long)rows / PG_ROWS + 2LL * n; }

/* ---- 24-bit fixed point in three balanced base-256 digits ----
 * n in [-127 * 65536, 127 * 65536 + 1]: n = 65536 a + 256 b + c with a, b, c in [-128, 127]. Adding 128 to the two lower digits makes
 * them the bytes of a plain number, and taking it off each byte again is an exclusive or. */
#define PG_FIX (127.0f * 65536.0f)
PG_FN unsigned pg_digits(int n) { return ((unsigned)n + 0x8080u) ^ 0x8080u; }

#endif
