/*
 * paged_plan.h - which rows of a paged cache a workgroup takes: the part of
 * the kernels of paged.hip that decides what they touch. Plain C++ for host
 * and device, so that a CPU test covers it with every length and page number.
 *
 * A sequence of `len` cached rows and a table of `stride` pages: rows
 * [lo, len) are visible, cut into units of PG_UNIT rows (64 codes rows, or 32
 * bf16 rows, what one round of matrix products takes), and the units into
 * chunks, one workgroup each. The lengths are on the device, so every
 * workgroup forms the cut for itself from the sum of all sequences' units:
 * chunks of equal length, as short as leaves at most `slots` whole chunks and
 * one short one a sequence.
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

/* units of a chunk */
PG_FN int pg_chunk(long long sum, int slots) {
    long long c = (sum + slots - 1) / slots;
    c = (c + PG_WAVES - 1) / PG_WAVES * PG_WAVES;
    return c < PG_WAVES ? PG_WAVES : (int)c;
}

/* chunks of a sequence: one at least, which takes the new token; none for what is no sequence */
PG_FN int pg_chunks(int len, int units, int chunk) { return len < 0 ? 0 : units == 0 ? 1 : (units + chunk - 1) / chunk; }

/* workgroups that the chunks of n sequences need at most */
PG_FN long long pg_max_chunks(int n, int slots) { return (long long)slots + n; }

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
/* pages of all runs at most: each row opens one, and a run's first and last may be parts */
PG_FN long long pg_max_run_pages(int n, int rows) { return (long long)rows / PG_ROWS + 2LL * n; }

/* ---- 24-bit fixed point in three balanced base-256 digits ----
 * n in [-127 * 65536, 127 * 65536 + 1]: n = 65536 a + 256 b + c with a, b, c in [-128, 127]. Adding 128 to the two lower digits makes
 * them the bytes of a plain number, and taking it off each byte again is an exclusive or. */
#define PG_FIX 8323072.0f /* 127 * 65536 */
PG_FN unsigned pg_digits(int n) { return ((unsigned)n + 0x8080u) ^ 0x8080u; }

#endif
