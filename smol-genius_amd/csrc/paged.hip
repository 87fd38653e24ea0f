/*
 * paged.hip - a KV cache in pages of 64 rows, bf16 or codes of 8 bits: rows
 * into their pages (k_pg_append) and back (k_pg_read), a decode step over them
 * (k_pg, k_pg_merge), and the choice of the pages that such a step reads
 * (k_pg_score, k_pg_select). Layouts: attn_internal.h; who takes what:
 * paged_plan.h.
 */
#include "attn_device.h"
#include "paged_plan.h"

namespace {

typedef int i4 __attribute__((ext_vector_type(4)));
typedef unsigned short u2v __attribute__((ext_vector_type(2)));

constexpr int PG_TPB = 64 * PG_WAVES;
constexpr int PG_HEADS = 16; /* query heads of a tile: the columns of a matrix product */

template <int HD>
struct PgGeom {
    static constexpr int NE = (HD + 63) / 64;  /* elements of a row that a lane of a wave holds */
    static constexpr int DT = (HD + 15) / 16;  /* 16-wide tiles of the output */
    static constexpr int XSTR = HD + 4;        /* LDS stride of a row */
    static constexpr int CH8 = (HD + 15) / 16; /* 16-byte pieces of a row of codes */
    static constexpr int CHB = HD / 8;         /* of a bf16 row */
    static constexpr int KS8 = (HD + 63) / 64; /* matrix steps of a score: codes */
    static constexpr int KSB = (HD + 31) / 32; /* bf16 */
};

/* bytes of K and of V of one (page, kv head) */
template <int HD, bool CODES>
struct PgBytes {
    static constexpr int K = (CODES ? PgGeom<HD>::CH8 : PgGeom<HD>::CHB) * PG_ROWS * 16;
    static constexpr int V = PG_ROWS * HD * (CODES ? 1 : 2);
};

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int sh = 32; sh; sh >>= 1) v += __shfl_xor(v, sh);
    return v;
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int sh = 32; sh; sh >>= 1) v += __shfl_xor(v, sh);
    return v;
}
__device__ __forceinline__ unsigned wave_max(unsigned v) {
#pragma unroll
    for (int sh = 32; sh; sh >>= 1) v = max(v, (unsigned)__shfl_xor((int)v, sh));
    return v;
}
/* the largest over the four lanes of a column; as whole numbers, so that a NaN's bits are the largest of all */
__device__ __forceinline__ unsigned row_maxu4(unsigned v) {
    const auto a = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = max(a[0], a[1]);
    const auto b = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return max(b[0], b[1]);
}

__device__ __forceinline__ float in_at(const void *x, int dtype, long long i) {
    return dtype == SMOL_IN_BF16 ? bf16_to_f32(((const uint16_t *)x)[i]) : ((const float *)x)[i];
}

/* LDS that the lanes of one wave write and then read of each other */
__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

__device__ __forceinline__ float sqrt_of(float x) { return sqrtf(x); }
__device__ __forceinline__ double sqrt_of(double x) { return sqrt(x); }

/* One head's row by one wave, in two parts so that many rows' loads are in flight: its elements lane, lane + 64, ..; then
 * dst[d] = f * rope(x w / sqrt(mean x^2 + eps)). T double where pages are chosen by what comes of it. */
template <int HD>
struct PgRow {
    float x[PgGeom<HD>::NE], w[PgGeom<HD>::NE];
    __device__ __forceinline__ void load(const void *base, int dtype, long long row, const float *norm) {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int e = 0; e < PgGeom<HD>::NE; e++) {
            const int d = lane + 64 * e;
            x[e] = HD % 64 == 0 || d < HD ? in_at(base, dtype, row + d) : 0.0f;
            if (norm) w[e] = HD % 64 == 0 || d < HD ? norm[d] : 0.0f;
        }
    }
};
template <int HD>
struct PgTurn {
    float c[PgGeom<HD>::NE], s[PgGeom<HD>::NE];
    __device__ __forceinline__ void load(const PgPool &p, int pos) {
        const int lane = threadIdx.x & 63;
        if (p.rope_kind == SMOL_ROPE_OFF) return;
#pragma unroll
        for (int e = 0; e < PgGeom<HD>::NE; e++) {
            const int d = lane + 64 * e;
            c[e] = HD % 64 == 0 || d < HD ? p.rope_cos[(long long)pos * HD + d] : 0.0f;
            s[e] = HD % 64 == 0 || d < HD ? p.rope_sin[(long long)pos * HD + d] : 0.0f;
        }
    }
};
template <int HD, class T>
__device__ __forceinline__ void pg_finish(const PgRow<HD> &r, bool norm, float eps, const PgTurn<HD> &turn, int kind, T f, T *dst) {
    constexpr int NE = PgGeom<HD>::NE;
    const int lane = threadIdx.x & 63;
    T x[NE];
#pragma unroll
    for (int e = 0; e < NE; e++) x[e] = (T)r.x[e];
    if (norm) {
        T ss = 0;
#pragma unroll
        for (int e = 0; e < NE; e++) ss += x[e] * x[e];
        const T ri = (T)1 / sqrt_of(wave_sum(ss) / (T)HD + (T)eps);
#pragma unroll
        for (int e = 0; e < NE; e++) x[e] = x[e] * (T)r.w[e] * ri;
    }
    if (kind == SMOL_ROPE_OFF) {
#pragma unroll
        for (int e = 0; e < NE; e++)
            if (HD % 64 == 0 || lane + 64 * e < HD) dst[lane + 64 * e] = x[e] * f;
        wave_fence();
        return;
    }
#pragma unroll
    for (int e = 0; e < NE; e++)
        if (HD % 64 == 0 || lane + 64 * e < HD) dst[lane + 64 * e] = x[e];
    wave_fence();
    T y[NE];
#pragma unroll
    for (int e = 0; e < NE; e++) {
        const int d = lane + 64 * e;
        if (HD % 64 != 0 && d >= HD) continue;
        const T other = dst[rope_partner(d, HD, kind)];
        const bool low = kind == SMOL_ROPE_NEOX_K ? d < HD / 2 : (d & 1) == 0;
        y[e] = (x[e] * (T)turn.c[e] + (low ? -other : other) * (T)turn.s[e]) * f;
    }
    wave_fence();
#pragma unroll
    for (int e = 0; e < NE; e++)
        if (HD % 64 == 0 || lane + 64 * e < HD) dst[lane + 64 * e] = y[e];
    wave_fence();
}

/* ---- rows of codes ----
 * s = amax / 127, code = rint(x (127 / amax)); nothing but zeros where amax is below 2^-90 (its quotients would leave fp32's
 * range), and a scale that is no number where an element is none or infinite: such a row then spoils what reads it. */
#define PG_TINY 8.077935669463161e-28f /* 2^-90 */
struct PgScale {
    float s, inv;
};
__device__ __forceinline__ PgScale pg_scale(unsigned amax_bits) {
    const float a = __uint_as_float(amax_bits);
    if (amax_bits >= 0x7F800000u) return {__uint_as_float(0x7FC00000u), 0.0f};
    if (a < PG_TINY) return {0.0f, 0.0f};
    return {a / 127.0f, 127.0f / a};
}
__device__ __forceinline__ int pg_code(float x, float inv) {
    /* inv 0 with an infinite x is no number: 0, its scale tells */
    const float y = rintf(x * inv);
    return y == y ? (int)fminf(fmaxf(y, -127.0f), 127.0f) : 0;
}
/* the next bf16 at or below / above x (a NaN stays one) */
__device__ __forceinline__ uint16_t bf16_down(float x) {
    const unsigned u = __float_as_uint(x);
    if (!(x == x)) return 0x7FC0;
    return (uint16_t)((u >> 16) + ((u & 0x80000000u) && (u & 0xFFFFu) ? 1u : 0u));
}
__device__ __forceinline__ uint16_t bf16_up(float x) {
    const unsigned u = __float_as_uint(x);
    if (!(x == x)) return 0x7FC0;
    return (uint16_t)((u >> 16) + (!(u & 0x80000000u) && (u & 0xFFFFu) ? 1u : 0u));
}
/* fp32 to bf16, nearest even, a NaN stays one */
__device__ __forceinline__ uint16_t bf16_of(float f) { return f == f ? f32_to_bf16(f) : 0x7FC0; }
/* the smaller / larger, no number if either is none */
__device__ __forceinline__ float min_nan(float a, float b) { return a != a ? a : b != b ? b : fminf(a, b); }
__device__ __forceinline__ float max_nan(float a, float b) { return a != a ? a : b != b ? b : fmaxf(a, b); }

/* One row (HD values in LDS) into row r of page `page`, by one wave: K pieces or V's column, scale, and for K the page's bounds */
template <int HD, bool CODES, bool KEY>
__device__ void pg_store_row(const PgPool &p, int page, int g, int r, const float *x) {
    const int lane = threadIdx.x & 63;
    const long long at = (long long)page * p.Hkv + g;
    PgScale sc = {0.0f, 0.0f};
    if (CODES) {
        unsigned m = 0;
        for (int d = lane; d < HD; d += 64) m = max(m, __float_as_uint(x[d]) & 0x7FFFFFFFu);
        sc = pg_scale(wave_max(m));
        if (lane == 0) p.scales[(at * 2 + (KEY ? 0 : 1)) * PG_ROWS + r] = sc.s;
    }
    unsigned char *base = KEY ? p.k + at * PgBytes<HD, CODES>::K : p.v + at * PgBytes<HD, CODES>::V;
    for (int d = lane; d < HD; d += 64) {
        float kept;
        if (CODES) {
            const int c = pg_code(x[d], sc.inv);
            kept = (float)c * sc.s;
            if (KEY) ((signed char *)base)[((d >> 4) * PG_ROWS + r) * 16 + (d & 15)] = (signed char)c;
            else ((signed char *)base)[d * PG_ROWS + pg_order(r, true)] = (signed char)c;
        } else {
            const uint16_t b = bf16_of(x[d]);
            kept = bf16_to_f32(b);
            if (KEY) ((uint16_t *)base)[((d >> 3) * PG_ROWS + r) * 8 + (d & 7)] = b;
            else ((uint16_t *)base)[((r >> 5) * HD + d) * 32 + (pg_order(r, false) & 31)] = b;
        }
        if (KEY) {
            uint16_t *lo = p.bounds + at * 2 * HD + d, *hi = lo + HD;
            const float a = r == 0 ? kept : min_nan(kept, bf16_to_f32(*lo)), b = r == 0 ? kept : max_nan(kept, bf16_to_f32(*hi));
            *lo = bf16_down(a);
            *hi = bf16_up(b);
        }
    }
    /* the padding of a row's last piece */
    if (KEY && CODES && HD % 16 != 0 && lane < 16 - HD % 16)
        ((signed char *)base)[((HD >> 4) * PG_ROWS + r) * 16 + HD % 16 + lane] = 0;
}

/* ---- the plan, by one wave: which chunk of which sequence workgroup u takes ---- */
struct PgItem {
    int seq, len;
    PgUnits units;
    int item0, chunks; /* its chunks are items item0 .. */
};
__device__ __forceinline__ int wave_scan(int v) { /* inclusive sums over the lanes */
#pragma unroll
    for (int sh = 1; sh < 64; sh <<= 1) {
        const int x = __shfl_up(v, sh);
        if ((int)(threadIdx.x & 63) >= sh) v += x;
    }
    return v;
}
__device__ __forceinline__ PgUnits pg_units_of(const PgParams &p, int len) {
    return pg_units(len, p.p.stride, p.p.positions, p.window, p.top, pg_unit(p.p.codes));
}
/* units of a chunk of this call */
__device__ __forceinline__ int pg_chunk_of(const PgParams &p) {
    const int lane = threadIdx.x & 63;
    long long sum = 0;
    for (int b = 0; b < p.p.n_seq; b += 64) {
        const int i = b + lane;
        const int n = i < p.p.n_seq ? pg_units_of(p, p.len[i]).n : 0;
        sum += __shfl(wave_scan(n), 63);
    }
    return __builtin_amdgcn_readfirstlane(pg_chunk(sum, p.slots));
}
/* by item: the one whose items hold u; otherwise sequence u itself. false: none */
template <bool BY_ITEM>
__device__ __forceinline__ bool pg_find(const PgParams &p, int u, int chunk, PgItem &it) {
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int b = 0; b < p.p.n_seq; b += 64) {
        const int i = b + lane;
        const int len = i < p.p.n_seq ? p.len[i] : -1;
        const PgUnits un = pg_units_of(p, len);
        const int n = pg_chunks(len, un.n, chunk);
        const int end = before + wave_scan(n);
        const unsigned long long hit = BY_ITEM ? __ballot(end - n <= u && u < end) : __ballot(i == u && n > 0);
        if (hit) {
            const int from = __ffsll(hit) - 1;
            it.seq = b + from;
            it.len = __builtin_amdgcn_readlane(len, from);
            it.units.first = __builtin_amdgcn_readlane(un.first, from);
            it.units.n = __builtin_amdgcn_readlane(un.n, from);
            it.item0 = __builtin_amdgcn_readlane(end - n, from);
            it.chunks = __builtin_amdgcn_readlane(n, from);
            return true;
        }
        if (!BY_ITEM && u < b + 64) return false;
        before = __builtin_amdgcn_readlane(end, 63);
    }
    return false;
}

/* ---- one wave's softmax state over the units it takes ---- */
template <int HD>
struct PgState {
    float m, l;
    f4 o[PgGeom<HD>::DT]; /* rows: dims 4 g + i of tile dt, column: head */
};

__device__ __forceinline__ float pg_capped(float s, float cap2) { return cap2 > 0.0f ? cap2 * tanhf(s / cap2) : s; }

/* new maximum of the state: what it holds is scaled down to it */
template <int HD>
__device__ __forceinline__ void pg_raise(PgState<HD> &st, float m) {
    if (!__any(m > st.m)) return;
    const float mn = fmaxf(st.m, m), a = __builtin_amdgcn_exp2f(st.m - mn);
    st.m = mn;
    st.l *= a;
#pragma unroll
    for (int dt = 0; dt < PgGeom<HD>::DT; dt++) st.o[dt] *= a;
}

} // namespace

/* ------------------------------------------------------------------ decode */

/* Q of a tile as the matrix operand */
template <int HD, bool CODES>
struct PgQ;
template <int HD>
struct PgQ<HD, true> {
    i4 part[3][PgGeom<HD>::KS8]; /* digits of 65536, 256, 1 */
    float unit;                  /* what the last digit stands for */
    __device__ __forceinline__ void make(const float *row, bool live, int g) {
        constexpr int KS = PgGeom<HD>::KS8;
        float x[KS][16];
        unsigned m = 0;
#pragma unroll
        for (int ks = 0; ks < KS; ks++)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const int d = 64 * ks + 16 * g + e;
                f4 v = {0.f, 0.f, 0.f, 0.f};
                if (live && (HD % 64 == 0 || d < HD)) v = *reinterpret_cast<const f4 *>(row + d);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    x[ks][e + i] = v[i];
                    m = max(m, __float_as_uint(v[i]) & 0x7FFFFFFFu);
                }
            }
        m = row_maxu4(m);
        const float a = __uint_as_float(m);
        /* 24-bit whole numbers against the row's largest element; a row with no number or an infinity: no numbers; one that is
         * all but zero: zeros */
        const float inv = m >= 0x7F800000u || a < PG_TINY ? 0.0f : PG_FIX / a;
        unit = m >= 0x7F800000u ? __uint_as_float(0x7FC00000u) : a < PG_TINY ? 0.0f : a / PG_FIX;
#pragma unroll
        for (int ks = 0; ks < KS; ks++)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                unsigned w[3] = {0, 0, 0};
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float y = rintf(x[ks][e + i] * inv);
                    const unsigned n = pg_digits(y == y ? (int)y : 0);
                    w[0] |= ((n >> 16) & 0xFFu) << 8 * i;
                    w[1] |= ((n >> 8) & 0xFFu) << 8 * i;
                    w[2] |= (n & 0xFFu) << 8 * i;
                }
#pragma unroll
                for (int q = 0; q < 3; q++) part[q][ks][e / 4] = (int)w[q];
            }
    }
};
template <int HD>
struct PgQ<HD, false> {
    b8 part[3][PgGeom<HD>::KSB];
    __device__ __forceinline__ void make(const float *row, bool live, int g) {
#pragma unroll
        for (int ks = 0; ks < PgGeom<HD>::KSB; ks++) {
            const int d = 32 * ks + 8 * g;
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = live && (HD % 32 == 0 || d < HD) ? row[d + e] : 0.0f;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const __bf16 a = (__bf16)x[e];
                const float r = x[e] - (float)a;
                const __bf16 b = (__bf16)r;
                part[0][ks][e] = a;
                part[1][ks][e] = b;
                part[2][ks][e] = (__bf16)(r - (float)b);
            }
        }
    }
};

/* one unit's rows in registers */
template <int HD, bool CODES>
struct PgUnitRegs;
template <int HD>
struct PgUnitRegs<HD, true> {
    i4 k[4][PgGeom<HD>::KS8], v[PgGeom<HD>::DT];
    f4 ks[4], vs[4];
    __device__ __forceinline__ void load(const PgPool &p, int page, int kvh, int half, int c, int g) {
        const long long at = (long long)page * p.Hkv + kvh;
        const unsigned char *kb = p.k + at * PgBytes<HD, true>::K, *vb = p.v + at * PgBytes<HD, true>::V;
        const float *sb = p.scales + at * 2 * PG_ROWS;
#pragma unroll
        for (int t = 0; t < 4; t++) ks[t] = *reinterpret_cast<const f4 *>(sb + 16 * t + 4 * g);
#pragma unroll
        for (int s = 0; s < PgGeom<HD>::KS8; s++)
#pragma unroll
            for (int t = 0; t < 4; t++) {
                const int ch = 4 * s + g;
                k[t][s] = i4{0, 0, 0, 0};
                if (HD % 64 == 0 || ch < PgGeom<HD>::CH8) k[t][s] = *reinterpret_cast<const i4 *>(kb + (ch * PG_ROWS + 16 * t + c) * 16);
            }
#pragma unroll
        for (int t = 0; t < 4; t++) vs[t] = *reinterpret_cast<const f4 *>(sb + PG_ROWS + 16 * t + 4 * g);
#pragma unroll
        for (int dt = 0; dt < PgGeom<HD>::DT; dt++) {
            const int d = 16 * dt + c;
            v[dt] = i4{0, 0, 0, 0};
            if (HD % 16 == 0 || d < HD) v[dt] = *reinterpret_cast<const i4 *>(vb + d * PG_ROWS + 16 * g);
        }
    }
};
template <int HD>
struct PgUnitRegs<HD, false> {
    uint4 k[2][PgGeom<HD>::KSB], v[PgGeom<HD>::DT];
    __device__ __forceinline__ void load(const PgPool &p, int page, int kvh, int half, int c, int g) {
        const long long at = (long long)page * p.Hkv + kvh;
        const unsigned char *kb = p.k + at * PgBytes<HD, false>::K + half * 512;
        const unsigned char *vb = p.v + at * PgBytes<HD, false>::V + half * HD * 64;
#pragma unroll
        for (int s = 0; s < PgGeom<HD>::KSB; s++)
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const int ch = 4 * s + g;
                k[t][s] = make_uint4(0, 0, 0, 0);
                if (HD % 32 == 0 || ch < PgGeom<HD>::CHB) k[t][s] = *reinterpret_cast<const uint4 *>(kb + (ch * PG_ROWS + 16 * t + c) * 16);
            }
#pragma unroll
        for (int dt = 0; dt < PgGeom<HD>::DT; dt++) {
            const int d = 16 * dt + c;
            v[dt] = make_uint4(0, 0, 0, 0);
            if (HD % 16 == 0 || d < HD) v[dt] = *reinterpret_cast<const uint4 *>(vb + d * 64 + 16 * g);
        }
    }
};

/* A unit of codes joins the state; visible rows of it [lo, hi).
 * A score is exact up to its last sum: K's codes and the digits of Q are whole numbers, and so are their dot products. The
 * weights p vs (vs: V's scales) are taken against the unit's largest as 24-bit whole numbers, digit by digit on the matrix
 * cores again, so V needs no conversion either. */
template <int HD>
__device__ __forceinline__ void pg_take(PgState<HD> &st, const PgQ<HD, true> &q, PgUnitRegs<HD, true> &u, float cap2, int g, int lo, int hi) {
    constexpr int DT = PgGeom<HD>::DT;
    const i4 zero = {0, 0, 0, 0};
    const bool part = lo > 0 || hi < 64;
    float s[4][4];
    if (part) { /* the scales of rows that are not seen could be anything */
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int r = 16 * t + 4 * g + i;
                if (r < lo || r >= hi) u.ks[t][i] = u.vs[t][i] = 0.0f;
            }
    }
    unsigned kbits = 0, vbits = 0;
#pragma unroll
    for (int t = 0; t < 4; t++) {
        i4 d0 = zero, d1 = zero, d2 = zero;
#pragma unroll
        for (int ks = 0; ks < PgGeom<HD>::KS8; ks++) {
            d0 = __builtin_amdgcn_mfma_i32_16x16x64_i8(u.k[t][ks], q.part[0][ks], d0, 0, 0, 0);
            d1 = __builtin_amdgcn_mfma_i32_16x16x64_i8(u.k[t][ks], q.part[1][ks], d1, 0, 0, 0);
            d2 = __builtin_amdgcn_mfma_i32_16x16x64_i8(u.k[t][ks], q.part[2][ks], d2, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            s[t][i] = fmaf((float)d0[i], 65536.0f, fmaf((float)d1[i], 256.0f, (float)d2[i])) * (q.unit * u.ks[t][i]);
            kbits = max(kbits, __float_as_uint(u.ks[t][i]));
            vbits = max(vbits, __float_as_uint(u.vs[t][i]));
        }
    }
    if (cap2 > 0.0f) {
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) s[t][i] = pg_capped(s[t][i], cap2);
    }
    if (part) {
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int r = 16 * t + 4 * g + i;
                if (r < lo || r >= hi) s[t][i] = -INFINITY;
            }
    }
    float mu = s[0][0];
#pragma unroll
    for (int e = 1; e < 16; e++) mu = fmaxf(mu, s[e >> 2][e & 3]);
    mu = row_max4(mu);
    vbits = row_maxu4(vbits);
    const float top = __uint_as_float(vbits), f = top > 0.0f ? 1.0f / top : 0.0f;
    float sum = 0.0f;
    i4 w0, w1, w2;
#pragma unroll
    for (int t = 0; t < 4; t++) {
        unsigned x[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float pr = __builtin_amdgcn_exp2f(s[t][i] - mu);
            sum += pr;
            /* 2^23 + n: the low bits of the sum are the whole number n, rounded to nearest */
            const float y = fmaf(pr * (u.vs[t][i] * f), PG_FIX, 8388608.0f);
            x[i] = (__float_as_uint(y) + 0x8080u) ^ 0x8080u;
        }
        const unsigned l01 = __builtin_amdgcn_perm(x[1], x[0], 0x05010400u), l23 = __builtin_amdgcn_perm(x[3], x[2], 0x05010400u);
        const unsigned h01 = __builtin_amdgcn_perm(x[1], x[0], 0x0c0c0602u), h23 = __builtin_amdgcn_perm(x[3], x[2], 0x0c0c0602u);
        w0[t] = (int)__builtin_amdgcn_perm(h23, h01, 0x05040100u);
        w1[t] = (int)__builtin_amdgcn_perm(l23, l01, 0x07060302u);
        w2[t] = (int)__builtin_amdgcn_perm(l23, l01, 0x05040100u);
    }
    pg_raise(st, mu);
    const float b = __builtin_amdgcn_exp2f(mu - st.m);
    /* a scale that is no number, or infinite, spoils the sum */
    st.l = fmaf(b, sum, st.l) + (0.0f * __uint_as_float(kbits) + 0.0f * top);
    const float bo = b * (top * (1.0f / PG_FIX));
#pragma unroll
    for (int dt = 0; dt < DT; dt++) {
        const i4 e0 = __builtin_amdgcn_mfma_i32_16x16x64_i8(u.v[dt], w0, zero, 0, 0, 0);
        const i4 e1 = __builtin_amdgcn_mfma_i32_16x16x64_i8(u.v[dt], w1, zero, 0, 0, 0);
        const i4 e2 = __builtin_amdgcn_mfma_i32_16x16x64_i8(u.v[dt], w2, zero, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 4; i++)
            st.o[dt][i] = fmaf(fmaf((float)e0[i], 65536.0f, fmaf((float)e1[i], 256.0f, (float)e2[i])), bo, st.o[dt][i]);
    }
}

/* A unit of 32 bf16 rows joins the state. Q and the weights are split into three bf16 parts each (24 bits). */
template <int HD>
__device__ __forceinline__ void pg_take(PgState<HD> &st, const PgQ<HD, false> &q, PgUnitRegs<HD, false> &u, float cap2, int g, int lo, int hi) {
    constexpr int DT = PgGeom<HD>::DT;
    const bool part = lo > 0 || hi < 32;
    f4 s[2];
#pragma unroll
    for (int t = 0; t < 2; t++) {
        s[t] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int pt = 2; pt >= 0; pt--)
#pragma unroll
            for (int ks = 0; ks < PgGeom<HD>::KSB; ks++)
                s[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_b8(u.k[t][ks]), q.part[pt][ks], s[t], 0, 0, 0);
    }
    float odd = 0.0f; /* no number if a visible score is none, or infinite */
    if (part) {
        /* rows that are not seen: no score, and zeros for values (0 times an infinity is no number) */
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int r = 16 * t + 4 * g + i;
                if (r < lo || r >= hi) s[t][i] = 0.0f;
            }
#pragma unroll
        for (int dt = 0; dt < DT; dt++) {
            unsigned w[4] = {u.v[dt].x, u.v[dt].y, u.v[dt].z, u.v[dt].w};
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int r = 16 * (e >> 2) + 4 * g + (e & 3);
                if (r < lo || r >= hi) w[e >> 1] &= e & 1 ? 0x0000FFFFu : 0xFFFF0000u;
            }
            u.v[dt] = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) odd = fmaf(s[t][i], 0.0f, odd);
    if (cap2 > 0.0f) {
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) s[t][i] = pg_capped(s[t][i], cap2);
    }
    if (part) {
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int r = 16 * t + 4 * g + i;
                if (r < lo || r >= hi) s[t][i] = -INFINITY;
            }
    }
    float mu = s[0][0];
#pragma unroll
    for (int e = 1; e < 8; e++) mu = fmaxf(mu, s[e >> 2][e & 3]);
    pg_raise(st, row_max4(mu));
    float sum = odd;
    b8 w[3];
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const float pr = __builtin_amdgcn_exp2f(s[e >> 2][e & 3] - st.m);
        sum += pr;
        const __bf16 a = (__bf16)pr;
        const float r = pr - (float)a;
        const __bf16 b = (__bf16)r;
        w[0][e] = a;
        w[1][e] = b;
        w[2][e] = (__bf16)(r - (float)b);
    }
    st.l += sum;
#pragma unroll
    for (int pt = 2; pt >= 0; pt--)
#pragma unroll
        for (int dt = 0; dt < DT; dt++) st.o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_b8(u.v[dt]), w[pt], st.o[dt], 0, 0, 0);
}

/* A chunk of a sequence's units against a tile of 16 heads of a kv head; the last chunk also takes the new token and stores
 * its row. */
template <int HD, bool CODES>
__global__ __launch_bounds__(PG_TPB) void k_pg(const PgParams p) {
    constexpr int XS = PgGeom<HD>::XSTR, DT = PgGeom<HD>::DT, U = CODES ? 64 : 32;
    /* the rows of Q (scaled), the new key; then the waves' outputs */
    __shared__ __align__(16) float s_mem[PG_WAVES * PG_HEADS * XS];
    __shared__ float s_v[HD], s_m[PG_WAVES + 1][PG_HEADS], s_l[PG_WAVES][PG_HEADS];
    __shared__ int s_bad[PG_HEADS];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, g = lane >> 4;
    const int kvh = blockIdx.y, tile = blockIdx.z, h0 = tile * PG_HEADS, R = min(PG_HEADS, p.G - h0);
    const int chunk = pg_chunk_of(p);
    PgItem it;
    if (!pg_find<true>(p, blockIdx.x, chunk, it)) return;
    const int nth = blockIdx.x - it.item0, u0 = nth * chunk, u1 = min(it.units.n, u0 + chunk);
    const bool ok = pg_len_ok(it.len, p.p.stride, p.p.positions), last = nth == it.chunks - 1;
    const int *row_table = p.p.table + (long long)it.seq * p.p.stride;
    const int *list = p.top > 0 ? p.list + ((long long)it.seq * p.p.Hkv + kvh) * p.top : nullptr;
    bool bad = !ok;

    /* the pages of this wave's first 64 units */
    int at = 0, page = 0; /* of unit u0 + wave + 4 lane: its first row, its page */
    auto pages = [&](int from) {
        const int un = from + PG_WAVES * lane;
        at = page = 0;
        if (un < u1) {
            const int row = list ? list[un / (PG_ROWS / U)] * PG_ROWS + un % (PG_ROWS / U) * U : (it.units.first + un) * U;
            at = row;
            page = row_table[row / PG_ROWS];
            if (pg_bad_page(page, p.p.n_pages)) {
                bad = true;
                page = 0;
            }
        }
    };
    pages(u0 + wave);
    int new_page = 0;
    if (last && ok) {
        new_page = row_table[it.len / PG_ROWS];
        if (pg_bad_page(new_page, p.p.n_pages)) {
            bad = true;
            new_page = -1;
        }
    }
    {
        /* rows of Q and the new key, normalised and rotated */
        constexpr int NR = (PG_HEADS + 1 + PG_WAVES - 1) / PG_WAVES;
        PgRow<HD> r[NR];
        PgTurn<HD> turn;
        const int n = R + (last ? 1 : 0), pos = ok ? it.len : 0;
#pragma unroll
        for (int k = 0; k < NR; k++) {
            const int i = wave + PG_WAVES * k;
            if (i < n) {
                const bool key = i == R;
                r[k].load(key ? p.k_in : p.q_in, p.in_dtype,
                          key ? ((long long)it.seq * p.p.Hkv + kvh) * HD : ((long long)it.seq * p.Hq + kvh * p.G + h0 + i) * HD,
                          key ? p.k_norm : p.q_norm);
            }
        }
        turn.load(p.p, pos);
        if (last)
            for (int d = tid; d < HD; d += PG_TPB) s_v[d] = in_at(p.v_in, p.in_dtype, ((long long)it.seq * p.p.Hkv + kvh) * HD + d);
#pragma unroll
        for (int k = 0; k < NR; k++) {
            const int i = wave + PG_WAVES * k;
            if (i < n) {
                const bool key = i == R;
                pg_finish<HD, float>(r[k], (key ? p.k_norm : p.q_norm) != nullptr, p.norm_eps, turn, p.p.rope_kind, key ? 1.0f : p.qscale,
                                     s_mem + i * XS);
            }
        }
    }
    if (tid < PG_HEADS) s_bad[tid] = 0;
    __syncthreads();
    PgQ<HD, CODES> q;
    q.make(s_mem + c * XS, c < R, g);

    PgState<HD> st;
    st.m = -INFINITY;
    st.l = 0.0f;
#pragma unroll
    for (int dt = 0; dt < DT; dt++) st.o[dt] = f4{0.f, 0.f, 0.f, 0.f};
    const int lo = p.top > 0 ? 0 : pg_first_row(it.len, p.window);
    for (int un = u0 + wave, n = 0; un < u1; un += PG_WAVES, n++) {
        if (n == 64) {
            pages(un);
            n = 0;
        }
        const int row = __builtin_amdgcn_readlane(at, n), pg = __builtin_amdgcn_readlane(page, n);
        if (row >= it.len) continue; /* the second half of a listed page that ends before it */
        PgUnitRegs<HD, CODES> u;
        u.load(p.p, pg, kvh, CODES ? 0 : row % PG_ROWS / 32, c, g);
        pg_take<HD>(st, q, u, p.cap2, g, max(0, lo - row), min(U, it.len - row));
    }
    if (__any(bad)) {
        if (lane == 0) *p.p.flag = 1;
        st.l = __uint_as_float(0x7FC00000u);
    }
    st.l = row_sum4(st.l);

    if (last) {
        /* the new token's scores, and its row into its page */
        for (int r = wave; r < R; r += PG_WAVES) {
            float d = 0.0f;
#pragma unroll
            for (int e = 0; e < PgGeom<HD>::NE; e++)
                if (HD % 64 == 0 || lane + 64 * e < HD) d = fmaf(s_mem[r * XS + lane + 64 * e], s_mem[R * XS + lane + 64 * e], d);
            d = wave_sum(d);
            /* an infinite score is no number, also behind a cap */
            if (lane == 0) s_m[PG_WAVES][r] = pg_capped(d, p.cap2) + 0.0f * d;
        }
        if (tile == 0 && ok && new_page >= 0) {
            if (wave == 2) pg_store_row<HD, CODES, true>(p.p, new_page, kvh, it.len % PG_ROWS, s_mem + R * XS);
            if (wave == 3) pg_store_row<HD, CODES, false>(p.p, new_page, kvh, it.len % PG_ROWS, s_v);
        }
    }
    __syncthreads();
    if (c < R) {
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
            if (HD % 16 == 0 || 16 * dt + 4 * g < HD) *reinterpret_cast<f4 *>(s_mem + (wave * PG_HEADS + c) * XS + 16 * dt + 4 * g) = st.o[dt];
        if (g == 0) {
            s_m[wave][c] = st.m;
            s_l[wave][c] = st.l;
        }
    }
    __syncthreads();
    /* the waves' states and the new token's as one */
    const bool whole = it.chunks == 1;
    const long long prow = ((long long)kvh * p.max_items + blockIdx.x) * p.G + h0;
    float *out = whole ? p.out + ((long long)it.seq * p.Hq + kvh * p.G + h0) * HD : p.part_o + prow * HD;
    constexpr int QD = HD / 4;
    auto join = [&](int e, f4 &o) {
        const int r = e / QD, d = e % QD * 4;
        float m = last ? s_m[PG_WAVES][r] : -INFINITY;
        const float mn = m;
#pragma unroll
        for (int w = 0; w < PG_WAVES; w++) m = fmaxf(m, s_m[w][r]);
        float l = 0.0f;
        o = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < PG_WAVES; w++) {
            const float lw = s_l[w][r], f = s_m[w][r] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(s_m[w][r] - m);
            l = fmaf(f, lw, l);
            if (lw != lw) l = lw; /* a wave that saw nothing but rows that are no numbers */
            o += *reinterpret_cast<const f4 *>(s_mem + (w * PG_HEADS + r) * XS + d) * f;
        }
        if (last) {
            const float f = mn != mn ? mn : __builtin_amdgcn_exp2f(mn - m);
            l += f;
            o += *reinterpret_cast<const f4 *>(s_v + d) * f;
        }
        if (!whole) {
            if (d == 0) {
                p.part_ml[(prow + r) * 2] = m;
                p.part_ml[(prow + r) * 2 + 1] = l;
            }
            return;
        }
        o *= 1.0f / l;
        /* what is not finite in one dim spoils the row */
        if (!(fabsf(o[0]) + fabsf(o[1]) + fabsf(o[2]) + fabsf(o[3]) < INFINITY)) s_bad[r] = 1;
    };
    constexpr int NJ = (PG_HEADS * QD + PG_TPB - 1) / PG_TPB;
    f4 o[NJ];
#pragma unroll
    for (int k = 0; k < NJ; k++)
        if (tid + k * PG_TPB < R * QD) join(tid + k * PG_TPB, o[k]);
    if (whole) __syncthreads();
#pragma unroll
    for (int k = 0; k < NJ; k++) {
        const int e = tid + k * PG_TPB;
        if (e >= R * QD) continue;
        if (whole && s_bad[e / QD]) o[k] = f4{NAN, NAN, NAN, NAN};
        *reinterpret_cast<f4 *>(out + (long long)e * 4) = o[k];
    }
}

/* Joins the chunks of a sequence that has more than one: a workgroup a (sequence, kv head) */
template <int HD>
__global__ __launch_bounds__(PG_TPB) void k_pg_merge(const PgParams p) {
    constexpr int QD = HD / 4;
    __shared__ int s_bad[PG_HEADS];
    const int tid = threadIdx.x, kvh = blockIdx.y, h0 = blockIdx.z * PG_HEADS, R = min(PG_HEADS, p.G - h0);
    const int chunk = pg_chunk_of(p);
    PgItem it;
    if (!pg_find<false>(p, blockIdx.x, chunk, it) || it.chunks == 1) return;
    if (tid < PG_HEADS) s_bad[tid] = 0;
    __syncthreads();
    const long long base = ((long long)kvh * p.max_items + it.item0) * p.G + h0;
    float *out = p.out + ((long long)it.seq * p.Hq + kvh * p.G + h0) * HD;
    constexpr int NJ = (PG_HEADS * QD + PG_TPB - 1) / PG_TPB;
    f4 o[NJ];
#pragma unroll
    for (int k = 0; k < NJ; k++) {
        const int e = tid + k * PG_TPB, r = e / QD, d = e % QD * 4;
        if (e >= R * QD) continue;
        float m = -INFINITY, l = 0.0f;
        f4 a = {0.f, 0.f, 0.f, 0.f};
        for (int n = 0; n < it.chunks; n++) {
            const long long row = base + (long long)n * p.G + r;
            const float mc = p.part_ml[row * 2], lc = p.part_ml[row * 2 + 1];
            const f4 oc = *reinterpret_cast<const f4 *>(p.part_o + row * HD + d);
            const float mn = fmaxf(m, mc), fa = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
            const float fb = mc == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mc - mn);
            l = l * fa + lc * fb;
            if (lc != lc) l = lc;
            a = a * fa + oc * fb;
            m = mn;
        }
        a *= 1.0f / l;
        if (!(fabsf(a[0]) + fabsf(a[1]) + fabsf(a[2]) + fabsf(a[3]) < INFINITY)) s_bad[r] = 1;
        o[k] = a;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < NJ; k++) {
        const int e = tid + k * PG_TPB;
        if (e >= R * QD) continue;
        if (s_bad[e / QD]) o[k] = f4{NAN, NAN, NAN, NAN};
        *reinterpret_cast<f4 *>(out + (long long)e * 4) = o[k];
    }
}

/* ------------------------------------------------------- which pages to read */

namespace {
constexpr int PS_PAGES = 64;   /* pages of a k_pg_score workgroup */
constexpr int PS_BINS = 2048;
constexpr int PS_LDS = 4096;   /* pages whose keys k_pg_select keeps in LDS */

__device__ __forceinline__ int pg_pages(int len) { return (len + PG_ROWS - 1) / PG_ROWS; }
} // namespace

/* score = sum over the heads of a kv head and the dims of max(q lo, q hi): an upper bound of the sum of a page's scores,
 * q+ . hi + q- . lo with q+ (q-) the sums of the heads' positive (negative) elements, so a page costs two products whatever the
 * number of heads. In 64 bits, and a page's terms in one order whatever the page: pages with equal bounds tie. */
template <int HD>
__global__ __launch_bounds__(PG_TPB) void k_pg_score(const PgParams p) {
    constexpr int LPP = HD <= 64 ? 8 : HD <= 128 ? 16 : 32, NE = PgGeom<HD>::NE;
    __shared__ double s_row[PG_WAVES][HD], s_sum[PG_WAVES][2][HD];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), kvh = blockIdx.y;
    const int blocks = (p.p.stride + PS_PAGES - 1) / PS_PAGES, seq = blockIdx.x / blocks, j0 = blockIdx.x % blocks * PS_PAGES;
    const int len = p.len[seq];
    if (!pg_len_ok(len, p.p.stride, p.p.positions)) return;
    const int pages = pg_pages(len);
    if (pages <= p.top || j0 >= pages) return;
    PgTurn<HD> turn;
    turn.load(p.p, len);
    double up[NE], dn[NE];
#pragma unroll
    for (int e = 0; e < NE; e++) up[e] = dn[e] = 0.0;
    for (int h = wave; h < p.G; h += PG_WAVES) {
        PgRow<HD> r;
        r.load(p.q_in, p.in_dtype, ((long long)seq * p.Hq + kvh * p.G + h) * HD, p.q_norm);
        pg_finish<HD, double>(r, p.q_norm != nullptr, p.norm_eps, turn, p.p.rope_kind, p.scale, s_row[wave]);
#pragma unroll
        for (int e = 0; e < NE; e++) {
            if (HD % 64 != 0 && lane + 64 * e >= HD) continue;
            const double x = s_row[wave][lane + 64 * e];
            up[e] += x > 0.0 ? x : 0.0; /* a NaN makes none of both */
            dn[e] += x > 0.0 ? 0.0 : x;
        }
    }
#pragma unroll
    for (int e = 0; e < NE; e++)
        if (HD % 64 == 0 || lane + 64 * e < HD) {
            s_sum[wave][0][lane + 64 * e] = up[e];
            s_sum[wave][1][lane + 64 * e] = dn[e];
        }
    __syncthreads();
    const int ch = lane % LPP;
    const bool live = 8 * ch < HD;
    double u[8], d[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        u[i] = d[i] = 0.0;
        if (!live) continue;
#pragma unroll
        for (int w = 0; w < PG_WAVES; w++) {
            u[i] += s_sum[w][0][8 * ch + i];
            d[i] += s_sum[w][1][8 * ch + i];
        }
    }
    const int *row_table = p.p.table + (long long)seq * p.p.stride;
    double *score = p.score + ((long long)seq * p.p.Hkv + kvh) * p.p.stride;
    for (int j = j0 + tid / LPP; j < min(j0 + PS_PAGES, (pages + 63) & ~63); j += PG_TPB / LPP) {
        double s = 0.0;
        bool bad = false;
        if (j < pages && live) {
            int page = row_table[j];
            if ((bad = pg_bad_page(page, p.p.n_pages))) page = 0;
            const uint16_t *b = p.p.bounds + ((long long)page * p.p.Hkv + kvh) * 2 * HD + 8 * ch;
            float lo[8], hi[8];
            unpack_bf16x8(*reinterpret_cast<const uint4 *>(b), lo);
            unpack_bf16x8(*reinterpret_cast<const uint4 *>(b + HD), hi);
#pragma unroll
            for (int i = 0; i < 8; i++) s = fma(u[i], (double)hi[i], fma(d[i], (double)lo[i], s));
        }
#pragma unroll
        for (int sh = LPP / 2; sh; sh >>= 1) s += __shfl_xor(s, sh);
        if (bad) s = __longlong_as_double(0x7FF8000000000000LL);
        if (j < pages && ch == 0) score[j] = s;
    }
}

namespace {
/* a score as a whole number of the same order: what stays by its place above all, then NaN, then the numbers (-0 as 0) */
__device__ __forceinline__ unsigned long long pg_key(double s, int j, int pages, int first, int recent) {
    if (j < first || j >= pages - recent) return ~0ULL;
    if (!(s == s)) return ~0ULL - 1;
    const unsigned long long u = s == 0.0 ? 0ULL : (unsigned long long)__double_as_longlong(s);
    return u >> 63 ? ~u : u | 0x8000000000000000ULL;
}
} // namespace

/* The `top` pages of the largest keys of one (sequence, kv head), in ascending order. The top-th largest key is found by the
 * highest eleven bits in which the keys still in question differ, again and again: a histogram of them in LDS says which bin
 * holds it. Mostly two rounds: the first leaves a few keys. */
template <bool LDS>
__global__ __launch_bounds__(PG_TPB) void k_pg_select(const PgParams p) {
    __shared__ unsigned long long s_key[LDS ? PS_LDS : 1], s_or[PG_WAVES], s_and[PG_WAVES];
    __shared__ int s_hist[PS_BINS], s_part[PG_WAVES], s_found[2];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, seq = blockIdx.x, kvh = blockIdx.y;
    const int len = p.len[seq];
    if (!pg_len_ok(len, p.p.stride, p.p.positions)) return;
    const int pages = pg_pages(len);
    int *list = p.list + ((long long)seq * p.p.Hkv + kvh) * p.top;
    if (pages <= p.top) {
        for (int j = tid; j < p.top; j += PG_TPB) list[j] = j < pages ? j : -1;
        return;
    }
    const double *score = p.score + ((long long)seq * p.p.Hkv + kvh) * p.p.stride;
    if (LDS) {
        for (int j = tid; j < pages; j += PG_TPB) s_key[j] = pg_key(score[j], j, pages, p.first, p.recent);
        __syncthreads();
    }
    auto key = [&](int j) { return LDS ? s_key[j] : pg_key(score[j], j, pages, p.first, p.recent); };
    unsigned long long prefix = 0, mask = 0; /* in question: keys with (key & mask) == prefix; larger ones are taken */
    int need = p.top, held = pages;          /* to take of those in question, and how many there are */
    while (held > need) {
        unsigned long long any = 0, all = ~0ULL;
        for (int j = tid; j < pages; j += PG_TPB) {
            const unsigned long long k = key(j);
            if ((k & mask) == prefix) {
                any |= k;
                all &= k;
            }
        }
#pragma unroll
        for (int sh = 32; sh; sh >>= 1) {
            any |= __shfl_xor(any, sh);
            all &= __shfl_xor(all, sh);
        }
        if (lane == 0) {
            s_or[wave] = any;
            s_and[wave] = all;
        }
        for (int b = tid; b < PS_BINS; b += PG_TPB) s_hist[b] = 0;
        __syncthreads();
        any = 0;
        all = ~0ULL;
#pragma unroll
        for (int w = 0; w < PG_WAVES; w++) {
            any |= s_or[w];
            all &= s_and[w];
        }
        const unsigned long long differ = any & ~all;
        if (differ == 0) break; /* all equal: the lowest pages of them */
        const int shift = max(0, 63 - __clzll(differ) - 10);
        for (int j = tid; j < pages; j += PG_TPB) {
            const unsigned long long k = key(j);
            if ((k & mask) == prefix) atomicAdd(&s_hist[(k >> shift) & (PS_BINS - 1)], 1);
        }
        __syncthreads();
        constexpr int NB = PS_BINS / PG_TPB;
        int cnt[NB], sum = 0;
#pragma unroll
        for (int b = 0; b < NB; b++) sum += cnt[b] = s_hist[PS_BINS - 1 - NB * tid - b];
        const int incl = wave_scan(sum);
        if (lane == 63) s_part[wave] = incl;
        __syncthreads();
        int above = incl - sum;
#pragma unroll
        for (int w = 0; w < PG_WAVES; w++)
            if (w < wave) above += s_part[w];
#pragma unroll
        for (int b = 0; b < NB; b++) {
            if (above < need && above + cnt[b] >= need) {
                s_found[0] = PS_BINS - 1 - NB * tid - b;
                s_found[1] = need - above;
            }
            above += cnt[b];
        }
        __syncthreads();
        const int bin = s_found[0];
        held = s_hist[bin];
        need = s_found[1];
        /* the bits at and above the bin's are known now: those above it are the same in all keys in question */
        mask = ~((1ULL << shift) - 1);
        prefix = (shift + 11 < 64 ? all >> (shift + 11) << (shift + 11) : 0ULL) | (unsigned long long)bin << shift;
        __syncthreads();
    }
    /* keys above the prefix, and the lowest `need` pages at it, by threads that take consecutive pages */
    const int per = (pages + PG_TPB - 1) / PG_TPB, b0 = min(pages, tid * per), b1 = min(pages, b0 + per);
    int eq = 0, more = 0;
    for (int j = b0; j < b1; j++) {
        const unsigned long long k = key(j) & mask;
        eq += k == prefix;
        more += k > prefix;
    }
    const int ie = wave_scan(eq);
    __syncthreads();
    if (lane == 63) s_part[wave] = ie;
    __syncthreads();
    int e = ie - eq;
#pragma unroll
    for (int w = 0; w < PG_WAVES; w++)
        if (w < wave) e += s_part[w];
    const int mine = more + max(0, min(need, e + eq) - min(need, e));
    const int im = wave_scan(mine);
    __syncthreads();
    if (lane == 63) s_part[wave] = im;
    __syncthreads();
    int at = im - mine;
#pragma unroll
    for (int w = 0; w < PG_WAVES; w++)
        if (w < wave) at += s_part[w];
    for (int j = b0; j < b1; j++) {
        const unsigned long long k = key(j) & mask;
        if (k > prefix || (k == prefix && e < need)) list[at++] = j;
        e += k == prefix;
    }
}

/* ------------------------------------------------------ rows in and out */

namespace {
struct PgRun {
    int seq, page, in0, r0, r1; /* rows [r0, r1) of `page`, from input row in0 */
};
/* page `u` of the runs of the batch, by one wave */
__device__ __forceinline__ bool pg_find_run(const PgRunParams &p, int u, PgRun &run) {
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int b = 0; b < p.p.n_seq; b += 64) {
        const int i = b + lane;
        int n = 0, start = 0, end = 0, pos = 0;
        if (i < p.p.n_seq) {
            start = p.starts[i];
            end = p.starts[i + 1];
            pos = p.pos[i];
            n = pg_run_pages(start, end, p.rows, pos, p.p.stride, p.p.positions);
            if (u == 0 && !pg_run_ok(start, end, p.rows, pos, p.p.stride, p.p.positions)) *p.p.flag = 1;
        }
        const int upto = before + wave_scan(n);
        const unsigned long long hit = __ballot(upto - n <= u && u < upto);
        if (hit) {
            const int from = __ffsll(hit) - 1;
            start = __builtin_amdgcn_readlane(start, from);
            end = __builtin_amdgcn_readlane(end, from);
            pos = __builtin_amdgcn_readlane(pos, from);
            const int first = __builtin_amdgcn_readlane(upto - n, from);
            const int page = pos / PG_ROWS + u - first, low = max(pos, page * PG_ROWS), high = min(pos + (end - start), (page + 1) * PG_ROWS);
            run.seq = b + from;
            run.page = page;
            run.in0 = start + (low - pos);
            run.r0 = low - page * PG_ROWS;
            run.r1 = high - page * PG_ROWS;
            if (u != 0) return true;
            /* workgroup 0 goes on: it looks at every run */
        }
        before = __builtin_amdgcn_readlane(upto, 63);
    }
    return u == 0 && before > 0;
}
} // namespace

template <int HD, bool CODES>
__global__ __launch_bounds__(PG_TPB) void k_pg_append(const PgRunParams p) {
    constexpr int XS = HD + 1; /* odd: columns without bank conflicts */
    __shared__ float s_x[PG_ROWS * XS];
    __shared__ float s_inv[PG_ROWS];
    const int tid = threadIdx.x, kvh = blockIdx.y;
    PgRun run;
    if (!pg_find_run(p, blockIdx.x, run)) return;
    const int page = p.p.table[(long long)run.seq * p.p.stride + run.page];
    if (pg_bad_page(page, p.p.n_pages)) {
        if (tid == 0) *p.p.flag = 1;
        return;
    }
    const int n = run.r1 - run.r0;
    const long long at = (long long)page * p.p.Hkv + kvh;
    unsigned char *kb = p.p.k + at * PgBytes<HD, CODES>::K, *vb = p.p.v + at * PgBytes<HD, CODES>::V;
    float *sb = CODES ? p.p.scales + at * 2 * PG_ROWS : nullptr;
    constexpr int C = HD / 8;
    auto fetch = [&](const void *x) {
        for (int e = tid; e < n * C; e += PG_TPB) {
            const int r = e / C, d = e % C * 8;
            float v[8];
            load8(x, p.dtype, ((long long)(run.in0 + r) * p.p.Hkv + kvh) * HD + d, v);
#pragma unroll
            for (int i = 0; i < 8; i++) s_x[r * XS + d + i] = v[i];
        }
        __syncthreads();
    };
    /* K: eight lanes a row, lane j the chunks j, j + 8, .. of 8 elements */
    fetch(p.k_in);
    const int j = tid & 7;
    constexpr int NC = (C + 7) / 8;
    for (int r0 = 0; r0 < n; r0 += PG_TPB / 8) {
        const int r = r0 + tid / 8;
        const bool live = r < n;
        float *x = s_x + min(r, n - 1) * XS;
        float y[NC][8];
        float ri = 1.0f;
        if (p.k_norm) {
            float ss = 0.0f;
            for (int d0 = 8 * j; d0 < HD; d0 += 64)
#pragma unroll
                for (int i = 0; i < 8; i++) ss = fmaf(x[d0 + i], x[d0 + i], ss);
            ss += __shfl_xor(ss, 1);
            ss += __shfl_xor(ss, 2);
            ss += __shfl_xor(ss, 4);
            ri = 1.0f / sqrtf(ss / (float)HD + p.norm_eps);
        }
        const long long pos = (long long)run.page * PG_ROWS + run.r0 + min(r, n - 1);
        unsigned m = 0;
#pragma unroll
        for (int k = 0; k < NC; k++) {
            const int d0 = 8 * j + 64 * k;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                y[k][i] = 0.0f;
                const int d = d0 + i;
                if (HD % 64 != 0 && d >= HD) continue;
                float a = x[d];
                if (p.k_norm) a = a * p.k_norm[d] * ri;
                if (p.p.rope_kind != SMOL_ROPE_OFF) {
                    const int pd = rope_partner(d, HD, p.p.rope_kind);
                    float b = x[pd];
                    if (p.k_norm) b = b * p.k_norm[pd] * ri;
                    const bool low = p.p.rope_kind == SMOL_ROPE_NEOX_K ? d < HD / 2 : (d & 1) == 0;
                    a = a * p.p.rope_cos[pos * HD + d] + (low ? -b : b) * p.p.rope_sin[pos * HD + d];
                }
                y[k][i] = a;
                m = max(m, __float_as_uint(a) & 0x7FFFFFFFu);
            }
        }
        m = max(m, (unsigned)__shfl_xor((int)m, 1));
        m = max(m, (unsigned)__shfl_xor((int)m, 2));
        m = max(m, (unsigned)__shfl_xor((int)m, 4));
        const PgScale sc = CODES ? pg_scale(m) : PgScale{1.0f, 1.0f};
        wave_fence(); /* the row's lanes have read their partners: the stored values take its place */
        if (live) {
            const int row = run.r0 + r;
            if (CODES && j == 0) sb[row] = sc.s;
#pragma unroll
            for (int k = 0; k < NC; k++) {
                const int d0 = 8 * j + 64 * k;
                if (HD % 64 != 0 && d0 >= HD) continue;
                if (CODES) {
                    unsigned w[2] = {0, 0};
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const int c = pg_code(y[k][i], sc.inv);
                        w[i >> 2] |= ((unsigned)c & 0xFFu) << 8 * (i & 3);
                        x[d0 + i] = (float)c * sc.s;
                    }
                    unsigned char *to = kb + ((d0 >> 4) * PG_ROWS + row) * 16 + (d0 & 8);
                    *reinterpret_cast<uint2 *>(to) = make_uint2(w[0], w[1]);
                    if (HD % 16 != 0 && d0 + 8 == HD) *reinterpret_cast<uint2 *>(to + 8) = make_uint2(0, 0);
                } else {
                    unsigned w[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const uint16_t a = bf16_of(y[k][2 * i]), b = bf16_of(y[k][2 * i + 1]);
                        w[i] = a | (unsigned)b << 16;
                        x[d0 + 2 * i] = bf16_to_f32(a);
                        x[d0 + 2 * i + 1] = bf16_to_f32(b);
                    }
                    *reinterpret_cast<uint4 *>(kb + ((d0 >> 3) * PG_ROWS + row) * 16) = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
        }
    }
    __syncthreads();
    for (int d = tid; d < HD; d += PG_TPB) {
        uint16_t *lo = p.p.bounds + at * 2 * HD + d, *hi = lo + HD;
        float a = INFINITY, b = -INFINITY;
        if (run.r0 > 0) {
            a = bf16_to_f32(*lo);
            b = bf16_to_f32(*hi);
        }
        for (int r = 0; r < n; r++) {
            a = min_nan(a, s_x[r * XS + d]);
            b = max_nan(b, s_x[r * XS + d]);
        }
        *lo = bf16_down(a);
        *hi = bf16_up(b);
    }
    __syncthreads();

    /* V */
    fetch(p.v_in);
    if (CODES) {
        for (int r0 = 0; r0 < n; r0 += PG_TPB / 8) {
            const int r = r0 + tid / 8;
            unsigned m = 0;
            if (r < n)
                for (int d0 = 8 * j; d0 < HD; d0 += 64)
#pragma unroll
                    for (int i = 0; i < 8; i++) m = max(m, __float_as_uint(s_x[r * XS + d0 + i]) & 0x7FFFFFFFu);
            m = max(m, (unsigned)__shfl_xor((int)m, 1));
            m = max(m, (unsigned)__shfl_xor((int)m, 2));
            m = max(m, (unsigned)__shfl_xor((int)m, 4));
            if (r < n && j == 0) {
                const PgScale sc = pg_scale(m);
                sb[PG_ROWS + run.r0 + r] = sc.s;
                s_inv[r] = sc.inv;
            }
        }
        __syncthreads();
    }
    /* a line of V in 16-byte pieces; pieces that hold other rows too by element */
    constexpr int E = CODES ? 16 : 8, P = PG_ROWS / E;
    for (int e = tid; e < HD * P; e += PG_TPB) {
        const int d = CODES ? e >> 2 : (e >> 2) % HD, half = CODES ? 0 : (e >> 2) / HD, g = e & 3;
        unsigned w[4] = {0, 0, 0, 0};
        unsigned char *to = CODES ? vb + d * PG_ROWS + 16 * g : vb + ((half * HD + d) * 32 + 8 * g) * 2;
        int rows[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < E; i++) {
            const int row = 32 * half + 16 * (i >> 2) + 4 * g + (i & 3), r = row - run.r0;
            const bool in = r >= 0 && r < n;
            rows[0] += in;
            const float v = in ? s_x[r * XS + d] : 0.0f;
            if (CODES) w[i >> 2] |= ((unsigned)(in ? pg_code(v, s_inv[r]) : 0) & 0xFFu) << 8 * (i & 3);
            else w[i >> 1] |= (unsigned)bf16_of(v) << 16 * (i & 1);
        }
        if (rows[0] == E) {
            *reinterpret_cast<uint4 *>(to) = make_uint4(w[0], w[1], w[2], w[3]);
        } else if (rows[0]) {
#pragma unroll
            for (int i = 0; i < E; i++) {
                const int row = 32 * half + 16 * (i >> 2) + 4 * g + (i & 3), r = row - run.r0;
                if (r < 0 || r >= n) continue;
                if (CODES) to[i] = (unsigned char)(w[i >> 2] >> 8 * (i & 3));
                else ((uint16_t *)to)[i] = (uint16_t)(w[i >> 1] >> 16 * (i & 1));
            }
        }
    }
}

template <int HD, bool CODES>
__global__ __launch_bounds__(PG_TPB) void k_pg_read(const PgRunParams p) {
    constexpr int XS = HD + 1;
    __shared__ float s_x[PG_ROWS * XS];
    const int tid = threadIdx.x, kvh = blockIdx.y;
    PgRun run;
    if (!pg_find_run(p, blockIdx.x, run)) return;
    const int page = p.p.table[(long long)run.seq * p.p.stride + run.page];
    const int n = run.r1 - run.r0;
    const bool bad = pg_bad_page(page, p.p.n_pages);
    if (bad && tid == 0) *p.p.flag = 1;
    const long long at = (long long)(bad ? 0 : page) * p.p.Hkv + kvh;
    const unsigned char *kb = p.p.k + at * PgBytes<HD, CODES>::K, *vb = p.p.v + at * PgBytes<HD, CODES>::V;
    const float *sb = CODES ? p.p.scales + at * 2 * PG_ROWS : nullptr;
    auto put = [&](void *out, int r, int d, float v) {
        const long long i = ((long long)(run.in0 + r) * p.p.Hkv + kvh) * HD + d;
        if (bad) v = __uint_as_float(0x7FC00000u);
        if (p.dtype == SMOL_IN_BF16) ((uint16_t *)out)[i] = bf16_of(v);
        else ((float *)out)[i] = v;
    };
    for (int e = tid; e < n * HD; e += PG_TPB) {
        const int r = e / HD, d = e % HD, row = run.r0 + r;
        if (CODES) put(p.k_out, r, d, (float)((const signed char *)kb)[((d >> 4) * PG_ROWS + row) * 16 + (d & 15)] * sb[row]);
        else put(p.k_out, r, d, bf16_to_f32(((const uint16_t *)kb)[((d >> 3) * PG_ROWS + row) * 8 + (d & 7)]));
    }
    for (int e = tid; e < HD * PG_ROWS; e += PG_TPB) {
        const int row = e % PG_ROWS, d = e / PG_ROWS, r = row - run.r0;
        if (r < 0 || r >= n) continue;
        if (CODES) s_x[r * XS + d] = (float)((const signed char *)vb)[d * PG_ROWS + pg_order(row, true)] * sb[PG_ROWS + row];
        else s_x[r * XS + d] = bf16_to_f32(((const uint16_t *)vb)[((row >> 5) * HD + d) * 32 + (pg_order(row, false) & 31)]);
    }
    __syncthreads();
    for (int e = tid; e < n * HD; e += PG_TPB) put(p.v_out, e / HD, e % HD, s_x[e / HD * XS + e % HD]);
}

/* ---------------------------------------------------------------- launches */

#define PG_BY_HD(hd, F) \
    switch (hd) { \
    case 64: F(64); break; \
    case 72: F(72); break; \
    case 80: F(80); break; \
    case 96: F(96); break; \
    case 128: F(128); break; \
    case 256: F(256); break; \
    default: return -1; \
    }

/* workgroups of k_pg on a compute unit */
extern "C" int smol_paged_occupancy(int hd, int codes) { return 2; }

extern "C" int smol_launch_pages(const PgRunParams *p, int hd, int write, hipStream_t st, hipEvent_t e0, hipEvent_t e1) {
    const dim3 grid((unsigned)pg_max_run_pages(p->p.n_seq, p->rows), p->p.Hkv), tpb(PG_TPB);
#define PG_RUN(HD) \
    if (write) { \
        if (p->p.codes) hipExtLaunchKernelGGL((k_pg_append<HD, true>), grid, tpb, 0, st, e0, e1, 0, *p); \
        else hipExtLaunchKernelGGL((k_pg_append<HD, false>), grid, tpb, 0, st, e0, e1, 0, *p); \
    } else { \
        if (p->p.codes) hipExtLaunchKernelGGL((k_pg_read<HD, true>), grid, tpb, 0, st, e0, e1, 0, *p); \
        else hipExtLaunchKernelGGL((k_pg_read<HD, false>), grid, tpb, 0, st, e0, e1, 0, *p); \
    }
    PG_BY_HD(hd, PG_RUN)
    return hipGetLastError() == hipSuccess ? 0 : -3;
}

extern "C" int smol_launch_paged(const PgParams *p, int hd, hipStream_t st, hipEvent_t e0, hipEvent_t e1) {
    const dim3 tpb(PG_TPB);
    hipEvent_t first = e0;
    if (p->top > 0) {
        const dim3 gs((unsigned)(p->p.n_seq * ((p->p.stride + PS_PAGES - 1) / PS_PAGES)), p->p.Hkv), gl(p->p.n_seq, p->p.Hkv);
#define PG_SCORE(HD) hipExtLaunchKernelGGL(k_pg_score<HD>, gs, tpb, 0, st, first, nullptr, 0, *p)
        PG_BY_HD(hd, PG_SCORE)
        first = nullptr;
        if (p->p.stride <= PS_LDS) hipExtLaunchKernelGGL(k_pg_select<true>, gl, tpb, 0, st, nullptr, nullptr, 0, *p);
        else hipExtLaunchKernelGGL(k_pg_select<false>, gl, tpb, 0, st, nullptr, nullptr, 0, *p);
    }
    const dim3 grid(p->max_items, p->p.Hkv, p->tiles), gm(p->p.n_seq, p->p.Hkv, p->tiles);
#define PG_STEP(HD) \
    if (p->p.codes) hipExtLaunchKernelGGL((k_pg<HD, true>), grid, tpb, 0, st, first, nullptr, 0, *p); \
    else hipExtLaunchKernelGGL((k_pg<HD, false>), grid, tpb, 0, st, first, nullptr, 0, *p); \
    hipExtLaunchKernelGGL(k_pg_merge<HD>, gm, tpb, 0, st, nullptr, e1, 0, *p)
    PG_BY_HD(hd, PG_STEP)
    return hipGetLastError() == hipSuccess ? 0 : -3;
}
