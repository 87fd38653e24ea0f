/*
 * paged.hip - a KV cache in pages of 64 rows, bf16 or codes of 8 bits: rows
 * into their pages (k_pg_append) and back (k_pg_read), a decode step over them
 * (k_pg), and the choice of the pages that such a step reads
 * (k_pg_choose). Layouts: attn_internal.h; who takes what:
 * paged_plan.h.
 */
#include "attn_device.h"
#include "paged_plan.h"

#include <algorithm>

namespace {

typedef int i4 __attribute__((ext_vector_type(4)));
typedef unsigned u2w __attribute__((ext_vector_type(2)));

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
    uint32_t x[PgGeom<HD>::NE]; /* as loaded: a conversion here would wait for each element */
    float w[PgGeom<HD>::NE];
    __device__ __forceinline__ void load(const void *base, int dtype, long long row, const float *norm) {
        const int lane = threadIdx.x & 63;
        if (dtype == SMOL_IN_BF16) {
#pragma unroll
            for (int e = 0; e < PgGeom<HD>::NE; e++) x[e] = HD % 64 == 0 || lane + 64 * e < HD ? ((const uint16_t *)base)[row + lane + 64 * e] : 0;
        } else {
#pragma unroll
            for (int e = 0; e < PgGeom<HD>::NE; e++) x[e] = HD % 64 == 0 || lane + 64 * e < HD ? ((const uint32_t *)base)[row + lane + 64 * e] : 0;
        }
        if (norm) {
#pragma unroll
            for (int e = 0; e < PgGeom<HD>::NE; e++) w[e] = HD % 64 == 0 || lane + 64 * e < HD ? norm[lane + 64 * e] : 0.0f;
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
__device__ __forceinline__ void pg_finish(const PgRow<HD> &r, int dtype, bool norm, float eps, const PgTurn<HD> &turn, int kind, T f, T *dst) {
    constexpr int NE = PgGeom<HD>::NE;
    const int lane = threadIdx.x & 63;
    T x[NE];
#pragma unroll
    for (int e = 0; e < NE; e++) x[e] = (T)__uint_as_float(dtype == SMOL_IN_BF16 ? r.x[e] << 16 : r.x[e]);
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
/* x inv, at most 127 in magnitude, plus 1.5 2^23: rounded to a whole number, whose two's complement is the low byte; what is no number
 * (inv 0 with an infinite x) leaves a zero there, and the row's scale tells */
#define PG_MAGIC 12582912.0f
__device__ __forceinline__ float pg_code(float x, float inv) {
#pragma clang fp contract(off) /* the fp32 product is what is rounded, as in the formula */
    return x * inv + PG_MAGIC;
}
/* the codes of four, packed */
__device__ __forceinline__ unsigned pg_pack4(float a, float b, float c, float d) {
    const unsigned lo = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x0c0c0400u);
    const unsigned hi = __builtin_amdgcn_perm(__float_as_uint(d), __float_as_uint(c), 0x0c0c0400u);
    return __builtin_amdgcn_perm(hi, lo, 0x05040100u);
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
    constexpr int NE = PgGeom<HD>::NE;
    const int lane = threadIdx.x & 63;
    const long long at = (long long)page * p.Hkv + g;
    uint16_t *bounds = p.bounds + at * 2 * HD;
    float lo[NE], hi[NE], v[NE];
    PgScale sc = {0.0f, 0.0f};
    unsigned m = 0;
#pragma unroll
    for (int e = 0; e < NE; e++) {
        const int d = lane + 64 * e;
        lo[e] = INFINITY;
        hi[e] = -INFINITY;
        v[e] = 0.0f;
        if (HD % 64 != 0 && d >= HD) continue;
        v[e] = x[d];
        if (KEY && r > 0) {
            lo[e] = bf16_to_f32(bounds[d]);
            hi[e] = bf16_to_f32(bounds[HD + d]);
        }
        m = max(m, __float_as_uint(v[e]) & 0x7FFFFFFFu);
    }
    if (CODES) {
        sc = pg_scale(wave_max(m));
        if (lane == 0) p.scales[(at * 2 + (KEY ? 0 : 1)) * PG_ROWS + r] = sc.s;
    }
    unsigned char *base = KEY ? p.k + at * PgBytes<HD, CODES>::K : p.v + at * PgBytes<HD, CODES>::V;
#pragma unroll
    for (int e = 0; e < NE; e++) {
        const int d = lane + 64 * e;
        if (HD % 64 != 0 && d >= HD) continue;
        if (CODES) {
            const float y = pg_code(v[e], sc.inv);
            const unsigned char c = (unsigned char)__float_as_uint(y);
            v[e] = (y - PG_MAGIC) * sc.s;
            if (KEY) base[((d >> 4) * PG_ROWS + r) * 16 + (d & 15)] = c;
            else base[d * PG_ROWS + pg_order(r, true)] = c;
        } else {
            const uint16_t b = bf16_of(v[e]);
            v[e] = bf16_to_f32(b);
            if (KEY) ((uint16_t *)base)[((d >> 3) * PG_ROWS + r) * 8 + (d & 7)] = b;
            else ((uint16_t *)base)[((r >> 5) * HD + d) * 32 + (pg_order(r, false) & 31)] = b;
        }
        if (KEY) {
            bounds[d] = bf16_down(min_nan(lo[e], v[e]));
            bounds[HD + d] = bf16_up(max_nan(hi[e], v[e]));
        }
    }
    /* the padding of a row's last piece */
    if (KEY && CODES && HD % 16 != 0 && lane < 16 - HD % 16) base[((HD >> 4) * PG_ROWS + r) * 16 + HD % 16 + lane] = 0;
}

/* inclusive sums over the lanes of a wave, without LDS */
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true); /* from 1, 2, 4, 8 lanes below, within 16 */
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false); /* the 16 lanes' sums to the next 16, then to the upper half */
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
    return v;
}

/* ---- the plan, by each wave: a lane's sequence of the 64 from b on ---- */
struct PgLane {
    int len, off; /* its first place on the line */
    PgUnits un;
    int end;      /* places of all sequences up to these 64's last */
    __device__ __forceinline__ void load(const PgParams &p, int b, int before) {
        const int i = b + (threadIdx.x & 63);
        len = i < p.p.n_seq ? p.len[i] : -1;
        place(p, before);
    }
    __device__ __forceinline__ void place(const PgParams &p, int before) {
        un = pg_units(len, p.p.stride, p.p.positions, p.window, p.top, pg_unit(p.p.codes));
        const int n = pg_places(len, un.n), upto = before + wave_scan(n);
        off = upto - n;
        end = __builtin_amdgcn_readlane(upto, 63);
    }
};
/* places of all sequences; s: the first 64 */
__device__ __forceinline__ int pg_line(const PgParams &p, PgLane &s) {
    s.load(p, 0, 0);
    int end = s.end;
    for (int b = 64; b < p.p.n_seq; b += 64) {
        PgLane t;
        t.load(p, b, end);
        end = t.end;
    }
    return end;
}

/* ---- one wave's softmax state over the units it takes ---- */
template <int HD>
struct PgState {
    float m, l, bad; /* bad: no number once a row was none (codes) */
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

namespace {
/* the bytes 2, 1 and 0 of four words, four of a kind in a word */
__device__ __forceinline__ void pg_split4(const unsigned (&x)[4], int &a, int &b, int &c) {
    const unsigned l01 = __builtin_amdgcn_perm(x[1], x[0], 0x05010400u), l23 = __builtin_amdgcn_perm(x[3], x[2], 0x05010400u);
    const unsigned h01 = __builtin_amdgcn_perm(x[1], x[0], 0x0c0c0602u), h23 = __builtin_amdgcn_perm(x[3], x[2], 0x0c0c0602u);
    a = (int)__builtin_amdgcn_perm(h23, h01, 0x05040100u);
    b = (int)__builtin_amdgcn_perm(l23, l01, 0x07060302u);
    c = (int)__builtin_amdgcn_perm(l23, l01, 0x05040100u);
}
} // namespace

/* Q of a tile as the matrix operand, three parts: in registers, or, at head_dim 256, where they would leave room for one wave a SIMD
 * alone, in LDS (a workgroup's waves read the same) */
template <int HD, bool CODES>
struct PgQ {
    static constexpr int KS = CODES ? PgGeom<HD>::KS8 : PgGeom<HD>::KSB;
    static constexpr bool FAR = HD > 128;
    static constexpr int LDS = FAR ? 3 * KS * 64 * 16 : 0; /* bytes */
    typedef typename std::conditional<CODES, i4, b8>::type Part;
    Part reg[FAR ? 1 : 3][FAR ? 1 : KS];
    const uint4 *lds;
    float unit; /* codes: what the last digit stands for */

    __device__ __forceinline__ Part part(int q, int ks) const {
        if constexpr (FAR) {
            const uint4 v = lds[(q * KS + ks) * 64 + (threadIdx.x & 63)];
            return *reinterpret_cast<const Part *>(&v);
        } else {
            return reg[q][ks];
        }
    }
    __device__ __forceinline__ void put(uint4 *to, int q, int ks, Part v) {
        if constexpr (FAR) {
            if (ks % PG_WAVES == (int)(threadIdx.x >> 6)) to[(q * KS + ks) * 64 + (threadIdx.x & 63)] = *reinterpret_cast<const uint4 *>(&v);
        } else {
            reg[q][ks] = v;
        }
    }
    /* of this lane's column's row; with FAR a barrier is needed before part() */
    __device__ __forceinline__ void make(const float *row, bool live, int g, uint4 *to) {
        lds = to;
        if constexpr (CODES) {
            unsigned m = 0;
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    const int d = 64 * ks + 16 * g + e;
                    f4 v = {0.f, 0.f, 0.f, 0.f};
                    if (live && (HD % 64 == 0 || d < HD)) v = *reinterpret_cast<const f4 *>(row + d);
#pragma unroll
                    for (int i = 0; i < 4; i++) m = max(m, __float_as_uint(v[i]) & 0x7FFFFFFFu);
                }
            m = row_maxu4(m);
            const float a = __uint_as_float(m);
            /* 24-bit whole numbers against the row's largest element; a row with no number or an infinity: no numbers; one that is
             * all but zero: zeros */
            const float inv = m >= 0x7F800000u || a < PG_TINY ? 0.0f : PG_FIX / a;
            unit = m >= 0x7F800000u ? __uint_as_float(0x7FC00000u) : a < PG_TINY ? 0.0f : a / PG_FIX;
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                i4 w[3];
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    const int d = 64 * ks + 16 * g + e;
                    f4 v = {0.f, 0.f, 0.f, 0.f};
                    if (live && (HD % 64 == 0 || d < HD)) v = *reinterpret_cast<const f4 *>(row + d);
                    unsigned n[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float y = rintf(v[i] * inv);
                        n[i] = pg_digits(y == y ? (int)y : 0);
                    }
                    int a, b, c;
                    pg_split4(n, a, b, c);
                    w[0][e / 4] = a;
                    w[1][e / 4] = b;
                    w[2][e / 4] = c;
                }
#pragma unroll
                for (int q = 0; q < 3; q++) put(to, q, ks, w[q]);
            }
        } else {
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                const int d = 32 * ks + 8 * g;
                b8 w[3];
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float x = live && (HD % 32 == 0 || d < HD) ? row[d + e] : 0.0f;
                    const __bf16 a = (__bf16)x;
                    const float r = x - (float)a;
                    const __bf16 b = (__bf16)r;
                    w[0][e] = a;
                    w[1][e] = b;
                    w[2][e] = (__bf16)(r - (float)b);
                }
#pragma unroll
                for (int q = 0; q < 3; q++) put(to, q, ks, w[q]);
            }
        }
    }
};

/* One unit's rows in registers, K and V apart: K of the next unit is requested when this one's scores are formed, V when this one's is
 * used, so something is always under way. Scales: one of K's and one of V's a lane (row = lane), laid out through LDS when needed. */
template <int HD, bool CODES>
struct PgUnitRegs;
template <int HD>
struct PgUnitRegs<HD, true> {
    i4 k[4][PgGeom<HD>::KS8], v[PgGeom<HD>::DT];
    float ks, vs;
    __device__ __forceinline__ void load_k(const PgPool &p, int page, int kvh, int half, int c, int g) {
        const long long at = (long long)page * p.Hkv + kvh;
        const unsigned char *kb = p.k + at * PgBytes<HD, true>::K;
        ks = p.scales[at * 2 * PG_ROWS + (threadIdx.x & 63)];
#pragma unroll
        for (int s = 0; s < PgGeom<HD>::KS8; s++)
#pragma unroll
            for (int t = 0; t < 4; t++) {
                const int ch = 4 * s + g;
                k[t][s] = i4{0, 0, 0, 0};
                if (HD % 64 == 0 || ch < PgGeom<HD>::CH8) k[t][s] = *reinterpret_cast<const i4 *>(kb + (ch * PG_ROWS + 16 * t + c) * 16);
            }
    }
    __device__ __forceinline__ void load_v(const PgPool &p, int page, int kvh, int half, int c, int g) {
        const long long at = (long long)page * p.Hkv + kvh;
        const unsigned char *vb = p.v + at * PgBytes<HD, true>::V;
        vs = p.scales[(at * 2 + 1) * PG_ROWS + (threadIdx.x & 63)];
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
    __device__ __forceinline__ void load_k(const PgPool &p, int page, int kvh, int half, int c, int g) {
        const unsigned char *kb = p.k + ((long long)page * p.Hkv + kvh) * PgBytes<HD, false>::K + half * 512;
#pragma unroll
        for (int s = 0; s < PgGeom<HD>::KSB; s++)
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const int ch = 4 * s + g;
                k[t][s] = make_uint4(0, 0, 0, 0);
                if (HD % 32 == 0 || ch < PgGeom<HD>::CHB) k[t][s] = *reinterpret_cast<const uint4 *>(kb + (ch * PG_ROWS + 16 * t + c) * 16);
            }
    }
    __device__ __forceinline__ void load_v(const PgPool &p, int page, int kvh, int half, int c, int g) {
        const unsigned char *vb = p.v + ((long long)page * p.Hkv + kvh) * PgBytes<HD, false>::V + half * HD * 64;
#pragma unroll
        for (int dt = 0; dt < PgGeom<HD>::DT; dt++) {
            const int d = 16 * dt + c;
            v[dt] = make_uint4(0, 0, 0, 0);
            if (HD % 16 == 0 || d < HD) v[dt] = *reinterpret_cast<const uint4 *>(vb + d * 64 + 16 * g);
        }
    }
};

/* The weights' unit is of 2^-100 at least, so that it and its inverse stay normal numbers: V's smallest scale is near 2^-97 (PG_TINY) */
#define PG_LEAST 7.888609052210118e-31f

/* A unit of codes joins the state; visible rows of it [lo, hi).
 * A score is exact up to its last sum: K's codes and the digits of Q are whole numbers, and so are their dot products. The
 * weights p vs (vs: V's scales) are taken against the largest product of the unit and head as 24-bit whole numbers, digit by digit on
 * the matrix cores again, so V needs no conversion either. The product, not the largest vs alone: the row that has the weight
 * may be one of small values (against the largest vs it would keep 14 of its bits where they are 1000 times smaller). */
template <int HD, class F>
__device__ __forceinline__ void pg_take(PgState<HD> &st, const PgQ<HD, true> &q, PgUnitRegs<HD, true> &u, float cap2, int g, int lo, int hi,
                                        float *lds, F next_k) {
    constexpr int DT = PgGeom<HD>::DT;
    const i4 zero = {0, 0, 0, 0};
    const bool part = lo > 0 || hi < 64;
    const int lane = threadIdx.x & 63;
    float s[4][4];
    /* the scales of rows that are not seen could be anything */
    float ksc[4][4], vsc[4][4];
    if (part && (lane < lo || lane >= hi)) u.ks = u.vs = 0.0f;
    lds[lane] = u.ks;
    lds[64 + lane] = u.vs;
    wave_fence();
#pragma unroll
    for (int t = 0; t < 4; t++) {
        const f4 a = *reinterpret_cast<const f4 *>(lds + 16 * t + 4 * g);
#pragma unroll
        for (int i = 0; i < 4; i++) ksc[t][i] = a[i];
    }
    /* a visible scale that is no number, or infinite, spoils the sum when the lanes' are joined */
    const float odd = 0.0f * u.ks + 0.0f * u.vs;
    i4 d[4][3];
#pragma unroll
    for (int t = 0; t < 4; t++) {
        d[t][0] = d[t][1] = d[t][2] = zero;
    }
#pragma unroll
    for (int ks = 0; ks < PgGeom<HD>::KS8; ks++)
#pragma unroll
        for (int pt = 0; pt < 3; pt++) {
            const i4 x = q.part(pt, ks);
#pragma unroll
            for (int t = 0; t < 4; t++) d[t][pt] = __builtin_amdgcn_mfma_i32_16x16x64_i8(u.k[t][ks], x, d[t][pt], 0, 0, 0);
            if (q.FAR && pt == 2) __builtin_amdgcn_sched_barrier(0); /* parts of Q are not read ahead: registers */
        }
#pragma unroll
    for (int t = 0; t < 4; t++)
#pragma unroll
        for (int i = 0; i < 4; i++)
            s[t][i] = fmaf((float)d[t][0][i], 65536.0f, fmaf((float)d[t][1][i], 256.0f, (float)d[t][2][i])) * (q.unit * ksc[t][i]);
    next_k();
#pragma unroll
    for (int t = 0; t < 4; t++) {
        const f4 a = *reinterpret_cast<const f4 *>(lds + 64 + 16 * t + 4 * g);
#pragma unroll
        for (int i = 0; i < 4; i++) vsc[t][i] = a[i];
    }
    wave_fence(); /* read before the next unit's are written */
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
    float sum = 0.0f, top = PG_LEAST;
#pragma unroll
    for (int t = 0; t < 4; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float pr = __builtin_amdgcn_exp2f(s[t][i] - mu);
            sum += pr;
            s[t][i] = pr * vsc[t][i];
            top = fmaxf(top, s[t][i]);
        }
    top = row_max4(top);
    const float f = 1.0f / top;
    i4 w0, w1, w2;
#pragma unroll
    for (int t = 0; t < 4; t++) {
        unsigned x[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            /* 2^23 + n: the low bits of the sum are the whole number n, rounded to nearest */
            const float y = fmaf(s[t][i] * f, PG_FIX, 8388608.0f);
            x[i] = (__float_as_uint(y) + 0x8080u) ^ 0x8080u;
        }
        int a, b, c;
        pg_split4(x, a, b, c);
        w0[t] = a;
        w1[t] = b;
        w2[t] = c;
    }
    pg_raise(st, mu);
    const float b = __builtin_amdgcn_exp2f(mu - st.m);
    st.l = fmaf(b, sum, st.l);
    st.bad += odd;
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
template <int HD, class F>
__device__ __forceinline__ void pg_take(PgState<HD> &st, const PgQ<HD, false> &q, PgUnitRegs<HD, false> &u, float cap2, int g, int lo, int hi,
                                        float *, F next_k) {
    constexpr int DT = PgGeom<HD>::DT;
    const bool part = lo > 0 || hi < 32;
    f4 s[2] = {};
#pragma unroll
    for (int pt = 2; pt >= 0; pt--)
#pragma unroll
        for (int ks = 0; ks < PgGeom<HD>::KSB; ks++) {
            const b8 x = q.part(pt, ks);
#pragma unroll
            for (int t = 0; t < 2; t++) s[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_b8(u.k[t][ks]), x, s[t], 0, 0, 0);
            if (q.FAR && ks % 4 == 3) __builtin_amdgcn_sched_barrier(0); /* parts of Q are not read ahead: registers */
        }
    next_k();
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

namespace {
/* O and (m, l) of a chunk go to the workgroup that joins them past the caches of the XCDs */
__device__ __forceinline__ void put_far(rsrc_t r, f4 v, unsigned off) {
    __builtin_amdgcn_raw_buffer_store_b128(u4v{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])}, r,
                                           off, 0, CPOL_SC1);
}
__device__ __forceinline__ f4 get_far(rsrc_t r, unsigned off) {
    const u4v v = __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, CPOL_SC1);
    return f4{__uint_as_float(v[0]), __uint_as_float(v[1]), __uint_as_float(v[2]), __uint_as_float(v[3])};
}
__device__ __forceinline__ void put_far(rsrc_t r, float m, float l, unsigned off) {
    __builtin_amdgcn_raw_buffer_store_b64(u2w{__float_as_uint(m), __float_as_uint(l)}, r, off, 0, CPOL_SC1);
}
__device__ __forceinline__ void get_far(rsrc_t r, unsigned off, float &m, float &l) {
    const u2w v = __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, CPOL_SC1);
    m = __uint_as_float(v[0]);
    l = __uint_as_float(v[1]);
}
/* What is not finite in one dim spoils its row. Each by itself: a sum of finite numbers may pass the largest */
__device__ __forceinline__ bool pg_odd(f4 a) { return 0.0f * a[0] + 0.0f * a[1] + 0.0f * a[2] + 0.0f * a[3] != 0.0f; }
template <int N>
using PgInt = std::integral_constant<int, N>;
} // namespace

/* A piece of the sequences' units against a tile of 16 heads of a kv head, sequence by sequence; a sequence's last chunk also takes the
 * new token and stores its row. Of a sequence with several chunks the workgroup that ends last joins them, in their order.
 *
 * One pass over the rows with the running maximum m and sum l of the softmax, O scaled down when m grows. Heads are the columns of the
 * matrix products (16, of which few may be live), so K and V come from memory straight into the operand's registers and each row is
 * read once for all heads that share it; the pages' layout is that operand's. The matrix cores are idle most of the time: what bounds
 * a batch is memory. 16 heads over 8 of 128, 64 sequences of 4000 to 16384 rows of codes (1.38 GB): 250 us, 5.5 TB/s of what has to be
 * read (the counters see 1.32 GB), where a plain read reaches 5.96; 16 sequences of 3000 to 4160 (121 MB): 36 us, of which 6 to 11 pass
 * before the first unit is there (plan 1.5, rows of Q 1 to 4) and 4 in the join. One sequence of 1024 bf16 rows: 12.8 us, all of it
 * latency; of codes 15: units of 64 rows share them out to half as many waves, and each weight has its digits to be formed.
 *
 * Equal pieces of one line, as many as the machine holds at once: with pieces a sequence (the first form) a second round of workgroups
 * cost 16 sequences 51 us instead of 37. A piece has at least PG_WAVES units: of 8, one sequence of 1024 rows takes 14.0 us instead
 * of 12.3, though one of 4096 bf16 rows gains (16.2 and 17.1). Two workgroups a compute unit up to head_dim 128 (256 registers
 * a lane, of which codes spill 5 at 96 and 8 at 128); at 256 the state and two units in flight take all 512 (one unit and Q's parts in LDS for a second workgroup: 78 us
 * where this takes 38, 24 sequences of 500 to 8191 rows). */
template <int HD, bool CODES>
__global__ __launch_bounds__(PG_TPB, HD > 128 ? 1 : 2) void k_pg(const PgParams p) {
    constexpr bool DEEP = HD > 128; /* one wave a SIMD, whose registers hold two units */
    constexpr int XS = PgGeom<HD>::XSTR, DT = PgGeom<HD>::DT, U = CODES ? 64 : 32, QD = HD / 4;
    /* Q's parts (head_dim 256); then the rows of Q (scaled), and when they are done with, the waves' outputs */
    extern __shared__ __align__(16) unsigned char s_dyn[];
    uint4 *s_q = reinterpret_cast<uint4 *>(s_dyn);
    float *s_mem = reinterpret_cast<float *>(s_dyn + PgQ<HD, CODES>::LDS);
    __shared__ __align__(16) float s_scale[PG_WAVES][CODES ? 128 : 4];
    __shared__ __align__(16) float s_k[HD], s_v[HD]; /* the new token */
    __shared__ float s_m[PG_WAVES + 1][PG_HEADS], s_l[PG_WAVES][PG_HEADS];
    __shared__ int s_bad[PG_HEADS], s_turn;
    const int kvh = blockIdx.y, tile = blockIdx.z, h0 = tile * PG_HEADS, R = min(PG_HEADS, p.G - h0);
    PgLane sl;
    const int piece = pg_piece(pg_line(p, sl), p.slots), w = blockIdx.x;
    int b0 = 0; /* the first of the 64 sequences in sl */
    unsigned long long todo = 0;
    bool fresh = true;
    for (;;) {
    /* hidden from the compiler, which else forms every address before the loop and has no registers left in it */
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, g = lane >> 4;
    /* the next sequence that this piece holds something of: the same for all waves */
    if (fresh) todo = __ballot(sl.len >= 0 && pg_cut(sl.off, sl.un.n, piece, w).mine);
    fresh = false;
    if (todo == 0) {
        b0 += 64;
        if (b0 >= p.p.n_seq || sl.end >= (w + 1) * piece) return;
        sl.load(p, b0, sl.end);
        fresh = true;
        continue;
    }
    struct {
        int seq, len, off;
        PgUnits units;
    } it;
    {
        const int from = __ffsll(todo) - 1;
        todo &= todo - 1;
        it.seq = b0 + from;
        it.len = __builtin_amdgcn_readlane(sl.len, from);
        it.off = __builtin_amdgcn_readlane(sl.off, from);
        it.units.first = __builtin_amdgcn_readlane(sl.un.first, from);
        it.units.n = __builtin_amdgcn_readlane(sl.un.n, from);
    }
    const PgCut cut = pg_cut(it.off, it.units.n, piece, w);
    const int u0 = cut.u0, u1 = cut.u1;
    const bool ok = pg_len_ok(it.len, p.p.stride, p.p.positions), last = cut.nth == cut.chunks - 1;
    const int *row_table = p.p.table + (long long)it.seq * p.p.stride;
    const int *list = p.top > 0 ? p.list + ((long long)it.seq * p.p.Hkv + kvh) * p.top : nullptr;
    bool bad = !ok;

    /* the pages of this wave's first 64 units */
    int at = 0, page = 0; /* of unit u0 + wave + 4 lane: its first row, its page */
    auto pages = [&](int from) {
        const int un = from + PG_WAVES * lane;
        at = page = 0;
        if (un < u1) {
            int row = (it.units.first + un) * U;
            if (list) {
                /* (a list that was written over meanwhile leads nowhere) */
                const int j = list[un / (PG_ROWS / U)];
                row = j >= 0 && j <= it.len / PG_ROWS ? j * PG_ROWS + un % (PG_ROWS / U) * U : it.len;
            }
            at = row;
            page = row_table[min(row, it.len) / PG_ROWS];
        }
    };
    auto checked = [&](int from) { /* once the numbers are here */
        if (from + PG_WAVES * lane < u1 && pg_bad_page(page, p.p.n_pages)) {
            bad = true;
            page = 0;
        }
    };
    pages(u0 + wave);
    int new_page = 0;
    if (last && ok) new_page = row_table[it.len / PG_ROWS];
    PgUnitRegs<HD, CODES> u[DEEP ? 2 : 1] = {}; /* (what is not set here would be carried from sequence to sequence) */
    auto load_k = [&](PgUnitRegs<HD, CODES> &to, int n) {
        const int row = __builtin_amdgcn_readlane(at, n), pg = __builtin_amdgcn_readlane(page, n);
        to.load_k(p.p, pg, kvh, CODES ? 0 : row % PG_ROWS / 32, c, g);
    };
    auto load_v = [&](PgUnitRegs<HD, CODES> &to, int n) {
        const int row = __builtin_amdgcn_readlane(at, n), pg = __builtin_amdgcn_readlane(page, n);
        to.load_v(p.p, pg, kvh, CODES ? 0 : row % PG_ROWS / 32, c, g);
    };
    {
        /* rows of Q and the new key, normalised and rotated */
        constexpr int NR = (PG_HEADS + 1 + PG_WAVES - 1) / PG_WAVES;
        PgRow<HD> r[NR] = {};
        PgTurn<HD> turn = {};
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
        uint32_t v_new = 0; /* HD <= PG_TPB: an element a thread */
        if (last && tid < HD) {
            const long long i = ((long long)it.seq * p.p.Hkv + kvh) * HD + tid;
            v_new = p.in_dtype == SMOL_IN_BF16 ? ((const uint16_t *)p.v_in)[i] : ((const uint32_t *)p.v_in)[i];
        }
        /* the first unit is requested behind them: a compute unit returns data in the order of its requests */
        __builtin_amdgcn_sched_barrier(0);
        checked(u0 + wave);
        if (u0 + wave < u1) {
            load_k(u[0], 0);
            load_v(u[0], 0);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int k = 0; k < NR; k++) {
            const int i = wave + PG_WAVES * k;
            if (i < n) {
                const bool key = i == R;
                pg_finish<HD, float>(r[k], p.in_dtype, (key ? p.k_norm : p.q_norm) != nullptr, p.norm_eps, turn, p.p.rope_kind, key ? 1.0f : p.qscale,
                                     key ? s_k : s_mem + i * XS);
            }
        }
        if (last && tid < HD) s_v[tid] = __uint_as_float(p.in_dtype == SMOL_IN_BF16 ? v_new << 16 : v_new);
    }
    if (last && ok && pg_bad_page(new_page, p.p.n_pages)) {
        bad = true;
        new_page = -1;
    }
    if (tid < PG_HEADS) s_bad[tid] = 0;
    __syncthreads();
    PgQ<HD, CODES> q;
    q.make(s_mem + c * XS, c < R, g, s_q);
    if (PgQ<HD, CODES>::FAR) __syncthreads();

    PgState<HD> st;
    st.m = -INFINITY;
    st.l = st.bad = 0.0f;
#pragma unroll
    for (int dt = 0; dt < DT; dt++) st.o[dt] = f4{0.f, 0.f, 0.f, 0.f};
    const int lo = p.top > 0 ? 0 : pg_first_row(it.len, p.window);
    int un = u0 + wave, n = 0;
    /* one unit, and the requests for the next: K when this one's scores are formed and V when this one's is used, into the same
     * registers, or (DEEP) both beforehand into others */
    auto step = [&](PgUnitRegs<HD, CODES> &cur, PgUnitRegs<HD, CODES> &next) {
        const int row = __builtin_amdgcn_readlane(at, n);
        n = (n + 1) & 63;
        un += PG_WAVES;
        const bool more = un < u1;
        if (more && n == 0) {
            pages(un);
            checked(un);
        }
        if (DEEP && more) {
            load_k(next, n);
            load_v(next, n);
        }
        if (DEEP) __builtin_amdgcn_sched_barrier(0);
        auto next_k = [&]() {
            if (!DEEP && more) load_k(next, n);
            __builtin_amdgcn_sched_barrier(0);
        };
        if (row < it.len) pg_take<HD>(st, q, cur, p.cap2, g, max(0, lo - row), min(U, it.len - row), s_scale[wave], next_k);
        else next_k(); /* the second half of a listed page that ends before it */
        if (!DEEP && more) load_v(next, n);
        __builtin_amdgcn_sched_barrier(0);
    };
    while (un < u1) {
        step(u[0], u[DEEP ? 1 : 0]);
        if (DEEP && un < u1) step(u[DEEP ? 1 : 0], u[0]);
    }
    st.l += st.bad;
    if (__any(bad || st.bad != st.bad)) st.l = __uint_as_float(0x7FC00000u);
    if (__any(bad) && lane == 0) *p.p.flag = 1;
    st.l = row_sum4(st.l);

    if (last) {
        /* the new token's scores */
        for (int r = wave; r < R; r += PG_WAVES) {
            float d = 0.0f;
#pragma unroll
            for (int e = 0; e < PgGeom<HD>::NE; e++)
                if (HD % 64 == 0 || lane + 64 * e < HD) d = fmaf(s_mem[r * XS + lane + 64 * e], s_k[lane + 64 * e], d);
            d = wave_sum(d);
            /* an infinite score is no number, also behind a cap */
            if (lane == 0) s_m[PG_WAVES][r] = pg_capped(d, p.cap2) + 0.0f * d;
        }
    }
    __syncthreads();
    if (c < R) {
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
            if (HD % 16 == 0 || 16 * dt + 4 * g < HD) *reinterpret_cast<f4 *>(s_mem + (wave * R + c) * XS + 16 * dt + 4 * g) = st.o[dt];
        if (g == 0) {
            s_m[wave][c] = st.m;
            s_l[wave][c] = st.l;
        }
    }
    __syncthreads();
    /* the waves' states and the new token's as one; a whole sequence's is the answer, others wait in memory */
    const bool whole = cut.chunks == 1;
    const int slot0 = it.units.n ? 2 * ((it.off + PG_EXTRA) / piece) : 0; /* the places of this sequence's chunks begin here */
    const long long first = ((long long)kvh * 2 * p.slots + slot0) * p.G + h0;
    const rsrc_t far = make_rsrc(p.part + first * PG_PART(HD), 1LL << 31);
    auto place = [&](int n, int r) { return ((pg_slot(it.off, piece, n) - slot0) * p.G + r) * PG_PART(HD) * 4; };
    float *out = p.out + ((long long)it.seq * p.Hq + kvh * p.G + h0) * HD;
    constexpr int NJ = (PG_HEADS * QD + PG_TPB - 1) / PG_TPB;
    f4 o[NJ] = {};
#pragma unroll
    for (int k = 0; k < NJ; k++) {
        const int e = tid + k * PG_TPB, r = e / QD, d = e % QD * 4;
        if (e >= R * QD) continue;
        const float mn = last ? s_m[PG_WAVES][r] : -INFINITY;
        float m = mn;
#pragma unroll
        for (int w = 0; w < PG_WAVES; w++) m = fmaxf(m, s_m[w][r]);
        float l = 0.0f;
        f4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < PG_WAVES; w++) {
            const float lw = s_l[w][r], f = s_m[w][r] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(s_m[w][r] - m);
            l = fmaf(f, lw, l);
            if (lw != lw) l = lw; /* a wave that saw nothing but rows that are no numbers */
            a += *reinterpret_cast<const f4 *>(s_mem + (w * R + r) * XS + d) * f;
        }
        if (last) {
            const float f = mn != mn ? mn : __builtin_amdgcn_exp2f(mn - m);
            l += f;
            a += *reinterpret_cast<const f4 *>(s_v + d) * f;
        }
        if (whole) {
            a *= 1.0f / l;
            if (pg_odd(a)) s_bad[r] = 1;
        } else {
            put_far(far, a, place(cut.nth, r) + d * 4);
            if (d == 0) put_far(far, m, l, place(cut.nth, r) + HD * 4);
        }
        o[k] = a;
    }
    if (!whole) {
        /* what this workgroup wrote has arrived where others read before it counts itself in; the count starts anew by itself */
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (tid == 0) s_turn = (int)atomicInc(p.count + ((long long)it.seq * p.p.Hkv + kvh) * p.tiles + tile, cut.chunks - 1);
        __syncthreads();
    }
    const bool answer = whole || s_turn == cut.chunks - 1;
    if (!whole && answer) {
        /* N places of the outputs a thread, B chunks in flight for each: what the chunks' round trips past the caches allow. At
         * head_dim 256 few heads leave registers for more of them (one sequence of 8191 rows, 67 chunks: 27.5 us, 8 in flight
         * 32.6); below, a second form of the loop costs what it saves */
        auto join = [&](auto n_of, auto b_of) {
            constexpr int N = decltype(n_of)::value, B = decltype(b_of)::value;
            float m[N], l[N];
#pragma unroll
            for (int k = 0; k < N; k++) {
                m[k] = -INFINITY;
                l[k] = 0.0f;
                o[k] = f4{0.f, 0.f, 0.f, 0.f};
            }
            for (int n0 = 0; n0 < cut.chunks; n0 += B) {
                float mc[N][B] = {}, lc[N][B] = {};
                f4 oc[N][B] = {};
#pragma unroll
                for (int k = 0; k < N; k++) {
                    const int e = min(tid + k * PG_TPB, R * QD - 1), r = e / QD, d = e % QD * 4;
                    if (k * PG_TPB >= R * QD) break;
#pragma unroll
                    for (int b = 0; b < B; b++) {
                        const int n = min(n0 + b, cut.chunks - 1);
                        get_far(far, place(n, r) + HD * 4, mc[k][b], lc[k][b]);
                        oc[k][b] = get_far(far, place(n, r) + d * 4);
                    }
                }
#pragma unroll
                for (int k = 0; k < N; k++) {
                    if (k * PG_TPB >= R * QD) break;
                    float mn = m[k];
#pragma unroll
                    for (int b = 0; b < B; b++) mn = fmaxf(mn, mc[k][b]);
                    const float fa = m[k] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[k] - mn);
                    l[k] *= fa;
                    o[k] *= fa;
#pragma unroll
                    for (int b = 0; b < B; b++) {
                        /* (places behind the last are the last once more; a branch here would send its loads one by one) */
                        const float f = n0 + b >= cut.chunks || mc[k][b] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mc[k][b] - mn);
                        l[k] = lc[k][b] != lc[k][b] ? lc[k][b] : fmaf(lc[k][b], f, l[k]);
                        o[k] += oc[k][b] * f;
                    }
                    m[k] = mn;
                }
            }
#pragma unroll
            for (int k = 0; k < N; k++) {
                if (tid + k * PG_TPB >= R * QD) continue;
                o[k] *= 1.0f / l[k];
                if (pg_odd(o[k])) s_bad[(tid + k * PG_TPB) / QD] = 1;
            }
        };
        if constexpr (DEEP) {
            if (R * QD <= PG_TPB) join(PgInt<1>(), PgInt<16>());
            else if (R * QD <= 2 * PG_TPB) join(PgInt<2>(), PgInt<16>());
            else join(PgInt<NJ>(), PgInt<8>());
        } else {
            join(PgInt<NJ>(), PgInt<8>());
        }
    }
    if (answer) {
        __syncthreads();
#pragma unroll
        for (int k = 0; k < NJ; k++) {
            const int e = tid + k * PG_TPB;
            if (e >= R * QD) continue;
            if (s_bad[e / QD]) o[k] = f4{NAN, NAN, NAN, NAN};
            *reinterpret_cast<f4 *>(out + (long long)e * 4) = o[k];
        }
    }
    /* the new row into its page, when nobody waits for it any more */
    if (last && tile == 0 && ok && new_page >= 0) {
        if (wave == 2) pg_store_row<HD, CODES, true>(p.p, new_page, kvh, it.len % PG_ROWS, s_k);
        if (wave == 3) pg_store_row<HD, CODES, false>(p.p, new_page, kvh, it.len % PG_ROWS, s_v);
    }
    __syncthreads();
    }
}

/* ------------------------------------------------------- which pages to read */

namespace {
constexpr int PS_BINS = 2048;
constexpr int PS_LDS = 4096; /* pages whose keys a choosing workgroup keeps in LDS */

__device__ __forceinline__ int pg_pages(int len) { return (len + PG_ROWS - 1) / PG_ROWS; }

/* score = sum over the heads of a kv head and the dims of max(q lo, q hi): an upper bound of any row's score, summed over the heads,
 * q+ . hi + q- . lo with q+ (q-) the sums of the heads' positive (negative) elements, so a page costs two products whatever the
 * number of heads. In 64 bits, and a page's terms in one order whatever the page: pages with equal bounds tie. */
template <int HD>
struct PgScore {
    static constexpr int LPP = HD <= 64 ? 8 : HD <= 128 ? 16 : 32; /* lanes of a page, eight dims each */
    double up[8], dn[8];

    /* q+ and q- of a sequence and kv head, the heads by the waves in turn, through LDS; then this lane's dims of them. All threads of
     * the workgroup call; next(): what is requested behind the first head's row */
    template <class F>
    __device__ __forceinline__ void make(const PgParams &p, int seq, int kvh, int len, double (*s_row)[HD], double (*s_sum)[2][HD], F next) {
        constexpr int NE = PgGeom<HD>::NE;
        const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        PgTurn<HD> turn;
        turn.load(p.p, len);
        double u[NE], d[NE];
#pragma unroll
        for (int e = 0; e < NE; e++) u[e] = d[e] = 0.0;
        PgRow<HD> r;
        auto request = [&](int h) { r.load(p.q_in, p.in_dtype, ((long long)seq * p.Hq + kvh * p.G + h) * HD, p.q_norm); };
        request(min(wave, p.G - 1));
        __builtin_amdgcn_sched_barrier(0);
        next();
        __builtin_amdgcn_sched_barrier(0);
        for (int h = wave; h < p.G; h += PG_WAVES) {
            const PgRow<HD> now = r;
            if (h + PG_WAVES < p.G) request(h + PG_WAVES);
            pg_finish<HD, double>(now, p.in_dtype, p.q_norm != nullptr, p.norm_eps, turn, p.p.rope_kind, p.scale, s_row[wave]);
#pragma unroll
            for (int e = 0; e < NE; e++) {
                if (HD % 64 != 0 && lane + 64 * e >= HD) continue;
                const double x = s_row[wave][lane + 64 * e];
                u[e] += x > 0.0 ? x : 0.0;
                d[e] += x > 0.0 ? 0.0 : x; /* takes a NaN */
            }
        }
#pragma unroll
        for (int e = 0; e < NE; e++)
            if (HD % 64 == 0 || lane + 64 * e < HD) {
                s_sum[wave][0][lane + 64 * e] = u[e];
                s_sum[wave][1][lane + 64 * e] = d[e];
            }
        __syncthreads();
        const int waves = min(p.G, PG_WAVES);
        for (int e = tid; e < 2 * HD; e += PG_TPB) {
            double x = s_sum[0][0][e];
            for (int w = 1; w < waves; w++) x += s_sum[w][0][e];
            s_sum[0][0][e] = x;
        }
        __syncthreads();
        const int ch = lane % LPP;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            up[i] = 8 * ch < HD ? s_sum[0][0][8 * ch + i] : 0.0;
            dn[i] = 8 * ch < HD ? s_sum[0][1][8 * ch + i] : 0.0;
        }
    }
    struct Bounds {
        uint4 lo, hi;
    };
    __device__ __forceinline__ void load(const PgPool &p, int page, int kvh, Bounds &b) const {
        const int ch = threadIdx.x % LPP;
        b.lo = b.hi = make_uint4(0, 0, 0, 0);
        if (8 * ch >= HD) return;
        const uint16_t *at = p.bounds + ((long long)page * p.Hkv + kvh) * 2 * HD + 8 * ch;
        b.lo = *reinterpret_cast<const uint4 *>(at);
        b.hi = *reinterpret_cast<const uint4 *>(at + HD);
    }
    /* the score, in all lanes of the page */
    __device__ __forceinline__ double of(const Bounds &b) const {
        float lo[8], hi[8];
        unpack_bf16x8(b.lo, lo);
        unpack_bf16x8(b.hi, hi);
        double s = 0.0;
#pragma unroll
        for (int i = 0; i < 8; i++) s = fma(up[i], (double)hi[i], fma(dn[i], (double)lo[i], s));
#pragma unroll
        for (int sh = LPP / 2; sh; sh >>= 1) s += __shfl_xor(s, sh);
        return s;
    }
    /* The score of a page for which of() is no number. An infinite bound that no head's element picks is none of the formula's terms:
     * its 0 times infinity is left out here. From memory and LDS once more, so that it costs the usual pages no registers (in of()
     * 32 of them: 64 sequences of 16384 rows 78 us instead of 74). */
    __device__ __forceinline__ double again(const PgPool &p, int page, int kvh, const double (*sum)[HD]) const {
        const int d0 = 8 * (threadIdx.x % LPP);
        const uint16_t *at = p.bounds + ((long long)page * p.Hkv + kvh) * 2 * HD + d0;
        double s = 0.0;
#pragma unroll 1
        for (int i = 0; i < 8 && d0 < HD; i++) {
            const float lo = bf16_to_f32(at[i]), hi = bf16_to_f32(at[HD + i]);
            const double u = sum[0][d0 + i], d = sum[1][d0 + i];
            if (u != 0.0 || fabsf(hi) != INFINITY) s += u * hi;
            if (d != 0.0 || fabsf(lo) != INFINITY) s += d * lo;
        }
#pragma unroll
        for (int sh = LPP / 2; sh; sh >>= 1) s += __shfl_xor(s, sh);
        return s;
    }
};

/* a score as a whole number of the same order: what stays by its place above all, then NaN, then the numbers (-0 as 0) */
__device__ __forceinline__ unsigned long long pg_key(double s, int j, int pages, int first, int recent) {
    if (j < first || j >= pages - recent) return ~0ULL;
    if (!(s == s)) return ~0ULL - 1;
    const unsigned long long u = s == 0.0 ? 0ULL : (unsigned long long)__double_as_longlong(s);
    return u >> 63 ? ~u : u | 0x8000000000000000ULL;
}

/* exclusive sums over the TPB threads, through s_part [TPB / 64]; the threads meet twice */
template <int TPB>
__device__ __forceinline__ int block_before(int v, int *s_part) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, incl = wave_scan(v);
    if (lane == 63) s_part[wave] = incl;
    __syncthreads();
    int at = incl - v;
#pragma unroll
    for (int w = 0; w < TPB / 64; w++)
        if (w < wave) at += s_part[w];
    __syncthreads();
    return at;
}

struct PgChoose {
    unsigned long long any[PG_WAVES], all[PG_WAVES];
    int hist[PS_BINS], part[PG_WAVES], found[2];
};

/* The `top` pages of the largest keys, in ascending order. The top-th largest key is found by the highest eleven bits in which the
 * keys still in question differ, again and again: a histogram of them in LDS says which bin holds it. Mostly two rounds: the first
 * leaves a few keys. */
template <int TPB, class F>
__device__ __forceinline__ void pg_choose(F key, int pages, int top, int *list, PgChoose &s) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    unsigned long long prefix = 0, mask = 0; /* in question: keys with (key & mask) == prefix; larger ones are taken */
    int need = top, held = pages;            /* to take of those in question, and how many there are */
    while (held > need) {
        unsigned long long any = 0, all = ~0ULL;
        for (int j = tid; j < pages; j += TPB) {
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
            s.any[wave] = any;
            s.all[wave] = all;
        }
        for (int b = tid; b < PS_BINS; b += TPB) s.hist[b] = 0;
        __syncthreads();
        any = 0;
        all = ~0ULL;
#pragma unroll
        for (int w = 0; w < TPB / 64; w++) {
            any |= s.any[w];
            all &= s.all[w];
        }
        const unsigned long long differ = any & ~all;
        if (differ == 0) break; /* all equal: the lowest pages of them */
        const int shift = max(0, 63 - __clzll(differ) - 10);
        for (int j = tid; j < pages; j += TPB) {
            const unsigned long long k = key(j);
            if ((k & mask) == prefix) atomicAdd(&s.hist[(k >> shift) & (PS_BINS - 1)], 1);
        }
        __syncthreads();
        constexpr int NB = PS_BINS / TPB;
        int cnt[NB], sum = 0;
#pragma unroll
        for (int b = 0; b < NB; b++) sum += cnt[b] = s.hist[PS_BINS - 1 - NB * tid - b];
        int above = block_before<TPB>(sum, s.part);
#pragma unroll
        for (int b = 0; b < NB; b++) {
            if (above < need && above + cnt[b] >= need) {
                s.found[0] = PS_BINS - 1 - NB * tid - b;
                s.found[1] = need - above;
            }
            above += cnt[b];
        }
        __syncthreads();
        const int bin = s.found[0];
        held = s.hist[bin];
        need = s.found[1];
        /* the bits at and above the bin's are known now: those above it are the same in all keys in question */
        mask = ~((1ULL << shift) - 1);
        prefix = (shift + 11 < 64 ? all >> (shift + 11) << (shift + 11) : 0ULL) | (unsigned long long)bin << shift;
        __syncthreads();
    }
    /* keys above the prefix, and the lowest `need` pages at it, by threads that take consecutive pages */
    const int per = (pages + TPB - 1) / TPB, b0 = min(pages, tid * per), b1 = min(pages, b0 + per);
    int eq = 0, more = 0;
    for (int j = b0; j < b1; j++) {
        const unsigned long long k = key(j) & mask;
        eq += k == prefix;
        more += k > prefix;
    }
    int e = block_before<TPB>(eq, s.part);
    int at = block_before<TPB>(more + max(0, min(need, e + eq) - min(need, e)), s.part);
    for (int j = b0; j < b1; j++) {
        const unsigned long long k = key(j) & mask;
        if (k > prefix || (k == prefix && e < need)) list[at++] = j;
        e += k == prefix;
    }
}
} // namespace

/* Scores of the pages, `per` of them a workgroup, and the choice by the workgroup of a (sequence, kv head) that ends last: one launch,
 * whose last part no other workgroup waits for. Few bytes (a page's bounds are 512 of head_dim 128), so what it takes is its chain of
 * round trips: Q's rows and their sums over the heads 5 us, the bounds 2, the scores past the caches 2, then the choice's rounds of LDS
 * and barriers 3: 11.5 us for 256 pages of one sequence, 18.5 for 250 to 512 of each of 16. Scores and choice by one workgroup of
 * 1024 threads were slower (one compute unit's 64-bit arithmetic). */
template <int HD>
__global__ __launch_bounds__(PG_TPB) void k_pg_choose(const PgParams p) {
    typedef PgScore<HD> Score;
    constexpr int LPP = Score::LPP, PP = PG_TPB / LPP, U = 64 / PP; /* pages of a step, such steps in flight */
    __shared__ union {
        struct {
            double row[PG_WAVES][HD];
            __align__(16) double sum[PG_WAVES][2][HD];
        } q;
        PgChoose c;
    } s;
    extern __shared__ __align__(16) unsigned char s_dyn[];
    unsigned long long *s_key = reinterpret_cast<unsigned long long *>(s_dyn); /* [min(stride, PS_LDS)] */
    __shared__ int s_turn;
    const int tid = threadIdx.x, kvh = blockIdx.y;
    const int blocks = (p.p.stride + p.per - 1) / p.per, seq = blockIdx.x / blocks, j0 = blockIdx.x % blocks * p.per;
    const int len = p.len[seq];
    if (len < 0) return;
    /* a length that is none: no page is chosen, and k_pg reports it */
    const int pages = pg_len_ok(len, p.p.stride, p.p.positions) ? pg_pages(len) : 0, j1 = min(pages, j0 + p.per);
    if (j0 >= pages && j0 > 0) return;
    const long long pair = (long long)seq * p.p.Hkv + kvh;
    int *list = p.list + pair * p.top;
    if (pages <= p.top) {
        if (j0 == 0)
            for (int j = tid; j < p.top; j += PG_TPB) list[j] = j < pages ? j : -1;
        return;
    }
    const int *row_table = p.p.table + (long long)seq * p.p.stride;
    Score sc;
    typename Score::Bounds b[U];
    bool bad[U];
    auto load = [&](int j) { /* the pages of a step whose first is j */
        int page[U];
#pragma unroll
        for (int u = 0; u < U; u++) page[u] = row_table[min(j + u * PP + tid / LPP, pages - 1)];
#pragma unroll
        for (int u = 0; u < U; u++) {
            bad[u] = pg_bad_page(page[u], p.p.n_pages);
            sc.load(p.p, bad[u] ? 0 : page[u], kvh, b[u]);
        }
    };
    sc.make(p, seq, kvh, len, s.q.row, s.q.sum, [&]() { load(j0); });
    const bool one = pages <= p.per;
    const rsrc_t far = make_rsrc(p.score + pair * p.p.stride, (long long)p.p.stride * 8);
    for (int j = j0; j < j1; j += 64) {
        double x[U];
        bool none = false;
#pragma unroll
        for (int u = 0; u < U; u++) {
            x[u] = sc.of(b[u]);
            none |= !(x[u] == x[u]);
        }
        if (__any(none)) {
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int page = row_table[min(j + u * PP + tid / LPP, pages - 1)]; /* looked at like the first time */
                const double y = sc.again(p.p, pg_bad_page(page, p.p.n_pages) ? 0 : page, kvh, s.q.sum[0]);
                if (!(x[u] == x[u])) x[u] = y;
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++)
            if (bad[u]) {
                /* chosen before numbers, so that the step meets it; reported here, since others without a number may leave no place */
                x[u] = __longlong_as_double(0x7FF8000000000000LL);
                *p.p.flag = 1;
            }
        if (j + 64 < j1) load(j + 64);
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int at = j + u * PP + tid / LPP;
            if (at >= j1 || tid % LPP) continue;
            const unsigned long long k = pg_key(x[u], at, pages, p.first, p.recent);
            if (one) s_key[at] = k;
            else __builtin_amdgcn_raw_buffer_store_b64(u2w{(unsigned)k, (unsigned)(k >> 32)}, far, at * 8, 0, CPOL_SC1);
        }
    }
    auto there = [&](int j) {
        const u2w v = __builtin_amdgcn_raw_buffer_load_b64(far, j * 8, 0, CPOL_SC1);
        return (unsigned long long)v[1] << 32 | v[0];
    };
    if (!one) {
        /* as in k_pg: what is written has arrived before the workgroup counts itself in */
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        const unsigned n = (pages + p.per - 1) / p.per;
        if (tid == 0) s_turn = (int)atomicInc(p.count + pair * p.tiles, n - 1);
        __syncthreads();
        if (s_turn != (int)n - 1) return;
        if (pages <= PS_LDS)
            for (int j = tid; j < pages; j += PG_TPB) s_key[j] = there(j);
    }
    __syncthreads();
    if (pages <= PS_LDS) pg_choose<PG_TPB>([&](int j) { return s_key[j]; }, pages, p.top, list, s.c);
    else pg_choose<PG_TPB>(there, pages, p.top, list, s.c);
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

namespace {
/* minimum and maximum that pass a NaN over, without the extra instruction that quiets a signalling one first */
__device__ __forceinline__ float min_num(float a, float b) {
    float r;
    asm("v_min_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}
__device__ __forceinline__ float max_num(float a, float b) {
    float r;
    asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}
/* a lane's value from the other half of its 16 lanes */
__device__ __forceinline__ float ror8(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x128, 0xF, 0xF, true));
}

/* Sixteen values a lane (f of two: their minimum or maximum) over the rows of a wave, LR lanes each, by halves: the upper and the
 * lower 32 lanes swap eight values each and keep eight, the lanes 16 apart four of those. Value e + 4 b4 + 8 b5 of the lanes with
 * bits 4 and 5 of b4 and b5 is left in v[e]: 28 instructions where a full exchange takes 16 times six. */
template <int LR, class F>
__device__ __forceinline__ void rows_join(float (&v)[16], F f) {
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[e]), __float_as_uint(v[e + 8]), false, false);
        v[e] = f(__uint_as_float(a[0]), __uint_as_float(a[1]));
    }
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[e]), __float_as_uint(v[e + 4]), false, false);
        v[e] = f(__uint_as_float(a[0]), __uint_as_float(a[1]));
        if (LR == 8) v[e] = f(v[e], ror8(v[e]));
    }
}

constexpr int PA_TPB = PG_APPEND_TPB, PA_WAVES = PA_TPB / 64; /* a k_pg_append workgroup */

template <int HD>
struct PgKGeom {
    static constexpr int C = HD / 8, LR = HD > 128 ? 16 : 8, NC = (C + LR - 1) / LR;
    static constexpr int RW = PA_TPB / LR, NP = PG_ROWS / RW; /* rows of a pass, passes of a page */
    static constexpr bool SAME = HD == 128 || HD == 256;      /* a NeoX partner is in the same lane */
};
/* the rotation's table for a row of a K workgroup, the same for all heads: lane j of the row's LR holds its chunks j, j + LR, .. of eight
 * elements (a wave's loads and stores are whole lines) */
template <int HD>
struct PgKTable {
    static constexpr int NC = PgKGeom<HD>::NC;
    float4 c[NC][2], s[NC][2];
    __device__ __forceinline__ void load(const PgRunParams &p, long long pos, int j) {
        const int kind = p.p.rope_kind;
        if (kind == SMOL_ROPE_OFF) return;
#pragma unroll
        for (int k = 0; k < NC; k++) {
            const int d0 = 8 * j + 8 * PgKGeom<HD>::LR * k;
            if (HD % 64 != 0 && d0 >= HD) continue;
            /* its rows repeat their first half (NeoX) */
            if (!PgKGeom<HD>::SAME || kind == SMOL_ROPE_INTERLEAVED_K || k < NC / 2) {
                const float4 *ct = reinterpret_cast<const float4 *>(p.p.rope_cos + pos * HD + d0);
                const float4 *st = reinterpret_cast<const float4 *>(p.p.rope_sin + pos * HD + d0);
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    c[k][i] = ct[i];
                    s[k][i] = st[i];
                }
            }
        }
    }
};
/* a row of a head. load() only requests, so that the next one's data is under way while this one's is worked on */
template <int HD, bool BF>
struct PgKStep {
    static constexpr int LR = PgKGeom<HD>::LR, NC = PgKGeom<HD>::NC;
    static constexpr bool SAME = PgKGeom<HD>::SAME;
    Raw8<BF> x[NC], pr[SAME ? 1 : NC];
    uint32_t pe[SAME ? 1 : NC][8];

    __device__ __forceinline__ void load(const PgRunParams &p, long long in, int j) {
        const int kind = p.p.rope_kind;
#pragma unroll
        for (int k = 0; k < NC; k++) {
            const int d0 = 8 * j + 8 * LR * k;
            if (HD % 64 != 0 && d0 >= HD) continue;
            raw_load<BF>(x[k], p.k_in, in + d0);
            if (!SAME && kind == SMOL_ROPE_NEOX_K) {
                if (HD % 16 == 0) { /* half a head is whole chunks */
                    raw_load<BF>(pr[k], p.k_in, in + (d0 < HD / 2 ? d0 + HD / 2 : d0 - HD / 2));
                } else {
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        pe[k][i] = __float_as_uint(in_at(p.k_in, BF ? SMOL_IN_BF16 : SMOL_IN_F32, in + rope_partner(d0 + i, HD, SMOL_ROPE_NEOX_K)));
                }
            }
        }
    }
    __device__ __forceinline__ static float at(const float4 (&v)[2], int i) {
        const float4 &q = v[i >> 2];
        return (i & 3) == 0 ? q.x : (i & 3) == 1 ? q.y : (i & 3) == 2 ? q.z : q.w;
    }
    /* y: the normalised, rotated chunks (zeros behind the row), in T. Codes take fp32, whose roundings are 2^-16 of a code's step;
     * bf16 rows 64 bits, so that they are the formula's own rounding (in fp32 one element of 16000 is a step beside it). */
    template <class T>
    __device__ __forceinline__ void finish(const PgRunParams &p, const PgKTable<HD> &t, int j, float (&y)[NC][8]) const {
        const int kind = p.p.rope_kind;
        T v[NC][8], o[SAME ? 1 : NC][8];
#pragma unroll
        for (int k = 0; k < NC; k++) {
            const int d0 = 8 * j + 8 * LR * k;
            float f[8] = {};
            if (HD % 64 == 0 || d0 < HD) raw_unpack<BF>(x[k], f);
#pragma unroll
            for (int i = 0; i < 8; i++) v[k][i] = (T)f[i];
            if (!SAME && kind == SMOL_ROPE_NEOX_K && (HD % 64 == 0 || d0 < HD)) {
                if (HD % 16 == 0) raw_unpack<BF>(pr[k], f);
#pragma unroll
                for (int i = 0; i < 8; i++) o[SAME ? 0 : k][i] = (T)(HD % 16 == 0 ? f[i] : __uint_as_float(pe[SAME ? 0 : k][i]));
            }
        }
        if (p.k_norm) {
            T ss[4] = {0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < NC; k++)
#pragma unroll
                for (int i = 0; i < 8; i++) ss[i & 3] += v[k][i] * v[k][i];
            T sum = (ss[0] + ss[1]) + (ss[2] + ss[3]);
#pragma unroll
            for (int sh = 1; sh < LR; sh <<= 1) sum += __shfl_xor(sum, sh);
            const T ri = (T)(1.0 / sqrt((double)sum / HD + (double)p.norm_eps)); /* in 64 bits: rounded once */
#pragma unroll
            for (int k = 0; k < NC; k++) {
                const int d0 = 8 * j + 8 * LR * k;
                if (HD % 64 != 0 && d0 >= HD) continue;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    v[k][i] *= (T)p.k_norm[d0 + i] * ri;
                    if (!SAME && kind == SMOL_ROPE_NEOX_K) o[SAME ? 0 : k][i] *= (T)p.k_norm[rope_partner(d0 + i, HD, SMOL_ROPE_NEOX_K)] * ri;
                }
            }
        }
#pragma unroll
        for (int k = 0; k < NC; k++) {
            constexpr int H = NC / 2 ? NC / 2 : 1;
            const int d0 = 8 * j + 8 * LR * k;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                T a = v[k][i];
                if (kind == SMOL_ROPE_NEOX_K) {
                    const T b = (SAME ? v[(k + H) % NC][i] : o[SAME ? 0 : k][i]) * (T)at(SAME ? t.s[k % H] : t.s[k], i);
                    a = a * (T)at(SAME ? t.c[k % H] : t.c[k], i) + ((SAME ? k < H : d0 + i < HD / 2) ? -b : b);
                } else if (kind == SMOL_ROPE_INTERLEAVED_K) {
                    const T b = v[k][i ^ 1] * (T)at(t.s[k], i);
                    a = a * (T)at(t.c[k], i) + (i & 1 ? b : -b);
                }
                y[k][i] = HD % 64 != 0 && d0 >= HD ? 0.0f : (float)a;
            }
        }
    }
};

/* K rows of heads [h0, h1) into a page, and its bounds */
template <int HD, bool CODES, bool BF>
__device__ __forceinline__ void pg_append_k(const PgRunParams &p, const PgRun &run, long long page, int h0, int h1) {
    typedef PgKStep<HD, BF> Step;
    typedef PgKGeom<HD> Geo;
    constexpr int C = Geo::C, LR = Geo::LR, NC = Geo::NC, RW = Geo::RW, NP = Geo::NP;
    __shared__ float s_lo[2][PA_WAVES][HD], s_hi[2][PA_WAVES][HD]; /* of the heads by turns: one barrier a head is enough */
    __shared__ unsigned s_none[2][PA_WAVES][C];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, j = tid & (LR - 1), n = run.r1 - run.r0;
    auto request = [&](Step &st, int h, int pass) {
        st.load(p, ((long long)(run.in0 + min(RW * pass + tid / LR, n - 1)) * p.p.Hkv + h) * HD, j);
    };
    Step next;
    request(next, h0, 0);
    PgKTable<HD> table[NP];
#pragma unroll
    for (int pass = 0; pass < NP; pass++)
        table[pass].load(p, (long long)run.page * PG_ROWS + run.r0 + min(RW * pass + tid / LR, n - 1), j);
    for (int h = h0; h < h1; h++) {
        const long long at = page * p.p.Hkv + h;
        const int turn = (h - h0) & 1;
        unsigned char *kb = p.p.k + at * PgBytes<HD, CODES>::K;
        float lo[16], hi[16]; /* element 8 k + i */
        unsigned none[NC];    /* elements that are no number in some row */
#pragma unroll
        for (int pass = 0; pass < NP; pass++) {
            if (RW * pass >= n) break;
            const Step cur = next;
            if (pass + 1 < NP && RW * (pass + 1) < n) request(next, h, pass + 1);
            else if (h + 1 < h1) request(next, h + 1, 0);
            /* lanes past the last row work on it once more: it changes no bound */
            const int r = RW * pass + tid / LR, row = run.r0 + r;
            float y[NC][8];
            cur.template finish<typename std::conditional<CODES, float, double>::type>(p, table[pass], j, y);
            PgScale sc = {1.0f, 1.0f};
            if (CODES) {
                unsigned m = 0;
#pragma unroll
                for (int k = 0; k < NC; k++)
#pragma unroll
                    for (int i = 0; i < 8; i++) m = max(m, __float_as_uint(y[k][i]) & 0x7FFFFFFFu);
#pragma unroll
                for (int sh = 1; sh < LR; sh <<= 1) m = max(m, (unsigned)__shfl_xor((int)m, sh));
                sc = pg_scale(m);
            }
            if (CODES && j == 0 && r < n) p.p.scales[at * 2 * PG_ROWS + row] = sc.s;
#pragma unroll
            for (int k = 0; k < NC; k++) {
                const int d0 = 8 * j + 8 * LR * k;
                const bool put = r < n && (HD % 64 == 0 || d0 < HD);
                float kept[8];
                unsigned bad = 0;
                if (CODES) {
                    float q[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        q[i] = pg_code(y[k][i], sc.inv);
                        kept[i] = (q[i] - PG_MAGIC) * sc.s;
                    }
                    unsigned char *to = kb + ((d0 >> 4) * PG_ROWS + row) * 16 + (d0 & 8);
                    if (put) *reinterpret_cast<uint2 *>(to) = make_uint2(pg_pack4(q[0], q[1], q[2], q[3]), pg_pack4(q[4], q[5], q[6], q[7]));
                    if (HD % 16 != 0 && put && d0 + 8 == HD) *reinterpret_cast<uint2 *>(to + 8) = make_uint2(0, 0);
                    bad = sc.s == sc.s ? 0u : 0xFFu;
                } else {
                    unsigned o[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const uint16_t a = bf16_of(y[k][2 * i]), b = bf16_of(y[k][2 * i + 1]);
                        o[i] = a | (unsigned)b << 16;
                        kept[2 * i] = bf16_to_f32(a);
                        kept[2 * i + 1] = bf16_to_f32(b);
                    }
                    if (put) *reinterpret_cast<uint4 *>(kb + ((d0 >> 3) * PG_ROWS + row) * 16) = make_uint4(o[0], o[1], o[2], o[3]);
#pragma unroll
                    for (int i = 0; i < 8; i++) bad |= kept[i] == kept[i] ? 0u : 1u << i;
                }
                none[k] = pass ? none[k] | bad : bad;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    lo[8 * k + i] = pass ? min_num(lo[8 * k + i], kept[i]) : kept[i];
                    hi[8 * k + i] = pass ? max_num(hi[8 * k + i], kept[i]) : kept[i];
                }
            }
        }
        if (NC == 1) /* the join takes sixteen */
#pragma unroll
            for (int e = 8; e < 16; e++) lo[e] = hi[e] = 0.0f;
        /* over the rows of the wave, then over the waves and what the page had */
#pragma unroll
        for (int k = 0; k < NC; k++) {
            unsigned b = none[k];
            if (LR == 8) b |= __shfl_xor((int)b, 8);
            b |= __shfl_xor((int)b, 16);
            b |= __shfl_xor((int)b, 32);
            const int d0 = 8 * j + 8 * LR * k;
            if (lane < LR && (HD % 64 == 0 || d0 < HD)) s_none[turn][wave][d0 / 8] = b;
        }
        rows_join<LR>(lo, min_num);
        rows_join<LR>(hi, max_num);
        if (LR == 16 || !(lane & 8)) {
            const int e0 = 4 * (lane >> 4 & 1) + 8 * (lane >> 5), d = 8 * j + 8 * LR * (e0 >> 3) + (e0 & 7);
            if (NC == 2 || e0 < 8)
                if (HD % 64 == 0 || d < HD)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        s_lo[turn][wave][d + e] = lo[e];
                        s_hi[turn][wave][d + e] = hi[e];
                    }
        }
        __syncthreads();
        for (int d = tid; d < HD; d += PA_TPB) {
            uint16_t *to = p.p.bounds + at * 2 * HD + d;
            float l = INFINITY, u = -INFINITY;
            bool bad = false;
            if (run.r0 > 0) {
                l = bf16_to_f32(to[0]);
                u = bf16_to_f32(to[HD]);
                bad = l != l || u != u;
            }
#pragma unroll
            for (int w = 0; w < PA_WAVES; w++) {
                l = min_num(l, s_lo[turn][w][d]);
                u = max_num(u, s_hi[turn][w][d]);
                bad |= s_none[turn][w][d / 8] >> (d & 7) & 1;
            }
            to[0] = bad ? 0x7FC0 : bf16_down(l);
            to[HD] = bad ? 0x7FC0 : bf16_up(u);
        }
    }
}

/* V rows of heads [h0, h1) into a page: a thread takes four dims of the eight rows 32 half + 16 t + 4 g + i, which lie side by side
 * along V's lines, and turns them round in its registers. 16 lanes hold 64 dims of a row, a wave half a page of them; what waves
 * are left take the next heads. */
template <int HD, bool CODES, bool BF>
__device__ __forceinline__ void pg_append_v(const PgRunParams &p, const PgRun &run, long long page, int h0, int h1) {
    constexpr int DB = (HD + 63) / 64, SUB = PA_WAVES / (2 * DB); /* blocks of 64 dims, heads at a time */
    static_assert(SUB >= 1, "a head's waves");
    __shared__ unsigned s_max[2][SUB][DB][PG_ROWS];
    __shared__ __align__(16) float s_inv[PA_WAVES][32];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane & 3, n = run.r1 - run.r0;
    const int half = wave & 1, block = wave / 2 % DB, sub = wave / (2 * DB), d = 64 * block + 4 * (lane >> 2);
    const bool mine = HD % 64 == 0 || d < HD;
    typedef typename std::conditional<BF, uint2, float4>::type Four;
    Four next[8];
    auto request = [&](int kvh) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int r = 32 * half + 16 * (e >> 2) + 4 * g + (e & 3) - run.r0;
            next[e] = Four{};
            if (kvh >= h1 || r < 0 || r >= n || !mine) continue;
            const long long in = ((long long)(run.in0 + r) * p.p.Hkv + kvh) * HD + d;
            next[e] = BF ? *reinterpret_cast<const Four *>((const uint16_t *)p.v_in + in) : *reinterpret_cast<const Four *>((const float *)p.v_in + in);
        }
    };
    request(h0 + sub);
    for (int hb = h0; hb < h1; hb += SUB) {
        const int kvh = hb + sub, turn = (hb - h0) / SUB & 1; /* by turns: one barrier a step is enough */
        const bool live = kvh < h1;
        const long long at = page * p.p.Hkv + kvh;
        unsigned char *vb = p.p.v + at * PgBytes<HD, CODES>::V;
        float x[8][4];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            if constexpr (BF) {
                x[e][0] = __uint_as_float(next[e].x << 16);
                x[e][1] = __uint_as_float(next[e].x & 0xFFFF0000u);
                x[e][2] = __uint_as_float(next[e].y << 16);
                x[e][3] = __uint_as_float(next[e].y & 0xFFFF0000u);
            } else {
                x[e][0] = next[e].x;
                x[e][1] = next[e].y;
                x[e][2] = next[e].z;
                x[e][3] = next[e].w;
            }
        }
        if (hb + SUB < h1) request(kvh + SUB);
        float inv[8];
#pragma unroll
        for (int e = 0; e < 8; e++) inv[e] = 0.0f;
        if (CODES) {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                unsigned m = 0;
#pragma unroll
                for (int i = 0; i < 4; i++) m = max(m, __float_as_uint(x[e][i]) & 0x7FFFFFFFu);
                /* lanes of the same g */
                m = max(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, 0x124, 0xF, 0xF, true));
                m = max(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, 0x128, 0xF, 0xF, true));
                m = row_maxu4(m);
                if (lane < 4) s_max[turn][sub][block][32 * half + 16 * (e >> 2) + 4 * g + (e & 3)] = m;
            }
            __syncthreads();
            /* a row's scale by one lane; its factor to the others of the wave */
            const int row = 32 * half + (lane & 31);
            unsigned m = 0;
#pragma unroll
            for (int b = 0; b < DB; b++) m = max(m, s_max[turn][sub][b][row]);
            const PgScale sc = pg_scale(m);
            if (lane < 32) {
                s_inv[wave][lane] = sc.inv;
                if (live && block == 0 && row >= run.r0 && row < run.r1) p.p.scales[(at * 2 + 1) * PG_ROWS + row] = sc.s;
            }
            wave_fence();
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const f4 v = *reinterpret_cast<const f4 *>(&s_inv[wave][16 * t + 4 * g]);
#pragma unroll
                for (int i = 0; i < 4; i++) inv[4 * t + i] = v[i];
            }
            wave_fence();
        }
        if (!live || !mine) continue;
        const bool all = run.r0 <= 32 * half + 4 * g && run.r1 >= 32 * half + 4 * g + 20;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            unsigned o[4];
            if constexpr (CODES) {
#pragma unroll
                for (int t = 0; t < 2; t++)
                    o[t] = pg_pack4(pg_code(x[4 * t][i], inv[4 * t]), pg_code(x[4 * t + 1][i], inv[4 * t + 1]),
                                    pg_code(x[4 * t + 2][i], inv[4 * t + 2]), pg_code(x[4 * t + 3][i], inv[4 * t + 3]));
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) o[e] = bf16_of(x[2 * e][i]) | (unsigned)bf16_of(x[2 * e + 1][i]) << 16;
            }
            unsigned char *to = CODES ? vb + (d + i) * PG_ROWS + 16 * g + 8 * half : vb + ((half * HD + d + i) * 32 + 8 * g) * 2;
            if (all) {
                if constexpr (CODES) *reinterpret_cast<uint2 *>(to) = make_uint2(o[0], o[1]);
                else *reinterpret_cast<uint4 *>(to) = make_uint4(o[0], o[1], o[2], o[3]);
            } else {
                /* the other rows' elements stay as they are */
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int row = 32 * half + 16 * (e >> 2) + 4 * g + (e & 3);
                    if (row < run.r0 || row >= run.r1) continue;
                    if (CODES) to[e] = (unsigned char)(o[e >> 2] >> 8 * (e & 3));
                    else ((uint16_t *)to)[e] = (uint16_t)(o[e >> 1] >> 16 * (e & 1));
                }
            }
        }
    }
}
} // namespace

/* A workgroup takes the K (z 0) or the V (z 1) rows of `heads` kv heads of one page: a page is the unit whose bounds and whose lines of V
 * belong to one sequence, so nothing is shared and every store but those at a run's ends is a whole line. K: a row by 8 (16) lanes, its
 * rotation table read once for all heads; V: turned round in registers. Memory, and behind it the vector instructions (60 of the 97 us):
 * 16 sequences of 2000 to 4096 bf16 rows of 8 heads of 128 into codes (310 MB) take 97 us, 3.2 TB/s, where a copy of as much takes
 * 66; a chunk of 26 rows 5.8. */
template <int HD, bool CODES, bool BF>
__global__ __launch_bounds__(PA_TPB, HD == 64 || (HD == 128 && CODES) ? 4 : 2) void k_pg_append(const PgRunParams p) {
    PgRun run;
    if (!pg_find_run(p, blockIdx.x, run)) return;
    const int page = p.p.table[(long long)run.seq * p.p.stride + run.page];
    if (pg_bad_page(page, p.p.n_pages)) {
        if (threadIdx.x == 0) *p.p.flag = 1;
        return;
    }
    const int h0 = blockIdx.y * p.heads, h1 = min(p.p.Hkv, h0 + p.heads);
    if (blockIdx.z == 0) pg_append_k<HD, CODES, BF>(p, run, page, h0, h1);
    else pg_append_v<HD, CODES, BF>(p, run, page, h0, h1);
}

namespace {
/* N values, times s, as the output's type */
template <bool BF, int N>
__device__ __forceinline__ void pg_put(void *out, long long i, const float (&v)[N], float s) {
    if (BF) {
        unsigned w[N / 2];
#pragma unroll
        for (int e = 0; e < N / 2; e++) w[e] = bf16_of(v[2 * e] * s) | (unsigned)bf16_of(v[2 * e + 1] * s) << 16;
        uint16_t *to = (uint16_t *)out + i;
        if constexpr (N == 4) {
            *reinterpret_cast<uint2 *>(to) = make_uint2(w[0], w[1]);
        } else {
#pragma unroll
            for (int e = 0; e < N / 8; e++) *reinterpret_cast<uint4 *>(to + 8 * e) = make_uint4(w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3]);
        }
    } else {
        float *to = (float *)out + i;
#pragma unroll
        for (int e = 0; e < N / 4; e++) *reinterpret_cast<f4 *>(to + 4 * e) = f4{v[4 * e] * s, v[4 * e + 1] * s, v[4 * e + 2] * s, v[4 * e + 3] * s};
    }
}
__device__ __forceinline__ float pg_byte(unsigned w, int i) { return (float)(int)(signed char)(w >> 8 * i & 0xFFu); }
} // namespace

/* A workgroup takes one page and kv head: K piece by piece (eight pieces of eight rows a wave: whole lines both ways), V four dims
 * of eight rows a thread, turned round in registers, as k_pg_append does. All of a thread's loads are requested before the first is
 * used. Memory: 8 sequences of 4000 to 8192 rows of codes, 8 heads of 128, to bf16 (303 MB): 60 us, 5.0 TB/s (a copy 4.7); 1500 rows of
 * 4 heads of 64: 5.4 us, latency. */
template <int HD, bool CODES, bool BF>
__global__ __launch_bounds__(PG_TPB) void k_pg_read(const PgRunParams p) {
    constexpr int E = CODES ? 16 : 8, CH = CODES ? PgGeom<HD>::CH8 : PgGeom<HD>::CHB;
    constexpr int CB = (CH + 7) / 8, NK = CB * 8 / PG_WAVES; /* (8 pieces, 8 rows) tasks of a wave */
    constexpr int DB = (HD + 63) / 64, NV = (2 * DB + PG_WAVES - 1) / PG_WAVES;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, kvh = blockIdx.y, g = lane & 3;
    PgRun run;
    if (!pg_find_run(p, blockIdx.x, run)) return;
    const int page = p.p.table[(long long)run.seq * p.p.stride + run.page];
    const bool bad = pg_bad_page(page, p.p.n_pages);
    if (bad && tid == 0) *p.p.flag = 1;
    const long long at = (long long)(bad ? 0 : page) * p.p.Hkv + kvh;
    const unsigned char *kb = p.p.k + at * PgBytes<HD, CODES>::K, *vb = p.p.v + at * PgBytes<HD, CODES>::V;
    const float *sb = CODES ? p.p.scales + at * 2 * PG_ROWS : nullptr;
    const float none = __uint_as_float(0x7FC00000u);
    auto index = [&](int row, int d) { return ((long long)(run.in0 + row - run.r0) * p.p.Hkv + kvh) * HD + d; };
    uint4 kw[NK];
    float ks[NK];
    unsigned vw[NV][4][CODES ? 2 : 4];
    f4 vs[NV][2];
#pragma unroll
    for (int k = 0; k < NK; k++) {
        const int task = wave + PG_WAVES * k, ch = task / 8 * 8 + (lane & 7), row = task % 8 * 8 + lane / 8;
        if (row < run.r0 || row >= run.r1 || (CH % 8 != 0 && ch >= CH)) continue;
        kw[k] = *reinterpret_cast<const uint4 *>(kb + (ch * PG_ROWS + row) * 16);
        ks[k] = CODES ? sb[row] : 1.0f;
    }
#pragma unroll
    for (int k = 0; k < NV; k++) {
        const int task = wave + PG_WAVES * k, h = task & 1, d = 64 * (task >> 1) + 4 * (lane >> 2), r0 = 32 * h + 4 * g;
        if (task >= 2 * DB || (HD % 64 != 0 && d >= HD) || r0 + 20 <= run.r0 || r0 >= run.r1) continue;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (CODES) {
                const uint2 v = *reinterpret_cast<const uint2 *>(vb + (d + i) * PG_ROWS + 16 * g + 8 * h);
                vw[k][i][0] = v.x;
                vw[k][i][1] = v.y;
            } else {
                const uint4 v = *reinterpret_cast<const uint4 *>(vb + ((h * HD + d + i) * 32 + 8 * g) * 2);
                vw[k][i][0] = v.x;
                vw[k][i][1] = v.y;
                vw[k][i][CODES ? 0 : 2] = v.z;
                vw[k][i][CODES ? 0 : 3] = v.w;
            }
        }
        if (CODES) {
#pragma unroll
            for (int t = 0; t < 2; t++) vs[k][t] = *reinterpret_cast<const f4 *>(sb + PG_ROWS + r0 + 16 * t);
        }
    }
#pragma unroll
    for (int k = 0; k < NK; k++) {
        const int task = wave + PG_WAVES * k, ch = task / 8 * 8 + (lane & 7), row = task % 8 * 8 + lane / 8;
        if (row < run.r0 || row >= run.r1 || (CH % 8 != 0 && ch >= CH)) continue;
        const unsigned w[4] = {kw[k].x, kw[k].y, kw[k].z, kw[k].w};
        const float s = bad ? none : ks[k];
        if constexpr (CODES) {
            float v[2][8];
#pragma unroll
            for (int i = 0; i < 16; i++) v[i >> 3][i & 7] = pg_byte(w[i >> 2], i & 3);
            pg_put<BF>(p.k_out, index(row, ch * E), v[0], s);
            if (HD % 16 == 0 || ch * E + 8 < HD) pg_put<BF>(p.k_out, index(row, ch * E + 8), v[1], s);
        } else {
            float v[8];
            unpack_bf16x8(kw[k], v);
            pg_put<BF>(p.k_out, index(row, ch * E), v, s);
        }
    }
#pragma unroll
    for (int k = 0; k < NV; k++) {
        const int task = wave + PG_WAVES * k, h = task & 1, d = 64 * (task >> 1) + 4 * (lane >> 2);
        if (task >= 2 * DB || (HD % 64 != 0 && d >= HD)) continue;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int row = 32 * h + 16 * (e >> 2) + 4 * g + (e & 3);
            if (row < run.r0 || row >= run.r1) continue;
            float v[4];
#pragma unroll
            for (int i = 0; i < 4; i++)
                v[i] = CODES ? pg_byte(vw[k][i][e >> 2], e & 3)
                             : __uint_as_float(e & 1 ? vw[k][i][CODES ? 0 : e >> 1] & 0xFFFF0000u : vw[k][i][CODES ? 0 : e >> 1] << 16);
            pg_put<BF>(p.v_out, index(row, d), v, bad ? none : CODES ? vs[k][e >> 2][e & 3] : 1.0f);
        }
    }
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

/* Workgroups (of one head) from which one takes two heads, and so on to eight: the rotation table and the run's search are then read
 * once, and the next head's rows are under way while one is worked on, as long as enough workgroups are left. 800 pages of 8 heads: one
 * head each 140 us, two 109, four (the rule) 97, eight 97. */
#define PG_HEADS_FROM 2048

/* workgroups of k_pg on a compute unit (registers) */
extern "C" int smol_paged_occupancy(int hd) { return hd > 128 ? 1 : 2; }

extern "C" int smol_launch_pages(const PgRunParams *pp, int hd, int write, hipStream_t st, hipEvent_t e0, hipEvent_t e1) {
    PgRunParams args = *pp, *p = &args;
    const long long pages = pg_max_run_pages(p->p.n_seq, p->rows);
    p->heads = 1;
    if (write)
        while (p->heads < 8 && 2 * p->heads <= p->p.Hkv && pages * p->p.Hkv / p->heads >= PG_HEADS_FROM) p->heads *= 2;
    const dim3 grid((unsigned)pages, (p->p.Hkv + p->heads - 1) / p->heads, write ? 2 : 1), tpb(write ? PA_TPB : PG_TPB);
    const bool bf = p->dtype == SMOL_IN_BF16;
#define PG_GO(HD, C, B) \
    if (write) hipExtLaunchKernelGGL((k_pg_append<HD, C, B>), grid, tpb, 0, st, e0, e1, 0, *p); \
    else hipExtLaunchKernelGGL((k_pg_read<HD, C, B>), grid, tpb, 0, st, e0, e1, 0, *p)
#define PG_RUN(HD) \
    if (p->p.codes && bf) { PG_GO(HD, true, true); } \
    else if (p->p.codes) { PG_GO(HD, true, false); } \
    else if (bf) { PG_GO(HD, false, true); } \
    else { PG_GO(HD, false, false); }
    PG_BY_HD(hd, PG_RUN)
    return hipGetLastError() == hipSuccess ? 0 : -3;
}

extern "C" int smol_launch_paged(const PgParams *p, int hd, hipStream_t st, hipEvent_t e0, hipEvent_t e1) {
    const dim3 tpb(PG_TPB);
    hipEvent_t first = e0;
    if (p->top > 0) {
        const dim3 gc((unsigned)(p->p.n_seq * ((p->p.stride + p->per - 1) / p->per)), p->p.Hkv);
#define PG_CHOOSE(HD) hipExtLaunchKernelGGL(k_pg_choose<HD>, gc, tpb, std::min(p->p.stride, PS_LDS) * 8, st, e0, nullptr, 0, *p)
        PG_BY_HD(hd, PG_CHOOSE)
        first = nullptr;
    }
    const dim3 grid(p->slots, p->p.Hkv, p->tiles);
    const int rows = PG_WAVES * std::min(p->G, PG_HEADS); /* of s_mem: the waves' outputs */
#define PG_STEP(HD) \
    if (p->p.codes) hipExtLaunchKernelGGL((k_pg<HD, true>), grid, tpb, PgQ<HD, true>::LDS + rows * PgGeom<HD>::XSTR * 4, st, first, e1, 0, *p); \
    else hipExtLaunchKernelGGL((k_pg<HD, false>), grid, tpb, PgQ<HD, false>::LDS + rows * PgGeom<HD>::XSTR * 4, st, first, e1, 0, *p)
    PG_BY_HD(hd, PG_STEP)
    return hipGetLastError() == hipSuccess ? 0 : -3;
}
