/*
 * attn_shared.hip - one decode step for a batch that shares a long prefix
 * (k_sh), and the step that also adds up the weight of every cached row
 * (k_sh as SH_SCORED); the rows that received little are taken out by
 * attn_evict.hip.
 *
 * Mathematics. Sequence i has own cache rows [0, l_i), the new token (row
 * l_i) and the prefix rows [0, P) that every sequence of the batch sees. With
 * s_j = scale q.k_j (cap tanh(s_j / cap) with a cap) over all of them,
 * out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m). A set of keys contributes
 * (m, l, O) = (max s, sum exp(s - m), sum exp(s - m) v), and two sets join by
 * rescaling to the larger m: so the prefix is one product of the batch's
 * n_seq x G rows of a kv head with its P keys, read once for all of them,
 * and each sequence's own rows are a product of G rows.
 *
 * Work split. A workgroup of four waves is one item: a chunk of the prefix
 * against a block of the batch's rows of a kv head, or a chunk of a
 * sequence's own rows against its G rows. Items need no table: the chunks are
 * equally long, so a workgroup finds its item from its number, and only the
 * sequences' (slot, length, position) travel with the call. Each item leaves
 * (m, l, O) of its rows in the workspace, and k_sh_merge joins a row's chunks.
 *   Narrow items (own rows; a prefix against at most 32 rows): all waves hold
 *     the same 16 rows and take 32-key slabs in turn, K and V^T fragments
 *     straight from the cache into registers; their states join in LDS. Bound
 *     by memory.
 *   Wide items (a prefix against more rows): the waves hold 16 rows each, 64
 *     together, and share every slab, which transfers bring into a ring in LDS
 *     in the order that its fragments are read without bank conflicts. Bound
 *     by the matrix cores and the softmax between their products, one after
 *     the other in a wave: three products for one (below).
 *
 * Measured on an MI355X (kernel time, head_dim 128, 16 heads over 8):
 * 4 sequences on 500 8.8 us and 16 on 4096 18.1 us (36 MB, 2.0 TB/s; the first
 * load waits for the sequences' table, a row and its turn, 3 to 5 us, and a
 * wave has one to four slabs); 64 on 16384 60 us (212 MB, 3.7 TB/s, matrix cores busy 26%;
 * a wide item 0.85 us a slab). head_dim 256, 8 heads over 1, 24 on 8191: 25.8 us,
 * one workgroup a compute unit, 2.6 us a wave's slab. Scored: 16 sequences of
 * 3000 to 4160 rows 56 us (244 MB, 4.4 TB/s). k_sh_merge 4 to 7 us, a launch's
 * and two round trips' time. Tried and not kept: a join by the last workgroup
 * instead of that launch, whose fences cost 1 us more at 4 sequences and 24 us
 * at 64; scores of the next slab beside the softmax of this one, a slab a step, 42.5
 * us a call against 38.2 for 64 on 16384 without own rows.
 *
 * Every lane loads, normalises and rotates exactly the elements of Q that its
 * fragments hold (row c, dims 32 ks + 8 j ..), so the prologue is one round of
 * loads without LDS or a barrier.
 *
 * Precision. K and V are the cache's bf16 bits. The fp32 side of each product
 * is split into bf16 parts that the matrix cores take exactly: Q into three
 * (24 bits, all of fp32), and so are the probabilities (two parts lose up to
 * 2^-16 of each, which measured 1.3e-6 of a row's norm where fp32 forms are
 * off by 5e-7). The new token's key and value are used in fp32 by the step
 * that appends them and rounded to nearest bf16 in the cache. Softmax state,
 * sums and the join are fp32.
 */
#include "attn_device.h"

#include <algorithm>

namespace {

constexpr int SH_NW = 4, SH_TPB = 64 * SH_NW;
constexpr int MASS_KEYS = 1024; /* rows whose weights a k_sh_merge workgroup adds up at a time */
constexpr int Q_PARTS = 3, P_PARTS = 3;

template <int HD>
struct ShGeom {
    static constexpr int KS = (HD + 31) / 32; /* 32-wide d chunks of a K fragment */
    static constexpr int DT = (HD + 15) / 16; /* 16-wide d tiles of the output */
    static constexpr int HALF = HD / 2;
    static constexpr int OSTR = DT * 16 + 4;  /* LDS row of a wave's output */
    static constexpr unsigned SLAB_BYTES = SMOL_SLAB * HD * 2;
    static constexpr bool POW2 = (HD & (HD - 1)) == 0; /* half a head is whole steps */
    static constexpr bool WIDE = HD == 64 || HD == 128; /* the sizes that have wide items */
    static constexpr int WS = 2;                       /* slabs of a wide item's step */
    static constexpr int STAGES = 2;
    static constexpr int CB_BYTES = (SH_NW * 16 * OSTR + 2 * SH_NW * 16) * 4; /* the waves' outputs, their m and l */
    static constexpr int RING_BYTES = WIDE ? STAGES * WS * 2 * (int)SLAB_BYTES : 0;
};

__device__ __forceinline__ void ld8f(const float *a, float *v) {
    const float4 x = *reinterpret_cast<const float4 *>(a), y = *reinterpret_cast<const float4 *>(a + 4);
    v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w; v[4] = y.x; v[5] = y.y; v[6] = y.z; v[7] = y.w;
}
/* x = p0 + p1 + p2 in bf16: each part is what the parts before it leave,
 * rounded to nearest, so three carry all 24 bits of x */
__device__ __forceinline__ void split8x3(const float *x, b8 &p0, b8 &p1, b8 &p2) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const __bf16 a = (__bf16)x[i];
        const float r = x[i] - (float)a;
        const __bf16 b = (__bf16)r;
        p0[i] = a;
        p1[i] = b;
        p2[i] = (__bf16)(r - (float)b);
    }
}

/* the bf16 values of word w (keys k and k + 1) outside [lo, hi) as zeros */
__device__ __forceinline__ unsigned keep_keys(unsigned w, int k, int lo, int hi) {
    return (k >= lo && k < hi ? w & 0xFFFFu : 0u) | (k + 1 >= lo && k + 1 < hi ? w & 0xFFFF0000u : 0u);
}
__device__ __forceinline__ uint4 keep_keys8(uint4 v, int k, int lo, int hi) {
    return make_uint4(keep_keys(v.x, k, lo, hi), keep_keys(v.y, k + 2, lo, hi), keep_keys(v.z, k + 4, lo, hi),
                      keep_keys(v.w, k + 6, lo, hi));
}
/* bit e: element e of the eight is not finite */
__device__ __forceinline__ unsigned not_finite8(uint4 v) {
    const unsigned a[4] = {v.x, v.y, v.z, v.w};
    unsigned bad = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        bad |= (a[i] & 0x7F80u) == 0x7F80u ? 1u << 2 * i : 0u;
        bad |= (a[i] & 0x7F800000u) == 0x7F800000u ? 2u << 2 * i : 0u;
    }
    return bad;
}

__device__ __forceinline__ ShSeq sh_seq(const ShParams &p, int i) {
    const int4 s = reinterpret_cast<const int4 *>(p.seqs_dev ? p.seqs_dev : p.seqs)[i];
    return ShSeq{s.x, s.y, s.z, s.w};
}
/* the sequence that own chunk u belongs to, when they are counted through: every wave compares 64 starts at a time */
__device__ __forceinline__ int sh_seq_of(const ShParams &p, int u) {
    const ShSeq *q = p.seqs_dev ? p.seqs_dev : p.seqs;
    int n = 0;
    for (int b = 0; b < p.n_seq; b += 64) {
        const int i = b + (threadIdx.x & 63);
        n += __popcll(__ballot(i < p.n_seq && q[min(i, p.n_seq - 1)].item0 <= u));
    }
    return __builtin_amdgcn_readfirstlane(n - 1);
}

/* the first of a sequence's own rows that its window leaves, down to a slab */
__device__ __forceinline__ int sh_own_first(const ShParams &p, const ShSeq &q) {
    return p.window > 0 ? max(0, q.pos - p.window + 1 - p.p_len) & ~(SMOL_SLAB - 1) : 0;
}
__device__ __forceinline__ int sh_own_chunks(const ShParams &p, const ShSeq &q) {
    return max(1, (q.len - sh_own_first(p, q) + p.s_chunk - 1) / p.s_chunk);
}

/* Elements [32 ks + 8 j, + 8) of a row for every ks, normalised (w: the norm's weights or null) and rotated to position
 * `pos`, the lanes j = 0 .. 3 (16 apart) of a column holding one row together; all of them call this. next(): what is
 * requested behind the row's own loads (a compute unit returns data in the order of its requests: the first slab in
 * front of them held the rows back by its whole transfer, 12 us instead of 5 with every compute unit streaming). */
template <int HD, class F>
__device__ __forceinline__ void sh_row(const ShParams &p, const void *x_in, long long row, const float *w, int pos, int j,
                                       float (&x)[ShGeom<HD>::KS][8], F next) {
    constexpr int KS = ShGeom<HD>::KS, HALF = ShGeom<HD>::HALF, KH = KS / 2;
    constexpr bool POW2 = ShGeom<HD>::POW2;
    const bool neox = p.rope_kind == SMOL_ROPE_NEOX_K, inter = p.rope_kind == SMOL_ROPE_INTERLEAVED_K;
    const float *ct = p.rope_cos + (long long)pos * HD, *st = p.rope_sin + (long long)pos * HD;
    /* the norm's weights and the table's row are requested with the row: behind the first slab they would wait for it */
    float wv[KS][8];
    float cv[KH][8], sn[KH][8]; /* the table repeats a row's first half in its second (NeoX), or every value (interleaved) */
#pragma unroll
    for (int ks = 0; ks < KS; ks++) {
        const int d0 = 32 * ks + 8 * j;
#pragma unroll
        for (int i = 0; i < 8; i++) x[ks][i] = 0.0f;
        if (HD % 32 == 0 || d0 < HD) load8(x_in, p.in_dtype, row + d0, x[ks]);
    }
    if (w) {
#pragma unroll
        for (int ks = 0; ks < KS; ks++)
            if (HD % 32 == 0 || 32 * ks + 8 * j < HD) ld8f(w + 32 * ks + 8 * j, wv[ks]);
    }
    if (POW2 && neox) {
#pragma unroll
        for (int ks = 0; ks < KH; ks++) {
            ld8f(ct + 32 * ks + 8 * j, cv[ks]);
            ld8f(st + 32 * ks + 8 * j, sn[ks]);
        }
    } else if (POW2 && inter) {
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            float c8[8], s8[8];
            ld8f(ct + 32 * ks + 8 * j, c8);
            ld8f(st + 32 * ks + 8 * j, s8);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                cv[ks / 2][ks % 2 * 4 + i] = c8[2 * i];
                sn[ks / 2][ks % 2 * 4 + i] = s8[2 * i];
            }
        }
    }
    next();
    float ri = 1.0f;
    if (__any(w != nullptr)) {
        float ss = 0.0f;
#pragma unroll
        for (int ks = 0; ks < KS; ks++)
#pragma unroll
            for (int i = 0; i < 8; i++) ss = fmaf(x[ks][i], x[ks][i], ss);
        ri = 1.0f / sqrtf(row_sum4(ss) / (float)HD + p.norm_eps);
        if (w) {
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                const int d0 = 32 * ks + 8 * j;
                if (HD % 32 == 0 || d0 < HD) {
#pragma unroll
                    for (int i = 0; i < 8; i++) x[ks][i] = x[ks][i] * wv[ks][i] * ri;
                }
            }
        }
    }
    if (POW2 && neox) {
        /* the partner half a head away is this lane's own */
#pragma unroll
        for (int ks = 0; ks < KH; ks++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float a = x[ks][i], b = x[ks + KH][i];
                x[ks][i] = fmaf(a, cv[ks][i], -(b * sn[ks][i]));
                x[ks + KH][i] = fmaf(b, cv[ks][i], a * sn[ks][i]);
            }
    } else if (POW2 && inter) {
#pragma unroll
        for (int ks = 0; ks < KS; ks++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float a = x[ks][2 * i], b = x[ks][2 * i + 1], c = cv[ks / 2][ks % 2 * 4 + i], d = sn[ks / 2][ks % 2 * 4 + i];
                x[ks][2 * i] = fmaf(a, c, -(b * d));
                x[ks][2 * i + 1] = fmaf(b, c, a * d);
            }
    } else if (inter || neox) {
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            const int d0 = 32 * ks + 8 * j;
            if (HD % 32 != 0 && d0 >= HD) continue;
            float c8[8], s8[8];
            ld8f(ct + d0, c8);
            ld8f(st + d0, s8);
            if (inter) {
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    const float a = x[ks][i], b = x[ks][i + 1];
                    x[ks][i] = fmaf(a, c8[i], -(b * s8[i]));
                    x[ks][i + 1] = fmaf(b, c8[i + 1], a * s8[i + 1]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int d = d0 + i, pd = d < HALF ? d + HALF : d - HALF;
                    float pr = p.in_dtype == SMOL_IN_BF16 ? bf16_to_f32(((const uint16_t *)x_in)[row + pd])
                                                          : ((const float *)x_in)[row + pd];
                    if (w) pr = pr * w[pd] * ri;
                    const float t = pr * s8[i];
                    x[ks][i] = fmaf(x[ks][i], c8[i], d < HALF ? -t : t);
                }
            }
        }
    }
}

/* One item: R rows against the keys [kb, ke) of the region at kc / vtc */
struct ShItem {
    bool prefix;
    int g;              /* kv head */
    int row0;           /* prefix: first row of the batch's n_seq G; own rows: first head of the group */
    int R;              /* rows */
    int seq;            /* own rows: the sequence */
    int kb, ke;
    const uint16_t *kc, *vtc;
    long long region_bytes;
    bool with_new;      /* own rows: this item takes the new token too */
    float *part_o, *part_ml; /* of its row 0 */
};

/* A wave's 16 rows: their fragments, the first key that each may see, and the softmax state */
template <int HD>
struct ShRows {
    static constexpr int KS = ShGeom<HD>::KS, DT = ShGeom<HD>::DT;
    b8 q[Q_PARTS][KS];
    int lo, lo_min, lo_max;
    float m, l;
    f4 o[DT];
};

constexpr int OWN_ROWS = 15; /* heads of an own-rows item: the 16th column holds the new key */

/* Column c: row r0 + c of the item, if it has one; its fp32 elements stay in y. The column behind an own-rows item's last
 * row holds the new key (normalised and rotated, not scaled), which takes no part in the products. */
template <int HD, class F>
__device__ __forceinline__ void sh_rows(const ShParams &p, const ShItem &it, int r0, int c, int j, ShRows<HD> &w,
                                        float (&y)[ShGeom<HD>::KS][8], F next) {
    constexpr int KS = ShGeom<HD>::KS, DT = ShGeom<HD>::DT;
    const bool live = r0 + c < it.R, is_k = it.with_new && c == it.R;
    const int r = live ? r0 + c : 0;
    const int seq = it.prefix ? (it.row0 + r) / p.G : it.seq;
    const int head = it.g * p.G + (it.prefix ? (it.row0 + r) % p.G : it.row0 + r);
    const int pos = sh_seq(p, seq).pos;
    sh_row<HD>(p, is_k ? p.k_in : p.q_in, is_k ? ((long long)seq * p.Hkv + it.g) * HD : ((long long)seq * p.Hq + head) * HD,
               is_k ? p.k_norm : p.q_norm, pos, j, y, next);
    const float f = live ? p.qscale : 1.0f;
#pragma unroll
    for (int ks = 0; ks < KS; ks++) {
        float z[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            y[ks][i] *= f;
            z[i] = live ? y[ks][i] : 0.0f;
        }
        split8x3(z, w.q[0][ks], w.q[1][ks], w.q[2][ks]);
    }
    w.lo = w.lo_min = w.lo_max = 0;
    if (p.window > 0) {
        const int lo = max(0, pos - p.window + 1 - (it.prefix ? 0 : p.p_len));
        w.lo = live ? lo : 0;
        w.lo_max = w.lo;
        w.lo_min = live ? lo : 1 << 30;
#pragma unroll
        for (int sh = 1; sh < 16; sh <<= 1) {
            w.lo_max = max(w.lo_max, __shfl_xor(w.lo_max, sh));
            w.lo_min = min(w.lo_min, __shfl_xor(w.lo_min, sh));
        }
        w.lo_max = __builtin_amdgcn_readfirstlane(w.lo_max);
        w.lo_min = __builtin_amdgcn_readfirstlane(w.lo_min);
    }
    w.m = -INFINITY;
    w.l = 0.0f;
#pragma unroll
    for (int dt = 0; dt < DT; dt++) w.o[dt] = f4{0.f, 0.f, 0.f, 0.f};
}

/* S^T = K.Q^T of one slab: the small parts of Q first */
template <int HD>
__device__ __forceinline__ void sh_qk(const ShRows<HD> &w, const uint4 (&k)[2][ShGeom<HD>::KS], f4 (&s)[2]) {
    s[0] = s[1] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int q = Q_PARTS - 1; q >= 0; q--)
#pragma unroll
        for (int ks = 0; ks < ShGeom<HD>::KS; ks++)
#pragma unroll
            for (int h = 0; h < 2; h++) s[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_b8(k[h][ks]), w.q[q][ks], s[h], 0, 0, 0);
}

/* The scores of NS slabs from key k0 on: capped, kept (logits: where this lane's go, or null), and -inf for keys that a row
 * does not see; nan: whether a row sees a value that is no number among those taken out. odd becomes the largest of the
 * scores' bits as whole numbers: MINUS_INF or more with a score of -inf (or of +inf and a cap, which makes a number of it), and
 * with no finite score. */
constexpr unsigned MINUS_INF = 0xFF800000u;
template <int HD, int NS, bool SC>
__device__ __forceinline__ bool sh_mask(const ShParams &p, const ShRows<HD> &w, int k0, int ke, int j, f4 (&s)[NS][2],
                                        uint4 (&v)[NS][ShGeom<HD>::DT], float *logits, unsigned &odd) {
    constexpr int DT = ShGeom<HD>::DT;
#pragma unroll
    for (int u = 0; u < NS; u++)
#pragma unroll
        for (int e = 0; e < 8; e++) odd = max(odd, __float_as_uint(s[u][e >> 2][e & 3]));
    asm volatile("" : "+v"(odd)); /* formed here: later, the scores as they were would hold registers */
    if (p.cap2 > 0.0f) {
#pragma unroll
        for (int u = 0; u < NS; u++)
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    odd = max(odd, s[u][h][i] == INFINITY ? MINUS_INF : 0u);
                    s[u][h][i] = p.cap2 * tanhf(s[u][h][i] / p.cap2);
                }
    }
    if (SC && logits) {
#pragma unroll
        for (int h = 0; h < 2; h++) *reinterpret_cast<f4 *>(logits + 4 * h) = s[0][h];
    }
    /* keys that some row does not see: their scores and, since 0 x inf is no number, their values */
    const bool low = k0 < w.lo_max;
    bool nan = false;
    if (low || k0 + NS * SMOL_SLAB > ke) {
#pragma unroll
        for (int u = 0; u < NS; u++) {
            const int ku = k0 + u * SMOL_SLAB + 8 * j;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int key = ku + e;
                s[u][e >> 2][e & 3] = key >= w.lo && key < ke ? s[u][e >> 2][e & 3] : -INFINITY;
            }
#pragma unroll
            for (int dt = 0; dt < DT; dt++) v[u][dt] = keep_keys8(v[u][dt], ku, w.lo_min, ke);
            if (low && w.lo_min < w.lo_max) {
                /* rows see different keys here: a key with a value that is not finite is taken out for all of them,
                 * and the rows that see it get a sum that is no number */
                unsigned bad = 0;
#pragma unroll
                for (int dt = 0; dt < DT; dt++) bad |= not_finite8(v[u][dt]);
                if (__any(bad != 0)) {
#pragma unroll
                    for (int sh = 1; sh < 16; sh <<= 1) bad |= __shfl_xor(bad, sh);
                    const uint4 keep = make_uint4((bad & 1 ? 0u : 0xFFFFu) | (bad & 2 ? 0u : 0xFFFF0000u),
                                                  (bad & 4 ? 0u : 0xFFFFu) | (bad & 8 ? 0u : 0xFFFF0000u),
                                                  (bad & 16 ? 0u : 0xFFFFu) | (bad & 32 ? 0u : 0xFFFF0000u),
                                                  (bad & 64 ? 0u : 0xFFFFu) | (bad & 128 ? 0u : 0xFFFF0000u));
#pragma unroll
                    for (int dt = 0; dt < DT; dt++)
                        v[u][dt] = make_uint4(v[u][dt].x & keep.x, v[u][dt].y & keep.y, v[u][dt].z & keep.z, v[u][dt].w & keep.w);
#pragma unroll
                    for (int e = 0; e < 8; e++) nan |= (bad >> e & 1) != 0 && ku + e >= w.lo;
                }
            }
        }
    }
    return nan;
}

/* softmax of NS slabs and O^T += V^T.P^T */
template <int HD, int NS>
__device__ __forceinline__ void sh_pv(ShRows<HD> &w, const f4 (&s)[NS][2], const uint4 (&v)[NS][ShGeom<HD>::DT], bool nan) {
    constexpr int DT = ShGeom<HD>::DT;
    float mx = -INFINITY;
#pragma unroll
    for (int u = 0; u < NS; u++)
#pragma unroll
        for (int e = 0; e < 8; e++) mx = fmaxf(mx, s[u][e >> 2][e & 3]);
    mx = row_max4(mx);
    const bool need = mx > w.m + LAZY_T;
    if (__any(need)) {
        const float m_new = need ? mx : w.m;
        const float alpha = need ? __builtin_amdgcn_exp2f(w.m - m_new) : 1.0f;
#pragma unroll
        for (int dt = 0; dt < DT; dt++) w.o[dt] *= alpha;
        w.l *= alpha;
        w.m = m_new;
    }
    const float m_use = w.m == -INFINITY ? 0.0f : w.m;
    float ps = nan ? __builtin_nanf("") : 0.0f;
    b8 pp[NS][P_PARTS];
#pragma unroll
    for (int u = 0; u < NS; u++) {
        float pv[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            pv[e] = __builtin_amdgcn_exp2f(s[u][e >> 2][e & 3] - m_use);
            ps += pv[e];
        }
        split8x3(pv, pp[u][0], pp[u][1], pp[u][2]);
    }
    w.l += ps;
#pragma unroll
    for (int u = 0; u < NS; u++)
#pragma unroll
        for (int q = P_PARTS - 1; q >= 0; q--)
#pragma unroll
            for (int dt = 0; dt < DT; dt++)
                w.o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_b8(v[u][dt]), pp[u][q], w.o[dt], 0, 0, 0);
}

/* Rows that see a key with an element that is not finite become NaN. Such a key's scores are not finite, for every row: NaN and
 * +inf go through the softmax, but -inf has no weight and a cap makes numbers of both. A finite product past fp32's range gives
 * them too. So the keys [k0, ke), a slab every `step`, are read again where odd tells of such a score. (A value that is not
 * finite shows in its dimension of the sum: k_sh_merge.) */
template <int HD>
__device__ __forceinline__ void sh_spoil(const ShItem &it, ShRows<HD> &w, unsigned odd, int k0, int step) {
    constexpr int PC = HD / 8;
    if (!__any(odd >= MINUS_INF)) return;
    const rsrc_t rs = make_rsrc(it.kc, it.region_bytes);
#pragma unroll 1
    for (; k0 < it.ke; k0 += step) {
        unsigned bad = 0; /* bit r: row r of the slab */
#pragma unroll 1
        for (int i = threadIdx.x & 63; i < SMOL_SLAB * PC; i += 64)
            if (not_finite8(bload(rs, i * 16, (unsigned)(k0 / SMOL_SLAB) * ShGeom<HD>::SLAB_BYTES))) bad |= 1u << i / PC;
#pragma unroll
        for (int sh = 1; sh < 64; sh <<= 1) bad |= __shfl_xor(bad, sh);
        const int lo = max(0, w.lo - k0), hi = min(SMOL_SLAB, it.ke - k0);
        const unsigned seen = lo < hi ? (~0u >> (SMOL_SLAB - hi)) & (~0u << lo) : 0u;
        if (bad & seen) w.l = __builtin_nanf("");
    }
}

/* At most 16 rows, the same in every wave; the waves take the slabs in turn */
template <int HD, bool SC>
__device__ __forceinline__ void sh_narrow(const ShParams &p, const ShItem &it, char *smem) {
    using Gm = ShGeom<HD>;
    constexpr int KS = Gm::KS, DT = Gm::DT, OSTR = Gm::OSTR;
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, j = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kt_row = 8 * (c >> 2) + (c & 3);
    unsigned vo_k[2][KS], vo_v[DT];
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            const int d0 = 32 * ks + 8 * j;
            vo_k[t][ks] = (HD % 32 == 0 || d0 < HD) ? (unsigned)(((kt_row + 4 * t) * HD + d0) * 2) : OOB_OFF;
        }
#pragma unroll
    for (int dt = 0; dt < DT; dt++) {
        const int d = 16 * dt + c;
        vo_v[dt] = (HD % 16 == 0 || d < HD) ? (unsigned)((d * SMOL_SLAB + 8 * j) * 2) : OOB_OFF;
    }
    uint4 k[2][KS], v[1][DT];
    /* a slab at or past ke has an empty range: its loads return zeros */
    auto issue_k = [&](int k0) __attribute__((always_inline)) {
        const bool live = k0 < it.ke;
        const rsrc_t rs = make_rsrc(it.kc, live ? it.region_bytes : 0);
        const unsigned so = live ? (unsigned)(k0 / SMOL_SLAB) * Gm::SLAB_BYTES : 0u;
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
                k[t][ks] = HD % 32 == 0 ? bload(rs, vo_k[0][0], so + (unsigned)((4 * t * HD + 32 * ks) * 2))
                                        : bload(rs, vo_k[t][ks], so);
    };
    auto issue_v = [&](int k0) __attribute__((always_inline)) {
        const bool live = k0 < it.ke;
        const rsrc_t rs = make_rsrc(it.vtc, live ? it.region_bytes : 0);
        const unsigned so = live ? (unsigned)(k0 / SMOL_SLAB) * Gm::SLAB_BYTES : 0u;
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
            v[0][dt] = HD % 16 == 0 ? bload(rs, vo_v[0], so + (unsigned)(16 * dt * SMOL_SLAB * 2)) : bload(rs, vo_v[dt], so);
    };
    int k0 = it.kb + wave * SMOL_SLAB;
    ShRows<HD> w;
    /* the new token is the last wave's, which has the fewest slabs: its key and value wait in LDS until the slabs are done */
    const bool add_new = it.with_new && wave == SH_NW - 1;
    float *s_kn = reinterpret_cast<float *>(smem + Gm::CB_BYTES), *s_vn = s_kn + KS * 32;
    const long long new_row = ((long long)it.seq * p.Hkv + it.g) * HD;
    {
        float y[KS][8], vn[(HD + 63) / 64];
        sh_rows<HD>(p, it, 0, c, j, w, y, [&]() __attribute__((always_inline)) {
            if (add_new) {
#pragma unroll
                for (int u = 0; u < (HD + 63) / 64; u++)
                    if (HD % 64 == 0 || 64 * u + lane < HD)
                        vn[u] = p.in_dtype == SMOL_IN_BF16 ? bf16_to_f32(((const uint16_t *)p.v_in)[new_row + 64 * u + lane])
                                                           : ((const float *)p.v_in)[new_row + 64 * u + lane];
            }
            issue_k(k0);
            if (HD <= 128) issue_v(k0); /* at 256 the rows' registers leave no room for both */
        });
        if (add_new) {
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
                if (c == it.R) {
                    *reinterpret_cast<f4 *>(s_kn + 32 * ks + 8 * j) = f4{y[ks][0], y[ks][1], y[ks][2], y[ks][3]};
                    *reinterpret_cast<f4 *>(s_kn + 32 * ks + 8 * j + 4) = f4{y[ks][4], y[ks][5], y[ks][6], y[ks][7]};
                }
#pragma unroll
            for (int u = 0; u < (HD + 63) / 64; u++)
                if (64 * u + lane < KS * 32) s_vn[64 * u + lane] = HD % 64 == 0 || 64 * u + lane < HD ? vn[u] : 0.0f;
        }
    }
    if (HD > 128) issue_v(k0);
    float *logits = SC && c < it.R
                        ? p.logits + ((long long)it.seq * p.Hq + it.g * p.G + it.row0 + c) * p.l_stride + 8 * j : nullptr;
    unsigned odd = 0;
    while (k0 < it.ke) {
        f4 s[1][2];
        sh_qk<HD>(w, k, s[0]);
        const int k1 = k0 + SMOL_SLAB * SH_NW;
        issue_k(k1);
        const bool nan = sh_mask<HD, 1, SC>(p, w, k0, it.ke, j, s, v, SC && logits ? logits + k0 : nullptr, odd);
        sh_pv<HD, 1>(w, s, v, nan);
        issue_v(k1);
        k0 = k1;
    }
    sh_spoil<HD>(it, w, odd, it.kb + wave * SMOL_SLAB, SMOL_SLAB * SH_NW);
    float lt = row_sum4(w.l);
    if (add_new) {
        /* the new token: its fp32 score of every row (the three parts hold the row whole), its share of the state, its
         * bf16 row in the cache */
        float sd = 0.0f, z = 0.0f; /* z: zero, or NaN with an element of the key that is not finite */
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            float kn[8];
            ld8f(s_kn + 32 * ks + 8 * j, kn);
            /* (formed here: in front of the slab loop the fp32 rows would hold registers through it) */
#pragma unroll
            for (int q = 0; q < Q_PARTS; q++) asm volatile("" : "+v"(w.q[q][ks]));
#pragma unroll
            for (int i = 0; i < 8; i++) {
                sd = fmaf(((float)w.q[0][ks][i] + (float)w.q[1][ks][i]) + (float)w.q[2][ks][i], kn[i], sd);
                z = fmaf(kn[i], 0.0f, z);
            }
        }
        sd = row_sum4(sd) + row_sum4(z);
        if (p.cap2 > 0.0f) sd = p.cap2 * tanhf(sd / p.cap2);
        if (SC && j == 0 && c < it.R) p.logit_new[(long long)it.seq * p.Hq + it.g * p.G + it.row0 + c] = sd;
        const float mm = fmaxf(w.m, sd), mu = mm == -INFINITY ? 0.0f : mm;
        const float alpha = __builtin_amdgcn_exp2f(w.m - mu), pn = __builtin_amdgcn_exp2f(sd - mu);
        lt = fmaf(lt, alpha, pn);
        w.m = mm;
#pragma unroll
        for (int dt = 0; dt < DT; dt++) w.o[dt] = w.o[dt] * alpha + *reinterpret_cast<const f4 *>(s_vn + 16 * dt + 4 * j) * pn;
        if (it.row0 == 0) {
            const ShSeq sq = sh_seq(p, it.seq);
            const long long base = (long long)sq.slot * p.c_slot_stride + (long long)it.g * p.cap * HD;
            if (lane < HD / 8) {
                float kn[8];
                ld8f(s_kn + 8 * lane, kn);
                *reinterpret_cast<uint4 *>(p.kc + base + (long long)sq.len * HD + 8 * lane) = pack_bf16x8(kn);
            }
            uint16_t *vt = p.vtc + base + (long long)(sq.len / SMOL_SLAB) * SMOL_SLAB * HD + sq.len % SMOL_SLAB;
            for (int d = lane; d < HD; d += 64) vt[(long long)d * SMOL_SLAB] = f32_to_bf16(s_vn[d]);
        }
    }

    /* the waves' states join */
    float *cb = reinterpret_cast<float *>(smem), *cm = cb + SH_NW * 16 * OSTR, *cl = cm + SH_NW * 16;
    if (j == 0) {
        cm[wave * 16 + c] = w.m;
        cl[wave * 16 + c] = lt;
    }
#pragma unroll
    for (int dt = 0; dt < DT; dt++) *reinterpret_cast<f4 *>(cb + (wave * 16 + c) * OSTR + 16 * dt + 4 * j) = w.o[dt];
    __syncthreads();
    for (int e = tid; e < it.R * (HD / 4); e += SH_TPB) {
        const int r = e / (HD / 4), d = (e - r * (HD / 4)) * 4;
        float mm = -INFINITY;
#pragma unroll
        for (int q = 0; q < SH_NW; q++) mm = fmaxf(mm, cm[q * 16 + r]);
        const float mu = mm == -INFINITY ? 0.0f : mm;
        f4 acc = {0.f, 0.f, 0.f, 0.f};
        float ls = 0.0f;
#pragma unroll
        for (int q = 0; q < SH_NW; q++) {
            const float f = __builtin_amdgcn_exp2f(cm[q * 16 + r] - mu);
            ls = fmaf(f, cl[q * 16 + r], ls);
            acc += f * *reinterpret_cast<f4 *>(cb + (q * 16 + r) * OSTR + d);
        }
        *reinterpret_cast<f4 *>(it.part_o + (long long)r * HD + d) = acc;
        if (d == 0) *reinterpret_cast<float2 *>(it.part_ml + r * 2) = make_float2(mm, ls);
    }
}

/* 64 rows of the batch, 16 a wave, against slabs that all waves share through LDS. The ring's 16-byte pieces are placed
 * so that the sixteen lanes that LDS serves together (c 0..3 and 12..15 of one j, c 4..11 of the next) fall in different
 * columns of its 256-byte lines: piece q of K row r at q ^ c(r) with the lane c that reads the row (c / 2 at head_dim 64,
 * whose lines hold two rows), piece j of V^T row d at j ^ (d >> 1 & 3); the conflict counter reads 0. A transfer writes its
 * lanes' pieces one after the other, so it is the lanes' source addresses that are permuted. */
template <int HD>
__device__ __forceinline__ void sh_wide(const ShParams &p, const ShItem &it, char *smem) {
    using Gm = ShGeom<HD>;
    constexpr int KS = Gm::KS, DT = Gm::DT, STAGES = Gm::STAGES, WS = Gm::WS, PC = HD / 8; /* PC: 16-byte pieces of a K row */
    constexpr int PART = Gm::SLAB_BYTES / 1024, ND = 2 * PART / SH_NW; /* 1 KB transfers of a slab's K (V^T); a wave's of a slab */
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, j = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = (it.ke - it.kb + SMOL_SLAB - 1) / SMOL_SLAB, first = it.kb / SMOL_SLAB;
    const rsrc_t rk = make_rsrc(it.kc, it.region_bytes), rv = make_rsrc(it.vtc, it.region_bytes);
    const unsigned lds0 = (unsigned)(size_t)smem;
    /* transfer t of a slab (K's first): lane l's piece at 16 l */
    unsigned voff[ND];
#pragma unroll
    for (int u = 0; u < ND; u++) {
        const int t = wave * ND + u, piece = t % PART * 64 + lane;
        if (t < PART) {
            const int r = piece / PC, q = piece % PC;
            voff[u] = (unsigned)((r * PC + (q ^ (HD == 128 ? (r & 3) | (r >> 3 & 3) << 2 : (r >> 1 & 1) | (r >> 3 & 3) << 1))) * 16);
        } else {
            const int d = piece / 4, q = piece % 4;
            voff[u] = (unsigned)((d * 4 + (q ^ (d >> 1 & 3))) * 16);
        }
    }
    auto fetch = [&](int i) __attribute__((always_inline)) {
#pragma unroll
        for (int s = 0; s < WS; s++) {
            /* past the last slab the last one again: every step has the same number of transfers in flight */
            const unsigned so = (unsigned)(first + min(i * WS + s, n - 1)) * Gm::SLAB_BYTES;
            const unsigned at = __builtin_amdgcn_readfirstlane(lds0 + (unsigned)((i % STAGES) * WS + s) * 2 * Gm::SLAB_BYTES + wave * ND * 1024);
#pragma unroll
            for (int u = 0; u < ND; u++) dma_1k(wave * ND + u < PART ? rk : rv, voff[u], so, at + u * 1024);
        }
    };
    ShRows<HD> w;
    {
        float y[KS][8];
        sh_rows<HD>(p, it, 16 * wave, c, j, w, y, []() {});
    }
    /* the compiler's own loads are done before the first transfer, so vmcnt counts transfers alone from here on */
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
    for (int i = 0; i < STAGES - 1; i++) fetch(i);
    const int kt_row = 8 * (c >> 2) + (c & 3), ksw = HD == 128 ? c : c >> 1;
    const int n_steps = (n + WS - 1) / WS;
    unsigned odd = 0;
    for (int i = 0; i < n_steps; i++) {
        /* this wave's part of step i has landed (later ones may be on their way); then everybody's has, and nobody
         * still reads the stage that the next transfers overwrite */
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((STAGES - 2) * WS * ND) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        fetch(i + STAGES - 1);
        const char *sk = smem + (i % STAGES) * WS * 2 * Gm::SLAB_BYTES;
        f4 s[WS][2];
        uint4 v[WS][DT];
#pragma unroll
        for (int u = 0; u < WS; u++) {
            uint4 k[2][KS];
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
#pragma unroll
                for (int t = 0; t < 2; t++) /* rows kt_row + 4 t: the swizzle's bits are c's */
                    k[t][ks] = *reinterpret_cast<const uint4 *>(sk + u * 2 * Gm::SLAB_BYTES +
                                                                ((kt_row + 4 * t) * PC + ((4 * ks + j) ^ ksw)) * 16);
            sh_qk<HD>(w, k, s[u]);
        }
#pragma unroll
        for (int u = 0; u < WS; u++)
#pragma unroll
            for (int dt = 0; dt < DT; dt++) {
                const int d = 16 * dt + c;
                v[u][dt] = *reinterpret_cast<const uint4 *>(sk + (2 * u + 1) * Gm::SLAB_BYTES + (d * 4 + (j ^ (d >> 1 & 3))) * 16);
            }
        /* a slab past the last one repeats it; its keys are past ke */
        const bool nan = sh_mask<HD, WS, false>(p, w, it.kb + i * WS * SMOL_SLAB, it.ke, j, s, v, nullptr, odd);
        sh_pv<HD, WS>(w, s, v, nan);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); /* no transfer outlives the workgroup */
    sh_spoil<HD>(it, w, odd, it.kb, SMOL_SLAB);
    const float lt = row_sum4(w.l);
    const int r = 16 * wave + c;
    if (r < it.R) {
#pragma unroll
        for (int dt = 0; dt < DT; dt++) *reinterpret_cast<f4 *>(it.part_o + (long long)r * HD + 16 * dt + 4 * j) = w.o[dt];
        if (j == 0) *reinterpret_cast<float2 *>(it.part_ml + r * 2) = make_float2(w.m, lt);
    }
}

} // namespace

/* KIND: what the call's prefix items are */
enum { SH_NARROW, SH_WIDE, SH_SCORED };
template <int HD, int KIND>
__global__ __launch_bounds__(SH_TPB, HD <= 128 ? 2 : 1) void k_sh(const ShParams p) {
    using Gm = ShGeom<HD>;
    constexpr int NARROW = Gm::CB_BYTES + 2 * Gm::KS * 32 * 4; /* the waves' states, the new key and value */
    constexpr int LDS = KIND == SH_WIDE && Gm::RING_BYTES > NARROW ? Gm::RING_BYTES : NARROW;
    constexpr int ROWS = KIND == SH_WIDE ? 16 * SH_NW : 16;
    __shared__ __attribute__((aligned(1024))) char smem[LDS];
    const int b = blockIdx.x;
    ShItem it;
    if constexpr (KIND != SH_SCORED) {
        if (b < p.n_pblocks) {
            /* workgroups b and b + 8 share an L2: the row blocks of one chunk follow each other there */
            const int rb = (b / 8) % p.n_rb, u = (b / (8 * p.n_rb)) * 8 + b % 8;
            const int g = u % p.Hkv, sp = u / p.Hkv;
            if (sp >= p.n_ps) return;
            it.prefix = true;
            it.g = g;
            it.row0 = rb * ROWS;
            it.R = min(ROWS, p.n_seq * p.G - it.row0);
            it.seq = 0;
            it.kb = p.p_first + sp * p.p_chunk;
            it.ke = min(p.p_len, it.kb + p.p_chunk);
            it.kc = p.pk + (long long)g * p.pcap * HD;
            it.vtc = p.pvt + (long long)g * p.pcap * HD;
            it.region_bytes = (long long)p.pcap * HD * 2;
            it.with_new = false;
            const long long row = ((long long)sp * p.Hkv + g) * p.n_seq * p.G + it.row0;
            it.part_o = p.p_o + row * HD;
            it.part_ml = p.p_ml + row * 2;
            if constexpr (KIND == SH_WIDE) sh_wide<HD>(p, it, smem);
            else sh_narrow<HD, false>(p, it, smem);
            return;
        }
    }
    const int a = b - p.n_pblocks;
    const int srb = a % p.s_rb, g = (a / p.s_rb) % p.Hkv, u = a / (p.s_rb * p.Hkv);
    const int i = p.n_own ? sh_seq_of(p, u) : u % p.n_seq;
    const ShSeq sq = sh_seq(p, i);
    const int sp = p.n_own ? u - sq.item0 : u / p.n_seq;
    if (sp >= sh_own_chunks(p, sq)) return;
    it.prefix = false;
    it.g = g;
    it.row0 = srb * OWN_ROWS;
    it.R = min(OWN_ROWS, p.G - it.row0);
    it.seq = i;
    it.kb = sh_own_first(p, sq) + sp * p.s_chunk;
    it.ke = min(sq.len, it.kb + p.s_chunk);
    const long long base = (long long)sq.slot * p.c_slot_stride + (long long)g * p.cap * HD;
    it.kc = p.kc + base;
    it.vtc = p.vtc + base;
    it.region_bytes = (long long)p.cap * HD * 2;
    it.with_new = sp == 0;
    const long long row = (((long long)i * p.Hkv + g) * p.n_ss + sp) * p.G + it.row0;
    it.part_o = p.s_o + row * HD;
    it.part_ml = p.s_ml + row * 2;
    sh_narrow<HD, KIND == SH_SCORED>(p, it, smem);
}

/* Joins the chunks of the output rows, one workgroup a row (a sequence's
 * head): (m, l) of every chunk first, then the outputs, as many chunks at a
 * time as there are lanes for. With mass (SH_SCORED): the workgroups behind
 * those add the weights exp2(s - m) / l of MASS_KEYS cached rows of a
 * (sequence, kv head), from the scores that k_sh left, in the heads' order;
 * the heads' (m, l) are found first, a wave a head, so that the scores of four
 * heads are under way at once (8 heads over 1: 5.2 us, 7.5 head after head). */

template <int HD>
__global__ __launch_bounds__(256) void k_sh_merge(const ShParams p) {
    constexpr int D4 = HD / 4, GL = HD <= 64 ? 16 : HD <= 128 ? 32 : 64, NG = 256 / GL;
    __shared__ __attribute__((aligned(16))) float s_w[2 * SH_MAX_SPLIT], s_red[NG * GL * 4], s_x[16];
    constexpr int MASS_HEADS = NG * GL * 2; /* heads whose state s_red holds */
    const int tid = threadIdx.x, wave = tid >> 6;
    const int n_out = p.n_seq * p.Hq;
    auto block_max = [&](float v) {
        for (int sh = 1; sh < 64; sh <<= 1) v = fmaxf(v, __shfl_xor(v, sh));
        if ((tid & 63) == 0) s_x[wave] = v;
        __syncthreads();
        return fmaxf(fmaxf(s_x[0], s_x[1]), fmaxf(s_x[2], s_x[3]));
    };
    auto block_sum = [&](float v) {
        for (int sh = 1; sh < 64; sh <<= 1) v += __shfl_xor(v, sh);
        if ((tid & 63) == 0) s_x[4 + wave] = v;
        __syncthreads();
        return (s_x[4] + s_x[5]) + (s_x[6] + s_x[7]);
    };
    if ((int)blockIdx.x < n_out) {
        const int i = blockIdx.x / p.Hq, head = blockIdx.x - i * p.Hq, g = head / p.G, h = head - g * p.G;
        const ShSeq sq = sh_seq(p, i);
        const int n = p.n_ps + sh_own_chunks(p, sq);
        auto row_of = [&](int k) -> long long {
            return k < p.n_ps ? (((long long)k * p.Hkv + g) * p.n_seq + i) * p.G + h
                              : (((long long)i * p.Hkv + g) * p.n_ss + (k - p.n_ps)) * p.G + h;
        };
        /* the first chunks' outputs are on their way while the weights are formed */
        constexpr int PRE = 4;
        const int q = tid / GL, d = (tid - q * GL) * 4;
        f4 pre[PRE];
#pragma unroll
        for (int u = 0; u < PRE; u++) {
            const int k = q + u * NG;
            pre[u] = f4{0.f, 0.f, 0.f, 0.f};
            if (d < HD && k < n) pre[u] = *reinterpret_cast<const f4 *>((k < p.n_ps ? p.p_o : p.s_o) + row_of(k) * HD + d);
        }
        float2 ml = make_float2(-INFINITY, 0.0f);
        if (tid < n) ml = *reinterpret_cast<const float2 *>((tid < p.n_ps ? p.p_ml : p.s_ml) + row_of(tid) * 2);
        const float M = block_max(ml.x), mu = M == -INFINITY ? 0.0f : M;
        const float w = tid < n ? __builtin_amdgcn_exp2f(ml.x - mu) : 0.0f;
        if (tid < n) s_w[tid] = w;
        const float L = block_sum(tid < n ? w * ml.y : 0.0f);
        f4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = 0; u < PRE; u++)
            if (q + u * NG < n) acc += s_w[q + u * NG] * pre[u];
        if (d < HD)
            for (int k = q + PRE * NG; k < n; k += NG)
                acc += s_w[k] * *reinterpret_cast<const f4 *>((k < p.n_ps ? p.p_o : p.s_o) + row_of(k) * HD + d);
        *reinterpret_cast<f4 *>(s_red + tid * 4) = acc;
        __syncthreads();
        if (tid < D4) {
            f4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < NG; k++) sum += *reinterpret_cast<const f4 *>(s_red + (k * GL + tid) * 4);
            /* a value that is not finite reached its dimension: the whole row becomes NaN (its threads are one wave) */
            const float z = ((sum[0] - sum[0]) + (sum[1] - sum[1])) + ((sum[2] - sum[2]) + (sum[3] - sum[3]));
            *reinterpret_cast<f4 *>(p.out + ((long long)i * p.Hq + head) * HD + tid * 4) = sum / (__any(z != 0.0f) ? __builtin_nanf("") : L);
        }
        return;
    }
    const int a = blockIdx.x - n_out, pair = a % (p.n_seq * p.Hkv);
    const int i = pair / p.Hkv, g = pair - i * p.Hkv;
    const ShSeq sq = sh_seq(p, i);
    const int ns = sh_own_chunks(p, sq);
    constexpr int KU = MASS_KEYS / 256;
    const int lane = tid & 63;
    const float *ml0 = p.s_ml + ((((long long)i * p.Hkv + g) * p.n_ss) * p.G) * 2;
    for (long long k0 = (long long)(a / (p.n_seq * p.Hkv)) * MASS_KEYS; k0 <= sq.len; k0 += (long long)p.m_chunks * MASS_KEYS) {
        float acc[KU] = {};
        for (int h0 = 0; h0 < p.G; h0 += MASS_HEADS) {
            const int hn = min(MASS_HEADS, p.G - h0);
            __syncthreads(); /* the last heads' state has been read */
            for (int h = wave; h < hn; h += 4) {
                const float2 ml = lane < ns ? *reinterpret_cast<const float2 *>(ml0 + ((long long)lane * p.G + h0 + h) * 2)
                                            : make_float2(-INFINITY, 0.0f);
                float M = ml.x;
#pragma unroll
                for (int sh = 1; sh < 64; sh <<= 1) M = fmaxf(M, __shfl_xor(M, sh));
                const float mu = M == -INFINITY ? 0.0f : M;
                float Ls = lane < ns ? __builtin_amdgcn_exp2f(ml.x - mu) * ml.y : 0.0f;
#pragma unroll
                for (int sh = 1; sh < 64; sh <<= 1) Ls += __shfl_xor(Ls, sh);
                if (lane == 0) *reinterpret_cast<float2 *>(s_red + 2 * h) = make_float2(mu, 1.0f / Ls);
            }
            __syncthreads();
#pragma unroll 4
            for (int h = 0; h < hn; h++) {
                const long long row = (long long)i * p.Hq + g * p.G + h0 + h;
                const float2 ml = *reinterpret_cast<const float2 *>(s_red + 2 * h);
#pragma unroll
                for (int u = 0; u < KU; u++) {
                    const long long key = k0 + u * 256 + tid;
                    const float x = key < sq.len ? p.logits[row * p.l_stride + key] : key == sq.len ? p.logit_new[row] : 0.0f;
                    acc[u] = fmaf(__builtin_amdgcn_exp2f(x - ml.x), ml.y, acc[u]);
                }
            }
        }
        float *mass = p.mass + ((long long)sq.slot * p.Hkv + g) * p.m_stride;
#pragma unroll
        for (int u = 0; u < KU; u++) {
            const long long key = k0 + u * 256 + tid;
            if (key < sq.len) {
                mass[key] = p.decay == 0.0f ? acc[u] : fmaf(mass[key], p.decay, acc[u]);
            } else if (key == sq.len) {
                mass[key] = acc[u];
                p.row_pos[((long long)sq.slot * p.Hkv + g) * p.m_stride + key] = sq.pos;
            }
        }
    }
}

template <int HD>
static int launch_hd(const ShParams *p, int tile_rows, hipStream_t st, hipEvent_t e0, hipEvent_t e1) {
    const unsigned blocks = (unsigned)p->n_pblocks + (unsigned)(p->n_own ? p->n_own : p->n_ss * p->n_seq) * p->Hkv * p->s_rb;
    if (p->mass) hipExtLaunchKernelGGL((k_sh<HD, SH_SCORED>), dim3(blocks), dim3(SH_TPB), 0, st, e0, nullptr, 0, *p);
    else if (tile_rows == 16) hipExtLaunchKernelGGL((k_sh<HD, SH_NARROW>), dim3(blocks), dim3(SH_TPB), 0, st, e0, nullptr, 0, *p);
    else if constexpr (ShGeom<HD>::WIDE) hipExtLaunchKernelGGL((k_sh<HD, SH_WIDE>), dim3(blocks), dim3(SH_TPB), 0, st, e0, nullptr, 0, *p);
    else return -1;
    if (hipGetLastError() != hipSuccess) return -3;
    unsigned mb = (unsigned)p->n_seq * p->Hq;
    if (p->mass) mb += (unsigned)p->n_seq * p->Hkv * p->m_chunks;
    hipExtLaunchKernelGGL((k_sh_merge<HD>), dim3(mb), dim3(256), 0, st, nullptr, e1, 0, *p);
    return hipGetLastError() == hipSuccess ? 0 : -3;
}

/* rows of a prefix item at head_dim hd, for a batch of `rows` rows a kv head: 64 for a wide item. Wide items read K and
 * V once for 64 rows where narrow ones do for 16 (64 sequences on 16384, head_dim 128, 128 rows a kv head: 71 us a call,
 * 93 with narrow ones; 32 rows on 4096: 20 either way). Not at 256, where a wave's state leaves one workgroup a compute
 * unit and its steps do not overlap (192 rows on 8191: 38 us, 31 narrow). 72, 80 and 96 have narrow items alone: the ring's
 * layout wants rows of 8 or 16 pieces, and slabs that the waves' 1 KB transfers share out evenly (192 rows of 4 kv heads on
 * 4096, a call: 20.8, 21.5 and 24.8 us narrow; 15.3 and 20.6 wide at 64 and 128). */
extern "C" int smol_shared_tile_rows(int hd, int rows) { return rows <= 32 || (hd != 64 && hd != 128) ? 16 : 16 * SH_NW; }

/* heads of an own-rows item */
extern "C" int smol_shared_own_rows(void) { return OWN_ROWS; }

/* workgroups for the weights of one (sequence, kv head), of `pairs`: one for every MASS_KEYS rows of the longest, but no
 * more than 4096 in all or one each, for most are empty where one sequence is long (1000 empty ones cost 1.1 us) */
extern "C" int smol_shared_mass_chunks(long long pairs, int max_len) {
    return (int)std::min<long long>(max_len / MASS_KEYS + 1, std::max(1LL, 4096 / pairs));
}

/* workgroups of a compute unit at once (k_sh's launch bounds) */
extern "C" int smol_shared_occupancy(int hd) { return hd <= 128 ? 2 : 1; }

extern "C" int smol_launch_shared(const ShParams *p, int hd, int tile_rows, hipStream_t st, hipEvent_t e0, hipEvent_t e1) {
    switch (hd) {
    case 64: return launch_hd<64>(p, tile_rows, st, e0, e1);
    case 72: return launch_hd<72>(p, tile_rows, st, e0, e1);
    case 80: return launch_hd<80>(p, tile_rows, st, e0, e1);
    case 96: return launch_hd<96>(p, tile_rows, st, e0, e1);
    case 128: return launch_hd<128>(p, tile_rows, st, e0, e1);
    case 256: return launch_hd<256>(p, tile_rows, st, e0, e1);
    default: return -1;
    }
}
