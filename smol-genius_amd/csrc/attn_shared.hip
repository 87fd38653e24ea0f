/*
 * attn_shared.hip - one decode step for a batch that shares a long prefix
 * (k_sh), and the step that also adds up the weight of every cached row
 * (k_sh with SC); the rows that received little are taken out by
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
 * Work split. A workgroup of four waves is one item: either (kv head, a tile
 * of 16 NT rows of the batch, a chunk of the prefix) or (sequence, kv head, a
 * chunk of its own rows). Its waves take 32-key slabs in turn, K and V^T
 * fragments straight from the cache into registers, as k_dec
 * (attn_decode.hip) does; their (m, l, O) join in LDS and go to the workspace,
 * and k_sh_merge joins an output row's chunks. Items need no table: the
 * chunks are equally long, so a workgroup finds its item from its number, and
 * only the sequences' (slot, length, position) travel with the call.
 *
 * Precision. K and V are the cache's bf16 bits. The fp32 side of each product
 * is split into bf16 parts that the matrix cores take exactly: Q into three
 * (24 bits, all of fp32), the probabilities into two (16 bits: at most 2^-16 of
 * each probability is lost, and their errors are independent).
 * The new token's key and value are used in fp32 by the step that appends
 * them and rounded to nearest bf16 in the cache. Softmax state, sums and the
 * join are fp32.
 */
#include "attn_device.h"

namespace {

template <int HD>
struct ShGeom {
    static constexpr int KS = (HD + 31) / 32; /* 32-wide d chunks of a K fragment */
    static constexpr int DT = (HD + 15) / 16; /* 16-wide d tiles of the output */
    static constexpr int HDP = KS * 32;
    static constexpr int QSTR = HDP + 4;      /* LDS row of a staged row */
    static constexpr int OSTR = DT * 16 + 4;  /* LDS row of a wave's output */
    static constexpr unsigned SLAB_BYTES = SMOL_SLAB * HD * 2;
};

constexpr int SH_NW = 4, SH_TPB = 64 * SH_NW;
constexpr int Q_PARTS = 3, P_PARTS = 3;

template <int HD, int NT>
struct ShLds {
    using Gm = ShGeom<HD>;
    static constexpr int TR = 16 * NT, CH8 = HD / 8;
    static constexpr int RAW = (TR + 1) * Gm::QSTR;               /* the rows times the norm's weights, the new key's behind */
    static constexpr int CB = SH_NW * 16 * Gm::OSTR + 2 * SH_NW * 16; /* a row tile's outputs of every wave, their m and l */
    static constexpr int UNI = RAW > CB ? RAW : CB;
    static constexpr int FRAG = Q_PARTS * Gm::KS * NT * 256;      /* Q fragments: 16 bytes a lane */
    static constexpr int SS = ((TR + 1) * CH8 + 3) & ~3;          /* a row's squares by chunk; then the new scores by chunk */
    static constexpr int FLOATS = UNI + FRAG + SS + 2 * Gm::HDP;  /* the new key and value last */
};

__device__ __forceinline__ void ld8f(const float *a, float *v) {
    const float4 x = *reinterpret_cast<const float4 *>(a), y = *reinterpret_cast<const float4 *>(a + 4);
    v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w; v[4] = y.x; v[5] = y.y; v[6] = y.z; v[7] = y.w;
}
__device__ __forceinline__ void st8f(float *a, const float *v) {
    *reinterpret_cast<float4 *>(a) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4 *>(a + 4) = make_float4(v[4], v[5], v[6], v[7]);
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
__device__ __forceinline__ bool any_not_finite(uint4 v) {
    const unsigned a[4] = {v.x, v.y, v.z, v.w};
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 4; i++) bad |= (a[i] & 0x7F80u) == 0x7F80u || (a[i] & 0x7F800000u) == 0x7F800000u;
    return bad;
}

__device__ __forceinline__ ShSeq sh_seq(const ShParams &p, int i) {
    const int4 s = reinterpret_cast<const int4 *>(p.seqs_dev ? p.seqs_dev : p.seqs)[i];
    return ShSeq{s.x, s.y, s.z, s.w};
}

/* the first of a sequence's own rows that its window leaves, down to a slab */
__device__ __forceinline__ int sh_own_first(const ShParams &p, const ShSeq &q) {
    return p.window > 0 ? max(0, q.pos - p.window + 1 - p.p_len) & ~(SMOL_SLAB - 1) : 0;
}
__device__ __forceinline__ int sh_own_chunks(const ShParams &p, const ShSeq &q) {
    return max(1, (q.len - sh_own_first(p, q) + p.s_chunk - 1) / p.s_chunk);
}

/* One item. NT row tiles of 16; rows r < R: sequence and head by `prefix`.
 * Keys [kb, ke) of the region at kbase / vbase (region_bytes each). */
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

template <int HD, int NT, bool SC>
__device__ __forceinline__ void sh_item(const ShParams &p, const ShItem &it, float *smem) {
    using Gm = ShGeom<HD>;
    using L = ShLds<HD, NT>;
    constexpr int KS = Gm::KS, DT = Gm::DT, HDP = Gm::HDP, QSTR = Gm::QSTR, OSTR = Gm::OSTR, TR = 16 * NT;
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, j = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int G = p.G, R = it.R;
    float *s_raw = smem;
    uint4 *s_frag = reinterpret_cast<uint4 *>(smem + L::UNI);
    float *s_ss = smem + L::UNI + L::FRAG, *s_knew = s_ss + L::SS, *s_vnew = s_knew + HDP;

    /* ---- the slab pipeline's loads ---- */
    struct KRaw { uint4 k[2][KS]; };
    struct VRaw { uint4 v[DT]; };
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
    /* a slab at or past ke has an empty range: its loads return zeros */
    auto issue_k = [&](int k0, KRaw &r) __attribute__((always_inline)) {
        const bool live = k0 < it.ke;
        const rsrc_t rs = make_rsrc(it.kc, live ? it.region_bytes : 0);
        const unsigned so = live ? (unsigned)(k0 / SMOL_SLAB) * Gm::SLAB_BYTES : 0u;
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
                r.k[t][ks] = HD % 32 == 0 ? bload(rs, vo_k[0][0], so + (unsigned)((4 * t * HD + 32 * ks) * 2))
                                          : bload(rs, vo_k[t][ks], so);
    };
    auto issue_v = [&](int k0, VRaw &r) __attribute__((always_inline)) {
        const bool live = k0 < it.ke;
        const rsrc_t rs = make_rsrc(it.vtc, live ? it.region_bytes : 0);
        const unsigned so = live ? (unsigned)(k0 / SMOL_SLAB) * Gm::SLAB_BYTES : 0u;
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
            r.v[dt] = HD % 16 == 0 ? bload(rs, vo_v[0], so + (unsigned)(16 * dt * SMOL_SLAB * 2)) : bload(rs, vo_v[dt], so);
    };
    int k0 = it.kb + wave * SMOL_SLAB;
    KRaw kr;
    VRaw vr;

    /* ---- stage the rows: normalised, rotated and split into fragments ----
     * Thread chunks of 8 elements; every load of a chunk (its row, the table
     * row, the weights) is issued before the first is used, and the first
     * slab's behind them. */
    constexpr int CH8 = HD / 8, HALF = HD / 2;
    constexpr int NQ = ((TR + 1) * CH8 + SH_TPB - 1) / SH_TPB;
    const int n_rows = R + (it.with_new ? 1 : 0); /* row R: the new key */
    auto row_seq = [&](int r) { return it.prefix ? (it.row0 + r) / G : it.seq; };
    auto row_head = [&](int r) { return it.g * G + (it.prefix ? (it.row0 + r) % G : it.row0 + r); };
    const bool rope = p.rope_kind != SMOL_ROPE_OFF;
    float x[NQ][8], cv[NQ][8], sn[NQ][8];
    ShSeq own;
    if (!it.prefix) own = sh_seq(p, it.seq);
#pragma unroll
    for (int u = 0; u < NQ; u++) {
        const int e = tid + SH_TPB * u, r = e / CH8, d0 = (e - r * CH8) * 8;
        if (e < n_rows * CH8) {
            const int sq = r < R ? row_seq(r) : it.seq;
            if (r < R) load8(p.q_in, p.in_dtype, (long long)sq * p.Hq * HD + (long long)row_head(r) * HD + d0, x[u]);
            else load8(p.k_in, p.in_dtype, ((long long)sq * p.Hkv + it.g) * HD + d0, x[u]);
            if (rope) {
                const long long at = (long long)(it.prefix ? sh_seq(p, sq).pos : own.pos) * HD + d0;
                ld8f(p.rope_cos + at, cv[u]);
                ld8f(p.rope_sin + at, sn[u]);
            }
        }
    }
    float vn[8];
    if (it.with_new && tid < CH8) load8(p.v_in, p.in_dtype, ((long long)it.seq * p.Hkv + it.g) * HD + tid * 8, vn);
    issue_k(k0, kr);
    issue_v(k0, vr);
    /* rows past R are zero columns */
    for (int e = tid; e < (TR - R) * 4 * KS * Q_PARTS; e += SH_TPB) {
        const int r = R + e % (TR - R), w = e / (TR - R), ks = w / 4 % KS, q = w / (4 * KS);
        s_frag[((q * KS + ks) * NT + (r >> 4)) * 64 + (w & 3) * 16 + (r & 15)] = make_uint4(0, 0, 0, 0);
    }
    if constexpr (HDP > HD) /* and so are columns past head_dim */
        for (int e = tid; e < R * (HDP - HD) / 8 * Q_PARTS; e += SH_TPB) {
            const int r = e % R, w = e / R, d0 = HD + w % ((HDP - HD) / 8) * 8, q = w / ((HDP - HD) / 8);
            s_frag[((q * KS + d0 / 32) * NT + (r >> 4)) * 64 + (d0 >> 3 & 3) * 16 + (r & 15)] = make_uint4(0, 0, 0, 0);
        }
#pragma unroll
    for (int u = 0; u < NQ; u++) {
        const int e = tid + SH_TPB * u, r = e / CH8, d0 = (e - r * CH8) * 8;
        if (e < n_rows * CH8) {
            const float *w = r < R ? p.q_norm : p.k_norm;
            if (w) {
                float ss = 0.0f, wv[8];
                ld8f(w + d0, wv);
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    ss = fmaf(x[u][i], x[u][i], ss);
                    x[u][i] *= wv[i];
                }
                s_ss[e] = ss;
            }
            st8f(s_raw + r * QSTR + d0, x[u]);
        }
    }
    if (it.with_new && tid < CH8) st8f(s_vnew + tid * 8, vn);
    __syncthreads();
#pragma unroll
    for (int u = 0; u < NQ; u++) {
        const int e = tid + SH_TPB * u, r = e / CH8, d0 = (e - r * CH8) * 8;
        if (e < n_rows * CH8) {
            const bool is_k = r >= R;
            float ri = is_k ? 1.0f : p.qscale;
            if (is_k ? p.k_norm != nullptr : p.q_norm != nullptr) {
                float ss = 0.0f;
#pragma unroll
                for (int i = 0; i < CH8; i++) ss += s_ss[r * CH8 + i];
                ri *= 1.0f / sqrtf(ss / (float)HD + p.norm_eps);
            }
            float y[8];
            if (!rope) {
#pragma unroll
                for (int i = 0; i < 8; i++) y[i] = x[u][i];
            } else if (p.rope_kind == SMOL_ROPE_INTERLEAVED_K) {
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    y[i] = fmaf(x[u][i], cv[u][i], -(x[u][i + 1] * sn[u][i]));
                    y[i + 1] = fmaf(x[u][i + 1], cv[u][i + 1], x[u][i] * sn[u][i + 1]);
                }
            } else {
                const float *row = s_raw + r * QSTR;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int d = d0 + i;
                    const float pr = row[d < HALF ? d + HALF : d - HALF];
                    y[i] = d < HALF ? fmaf(x[u][i], cv[u][i], -(pr * sn[u][i])) : fmaf(x[u][i], cv[u][i], pr * sn[u][i]);
                }
            }
#pragma unroll
            for (int i = 0; i < 8; i++) x[u][i] = y[i] * ri;
            if (is_k) {
                st8f(s_knew + d0, x[u]);
            } else {
                b8 f[Q_PARTS];
                split8x3(x[u], f[0], f[1], f[2]);
                const int ks = d0 / 32, at = ((d0 >> 3) & 3) * 16 + (r & 15);
#pragma unroll
                for (int q = 0; q < Q_PARTS; q++)
                    s_frag[((q * KS + ks) * NT + (r >> 4)) * 64 + at] = *reinterpret_cast<uint4 *>(&f[q]);
            }
        }
    }
    __syncthreads();
    if (it.with_new) {
        /* the new key's fp32 score by chunks: row_new() sums them */
#pragma unroll
        for (int u = 0; u < NQ; u++) {
            const int e = tid + SH_TPB * u, r = e / CH8, d0 = (e - r * CH8) * 8;
            if (r < R) {
                float kn[8], sd = 0.0f;
                ld8f(s_knew + d0, kn);
#pragma unroll
                for (int i = 0; i < 8; i++) sd = fmaf(x[u][i], kn[i], sd);
                s_ss[e] = sd;
            }
        }
    }
    auto row_new = [&](int r) __attribute__((always_inline)) {
        float sd = 0.0f;
#pragma unroll
        for (int i = 0; i < CH8; i++) sd += s_ss[r * CH8 + i];
        return p.cap2 > 0.0f ? p.cap2 * tanhf(sd / p.cap2) : sd;
    };

    /* ---- row ranges, state ---- */
    float m[NT], l[NT];
    f4 o[NT][DT];
    int lo[NT], lo_min = 1 << 30, lo_max = 0; /* window: the first key that a row sees */
#pragma unroll
    for (int t = 0; t < NT; t++) {
        m[t] = -INFINITY;
        l[t] = 0.0f;
        lo[t] = 0;
        if (p.window > 0) {
            const int r = t * 16 + c;
            if (r < R) lo[t] = max(0, sh_seq(p, row_seq(r)).pos - p.window + 1 - (it.prefix ? 0 : p.p_len));
            lo_max = max(lo_max, lo[t]);
            lo_min = min(lo_min, r < R ? lo[t] : 1 << 30);
        }
#pragma unroll
        for (int dt = 0; dt < DT; dt++) o[t][dt] = f4{0.f, 0.f, 0.f, 0.f};
    }
    if (p.window > 0) {
#pragma unroll
        for (int sh = 1; sh < 16; sh <<= 1) {
            lo_max = max(lo_max, __shfl_xor(lo_max, sh));
            lo_min = min(lo_min, __shfl_xor(lo_min, sh));
        }
        lo_max = __builtin_amdgcn_readfirstlane(lo_max);
        lo_min = __builtin_amdgcn_readfirstlane(lo_min);
    } else {
        lo_min = 0;
    }

    /* ---- the wave's slabs ---- */
    while (k0 < it.ke) {
        /* Q's fragments are read from LDS in every slab: kept in registers
         * they would take 48 NT of them at head_dim 128 (the fence keeps the
         * compiler from moving the reads in front of the loop) */
        asm volatile("" ::: "memory");
        f4 sacc[NT][2];
#pragma unroll
        for (int t = 0; t < NT; t++) {
            sacc[t][0] = sacc[t][1] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int q = Q_PARTS - 1; q >= 0; q--)
#pragma unroll
                for (int ks = 0; ks < KS; ks++) {
                    const b8 f = as_b8(s_frag[((q * KS + ks) * NT + t) * 64 + lane]);
#pragma unroll
                    for (int h = 0; h < 2; h++)
                        sacc[t][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_b8(kr.k[h][ks]), f, sacc[t][h], 0, 0, 0);
                }
        }
        const int k1 = k0 + SMOL_SLAB * SH_NW;
        issue_k(k1, kr);
        /* keys of the slab that some row does not see */
        const bool low = k0 < lo_max, tail = k0 + SMOL_SLAB > it.ke;
        bool apart = false; /* a value that is not finite in a slab whose rows see different keys */
        if (low || tail) {
#pragma unroll
            for (int dt = 0; dt < DT; dt++) vr.v[dt] = keep_keys8(vr.v[dt], k0 + 8 * j, lo_min, it.ke);
            if (low && lo_min < lo_max) {
                bool bad = false;
#pragma unroll
                for (int dt = 0; dt < DT; dt++) bad |= any_not_finite(vr.v[dt]);
                apart = __any(bad);
            }
        }
#pragma unroll
        for (int t = 0; t < NT; t++) {
            float sv[8];
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int i = 0; i < 4; i++) sv[4 * h + i] = sacc[t][h][i];
            if (p.cap2 > 0.0f) {
#pragma unroll
                for (int e = 0; e < 8; e++) sv[e] = p.cap2 * tanhf(sv[e] / p.cap2);
            }
            if constexpr (SC) {
                if (c < R) {
                    float *lg = p.logits + ((long long)it.seq * p.Hq + row_head(c)) * p.l_stride + k0 + 8 * j;
                    st8f(lg, sv);
                }
            }
            if (low || tail) {
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int key = k0 + 8 * j + e;
                    sv[e] = key >= lo[t] && key < it.ke ? sv[e] : -INFINITY;
                }
            }
            float mx = sv[0];
#pragma unroll
            for (int e = 1; e < 8; e++) mx = fmaxf(mx, sv[e]);
            mx = row_max4(mx);
            const bool need = mx > m[t] + LAZY_T;
            if (__any(need)) {
                const float m_new = need ? mx : m[t];
                const float alpha = need ? __builtin_amdgcn_exp2f(m[t] - m_new) : 1.0f;
#pragma unroll
                for (int dt = 0; dt < DT; dt++) o[t][dt] *= alpha;
                l[t] *= alpha;
                m[t] = m_new;
            }
            const float m_use = m[t] == -INFINITY ? 0.0f : m[t];
            float pv[8], ps = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                pv[e] = __builtin_amdgcn_exp2f(sv[e] - m_use);
                ps += pv[e];
            }
            l[t] += ps;
            b8 pp[P_PARTS];
            split8x3(pv, pp[0], pp[1], pp[2]);
            if (apart) {
                /* a row must not meet 0 x inf: one row at a time, against
                 * the values that it sees */
                for (int r = 0; r < 16; r++) {
                    const int lo_r = __builtin_amdgcn_readlane(lo[t], r);
#pragma unroll
                    for (int dt = 0; dt < DT; dt++) {
                        const b8 v = as_b8(keep_keys8(vr.v[dt], k0 + 8 * j, lo_r, it.ke));
                        f4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int q = P_PARTS - 1; q >= 0; q--) a = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, pp[q], a, 0, 0, 0);
                        if (c == r) o[t][dt] += a;
                    }
                }
            } else {
#pragma unroll
                for (int q = P_PARTS - 1; q >= 0; q--)
#pragma unroll
                    for (int dt = 0; dt < DT; dt++)
                        o[t][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_b8(vr.v[dt]), pp[q], o[t][dt], 0, 0, 0);
            }
        }
        issue_v(k1, vr);
        k0 = k1;
    }

    /* ---- the waves' states (and the new token's) join, one row tile at a time ---- */
    float *cb = smem, *cm = smem + SH_NW * 16 * OSTR, *cl = cm + SH_NW * 16;
    for (int t = 0; t < NT; t++) {
        __syncthreads();
#pragma unroll
        for (int tt = 0; tt < NT; tt++)
            if (tt == t) {
                const float lt = row_sum4(l[tt]);
                if (j == 0) {
                    cm[wave * 16 + c] = m[tt];
                    cl[wave * 16 + c] = lt;
                }
#pragma unroll
                for (int dt = 0; dt < DT; dt++)
                    *reinterpret_cast<f4 *>(cb + (wave * 16 + c) * OSTR + 16 * dt + 4 * j) = o[tt][dt];
            }
        __syncthreads();
        for (int e = tid; e < 16 * (HD / 4); e += SH_TPB) {
            const int r = e / (HD / 4), d = (e - r * (HD / 4)) * 4;
            if (t * 16 + r >= R) continue;
            const float s_new = it.with_new ? row_new(r) : -INFINITY;
            float mm = s_new;
#pragma unroll
            for (int w = 0; w < SH_NW; w++) mm = fmaxf(mm, cm[w * 16 + r]);
            const float mu = mm == -INFINITY ? 0.0f : mm;
            f4 acc = {0.f, 0.f, 0.f, 0.f};
            float ls = 0.0f;
            if (it.with_new) {
                ls = __builtin_amdgcn_exp2f(s_new - mu);
                acc = *reinterpret_cast<f4 *>(s_vnew + d) * ls;
            }
#pragma unroll
            for (int w = 0; w < SH_NW; w++) {
                const float f = __builtin_amdgcn_exp2f(cm[w * 16 + r] - mu);
                ls += f * cl[w * 16 + r];
                acc += f * *reinterpret_cast<f4 *>(cb + (w * 16 + r) * OSTR + d);
            }
            *reinterpret_cast<f4 *>(it.part_o + (long long)(t * 16 + r) * HD + d) = acc;
            if (d == 0) {
                *reinterpret_cast<float2 *>(it.part_ml + (t * 16 + r) * 2) = make_float2(mm, ls);
                if (SC && it.with_new) p.logit_new[(long long)it.seq * p.Hq + row_head(r)] = s_new;
            }
        }
    }
    if (it.with_new && it.row0 == 0) {
        const ShSeq sq = sh_seq(p, it.seq);
        for (int d0 = tid * 8; d0 < HD; d0 += SH_TPB * 8) {
            const long long base = (long long)sq.slot * p.c_slot_stride + (long long)it.g * p.cap * HD;
            float y[8];
            ld8f(s_knew + d0, y);
            *reinterpret_cast<uint4 *>(p.kc + base + (long long)sq.len * HD + d0) = pack_bf16x8(y);
            uint16_t *vt = p.vtc + base + (long long)(sq.len / SMOL_SLAB) * SMOL_SLAB * HD + sq.len % SMOL_SLAB;
#pragma unroll
            for (int i = 0; i < 8; i++) vt[(long long)(d0 + i) * SMOL_SLAB] = f32_to_bf16(s_vnew[d0 + i]);
        }
    }
}

} // namespace

template <int HD, int NT, bool SC>
__global__ __launch_bounds__(SH_TPB, HD <= 128 && NT <= 2 ? 2 : 1) void k_sh(const ShParams p) {
    __shared__ __attribute__((aligned(16))) float smem[ShLds<HD, NT>::FLOATS];
    const int b = blockIdx.x;
    ShItem it;
    if (NT > 1 || !SC) {
        if (b < p.n_pblocks) {
            /* workgroups b and b + 8 share an L2: the row blocks of one chunk follow each other there */
            const int rb = (b / 8) % p.n_rb, u = (b / (8 * p.n_rb)) * 8 + b % 8;
            const int g = u % p.Hkv, sp = u / p.Hkv;
            if (sp >= p.n_ps) return;
            it.prefix = true;
            it.g = g;
            it.row0 = rb * 16 * NT;
            it.R = min(16 * NT, p.n_seq * p.G - it.row0);
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
            sh_item<HD, NT, false>(p, it, smem);
            return;
        }
    }
    const int a = b - p.n_pblocks;
    const int srb = a % p.s_rb, g = (a / p.s_rb) % p.Hkv, i = (a / (p.s_rb * p.Hkv)) % p.n_seq;
    const int sp = a / (p.s_rb * p.Hkv * p.n_seq);
    const ShSeq sq = sh_seq(p, i);
    if (sp >= sh_own_chunks(p, sq)) return;
    it.prefix = false;
    it.g = g;
    it.row0 = srb * 16;
    it.R = min(16, p.G - it.row0);
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
    sh_item<HD, 1, SC>(p, it, smem);
}

/* Joins the chunks of the output rows, one workgroup a row (a sequence's
 * head): (m, l) of every chunk first, then the outputs, as many chunks at a
 * time as there are lanes for. With mass (k_sh's SC): the workgroups behind
 * those add the weights exp2(s - m) / l of MASS_KEYS cached rows of a
 * (sequence, kv head), from the scores that k_sh left, in the heads' order. */
constexpr int MASS_KEYS = 1024;

template <int HD>
__global__ __launch_bounds__(256) void k_sh_merge(const ShParams p) {
    constexpr int D4 = HD / 4, GL = HD <= 64 ? 16 : HD <= 128 ? 32 : 64, NG = 256 / GL;
    __shared__ __attribute__((aligned(16))) float s_w[2 * SH_MAX_SPLIT], s_red[NG * GL * 4], s_x[16];
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
        float2 ml = make_float2(-INFINITY, 0.0f);
        if (tid < n) ml = *reinterpret_cast<const float2 *>((tid < p.n_ps ? p.p_ml : p.s_ml) + row_of(tid) * 2);
        const float M = block_max(ml.x), mu = M == -INFINITY ? 0.0f : M;
        const float w = tid < n ? __builtin_amdgcn_exp2f(ml.x - mu) : 0.0f;
        if (tid < n) s_w[tid] = w;
        const float L = block_sum(tid < n ? w * ml.y : 0.0f);
        const int q = tid / GL, d = (tid - q * GL) * 4;
        f4 acc = {0.f, 0.f, 0.f, 0.f};
        if (d < HD)
            for (int k = q; k < n; k += NG)
                acc += s_w[k] * *reinterpret_cast<const f4 *>((k < p.n_ps ? p.p_o : p.s_o) + row_of(k) * HD + d);
        *reinterpret_cast<f4 *>(s_red + tid * 4) = acc;
        __syncthreads();
        if (tid < D4) {
            f4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < NG; k++) sum += *reinterpret_cast<const f4 *>(s_red + (k * GL + tid) * 4);
            *reinterpret_cast<f4 *>(p.out + ((long long)i * p.Hq + head) * HD + tid * 4) = sum / L;
        }
        return;
    }
    const int a = blockIdx.x - n_out, pair = a % (p.n_seq * p.Hkv), chunk = a / (p.n_seq * p.Hkv);
    const int i = pair / p.Hkv, g = pair - i * p.Hkv;
    const ShSeq sq = sh_seq(p, i);
    if (chunk * MASS_KEYS > sq.len) return;
    const int ns = sh_own_chunks(p, sq);
    float acc[MASS_KEYS / 256] = {};
    for (int h = 0; h < p.G; h++) {
        /* every wave finds (m, l) by itself: the same order, so the same bits in each */
        const float *ml = p.s_ml + ((((long long)i * p.Hkv + g) * p.n_ss) * p.G + h) * 2;
        const int lane = tid & 63;
        const float2 x = lane < ns ? *reinterpret_cast<const float2 *>(ml + (long long)lane * p.G * 2)
                                   : make_float2(-INFINITY, 0.0f);
        float M = x.x;
        for (int sh = 1; sh < 64; sh <<= 1) M = fmaxf(M, __shfl_xor(M, sh));
        const float mu = M == -INFINITY ? 0.0f : M;
        float Ls = lane < ns ? __builtin_amdgcn_exp2f(x.x - mu) * x.y : 0.0f;
        for (int sh = 1; sh < 64; sh <<= 1) Ls += __shfl_xor(Ls, sh);
        const long long row = (long long)i * p.Hq + g * p.G + h;
#pragma unroll
        for (int u = 0; u < MASS_KEYS / 256; u++) {
            const int key = chunk * MASS_KEYS + u * 256 + tid;
            if (key <= sq.len)
                acc[u] += __builtin_amdgcn_exp2f((key < sq.len ? p.logits[row * p.l_stride + key] : p.logit_new[row]) - mu) / Ls;
        }
    }
    float *mass = p.mass + ((long long)sq.slot * p.Hkv + g) * p.m_stride;
#pragma unroll
    for (int u = 0; u < MASS_KEYS / 256; u++) {
        const int key = chunk * MASS_KEYS + u * 256 + tid;
        if (key < sq.len) {
            mass[key] = p.decay == 0.0f ? acc[u] : fmaf(mass[key], p.decay, acc[u]);
        } else if (key == sq.len) {
            mass[key] = acc[u];
            p.row_pos[((long long)sq.slot * p.Hkv + g) * p.m_stride + key] = sq.pos;
        }
    }
}

template <int HD>
static int launch_hd(const ShParams *p, int nt, int max_len, hipStream_t st, hipEvent_t e0, hipEvent_t e1) {
    const unsigned blocks = (unsigned)p->n_pblocks + (unsigned)p->n_ss * p->n_seq * p->Hkv * p->s_rb;
    if (p->mass) hipExtLaunchKernelGGL((k_sh<HD, 1, true>), dim3(blocks), dim3(SH_TPB), 0, st, e0, nullptr, 0, *p);
    else if (nt == 1) hipExtLaunchKernelGGL((k_sh<HD, 1, false>), dim3(blocks), dim3(SH_TPB), 0, st, e0, nullptr, 0, *p);
    else if (nt == 4 && HD <= 128) {
        if constexpr (HD <= 128) hipExtLaunchKernelGGL((k_sh<HD, 4, false>), dim3(blocks), dim3(SH_TPB), 0, st, e0, nullptr, 0, *p);
    } else if (nt == 2 && HD == 256) {
        if constexpr (HD == 256) hipExtLaunchKernelGGL((k_sh<HD, 2, false>), dim3(blocks), dim3(SH_TPB), 0, st, e0, nullptr, 0, *p);
    }
    else if constexpr (HD <= 128) hipExtLaunchKernelGGL((k_sh<HD, 2, false>), dim3(blocks), dim3(SH_TPB), 0, st, e0, nullptr, 0, *p);
    else return -1;
    if (hipGetLastError() != hipSuccess) return -3;
    unsigned mb = (unsigned)p->n_seq * p->Hq;
    if (p->mass) mb += (unsigned)p->n_seq * p->Hkv * (max_len / MASS_KEYS + 1);
    hipExtLaunchKernelGGL((k_sh_merge<HD>), dim3(mb), dim3(256), 0, st, nullptr, e1, 0, *p);
    return hipGetLastError() == hipSuccess ? 0 : -3;
}

/* rows of a prefix item's tile at head_dim hd, for a batch of `rows` rows a kv head */
extern "C" int smol_shared_tile_rows(int hd, int rows) { return rows <= 16 || hd > 128 ? 16 : 32; }

/* workgroups of a compute unit at once (k_sh's launch bounds) */
extern "C" int smol_shared_occupancy(int hd) { return hd <= 128 ? 2 : 1; }

extern "C" int smol_launch_shared(const ShParams *p, int hd, int tile_rows, int max_len, hipStream_t st, hipEvent_t e0,
                                  hipEvent_t e1) {
    const int nt = tile_rows / 16;
    switch (hd) {
    case 64: return launch_hd<64>(p, nt, max_len, st, e0, e1);
    case 72: return launch_hd<72>(p, nt, max_len, st, e0, e1);
    case 80: return launch_hd<80>(p, nt, max_len, st, e0, e1);
    case 96: return launch_hd<96>(p, nt, max_len, st, e0, e1);
    case 128: return launch_hd<128>(p, nt, max_len, st, e0, e1);
    case 256: return launch_hd<256>(p, nt, max_len, st, e0, e1);
    default: return -1;
    }
}
