/*
 * attn_evict.hip - takes the rows that received little attention out of a KV
 * cache (smol_kv_cache_evict).
 *
 * Of the n rows of a (slot, kv head), `keep` stay: by the order (protected,
 * mass, lower row). Attention does not depend on the order of its keys (their
 * positions are rotated into K), so a kept row below `keep` stays where it
 * is and the kept rows at or above `keep` fill the holes, both in ascending
 * order: at most min(keep, n - keep) rows move, where closing the gaps would
 * move almost all of them.
 *
 * k_evict_select, one workgroup a (sequence, kv head): a row's rank becomes a
 * 32-bit whole number of the same order, and the keep-th largest is found by
 * its digits (11, 11 and 10 bits) from histograms in LDS. Ties and the two
 * lists need counts in row order: each thread takes a run of consecutive rows
 * (an odd number of them, so the threads' LDS reads fall in different banks)
 * and one scan over the threads' counts gives every run its start.
 * k_evict_move then moves K rows in 16-byte pieces and V^T columns by element,
 * neighbouring rows in neighbouring lanes, since the rows of one slab share
 * the 64 bytes of a column.
 */
#include "attn_device.h"

namespace {

constexpr int EV_TPB = 1024;
constexpr int EV_BINS = 2048;
constexpr int EV_MOVES = 32;       /* moves of a k_evict_move workgroup */

__device__ __forceinline__ ShSeq ev_seq(const EvictParams &p, int i) {
    const int4 s = reinterpret_cast<const int4 *>(p.seqs_dev ? p.seqs_dev : p.seqs)[i];
    return ShSeq{s.x, s.y, s.z, s.w};
}

/* The row's rank: protected rows above all, then NaN, then the floats in their order (-0 as 0) */
__device__ __forceinline__ unsigned ev_rank(float m, int pos, int first, int from) {
    if (pos < first || pos >= from) return 0xFFFFFFFFu;
    if (!(m == m)) return 0xFFFFFFFEu;
    const unsigned u = m == 0.0f ? 0u : __float_as_uint(m);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

/* exclusive prefix sums over the workgroup's threads of (a, b); ta, tb: the totals */
__device__ __forceinline__ void ev_scan2(int &a, int &b, int &ta, int &tb, int *s_part) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int ia = a, ib = b;
#pragma unroll
    for (int sh = 1; sh < 64; sh <<= 1) {
        const int xa = __shfl_up(ia, sh), xb = __shfl_up(ib, sh);
        if (lane >= sh) {
            ia += xa;
            ib += xb;
        }
    }
    __syncthreads();
    if (lane == 63) {
        s_part[wave] = ia;
        s_part[16 + wave] = ib;
    }
    __syncthreads();
    int oa = 0, ob = 0;
    ta = tb = 0;
#pragma unroll
    for (int w = 0; w < EV_TPB / 64; w++) {
        if (w == wave) {
            oa = ta;
            ob = tb;
        }
        ta += s_part[w];
        tb += s_part[16 + w];
    }
    a = oa + ia - a;
    b = ob + ib - b;
}

} // namespace

/* ROWS: the longest sequence whose ranks stay in LDS; 0: any, its ranks formed again at each reading */
template <int ROWS>
__global__ __launch_bounds__(EV_TPB) void k_evict_select(const EvictParams p) {
    constexpr bool LDS = ROWS > 0;
    __shared__ unsigned s_rank[LDS ? ROWS : 1];
    __shared__ int s_hist[EV_BINS], s_part[32], s_found[3];
    const int tid = threadIdx.x, pair = blockIdx.x, i = pair / p.Hkv, g = pair - i * p.Hkv;
    const ShSeq sq = ev_seq(p, i);
    const int n = sq.len, keep = p.keep, left = min(n, keep);
    const long long at = ((long long)sq.slot * p.Hkv + g) * p.m_stride;
    const float *mass = p.mass + at;
    const int *pos = p.row_pos + at;
    float *mo = p.mass_out + at;
    int *po = p.pos_out + at;
    const bool apart = p.mass_out != p.mass;
    if (n <= keep) {
        if (tid == 0) p.n_moves[pair] = 0;
        if (apart)
            for (int r = tid; r < n; r += EV_TPB) {
                mo[r] = mass[r];
                po[r] = pos[r];
            }
        return;
    }
    const int from = sq.pos - p.recent; /* sq.pos: one past the newest position */
    auto rank_at = [&](int r) { return LDS ? s_rank[r] : ev_rank(mass[r], pos[r], p.first, from); };

    /* the keep-th largest rank, digit by digit */
    unsigned prefix = 0;
    int need = keep; /* rows still to take among those whose higher digits are `prefix` */
#pragma unroll
    for (int pass = 0; pass < 3; pass++) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
        for (int b = tid; b < EV_BINS; b += EV_TPB) s_hist[b] = 0;
        __syncthreads();
        for (int r0 = 0; r0 < n; r0 += EV_TPB) {
            const int r = r0 + tid;
            unsigned v = 0;
            bool live = r < n;
            if (live) {
                if (LDS && pass == 0) {
                    v = ev_rank(mass[r], pos[r], p.first, from);
                    s_rank[r] = v;
                } else {
                    v = rank_at(r);
                }
                live = pass == 0 || (v >> (shift + bits)) == (prefix >> (shift + bits));
            }
            /* a wave whose rows share a bin adds them at once */
            const unsigned bin = (v >> shift) & ((1u << bits) - 1);
            const unsigned long long who = __ballot(live);
            if (who) {
                const int lead = __ffsll(who) - 1;
                const unsigned b0 = __shfl(bin, lead);
                if (__ballot(live && bin == b0) == who) {
                    if ((tid & 63) == lead) atomicAdd(&s_hist[b0], __popcll(who));
                } else if (live) {
                    atomicAdd(&s_hist[bin], 1);
                }
            }
        }
        __syncthreads();
        /* thread t holds the bins 2 (1023 - t) + 1 and 2 (1023 - t): an exclusive scan counts the rows above them */
        const int hi = 2 * (EV_TPB - 1 - tid) + 1;
        const int ch = s_hist[hi], cl = s_hist[hi - 1];
        int above = ch + cl, z = 0, ta, tb;
        ev_scan2(above, z, ta, tb, s_part);
        if (above < need && above + ch + cl >= need) {
            const bool in_hi = above + ch >= need;
            s_found[0] = in_hi ? hi : hi - 1;
            s_found[1] = need - (in_hi ? above : above + ch);
        }
        __syncthreads();
        prefix |= (unsigned)s_found[0] << shift;
        need = s_found[1];
        __syncthreads();
    }

    /* rows above the threshold stay, and the lowest `need` rows at it */
    const int per = ((n + EV_TPB - 1) / EV_TPB) | 1, b0 = min(n, tid * per), b1 = min(n, b0 + per);
    int eq = 0, z = 0, te, tz;
    for (int r = b0; r < b1; r++) eq += rank_at(r) == prefix;
    ev_scan2(eq, z, te, tz, s_part);
    auto walk = [&](auto f) __attribute__((always_inline)) {
        int e = eq;
        for (int r = b0; r < b1; r++) {
            const unsigned v = rank_at(r);
            const bool kept = v > prefix || (v == prefix && e < need);
            e += v == prefix;
            f(r, kept);
        }
    };
    int holes = 0, movers = 0, th, tm;
    walk([&](int r, bool kept) {
        holes += r < keep && !kept;
        movers += r >= keep && kept;
    });
    ev_scan2(holes, movers, th, tm, s_part);
    int *dst = p.moves + (long long)pair * 2 * p.max_moves, *src = dst + p.max_moves;
    walk([&](int r, bool kept) {
        if (r < keep && !kept) dst[holes++] = r;
        if (r >= keep && kept) src[movers++] = r;
    });
    if (tid == 0) p.n_moves[pair] = th;
    /* the rows that stay in place; k_evict_move writes the holes (in a launch behind this one) */
    if (apart)
        for (int r = tid; r < left; r += EV_TPB) {
            mo[r] = mass[r];
            po[r] = pos[r];
        }
}

__global__ __launch_bounds__(256) void k_evict_move(const EvictParams p) {
    __shared__ int s_dst[EV_MOVES], s_src[EV_MOVES];
    const int pairs = p.n_seq * p.Hkv, pair = blockIdx.x % pairs, m0 = blockIdx.x / pairs * EV_MOVES;
    const int total = p.n_moves[pair];
    if (m0 >= total) return;
    const int tid = threadIdx.x, i = pair / p.Hkv, g = pair - i * p.Hkv, n = min(EV_MOVES, total - m0);
    const ShSeq sq = ev_seq(p, i);
    const int *dst = p.moves + (long long)pair * 2 * p.max_moves + m0, *src = dst + p.max_moves;
    const long long at = ((long long)sq.slot * p.Hkv + g) * p.m_stride;
    if (tid < n) {
        const int d = dst[tid], s = src[tid];
        s_dst[tid] = d;
        s_src[tid] = s;
        p.mass_out[at + d] = p.mass[at + s];
        p.pos_out[at + d] = p.row_pos[at + s];
    }
    __syncthreads();
    const int hd = p.hd, pieces = hd / 8;
    const long long base = (long long)sq.slot * p.c_slot_stride + (long long)g * p.cap * hd;
    uint16_t *kc = p.kc + base, *vt = p.vtc + base;
    for (int e = tid; e < n * pieces; e += 256) {
        const int m = e / pieces, d0 = (e - m * pieces) * 8;
        *reinterpret_cast<uint4 *>(kc + (long long)s_dst[m] * hd + d0) =
            *reinterpret_cast<const uint4 *>(kc + (long long)s_src[m] * hd + d0);
    }
    const int m = tid % EV_MOVES;
    if (m < n) {
        const long long so = (long long)(s_src[m] / SMOL_SLAB) * SMOL_SLAB * hd + s_src[m] % SMOL_SLAB;
        const long long to = (long long)(s_dst[m] / SMOL_SLAB) * SMOL_SLAB * hd + s_dst[m] % SMOL_SLAB;
        /* eight loads in flight before the first store (source and target could be the same row for all the compiler
         * knows) */
        constexpr int DS = 256 / EV_MOVES;
        for (int d0 = tid / EV_MOVES; d0 < hd; d0 += 8 * DS) {
            uint16_t x[8];
#pragma unroll
            for (int u = 0; u < 8; u++) x[u] = d0 + u * DS < hd ? vt[so + (d0 + u * DS) * SMOL_SLAB] : (uint16_t)0;
#pragma unroll
            for (int u = 0; u < 8; u++)
                if (d0 + u * DS < hd) vt[to + (d0 + u * DS) * SMOL_SLAB] = x[u];
        }
    }
}

/* max_rows: rows of the longest sequence */
extern "C" int smol_launch_evict(const EvictParams *p, int max_rows, hipStream_t st, hipEvent_t e0, hipEvent_t e1) {
    const unsigned pairs = (unsigned)p->n_seq * p->Hkv;
    if (max_rows <= 4096) hipExtLaunchKernelGGL((k_evict_select<4096>), dim3(pairs), dim3(EV_TPB), 0, st, e0, nullptr, 0, *p);
    else if (max_rows <= 32768) hipExtLaunchKernelGGL((k_evict_select<32768>), dim3(pairs), dim3(EV_TPB), 0, st, e0, nullptr, 0, *p);
    else hipExtLaunchKernelGGL((k_evict_select<0>), dim3(pairs), dim3(EV_TPB), 0, st, e0, nullptr, 0, *p);
    if (hipGetLastError() != hipSuccess) return -3;
    const unsigned blocks = pairs * (unsigned)((p->max_moves + EV_MOVES - 1) / EV_MOVES);
    if (blocks == 0) return 0;
    hipExtLaunchKernelGGL(k_evict_move, dim3(blocks), dim3(256), 0, st, nullptr, e1, 0, *p);
    return hipGetLastError() == hipSuccess ? 0 : -3;
}
