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
 * and one scan over the threads' counts gives every run its start. A few moves
 * (EV_FUSED) are made by the same workgroup; more go to k_evict_move, which has
 * a workgroup for every EV_MOVES of them. K rows move in 16-byte pieces, V^T
 * columns by element with neighbouring rows in neighbouring lanes, since the
 * rows of one slab share the 64 bytes of a column.
 *
 * What bounds it: the ranks are latency (loads, about a dozen barriers); the
 * moves are memory traffic in pieces of 64 bytes. A moved row's V touches one
 * such piece per column, so rows far apart cost 32 times their bytes: 8192 rows
 * cut to 1024 read 1.8 MB of V^T a head for 0.2 MB of moved values.
 * Measured on an MI355X (head_dim 128, 8 kv heads): 16 sequences, 4160 rows cut
 * to 4096, 26 us in k_evict_select, 12 of them for the ranks; 32 sequences,
 * 8192 cut to 1024, 18 us and 156 us in k_evict_move for 703 MB of traffic
 * (4.5 TB/s; a large copy reaches 4.7).
 */
#include "attn_device.h"

namespace {

constexpr int EV_BINS = 2048;
constexpr int EV_MOVES = 32;  /* moves of a k_evict_move workgroup */
constexpr int EV_TPB = 1024;  /* threads of k_evict_select (256: 11.5 us for 300 rows cut to 256, 1024: 10) */
/* Moves that k_evict_select makes itself, which saves a launch (2.4 us) and a start-up: head_dim 128, 16 sequences of 8 kv heads,
 * 32 moves 19.3 us against 28.7 in two kernels, 128 moves 38.6 against 43.2, 256 moves 56.2 against 55.2; one sequence, 128 moves
 * 21.3 against 20.6, 256 moves 30.2 against 22.2. */
constexpr int EV_FUSED = 128;

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

/* inclusive sums over the lanes of a wave */
__device__ __forceinline__ int ev_wave_sum(int v) {
#pragma unroll
    for (int sh = 1; sh < 64; sh <<= 1) {
        const int x = __shfl_up(v, sh);
        if ((threadIdx.x & 63) >= sh) v += x;
    }
    return v;
}

/* exclusive prefix sums of (a, b) over the TPB threads, through s_part [2][TPB / 64] of this scan's own */
template <int TPB>
__device__ __forceinline__ void ev_scan2(int &a, int &b, int *s_part) {
    constexpr int NW = TPB / 64;
    const int wave = threadIdx.x >> 6, ia = ev_wave_sum(a), ib = ev_wave_sum(b);
    if ((threadIdx.x & 63) == 63) {
        s_part[wave] = ia;
        s_part[NW + wave] = ib;
    }
    __syncthreads();
    int oa = 0, ob = 0;
#pragma unroll
    for (int w = 0; w < NW; w++)
        if (w < wave) {
            oa += s_part[w];
            ob += s_part[NW + w];
        }
    a = oa + ia - a;
    b = ob + ib - b;
}

/* V^T elements and K pieces of n moves (dst, src: shared memory) by TPB threads, and their mass and position, MB moves at
 * a time. All loads of a round go out before its first store (source and target could be the same row for all the
 * compiler knows). */
template <int TPB, int MB>
__device__ __forceinline__ void ev_move(const EvictParams &p, const ShSeq &sq, int g, const int *dst, const int *src, int n) {
    const int tid = threadIdx.x, hd = p.hd;
    const long long at = ((long long)sq.slot * p.Hkv + g) * p.m_stride;
    const long long base = (long long)sq.slot * p.c_slot_stride + (long long)g * p.cap * hd;
    uint16_t *kc = p.kc + base, *vt = p.vtc + base;
    constexpr int DS = TPB / MB, U = 128 / DS, KU = 2;
    const int pieces = hd / 8;
    for (int m0 = 0; m0 < n; m0 += MB) {
        const int mn = min(MB, n - m0), m = m0 + tid % MB;
        const bool mine = m < n;
        uint4 kx[KU];
#pragma unroll
        for (int u = 0; u < KU; u++) {
            const int e = tid + u * TPB;
            if (e < mn * pieces) kx[u] = *reinterpret_cast<const uint4 *>(kc + (long long)src[m0 + e / pieces] * hd + e % pieces * 8);
        }
        float mass = 0.0f;
        int pos = 0;
        if (tid < mn) {
            mass = p.mass[at + src[m0 + tid]];
            pos = p.row_pos[at + src[m0 + tid]];
        }
        const int sm = mine ? src[m] : 0, dm = mine ? dst[m] : 0;
        const long long so = (long long)(sm / SMOL_SLAB) * SMOL_SLAB * hd + sm % SMOL_SLAB;
        const long long to = (long long)(dm / SMOL_SLAB) * SMOL_SLAB * hd + dm % SMOL_SLAB;
        for (int d0 = tid / MB; d0 < hd; d0 += U * DS) {
            uint16_t x[U];
#pragma unroll
            for (int u = 0; u < U; u++) x[u] = mine && d0 + u * DS < hd ? vt[so + (d0 + u * DS) * SMOL_SLAB] : (uint16_t)0;
#pragma unroll
            for (int u = 0; u < U; u++)
                if (mine && d0 + u * DS < hd) vt[to + (d0 + u * DS) * SMOL_SLAB] = x[u];
        }
#pragma unroll
        for (int u = 0; u < KU; u++) {
            const int e = tid + u * TPB;
            if (e < mn * pieces) *reinterpret_cast<uint4 *>(kc + (long long)dst[m0 + e / pieces] * hd + e % pieces * 8) = kx[u];
        }
        for (int e = tid + KU * TPB; e < mn * pieces; e += TPB) /* head_dim 256 in few threads */
            *reinterpret_cast<uint4 *>(kc + (long long)dst[m0 + e / pieces] * hd + e % pieces * 8) =
                *reinterpret_cast<const uint4 *>(kc + (long long)src[m0 + e / pieces] * hd + e % pieces * 8);
        if (tid < mn) {
            p.mass_out[at + dst[m0 + tid]] = mass;
            p.pos_out[at + dst[m0 + tid]] = pos;
        }
    }
}

} // namespace

/* ROWS: the longest sequence whose ranks stay in LDS; 0: any, its ranks formed again at each reading */
template <int ROWS>
__global__ __launch_bounds__(EV_TPB) void k_evict_select(const EvictParams p) {
    constexpr int TPB = EV_TPB;
    constexpr bool LDS = ROWS > 0;
    constexpr int NW = TPB / 64, NB = EV_BINS / TPB, U = 8;
    __shared__ unsigned s_rank[LDS ? ROWS : 1];
    __shared__ int s_hist[3][EV_BINS], s_part[5][2 * NW], s_found[3][2];
    const int tid = threadIdx.x, pair = blockIdx.x, i = pair / p.Hkv, g = pair - i * p.Hkv;
    const int lane = tid & 63, wave = tid >> 6;
    const ShSeq sq = ev_seq(p, i);
    const int n = sq.len, keep = p.keep, left = min(n, keep);
    const long long at = ((long long)sq.slot * p.Hkv + g) * p.m_stride;
    const float *mass = p.mass + at;
    const int *pos = p.row_pos + at;
    float *mo = p.mass_out + at;
    int *po = p.pos_out + at;
    const bool apart = p.mass_out != p.mass;
    if (n <= keep) {
        if (tid == 0 && !p.fused) p.n_moves[pair] = 0;
        if (apart)
            for (int r = tid; r < n; r += TPB) {
                mo[r] = mass[r];
                po[r] = pos[r];
            }
        return;
    }
    const int from = sq.pos - p.recent; /* sq.pos: one past the newest position */
    auto rank_at = [&](int r) { return LDS ? s_rank[r] : ev_rank(mass[r], pos[r], p.first, from); };
    for (int b = tid; b < 3 * EV_BINS; b += TPB) s_hist[0][b] = 0;
    __syncthreads();

    /* adds one to the bin of every live lane; a wave whose rows share a bin adds them at once */
    auto count = [&](int *hist, unsigned bin, bool live) __attribute__((always_inline)) {
        const unsigned long long who = __ballot(live);
        if (!who) return;
        const int lead = __ffsll(who) - 1;
        const unsigned b0 = __shfl(bin, lead);
        if (__ballot(live && bin == b0) == who) {
            if (lane == lead) atomicAdd(&hist[b0], __popcll(who));
        } else if (live) {
            atomicAdd(&hist[bin], 1);
        }
    };
    /* the ranks and their first digits, U rows a thread in flight; the rows that stay in place are written where the
     * arrays are apart (the holes are written again, later) */
    for (int r0 = tid; r0 - tid < n; r0 += U * TPB) {
        float m[U];
        int q[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int r = min(r0 + u * TPB, n - 1);
            m[u] = mass[r];
            q[u] = pos[r];
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int r = r0 + u * TPB;
            if (r - tid >= n) break;
            const unsigned v = ev_rank(m[u], q[u], p.first, from);
            if (LDS && r < n) s_rank[r] = v;
            count(s_hist[0], v >> 21, r < n);
            if (apart && r < left) {
                mo[r] = m[u];
                po[r] = q[u];
            }
        }
    }
    __syncthreads();

    /* the keep-th largest rank, digit by digit */
    unsigned prefix = 0;
    int need = keep; /* rows still to take among those whose higher digits are `prefix` */
#pragma unroll
    for (int pass = 0; pass < 3; pass++) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
        if (pass > 0) {
            for (int r0 = 0; r0 < n; r0 += TPB) {
                const int r = r0 + tid;
                const unsigned v = r < n ? rank_at(r) : 0;
                count(s_hist[pass], (v >> shift) & ((1u << bits) - 1),
                      r < n && (v >> (shift + bits)) == (prefix >> (shift + bits)));
            }
            __syncthreads();
        }
        /* thread t holds NB bins, the highest first: the rows in the bins above them are the threads' before it */
        int cnt[NB], sum = 0;
#pragma unroll
        for (int b = 0; b < NB; b++) sum += cnt[b] = s_hist[pass][EV_BINS - 1 - NB * tid - b];
        const int incl = ev_wave_sum(sum);
        if (lane == 63) s_part[pass][wave] = incl;
        __syncthreads();
        int above = incl - sum;
#pragma unroll
        for (int w = 0; w < NW; w++)
            if (w < wave) above += s_part[pass][w];
#pragma unroll
        for (int b = 0; b < NB; b++) {
            if (above < need && above + cnt[b] >= need) {
                s_found[pass][0] = EV_BINS - 1 - NB * tid - b;
                s_found[pass][1] = need - above;
            }
            above += cnt[b];
        }
        __syncthreads();
        prefix |= (unsigned)s_found[pass][0] << shift;
        need = s_found[pass][1];
    }

    /* rows above the threshold stay, and the lowest `need` rows at it */
    const int per = ((n + TPB - 1) / TPB) | 1, b0 = min(n, tid * per), b1 = min(n, b0 + per);
    int eq = 0, z = 0;
    for (int r = b0; r < b1; r++) eq += rank_at(r) == prefix;
    ev_scan2<TPB>(eq, z, s_part[3]);
    auto walk = [&](auto f) __attribute__((always_inline)) {
        int e = eq;
        for (int r = b0; r < b1; r++) {
            const unsigned v = rank_at(r);
            const bool kept = v > prefix || (v == prefix && e < need);
            e += v == prefix;
            f(r, kept);
        }
    };
    int holes = 0, movers = 0;
    walk([&](int r, bool kept) {
        holes += r < keep && !kept;
        movers += r >= keep && kept;
    });
    ev_scan2<TPB>(holes, movers, s_part[4]);
    if (p.fused) {
        walk([&](int r, bool kept) {
            if (r < keep && !kept) s_hist[0][holes++] = r;
            if (r >= keep && kept) s_hist[1][movers++] = r;
        });
    } else {
        int *dst = p.moves + (long long)pair * 2 * p.max_moves, *src = dst + p.max_moves;
        walk([&](int r, bool kept) {
            if (r < keep && !kept) dst[holes++] = r;
            if (r >= keep && kept) src[movers++] = r;
        });
    }
    /* as many holes as movers; the last thread's counts are the totals */
    if (tid == TPB - 1) {
        if (p.fused) s_found[0][0] = holes;
        else p.n_moves[pair] = holes;
    }
    if (!p.fused) return;
    __syncthreads();
    ev_move<TPB, EV_MOVES>(p, sq, g, s_hist[0], s_hist[1], s_found[0][0]);
}

__global__ __launch_bounds__(256) void k_evict_move(const EvictParams p) {
    __shared__ int s_dst[EV_MOVES], s_src[EV_MOVES];
    const int pairs = p.n_seq * p.Hkv, pair = blockIdx.x % pairs, m0 = blockIdx.x / pairs * EV_MOVES;
    const int total = p.n_moves[pair];
    if (m0 >= total) return;
    const int tid = threadIdx.x, i = pair / p.Hkv, g = pair - i * p.Hkv, n = min(EV_MOVES, total - m0);
    if (tid < n) {
        const int *dst = p.moves + (long long)pair * 2 * p.max_moves + m0 + tid;
        s_dst[tid] = dst[0];
        s_src[tid] = dst[p.max_moves];
    }
    __syncthreads();
    ev_move<256, EV_MOVES>(p, ev_seq(p, i), g, s_dst, s_src, n);
}

extern "C" int smol_evict_fused(int max_moves) { return max_moves <= EV_FUSED; }

/* max_rows: rows of the longest sequence */
extern "C" int smol_launch_evict(const EvictParams *p, int max_rows, hipStream_t st, hipEvent_t e0, hipEvent_t e1) {
    const unsigned pairs = (unsigned)p->n_seq * p->Hkv;
    const hipEvent_t e = p->fused ? e1 : nullptr;
    const dim3 g(pairs), b(EV_TPB);
    if (max_rows <= 8192) hipExtLaunchKernelGGL(k_evict_select<8192>, g, b, 0, st, e0, e, 0, *p);
    else if (max_rows <= 32768) hipExtLaunchKernelGGL(k_evict_select<32768>, g, b, 0, st, e0, e, 0, *p);
    else hipExtLaunchKernelGGL(k_evict_select<0>, g, b, 0, st, e0, e, 0, *p);
    if (hipGetLastError() != hipSuccess) return -3;
    if (p->fused) return 0;
    const unsigned blocks = pairs * (unsigned)((p->max_moves + EV_MOVES - 1) / EV_MOVES);
    hipExtLaunchKernelGGL(k_evict_move, dim3(blocks), dim3(256), 0, st, nullptr, e1, 0, *p);
    return hipGetLastError() == hipSuccess ? 0 : -3;
}
