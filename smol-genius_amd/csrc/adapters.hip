/*
 * adapters.hip - a shared bf16 projection with a low-rank adapter of its own
 * for every row (smol_linear_adapters_dev): for row s with adapter a,
 *     y_s = W x_s + bias + scale_a B_a (A_a x_s),   A_a [rank][in], B_a [out][rank].
 *
 * The low-rank part works on tiles of 16 rows that share an adapter (the host
 * sorts the rows; the rows of a tile need not follow each other):
 *   k_adapt_in   t = A x, the in_dim cut into chunks so that few tiles still fill
 *                the device; each chunk writes its own partial t, so the sum's
 *                order is fixed.
 * A few rows with few ranks run in one launch, k_adapt_one, whose workgroups
 * each form t themselves.
 * Up to AD_FEW rows the rest is one launch, k_adapt_few: W streams once from
 * memory through the matrix cores against all rows (k_adapt_in's launch has
 * laid x out as bf16 parts for it), the waves' sums meet in LDS, and scale B t
 * and the bias join them there. More rows run the library's own product
 * (linear.hip) and then k_adapt_out, which adds scale B t to it.
 * All run on v_mfma_f32_16x16x32_bf16 with the weights as the A operand, so a
 * lane holds four consecutive ranks (outputs) of one row. An fp32 x and t are
 * split into three bf16 parts (24 bits), so these products are as exact as
 * fp32 products of the bf16 weights.
 *
 * The weights of a set are packed once, at its creation: ranks padded with
 * zeros to the matrix instruction's sizes, so no load needs a bound.
 *
 * Measured on an MI355X: 3 rows of 1024 -> 2048, rank 8: k_adapt_one 8.2 us; 32
 * rows of 1024 -> 4096, fp32, rank 16: 4.6 + 7.6 us (W's 8.4 MB; the bf16 parts
 * of x, read again by every workgroup from L2, are 50 MB); 3 rows of 4096 ->
 * 4096: 4.6 + 11 us (33.6 MB of W at 3.0 TB/s). 1536 rows of 1024 -> 2048,
 * bf16, rank 32: 4.9 us, the library's product 20.5, k_adapt_out 8.5 us (26 MB,
 * 3.1 TB/s).
 */
#include "attn_device.h"

#include <limits.h>
#include <stdio.h>
#include <string.h>

#include <algorithm>
#include <vector>

#include "../../include/smol_linear.h"

extern "C" int smol_internal_fail(int code, const char *msg);
extern "C" int smol_internal_ctx_device(smol_attn_ctx *ctx);
extern "C" int smol_internal_ctx_cus(smol_attn_ctx *ctx);
extern "C" void smol_internal_timing_events(smol_attn_ctx *ctx, int kind, hipEvent_t *a, hipEvent_t *b);
extern "C" int smol_internal_work(smol_attn_ctx *ctx, size_t bytes, void **p);
extern "C" int smol_internal_upload(smol_attn_ctx *ctx, const void *host, size_t bytes, const void **dev);

namespace {

constexpr int AD_MAX_RANK = 128;
constexpr int AD_TPB = 256, AD_NW = AD_TPB / 64;
constexpr int AD_ARG_TILES = 40, AD_ARG_RUNS = 400;
/* Rows that k_adapt_few takes. It keeps fp32 x at 24 bits and is two launches instead of three or four; against the library's
 * product and k_adapt_out (kernel time, fp32 x, rank 16): 1024 -> 4096 16 rows 10.6 us against 14.2, 32 rows 12.2 against 14.6,
 * 64 rows 15.5 against 16.2; 2048 -> 1024, where its workgroups are few, 64 rows 19.4 against 15.8, which the 24 bits cost
 * there. A bf16 x, a call of 64 rows here and one of 65 the other way: 1024 -> 1024 11.2 us and 15.2, 2048 -> 1024 12.7 and
 * 15.6, 1024 -> 4096 11.3 and 15.7, 1024 -> 6144 15.0 and 16.2. It re-reads x for every 16 outputs, so it only loses more
 * beyond. */
constexpr int AD_FEW = 64;
constexpr int AD_TIMING_KIND = 2;

struct AdTile {
    int adapter, n, rank; /* adapter -1: rows without one, whose product k_adapt_out truncates */
    float scale;
    int row[16]; /* rows past n repeat the first */
};
/* a tile of rows that follow each other (prompts one after the other): more of them fit the kernel arguments */
struct AdRun {
    int row0;
    short adapter, n;
};

struct AdParams {
    const void *x; int x_bf16; int vec;
    const uint16_t *w; int w_vec; const float *bias;
    uint16_t *xs;                    /* few rows: x as B fragments [16-row tile][32-wide step][part][lane][8], zeros past
                                      * in_dim and seq */
    int in_blocks;                   /* workgroups of k_adapt_in on tiles; those behind them lay x out */
    int in_dim, out_dim, seq;
    const uint16_t *a; int ra, kp;   /* [adapter][ra][kp] */
    const uint16_t *b; int np, rp;   /* [adapter][np][rp] */
    const float *scale; const int *rank; /* [adapter] */
    float *t; int n_tiles, n_chunks, chunk; /* [chunk][seq][ra]; chunk: 32-wide steps of in_dim */
    int n_out;                       /* tiles of k_adapt_out: behind the n_tiles those without an adapter */
    unsigned has[2];                 /* few rows: the rows that have an adapter */
    const float *base;               /* fp32 [seq][out] that the low-rank part is added to */
    void *y; int y_bf16;             /* fp32 y is base itself */
    const AdTile *tiles_dev;
    int runs_only;                   /* the tiles are runs[] */
    union {
        AdTile tiles[AD_ARG_TILES];
        AdRun runs[AD_ARG_RUNS];
    };
};

static_assert(sizeof(AdParams) <= 4096, "kernel arguments");

struct AdAt {
    int adapter, n, rank;
    float scale;
    int row; /* of this lane's column c */
};
__device__ __forceinline__ AdAt ad_at(const AdParams &p, int tile, int c) {
    if (p.runs_only) {
        const AdRun r = p.runs[tile];
        const int row = r.row0 + (c < r.n ? c : 0);
        return r.adapter < 0 ? AdAt{-1, r.n, 0, 0.0f, row} : AdAt{r.adapter, r.n, p.rank[r.adapter], p.scale[r.adapter], row};
    }
    const AdTile *t = (p.tiles_dev ? p.tiles_dev : p.tiles) + tile;
    return AdAt{t->adapter, t->n, t->rank, t->scale, t->row[c]};
}

/* x = p0 + p1 + p2 in bf16, each part what the parts before it leave, rounded to nearest: 24 bits. The first two are held to
 * bf16's largest finite value: a finite x beyond it would round to infinity, and inf - inf is no number. An infinite x so goes
 * into p2 whole, beside finite parts of its sign, and its products are infinities of the right sign. */
__device__ __forceinline__ void ad_split3(const float *x, b8 &p0, b8 &p1, b8 &p2) {
    constexpr float BF16_MAX = 3.3895313892515355e38f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const __bf16 a = (__bf16)__builtin_amdgcn_fmed3f(x[i], -BF16_MAX, BF16_MAX);
        const float r = x[i] - (float)a;
        const __bf16 b = (__bf16)__builtin_amdgcn_fmed3f(r, -BF16_MAX, BF16_MAX);
        p0[i] = a;
        p1[i] = b;
        p2[i] = (__bf16)(r - (float)b);
    }
}

/* elements [k0, k0 + 8) of row `row` of x as bf16 parts, zeros past in_dim; vec: in_dim is a multiple of 8 and x
 * aligned */
template <bool XBF>
__device__ __forceinline__ void ad_x8(const AdParams &p, long long row, int k0, b8 *xp) {
    if constexpr (XBF) {
        const uint16_t *x = (const uint16_t *)p.x + row * p.in_dim + k0;
        uint4 w = make_uint4(0, 0, 0, 0);
        if (p.vec) {
            if (k0 < p.in_dim) w = *reinterpret_cast<const uint4 *>(x);
        } else {
            uint32_t v[8];
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = k0 + i < p.in_dim ? x[i] : 0u;
            w = make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
        }
        xp[0] = as_b8(w);
    } else {
        const float *x = (const float *)p.x + row * p.in_dim + k0;
        float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (p.vec) {
            if (k0 < p.in_dim) {
                const float4 u = *reinterpret_cast<const float4 *>(x), w = *reinterpret_cast<const float4 *>(x + 4);
                v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w; v[4] = w.x; v[5] = w.y; v[6] = w.z; v[7] = w.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (k0 + i < p.in_dim) v[i] = x[i];
        }
        ad_split3(v, xp[0], xp[1], xp[2]);
    }
}

/* NT: rank tiles of 16 that the accumulators hold */
template <int NT, bool XBF>
__global__ __launch_bounds__(AD_TPB) void k_adapt_in(const AdParams p) {
    constexpr int PARTS = XBF ? 1 : 3;
    __shared__ __attribute__((aligned(16))) float s_t[AD_NW * 16 * NT * 16];
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, j = lane >> 4;
    if ((int)blockIdx.x >= p.in_blocks) {
        /* a wave a fragment: lane (c, j) holds row c's elements 8 j .. + 7 of the step */
        const int f = (blockIdx.x - p.in_blocks) * AD_NW + (tid >> 6), steps = p.kp / 32, t = f / steps, s = f - t * steps;
        const int row = 16 * t + c;
        if (t >= (p.seq + 15) / 16) return;
        b8 xp[PARTS];
        ad_x8<XBF>(p, min(row, p.seq - 1), row < p.seq ? 32 * s + 8 * j : p.kp, xp);
#pragma unroll
        for (int q = 0; q < PARTS; q++) *reinterpret_cast<b8 *>(p.xs + ((((long long)t * steps + s) * PARTS + q) * 64 + lane) * 8) = xp[q];
        return;
    }
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int tile = blockIdx.x % p.n_tiles, chunk = blockIdx.x / p.n_tiles;
    const AdAt tl = ad_at(p, tile, c);
    const int n = tl.n, nt = (tl.rank + 15) / 16;
    const long long row = tl.row;
    const uint16_t *a = p.a + ((long long)tl.adapter * p.ra + c) * p.kp + 8 * j;
    f4 acc[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) acc[t] = f4{0.f, 0.f, 0.f, 0.f};
    const int s1 = min((chunk + 1) * p.chunk, p.kp / 32);
    constexpr int US = NT <= 4 ? 4 : 2; /* steps in flight */
    for (int s0 = chunk * p.chunk + wave * US; s0 < s1; s0 += AD_NW * US) {
        b8 xp[US][PARTS], w[US][NT];
#pragma unroll
        for (int u = 0; u < US; u++) {
            const bool live = s0 + u < s1;
            const int k0 = live ? 32 * (s0 + u) : 0;
#pragma unroll
            for (int t = 0; t < NT; t++)
                if (t < nt) w[u][t] = as_b8(*reinterpret_cast<const uint4 *>(a + (long long)t * 16 * p.kp + k0));
            ad_x8<XBF>(p, row, live ? k0 + 8 * j : p.kp, xp[u]); /* past the chunk: zeros */
        }
#pragma unroll
        for (int u = 0; u < US; u++)
#pragma unroll
            for (int t = 0; t < NT; t++) {
                if (t >= nt) break;
#pragma unroll
                for (int q = PARTS - 1; q >= 0; q--) acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[u][t], xp[u][q], acc[t], 0, 0, 0);
            }
    }
    /* lane (c, j): ranks 16 t + 4 j .. + 3 of row c */
#pragma unroll
    for (int t = 0; t < NT; t++)
        *reinterpret_cast<f4 *>(s_t + ((wave * 16 + c) * NT + t) * 16 + 4 * j) = acc[t];
    __syncthreads();
    for (int e = tid; e < n * nt * 4; e += AD_TPB) {
        const int r = e / (nt * 4), q = e - r * nt * 4;
        f4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < AD_NW; w++) sum += *reinterpret_cast<f4 *>(s_t + ((w * 16 + r) * NT) * 16 + 4 * q);
        *reinterpret_cast<f4 *>(p.t + ((long long)chunk * p.seq + ad_at(p, tile, r).row) * p.ra + 4 * q) = sum;
    }
}

/* scale t of row `row`, ranks [8 j', 8 j' + 8) of each 32-wide step, as bf16 parts: the chunks' partial sums, four at a
 * time in flight. Ranks past the adapter's are zeros: an infinite x makes NaN of the padding's 0 x there */
template <int KS>
__device__ __forceinline__ void ad_t(const AdParams &p, long long row, int rank, float scale, bool live, int j, b8 (*tp)[3]) {
    const long long step = (long long)p.seq * p.ra;
#pragma unroll
    for (int ks = 0; ks < KS; ks++) {
        const int r = 32 * ks + 8 * j;
        float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        /* k_adapt_in writes whole tiles of 16 ranks */
        if (live && r < ((rank + 15) & ~15)) {
            const float *t = p.t + row * p.ra + r;
            for (int q = 0; q < p.n_chunks; q += 4) {
                f4 x[4], z[4];
#pragma unroll
                for (int u = 0; u < 4; u++)
                    if (q + u < p.n_chunks) {
                        x[u] = *reinterpret_cast<const f4 *>(t + (q + u) * step);
                        z[u] = *reinterpret_cast<const f4 *>(t + (q + u) * step + 4);
                    }
#pragma unroll
                for (int u = 0; u < 4; u++)
                    if (q + u < p.n_chunks) {
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            v[i] += x[u][i];
                            v[4 + i] += z[u][i];
                        }
                    }
            }
        }
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = r + i < rank ? v[i] * scale : 0.0f;
        ad_split3(v, tp[ks][0], tp[ks][1], tp[ks][2]);
    }
}

/* elements [8 j, 8 j + 8) of step s of W's row (w: its element 8 j), zeros past in_dim */
__device__ __forceinline__ uint4 ad_w8(const AdParams &p, const uint16_t *w, int s, int j) {
    const int k0 = 32 * s + 8 * j;
    if (p.w_vec) return k0 < p.in_dim ? *reinterpret_cast<const uint4 *>(w + 32 * s) : make_uint4(0, 0, 0, 0);
    uint32_t x[8];
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = k0 + i < p.in_dim ? w[32 * s + i] : 0u;
    return make_uint4(x[0] | x[1] << 16, x[2] | x[3] << 16, x[4] | x[5] << 16, x[6] | x[7] << 16);
}

/* Up to 16 RT rows against 16 outputs a workgroup. Its waves share in_dim out by runs of US 32-wide steps (whole cache lines of
 * W's rows), a run in flight; the sums of every wave are added in LDS in wave order, the adapters' tiles (one wave each) add their
 * part, and each output is written once. */
template <int RT, bool XBF>
struct Few {
    /* sixteen waves, eight where their sums fill more LDS than their loads gain (1024 -> 4096, fp32 x: 16 rows 6.3 us against 7.0
     * with eight, 32 rows 7.5 against 8.2, 64 rows 11.9 against 10.9; bf16 x: 64 rows 7.3 against 8.2) */
    static constexpr int NW = RT == 4 && !XBF ? 8 : 16;
    static constexpr int US = RT == 1 || (RT == 2 && XBF) ? 4 : 2;
};
template <int RT, bool XBF, int KS>
__global__ __launch_bounds__((64 * Few<RT, XBF>::NW)) void k_adapt_few(const AdParams p) {
    constexpr int FEW_NW = Few<RT, XBF>::NW, PARTS = XBF ? 1 : 3, US = Few<RT, XBF>::US, STR = 20;
    __shared__ __attribute__((aligned(16))) float s_y[(FEW_NW + 1) * RT * 16 * STR];
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, j = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int o0 = blockIdx.x * 16, steps = p.kp / 32;
    const uint16_t *w = p.w + (long long)min(o0 + c, p.out_dim - 1) * p.in_dim + 8 * j;
    f4 acc[RT];
#pragma unroll
    for (int t = 0; t < RT; t++) acc[t] = f4{0.f, 0.f, 0.f, 0.f};
    /* columns past the last row take the last row's x: results that no one reads, without reading their padding */
    int xo[RT];
#pragma unroll
    for (int t = 0; t < RT; t++) xo[t] = (16 * j + max(0, min(c, p.seq - 1 - 16 * t))) * 8;
    const int tiles_x = (p.seq + 15) / 16;
    for (int s0 = wave * US; s0 < steps; s0 += FEW_NW * US) {
        uint4 wv[US];
        b8 xf[US][RT][PARTS];
#pragma unroll
        for (int u = 0; u < US; u++) {
            const int s = s0 + u;
            wv[u] = s < steps ? ad_w8(p, w, s, j) : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int t = 0; t < RT; t++)
#pragma unroll
                for (int q = 0; q < PARTS; q++)
                    xf[u][t][q] = as_b8(s < steps && t < tiles_x
                                            ? *reinterpret_cast<const uint4 *>(
                                                  p.xs + (((long long)t * steps + s) * PARTS + q) * 512 + xo[t])
                                            : make_uint4(0, 0, 0, 0));
        }
#pragma unroll
        for (int u = 0; u < US; u++)
#pragma unroll
            for (int t = 0; t < RT; t++)
#pragma unroll
                for (int q = PARTS - 1; q >= 0; q--)
                    acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_b8(wv[u]), xf[u][t][q], acc[t], 0, 0, 0);
    }
#pragma unroll
    for (int t = 0; t < RT; t++) *reinterpret_cast<f4 *>(s_y + ((wave * RT + t) * 16 + c) * STR + 4 * j) = acc[t];
    /* the low-rank part, by row, behind the waves' sums (rows without an adapter are not read there) */
    float *s_low = s_y + FEW_NW * RT * 16 * STR;
    for (int tile = wave; tile < p.n_tiles; tile += FEW_NW) {
        const AdAt tl = ad_at(p, tile, c);
        const int row = tl.row;
        const bool live = c < tl.n;
        const uint16_t *b = p.b + ((long long)tl.adapter * p.np + o0 + c) * p.rp + 8 * j;
        b8 bw[KS], tp[KS][3];
#pragma unroll
        for (int ks = 0; ks < KS; ks++) bw[ks] = as_b8(*reinterpret_cast<const uint4 *>(b + 32 * ks));
        ad_t<KS>(p, row, tl.rank, tl.scale, live, j, tp);
        f4 low = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ks++)
#pragma unroll
            for (int q = 2; q >= 0; q--) low = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bw[ks], tp[ks][q], low, 0, 0, 0);
        if (live) *reinterpret_cast<f4 *>(s_low + row * STR + 4 * j) = low;
    }
    __syncthreads();
    for (int e = tid; e < p.seq * 16; e += 64 * FEW_NW) {
        const int r = e / 16, o = e % 16;
        if (o0 + o >= p.out_dim) continue;
        float v = 0.0f;
#pragma unroll
        for (int q = 0; q < FEW_NW; q++) v += s_y[(q * RT * 16 + r) * STR + o];
        if (p.bias) v += p.bias[o0 + o];
        if (p.has[r >> 5] >> (r & 31) & 1) v += s_low[r * STR + o];
        const long long at = (long long)r * p.out_dim + o0 + o;
        if (p.y_bf16) ((uint16_t *)p.y)[at] = (uint16_t)(__float_as_uint(v) >> 16);
        else ((float *)p.y)[at] = v;
    }
}

/* Up to 16 rows with up to ONE_SLOTS tiles of 16 ranks among their adapters, all in one launch: every workgroup (16 outputs)
 * forms A x of those tiles by itself, for all rows, beside its outputs of W x. Its waves share in_dim out; their sums meet in
 * LDS in wave order, t is split there for B. What a workgroup reads again of A and x bounds it, so only little of both
 * (ONE_WORK, in_dim times 4 for a slot and 1 for a row; kernel time here and in two launches, whatever out_dim up to 4096: one
 * row and slot of 1024 6.9 and 9.6 us, of 4096 13.9 and 13.9; three and three of 1024 8.2 and 9.7, of 2048 12.0 and 11.4; four
 * rows and slots of 1024 10.7 and 11.3, of 2048 15.9 and 14.1; 16 rows and four slots of 512 9.1 and 9.2, of 1024 12.4 and 10.1;
 * a second launch costs the host 2.4 us besides). */
constexpr int ONE_SLOTS = 4, ONE_NW = 16;
constexpr long long ONE_WORK = 20480;
template <bool XBF>
__global__ __launch_bounds__(64 * ONE_NW) void k_adapt_one(const AdParams p) {
    constexpr int PARTS = XBF ? 1 : 3, US = 2, STR = 20, NS = 1 + ONE_SLOTS, TSTR = ONE_SLOTS * 16 + 4;
    __shared__ __attribute__((aligned(16))) float s_y[ONE_NW * NS * 16 * STR], s_t[16 * TSTR], s_low[16 * STR];
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, j = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int o0 = blockIdx.x * 16, steps = p.kp / 32;
    const uint16_t *w = p.w + (long long)min(o0 + c, p.out_dim - 1) * p.in_dim + 8 * j;
    /* slot q: tile q's first ranks, and so on: the tiles' slots follow each other */
    const uint16_t *a[ONE_SLOTS];
    int n_slots = 0;
#pragma unroll
    for (int q = 0; q < ONE_SLOTS; q++) a[q] = p.a;
    for (int t = 0; t < p.n_tiles; t++)
        for (int r = 0; r < p.tiles[t].rank; r += 16, n_slots++)
#pragma unroll
            for (int q = 0; q < ONE_SLOTS; q++)
                if (q == n_slots) a[q] = p.a + ((long long)p.tiles[t].adapter * p.ra + r + c) * p.kp + 8 * j;
    const long long row = min(c, p.seq - 1); /* columns past the last row: results that no one reads */
    f4 acc[NS];
#pragma unroll
    for (int q = 0; q < NS; q++) acc[q] = f4{0.f, 0.f, 0.f, 0.f};
    for (int s0 = wave * US; s0 < steps; s0 += ONE_NW * US) {
        uint4 wv[US];
        b8 xp[US][PARTS], av[US][ONE_SLOTS];
#pragma unroll
        for (int u = 0; u < US; u++) {
            const bool live = s0 + u < steps;
            const int s = live ? s0 + u : 0;
            wv[u] = ad_w8(p, w, s, j);
#pragma unroll
            for (int q = 0; q < ONE_SLOTS; q++)
                if (q < n_slots) av[u][q] = as_b8(*reinterpret_cast<const uint4 *>(a[q] + 32 * s));
            ad_x8<XBF>(p, row, live ? 32 * s + 8 * j : p.kp, xp[u]); /* past the last step: zeros */
        }
#pragma unroll
        for (int u = 0; u < US; u++)
#pragma unroll
            for (int q = PARTS - 1; q >= 0; q--) {
                acc[0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_b8(wv[u]), xp[u][q], acc[0], 0, 0, 0);
#pragma unroll
                for (int t = 0; t < ONE_SLOTS; t++)
                    if (t < n_slots) acc[1 + t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(av[u][t], xp[u][q], acc[1 + t], 0, 0, 0);
            }
    }
#pragma unroll
    for (int q = 0; q < NS; q++)
        if (q <= n_slots) *reinterpret_cast<f4 *>(s_y + ((wave * NS + q) * 16 + c) * STR + 4 * j) = acc[q];
    __syncthreads();
    /* t of every row and slot: a thread a rank */
    for (int e = tid; e < n_slots * 256; e += 64 * ONE_NW) {
        const int q = e / 256, r = e / 16 % 16, k = e % 16;
        float v = 0.0f;
#pragma unroll
        for (int u = 0; u < ONE_NW; u++) v += s_y[((u * NS + 1 + q) * 16 + r) * STR + k];
        s_t[r * TSTR + q * 16 + k] = v;
    }
    __syncthreads();
    /* B t by tile, a wave each */
    for (int tile = wave; tile < p.n_tiles; tile += ONE_NW) {
        int slot = 0;
        for (int t = 0; t < tile; t++) slot += (p.tiles[t].rank + 15) / 16;
        const AdAt tl = ad_at(p, tile, c);
        const uint16_t *b = p.b + ((long long)tl.adapter * p.np + o0 + c) * p.rp + 8 * j;
        f4 low = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < ONE_SLOTS / 2; ks++) {
            if (32 * ks >= tl.rank) break;
            const int r = 32 * ks + 8 * j;
            float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
            if (r < ((tl.rank + 15) & ~15)) {
                const f4 x = *reinterpret_cast<const f4 *>(s_t + tl.row * TSTR + slot * 16 + r);
                const f4 y = *reinterpret_cast<const f4 *>(s_t + tl.row * TSTR + slot * 16 + r + 4);
#pragma unroll
                for (int i = 0; i < 4; i++) { /* ranks past the adapter's: as in ad_t */
                    v[i] = r + i < tl.rank ? x[i] * tl.scale : 0.0f;
                    v[4 + i] = r + 4 + i < tl.rank ? y[i] * tl.scale : 0.0f;
                }
            }
            b8 tp[3];
            ad_split3(v, tp[0], tp[1], tp[2]);
            const b8 bw = as_b8(*reinterpret_cast<const uint4 *>(b + 32 * ks));
#pragma unroll
            for (int q = 2; q >= 0; q--) low = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bw, tp[q], low, 0, 0, 0);
        }
        if (c < tl.n) *reinterpret_cast<f4 *>(s_low + tl.row * STR + 4 * j) = low;
    }
    __syncthreads();
    for (int e = tid; e < p.seq * 16; e += 64 * ONE_NW) {
        const int r = e / 16, o = e % 16;
        if (o0 + o >= p.out_dim) continue;
        float v = 0.0f;
#pragma unroll
        for (int q = 0; q < ONE_NW; q++) v += s_y[(q * NS * 16 + r) * STR + o];
        if (p.bias) v += p.bias[o0 + o];
        if (p.has[0] >> r & 1) v += s_low[r * STR + o];
        const long long at = (long long)r * p.out_dim + o0 + o;
        if (p.y_bf16) ((uint16_t *)p.y)[at] = (uint16_t)(__float_as_uint(v) >> 16);
        else ((float *)p.y)[at] = v;
    }
}

constexpr int AD_OUT = 64; /* outputs of a k_adapt_out wave */

/* y = base + scale B t for a tile's rows and 256 outputs. The products leave the matrix cores with a row's outputs spread
 * over lanes 16 apart; they pass through LDS so that base and y move as whole lines (16 rows of 1 KB). Bound by base and y.
 * KS: 32-wide steps over the rank */
template <int KS>
__global__ __launch_bounds__(AD_TPB) void k_adapt_out(const AdParams p) {
    constexpr int W = AD_OUT * AD_NW, STR = W + 4, U = AD_OUT / 16, NB = 16 * W / 4 / AD_TPB;
    __shared__ __attribute__((aligned(16))) float s_d[16 * STR];
    __shared__ int s_row[16];
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, j = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int tile = blockIdx.x % p.n_out, w0 = blockIdx.x / p.n_out * W, o0 = w0 + wave * AD_OUT;
    const AdAt tl = ad_at(p, tile, c);
    const long long row = tl.row;
    if (tid < 16) s_row[tid] = tl.row;
    const bool live = c < tl.n, mine = o0 < p.out_dim; /* B has whole tiles of AD_OUT rows and 32 ranks */
    if (tl.adapter < 0) {
        /* what adds nothing to any value, its sign included */
        for (int e = tid; e < 16 * STR; e += AD_TPB) s_d[e] = -0.0f;
    } else {
        b8 w[U][KS], tp[KS][3];
        const uint16_t *b = p.b + ((long long)tl.adapter * p.np + (mine ? o0 : 0) + c) * p.rp + 8 * j;
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int ks = 0; ks < KS; ks++) w[u][ks] = as_b8(*reinterpret_cast<const uint4 *>(b + (long long)16 * u * p.rp + 32 * ks));
        ad_t<KS>(p, row, tl.rank, tl.scale, live, j, tp);
#pragma unroll
        for (int u = 0; u < U; u++) {
            f4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
#pragma unroll
                for (int q = 2; q >= 0; q--) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[u][ks], tp[ks][q], acc, 0, 0, 0);
            *reinterpret_cast<f4 *>(s_d + c * STR + wave * AD_OUT + 16 * u + 4 * j) = acc;
        }
    }
    __syncthreads();
    /* a wave a row at a time, a lane four outputs */
    const bool quads = (p.out_dim & 3) == 0;
    f4 base[NB];
#pragma unroll
    for (int u = 0; u < NB; u++) {
        const int e = tid + u * AD_TPB, r = e / (W / 4), o = w0 + e % (W / 4) * 4;
        if (r >= tl.n) continue;
        const long long at = (long long)s_row[r] * p.out_dim + o;
        if (quads) {
            if (o < p.out_dim) base[u] = *reinterpret_cast<const f4 *>(p.base + at);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (o + i < p.out_dim) base[u][i] = p.base[at + i];
        }
    }
#pragma unroll
    for (int u = 0; u < NB; u++) {
        const int e = tid + u * AD_TPB, r = e / (W / 4), o = w0 + e % (W / 4) * 4;
        if (r >= tl.n) continue;
        const long long at = (long long)s_row[r] * p.out_dim + o;
        const f4 v = base[u] + *reinterpret_cast<const f4 *>(s_d + r * STR + o - w0);
        if (quads && o < p.out_dim) {
            if (p.y_bf16)
                *reinterpret_cast<uint2 *>((uint16_t *)p.y + at) =
                    make_uint2(__float_as_uint(v[0]) >> 16 | (__float_as_uint(v[1]) & 0xFFFF0000u),
                               __float_as_uint(v[2]) >> 16 | (__float_as_uint(v[3]) & 0xFFFF0000u));
            else
                *reinterpret_cast<f4 *>((float *)p.y + at) = v;
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (o + i < p.out_dim) {
                    if (p.y_bf16) ((uint16_t *)p.y)[at + i] = (uint16_t)(__float_as_uint(v[i]) >> 16);
                    else ((float *)p.y)[at + i] = v[i];
                }
        }
    }
}

/* dst [rows][stride] = src [rows][cols], zeros behind; rows past src_rows are zeros */
template <typename T>
__global__ __launch_bounds__(256) void k_adapt_pack(T *dst, const T *src, int rows, int stride, int src_rows,
                                                    int cols) {
    for (int r = blockIdx.x; r < rows; r += gridDim.x) {
        const T *s = src + (long long)r * cols;
        for (int q = threadIdx.x; q < stride; q += 256) dst[(long long)r * stride + q] = r < src_rows && q < cols ? s[q] : (T)0;
    }
}

int afail(int code, const char *msg) { return smol_internal_fail(code, msg); }

#define AHIP(expr)                                                                          \
    do {                                                                                    \
        hipError_t e_ = (expr);                                                             \
        if (e_ != hipSuccess) return afail(SMOL_ATTN_ERR_DEVICE, hipGetErrorString(e_));    \
    } while (0)

} // namespace

struct smol_adapters {
    smol_attn_ctx *ctx;
    int device;
    hipStream_t stream;
    int n, in_dim, out_dim, max_rank, ra, rp, kp, np;
    void *mem = nullptr;
    uint16_t *a, *b;
    float *scale;
    int *rank;
    std::vector<float> h_scale;
    std::vector<int> h_rank;
};

extern "C" int smol_adapters_destroy(smol_adapters *s) {
    if (!s) return SMOL_ATTN_OK;
    (void)hipSetDevice(s->device);
    (void)hipStreamSynchronize(s->stream);
    if (s->mem) (void)hipFree(s->mem);
    delete s;
    return SMOL_ATTN_OK;
}

extern "C" int smol_adapters_create(smol_attn_ctx *ctx, int n, int in_dim, int out_dim, const uint16_t *const *a,
                                    const uint16_t *const *b, const int *rank, const float *scale, smol_adapters **out) {
    if (!ctx || !out) return afail(SMOL_ATTN_ERR_ARG, "smol_adapters_create: null context or result");
    *out = nullptr;
    if (n <= 0 || in_dim <= 0 || out_dim <= 0 || !a || !b || !rank || !scale)
        return afail(SMOL_ATTN_ERR_ARG, "smol_adapters_create: sizes or null arrays");
    /* what no call of one row could take; the padded sizes stay below 31 bits */
    if (in_dim > INT_MAX / 4 || out_dim > INT_MAX / 4 || (long long)out_dim * in_dim > (1LL << 40))
        return afail(SMOL_ATTN_ERR_UNSUPPORTED, "smol_adapters_create: sizes beyond the supported range");
    int max_rank = 0;
    for (int i = 0; i < n; i++) {
        if (rank[i] < 1 || rank[i] > AD_MAX_RANK) return afail(SMOL_ATTN_ERR_UNSUPPORTED, "smol_adapters_create: a rank outside 1 .. 128");
        if (!a[i] || !b[i]) return afail(SMOL_ATTN_ERR_ARG, "smol_adapters_create: null weights");
        max_rank = std::max(max_rank, rank[i]);
    }
    AHIP(hipSetDevice(smol_internal_ctx_device(ctx)));
    smol_adapters *s = new smol_adapters();
    s->ctx = ctx;
    s->device = smol_internal_ctx_device(ctx);
    s->stream = static_cast<hipStream_t>(smol_attn_ctx_stream(ctx));
    s->n = n;
    s->in_dim = in_dim;
    s->out_dim = out_dim;
    s->max_rank = max_rank;
    s->h_scale.assign(scale, scale + n);
    s->h_rank.assign(rank, rank + n);
    s->ra = (max_rank + 15) & ~15;
    s->rp = (max_rank + 31) & ~31;
    s->kp = (int)(((long long)in_dim + 31) & ~31LL);
    s->np = (int)(((long long)out_dim + AD_OUT - 1) / AD_OUT * AD_OUT);
    const size_t ab = ((size_t)n * s->ra * s->kp * 2 + 255) & ~(size_t)255, bb = ((size_t)n * s->np * s->rp * 2 + 255) & ~(size_t)255;
    const size_t sb = ((size_t)n * 4 + 255) & ~(size_t)255;
    hipError_t e = hipMalloc(&s->mem, ab + bb + 2 * sb);
    if (e != hipSuccess) {
        delete s;
        (void)hipGetLastError();
        return afail(e == hipErrorOutOfMemory ? SMOL_ATTN_ERR_NOMEM : SMOL_ATTN_ERR_DEVICE, "smol_adapters_create: device memory");
    }
    s->a = static_cast<uint16_t *>(s->mem);
    s->b = reinterpret_cast<uint16_t *>(static_cast<char *>(s->mem) + ab);
    s->scale = reinterpret_cast<float *>(static_cast<char *>(s->mem) + ab + bb);
    s->rank = reinterpret_cast<int *>(static_cast<char *>(s->mem) + ab + bb + sb);
    for (int i = 0; i < n && e == hipSuccess; i++) {
        auto pack = [&](uint16_t *dst, const uint16_t *src, int rows, int stride, int src_rows, int cols) {
            hipLaunchKernelGGL(k_adapt_pack<uint16_t>, dim3((unsigned)std::min(rows, 4096)), dim3(256), 0, s->stream, dst, src, rows, stride, src_rows, cols);
        };
        pack(s->a + (size_t)i * s->ra * s->kp, a[i], s->ra, s->kp, rank[i], in_dim);
        pack(s->b + (size_t)i * s->np * s->rp, b[i], s->np, s->rp, out_dim, rank[i]);
        e = hipGetLastError();
    }
    /* pageable host memory: the copies return when they have been made */
    if (e == hipSuccess) e = hipMemcpyAsync(s->scale, scale, (size_t)n * 4, hipMemcpyHostToDevice, s->stream);
    if (e == hipSuccess) e = hipMemcpyAsync(s->rank, rank, (size_t)n * 4, hipMemcpyHostToDevice, s->stream);
    if (e == hipSuccess) e = hipStreamSynchronize(s->stream);
    if (e != hipSuccess) {
        smol_adapters_destroy(s);
        return afail(SMOL_ATTN_ERR_DEVICE, hipGetErrorString(e));
    }
    *out = s;
    return SMOL_ATTN_OK;
}

template <int RT, bool XBF>
static void launch_few(const AdParams &p, int ks, hipStream_t st) {
    const dim3 g((unsigned)((p.out_dim + 15) / 16)), b(64 * Few<RT, XBF>::NW);
    switch (ks) {
    case 1: hipLaunchKernelGGL((k_adapt_few<RT, XBF, 1>), g, b, 0, st, p); break;
    case 2: hipLaunchKernelGGL((k_adapt_few<RT, XBF, 2>), g, b, 0, st, p); break;
    default: hipLaunchKernelGGL((k_adapt_few<RT, XBF, 4>), g, b, 0, st, p); break;
    }
}

template <int NT>
static void launch_in(const AdParams &p, unsigned blocks, hipStream_t st) {
    if (p.x_bf16) hipLaunchKernelGGL((k_adapt_in<NT, true>), dim3(blocks), dim3(AD_TPB), 0, st, p);
    else hipLaunchKernelGGL((k_adapt_in<NT, false>), dim3(blocks), dim3(AD_TPB), 0, st, p);
}

extern "C" int smol_linear_adapters_dev(smol_attn_ctx *ctx, void *y, int y_dtype, const void *x, int x_dtype, const uint16_t *w,
                                        const float *bias, int seq, int in_dim, int out_dim, const smol_adapters *set,
                                        const int *ids) {
    if (!ctx) return afail(SMOL_ATTN_ERR_ARG, "smol_linear_adapters_dev: null context");
    if ((x_dtype != SMOL_ATTN_F32 && x_dtype != SMOL_ATTN_BF16) || (y_dtype != SMOL_ATTN_F32 && y_dtype != SMOL_ATTN_BF16))
        return afail(SMOL_ATTN_ERR_ARG, "smol_linear_adapters_dev: dtype");
    if (!set || (!ids && seq != 0)) return afail(SMOL_ATTN_ERR_ARG, "smol_linear_adapters_dev: null adapters or ids");
    if (set->ctx != ctx) return afail(SMOL_ATTN_ERR_ARG, "smol_linear_adapters_dev: adapters of another context");
    if (seq < 0 || in_dim != set->in_dim || out_dim != set->out_dim)
        return afail(SMOL_ATTN_ERR_ARG, "smol_linear_adapters_dev: sizes differ from the adapters'");
    if (seq == 0) return SMOL_ATTN_OK;
    if (!y || !x || !w) return afail(SMOL_ATTN_ERR_ARG, "smol_linear_adapters_dev: null pointer");
    const int xs = x_dtype == SMOL_ATTN_BF16 ? 2 : 4, ys = y_dtype == SMOL_ATTN_BF16 ? 2 : 4;
    if (((uintptr_t)x & (xs - 1)) || ((uintptr_t)y & 15)) return afail(SMOL_ATTN_ERR_ARG, "smol_linear_adapters_dev: alignment");
    if ((long long)seq * in_dim > INT_MAX / 4 || (long long)seq * out_dim > INT_MAX / 4)
        return afail(SMOL_ATTN_ERR_UNSUPPORTED, "smol_linear_adapters_dev: sizes beyond the supported range");
    if ((const char *)x < (const char *)y + (size_t)seq * out_dim * ys && (const char *)y < (const char *)x + (size_t)seq * in_dim * xs)
        return afail(SMOL_ATTN_ERR_ARG, "smol_linear_adapters_dev: y overlaps x");
    if ((const char *)w < (const char *)y + (size_t)seq * out_dim * ys && (const char *)y < (const char *)w + (size_t)out_dim * in_dim * 2)
        return afail(SMOL_ATTN_ERR_ARG, "smol_linear_adapters_dev: y overlaps W");
    /* the rows by adapter, tiles of at most 16 */
    std::vector<int> count(set->n + 1, 0);
    int bare = 0;
    for (int s = 0; s < seq; s++) {
        if (ids[s] < -1 || ids[s] >= set->n) return afail(SMOL_ATTN_ERR_ARG, "smol_linear_adapters_dev: an id outside the set");
        if (ids[s] < 0) bare++;
        else count[ids[s]]++;
    }
    if (bare == seq) return smol_linear_dev(ctx, y, y_dtype, x, x_dtype, w, bias, seq, in_dim, out_dim);
    /* rows without one are k_adapt_out's too where y is not the product itself */
    const bool casts = bare && y_dtype == SMOL_ATTN_BF16 && seq > AD_FEW;
    std::vector<int> first(set->n + 1, 0);
    int n_tiles = 0;
    for (int i = 0; i < set->n; i++) {
        first[i] = n_tiles;
        n_tiles += (count[i] + 15) / 16;
        count[i] = 0;
    }
    const int n_out = n_tiles + (casts ? (bare + 15) / 16 : 0);
    first[set->n] = n_tiles;
    std::vector<AdTile> tiles(n_out);
    bool runs_only = set->n <= SHRT_MAX;
    for (int s = 0; s < seq; s++) {
        if (ids[s] < 0 && !casts) continue;
        const int id = ids[s] < 0 ? set->n : ids[s];
        AdTile &t = tiles[first[id] + count[id] / 16];
        const int k = count[id]++ % 16;
        if (k == 0) {
            t.adapter = ids[s];
            t.rank = ids[s] < 0 ? 0 : set->h_rank[id];
            t.scale = ids[s] < 0 ? 0.0f : set->h_scale[id];
            for (int i = 0; i < 16; i++) t.row[i] = s;
        }
        runs_only &= s == t.row[0] + k;
        t.row[k] = s;
        t.n = k + 1;
    }

    AHIP(hipSetDevice(smol_internal_ctx_device(ctx)));
    hipStream_t st = static_cast<hipStream_t>(smol_attn_ctx_stream(ctx));
    AdParams p;
    memset(&p, 0, offsetof(AdParams, tiles));
    p.x = x;
    p.x_bf16 = x_dtype == SMOL_ATTN_BF16;
    p.vec = in_dim % 8 == 0 && ((uintptr_t)x & 15) == 0;
    p.in_dim = in_dim;
    p.out_dim = out_dim;
    p.seq = seq;
    p.a = set->a; p.ra = set->ra; p.kp = set->kp;
    p.b = set->b; p.np = set->np; p.rp = set->rp;
    p.scale = set->scale;
    p.rank = set->rank;
    p.n_tiles = n_tiles;
    p.n_out = n_out;
    /* A step a wave at least. Few tiles: workgroups for a quarter of the compute units, since every chunk is another partial
     * sum for each of the readers (64 rows of 2048 and 1024: a quarter, half, all of them 19.4, 20.2, 22.6 and 15.5, 16.4,
     * 16.4 us in both kernels). Many tiles (more rows than k_adapt_few takes) have few readers a row: all compute units
     * (1536 rows: k_adapt_in 4.8 us, a quarter of them 6.1). */
    const int steps = set->kp / 32, cus = smol_internal_ctx_cus(ctx);
    const int chunks = std::max(1, std::min({n_tiles > 32 ? cus / n_tiles : cus / 4 / n_tiles, (steps + AD_NW - 1) / AD_NW, 16}));
    p.chunk = (steps + chunks - 1) / chunks;
    p.n_chunks = (steps + p.chunk - 1) / p.chunk;
    const bool ybf = y_dtype == SMOL_ATTN_BF16, few = seq <= AD_FEW;
    int slots = 0;
    for (const AdTile &t : tiles) slots += (t.rank + 15) / 16;
    const bool one = seq <= 16 && slots <= ONE_SLOTS && (4LL * slots + seq) * in_dim <= ONE_WORK;
    /* more rows than k_adapt_few takes, and operands that the library's product cannot stage (16-byte pieces): x and W
     * are copied with padded rows first */
    const bool pad = !few && (in_dim % 8 != 0 || ((uintptr_t)x & 15) || ((uintptr_t)w & 15));
    const int kp = set->kp, parts = p.x_bf16 ? 1 : 3;
    auto up = [](size_t n) { return (n + 255) & ~(size_t)255; };
    const size_t tb = up((size_t)p.n_chunks * seq * set->ra * 4), yb = up(!few && ybf ? (size_t)seq * out_dim * 4 : 0);
    const size_t xb = up(few ? (size_t)parts * ((seq + 15) & ~15) * kp * 2 : pad ? (size_t)seq * kp * xs : 0);
    void *work;
    if (int rc = smol_internal_work(ctx, tb + yb + xb + (pad ? (size_t)out_dim * kp * 2 : 0), &work)) return rc;
    p.t = static_cast<float *>(work);
    float *base = yb ? reinterpret_cast<float *>(static_cast<char *>(work) + tb) : static_cast<float *>(y);
    void *x_own = static_cast<char *>(work) + tb + yb;
    uint16_t *w_own = reinterpret_cast<uint16_t *>(static_cast<char *>(work) + tb + yb + xb);
    p.w = w;
    p.w_vec = in_dim % 8 == 0 && ((uintptr_t)w & 15) == 0;
    p.bias = bias;
    p.xs = static_cast<uint16_t *>(x_own);
    if (few)
        for (int s = 0; s < seq; s++)
            if (ids[s] >= 0) p.has[s >> 5] |= 1u << (s & 31);
    p.base = base;
    p.y = y;
    p.y_bf16 = ybf;
    if (n_out > AD_ARG_TILES && n_out <= AD_ARG_RUNS && runs_only) {
        p.runs_only = 1;
        for (int i = 0; i < n_out; i++) p.runs[i] = {tiles[i].row[0], (short)tiles[i].adapter, (short)tiles[i].n};
    } else if (n_out <= AD_ARG_TILES) {
        memcpy(p.tiles, tiles.data(), n_out * sizeof(AdTile));
    } else {
        const void *dev;
        if (int rc = smol_internal_upload(ctx, tiles.data(), n_out * sizeof(AdTile), &dev)) return rc;
        p.tiles_dev = static_cast<const AdTile *>(dev);
    }
    hipEvent_t e0 = nullptr, e1 = nullptr;
    if (few) {
        smol_internal_timing_events(ctx, AD_TIMING_KIND, &e0, &e1);
        if (e0) AHIP(hipEventRecord(e0, st));
    } else {
        const void *bx = x;
        const uint16_t *bw = w;
        int bk = in_dim;
        if (pad) {
            const unsigned xg = (unsigned)std::min(seq, 4096), wg = (unsigned)std::min(out_dim, 4096);
            if (p.x_bf16) hipLaunchKernelGGL(k_adapt_pack<uint16_t>, dim3(xg), dim3(256), 0, st, static_cast<uint16_t *>(x_own), (const uint16_t *)x, seq, kp, seq, in_dim);
            else hipLaunchKernelGGL(k_adapt_pack<uint32_t>, dim3(xg), dim3(256), 0, st, static_cast<uint32_t *>(x_own), (const uint32_t *)x, seq, kp, seq, in_dim);
            hipLaunchKernelGGL(k_adapt_pack<uint16_t>, dim3(wg), dim3(256), 0, st, w_own, w, out_dim, kp, out_dim, in_dim);
            AHIP(hipGetLastError());
            bx = x_own;
            bw = w_own;
            bk = kp;
        }
        if (int rc = smol_linear_dev(ctx, base, SMOL_ATTN_F32, bx, x_dtype, bw, bias, seq, bk, out_dim)) return rc;
        smol_internal_timing_events(ctx, AD_TIMING_KIND, &e0, &e1);
        if (e0) AHIP(hipEventRecord(e0, st));
    }
    if (one) {
        const dim3 g((unsigned)((out_dim + 15) / 16)), b(64 * ONE_NW);
        if (p.x_bf16) hipLaunchKernelGGL(k_adapt_one<true>, g, b, 0, st, p);
        else hipLaunchKernelGGL(k_adapt_one<false>, g, b, 0, st, p);
        AHIP(hipGetLastError());
        if (e1) AHIP(hipEventRecord(e1, st));
        return SMOL_ATTN_OK;
    }
    p.in_blocks = n_tiles * p.n_chunks;
    const unsigned in_blocks = (unsigned)p.in_blocks + (few ? ((unsigned)((seq + 15) / 16) * (kp / 32) + AD_NW - 1) / AD_NW : 0);
    const int nt = set->ra / 16;
    if (nt <= 1) launch_in<1>(p, in_blocks, st);
    else if (nt <= 2) launch_in<2>(p, in_blocks, st);
    else if (nt <= 4) launch_in<4>(p, in_blocks, st);
    else launch_in<8>(p, in_blocks, st);
    AHIP(hipGetLastError());
    if (few) {
        const int ks = set->rp / 32;
        if (p.x_bf16) {
            if (seq <= 16) launch_few<1, true>(p, ks, st);
            else if (seq <= 32) launch_few<2, true>(p, ks, st);
            else launch_few<4, true>(p, ks, st);
        } else {
            if (seq <= 16) launch_few<1, false>(p, ks, st);
            else if (seq <= 32) launch_few<2, false>(p, ks, st);
            else launch_few<4, false>(p, ks, st);
        }
        AHIP(hipGetLastError());
        if (e1) AHIP(hipEventRecord(e1, st));
        return SMOL_ATTN_OK;
    }
    const unsigned out_blocks = (unsigned)n_out * ((out_dim + AD_OUT * AD_NW - 1) / (AD_OUT * AD_NW));
    switch (set->rp / 32) {
    case 1: hipLaunchKernelGGL(k_adapt_out<1>, dim3(out_blocks), dim3(AD_TPB), 0, st, p); break;
    case 2: hipLaunchKernelGGL(k_adapt_out<2>, dim3(out_blocks), dim3(AD_TPB), 0, st, p); break;
    default: hipLaunchKernelGGL(k_adapt_out<4>, dim3(out_blocks), dim3(AD_TPB), 0, st, p); break;
    }
    AHIP(hipGetLastError());
    if (e1) AHIP(hipEventRecord(e1, st));
    return SMOL_ATTN_OK;
}
