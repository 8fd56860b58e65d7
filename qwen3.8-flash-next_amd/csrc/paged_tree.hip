/*
 * paged_tree.hip -- decoding with drafted tokens on a paged cache: appending
 * rows with the position rotation applied on the way, what the rows of a tree
 * of drafted tokens see (their attention is paged_attn.hip's), the path that
 * the target's choices take through it, and keeping that path's rows.
 *
 * As in paged_pages.hip, lengths and tables stay on the device, and every
 * result is the same from call to call.
 */
#include "qk_device.h"
#include "gemv_parts.h"
#include "paged_parts.h"

/* ------------------------------------------------------------ rotation
 * A workgroup per new row (of four in long calls): cos and sin of its rot / 2
 * angles once, then its heads of q, k and v, 8 elements a lane.  A head of q or
 * k is normed first where a weight is given: y = x / sqrt(mean x^2 + eps) * w,
 * the sum in fp32 over the head's lanes.  Pairs (a, b) become (a cos - b sin, a
 * sin + b cos); in halves (i, i + rot / 2) a lane's partners lie with others
 * and come through LDS.  The heads' loads need no position and go out first;
 * the sequence is found by a wave, 64 starts at a time.
 * Bound: latency in short calls, 4.2 us for a row, 6.9 for 900 drafts of 64
 * sequences (14 MB; of a wave of 256 threads for every row 5.0 and 7.4, found
 * after the heads' loads by a search of one start at a time 5.8 and 9.6); HBM
 * in long ones, prompts of 266 MB read and written 52 us, 5.1 TB/s (a row a
 * workgroup 57), as much as a copy. */
struct PgRotary {
    pg_cache c;
    const void *q, *k, *v;
    void *out;
    int64_t q_token, q_head, k_token, k_head, v_token, v_head, o_token, o_head; /* elements */
    const float *freqs, *q_norm, *k_norm;
    const int32_t *starts, *slots, *status, *depths;
    float eps;
    int n, n_seqs, h, half, inter; /* half = rot / 2 */
    pg_div per_row;      /* heads of q, k and v of a token */
};
#define PG_ROTARY_MANY 2048 /* rows from which a workgroup has four: as many as the card holds workgroups */

/* cos and sin of position * freq, whose fp32 value is off by a radian at far
 * positions: x = position * freq in 64 bits (exact up to position 2^29: 29 and
 * 24 bits), x / 2 pi in two parts, so that no bit of it is lost with the whole
 * turns (up to 2^77 radians, where the second part's own rounding reaches a
 * tenth of a step of fp32), and the nearest quarter turn taken off.  What is
 * left, at most 1/8, is rounded to fp32, and sin and cos of 2 pi r are their
 * Taylor series (the first term left out is below 2e-9, the sums are off by
 * about one step of fp32). */
__device__ __forceinline__ float2 pg_turn(int pos, float freq) {
    const double x = (double)pos * (double)freq;
    const double t = x * 0x1.45f306dc9c883p-3, e = fma(x, 0x1.45f306dc9c883p-3, -t) + x * -0x1.6b01ec5417056p-57;
    const double whole = rint(t), f = (t - whole) + e, quarter = rint(4.0 * f);
    const float r = (float)(f - 0.25 * quarter), r2 = r * r;
    float s = fmaf(r2, 4.205869394e+01f, -7.670585975e+01f);
    s = fmaf(r2, s, 8.160524928e+01f);
    s = fmaf(r2, s, -4.134170224e+01f);
    s = fmaf(r2, s, 6.283185307e+00f) * r;
    float c = fmaf(r2, -2.642625678e+01f, 6.024464137e+01f);
    c = fmaf(r2, c, -8.545681721e+01f);
    c = fmaf(r2, c, 6.493939402e+01f);
    c = fmaf(r2, c, -1.973920880e+01f);
    c = fmaf(r2, c, 1.0f);
    const int n = (int)quarter & 3;
    const float a = n & 1 ? s : c, b = n & 1 ? c : s;
    /* (c, s) turned by n quarters: (c, s), (-s, c), (-c, -s), (s, -c) */
    return make_float2(n == 1 || n == 2 ? -a : a, n & 2 ? -b : b);
}

template <typename T>
__device__ __forceinline__ void pg_get8(const T *p, float x[8]) {
    if constexpr (sizeof(T) == 2) {
        const uint4 w = qk_ld((const uint4 *)p);
        x[0] = qk_bf16_lo(w.x); x[1] = qk_bf16_hi(w.x); x[2] = qk_bf16_lo(w.y); x[3] = qk_bf16_hi(w.y);
        x[4] = qk_bf16_lo(w.z); x[5] = qk_bf16_hi(w.z); x[6] = qk_bf16_lo(w.w); x[7] = qk_bf16_hi(w.w);
    } else {
        const float4 a = qk_ld((const float4 *)p), b = qk_ld((const float4 *)p + 1);
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
        x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    }
}
/* f32 -> bf16 rounds to nearest even: the page type's own rounding */
template <typename T>
__device__ __forceinline__ void pg_put8(T *p, const float x[8]) {
    if constexpr (sizeof(T) == 2) {
        const uint4 w = make_uint4(qk_cvt_pk_bf16(x[0], x[1]), qk_cvt_pk_bf16(x[2], x[3]), qk_cvt_pk_bf16(x[4], x[5]),
                                   qk_cvt_pk_bf16(x[6], x[7]));
        qk_st((float4 *)p, __builtin_bit_cast(float4, w));
    } else {
        qk_st((float4 *)p, make_float4(x[0], x[1], x[2], x[3]));
        qk_st((float4 *)p + 1, make_float4(x[4], x[5], x[6], x[7]));
    }
}

/* the sequence that has row t, as pg_find, by a whole wave: 64 starts at a time */
__device__ __forceinline__ int pg_find_wave(const int32_t *starts, int n_seqs, int t) {
    const int lane = threadIdx.x & 63;
    const int end = qk_ld(starts + n_seqs); /* in flight beside the first round */
    int lo = 0, span = n_seqs;
    while (true) {
        const int step = (span + 63) >> 6, i = lo + lane * step;
        const int c = __popcll(__ballot(lane * step < span && qk_ld(starts + min(i, n_seqs - 1)) <= t));
        if (c == 0) return n_seqs;
        lo += (c - 1) * step;
        if (step == 1) return t < end ? lo : n_seqs;
        span = min(step, span - (c - 1) * step);
    }
}

/* lanes of a head; of 192, 24 of them hold elements */
constexpr int pg_head_lanes(int hd) { return hd <= 64 ? 8 : hd <= 128 ? 16 : 32; }

template <typename S, typename D, int HD, int TOK>
__global__ __launch_bounds__(512) void k_pg_rotary(PgRotary a) {
    constexpr int LP = pg_head_lanes(HD);
    const int threads = blockDim.x, RP = threads / LP;
    struct Row {
        int64_t at;   /* of its place in the pages, or -1 */
        int pos;      /* -1: nothing of it is written */
    };
    __shared__ __attribute__((aligned(16))) float cs[TOK][HD / 2], sn[TOK][HD / 2], buf[512 / LP][HD + 4];
    __shared__ Row rows[TOK];
    const int tid = threadIdx.x, wave = tid >> 6, slot = tid / LP, e0 = 8 * (tid % LP), rot = 2 * a.half;
    const bool on = HD != 192 || e0 < HD;
    const int e1 = on ? e0 : 0, t0 = blockIdx.x * TOK, R = (int)a.per_row.d, end = min(TOK, a.n - t0) * R;
    /* a head of the workgroup's tokens: which of q, k and v, and where it lies; their loads need
     * no position and go out first */
    struct Head {
        int t, which, hd;
    };
    auto head = [&](int r) {
        Head h;
        h.t = TOK == 1 ? 0 : (int)pg_div_of(a.per_row, (uint32_t)r);
        const int x = r - h.t * R;
        h.which = x < a.h ? 0 : x < a.h + a.c.kvh ? 1 : 2;
        h.hd = x - (h.which == 0 ? 0 : h.which == 1 ? a.h : a.h + a.c.kvh);
        return h;
    };
    auto load = [&](int r, float x[8]) {
        const Head h = head(min(r, end - 1));
        const int64_t t = t0 + h.t;
        pg_get8((h.which == 0 ? (const S *)a.q + t * a.q_token + h.hd * a.q_head
                              : h.which == 1 ? (const S *)a.k + t * a.k_token + h.hd * a.k_head
                                             : (const S *)a.v + t * a.v_token + h.hd * a.v_head) + e1, x);
    };
    float next[8];
    load(slot, next);
    const float freq = qk_ld(a.freqs + (tid < TOK * a.half ? tid % a.half : 0));
    const int refused = a.status ? qk_ld(a.status) : 0;
    for (int k = wave; k < TOK; k += threads >> 6) {
        const int t = t0 + k, s = t < a.n ? pg_find_wave(a.starts, a.n_seqs, t) : a.n_seqs;
        Row w = {-1, -1};
        if (s < a.n_seqs && !refused) {
            const int depth = a.depths ? qk_ld(a.depths + t) : 0;
            const pg_seq q = pg_seq_at(&a.c, a.starts, a.slots, a.n, s);
            const int first = q.len - q.count, row = t - q.start, place = first + row;
            if (q.slot >= 0 && row >= 0 && row < q.count && place >= 0 && depth >= 0) {
                w.at = pg_row_at(&a.c, a.c.table + q.slot * a.c.table_stride, place);
                w.pos = a.depths ? first + min(depth, row) : place; /* below 0: a node before the first row */
            }
        }
        if ((tid & 63) == 0) rows[k] = w;
    }
    __syncthreads();
    for (int i = tid; i < TOK * a.half; i += threads) {
        const int k = i / a.half, f = i - k * a.half;
        const float2 c = pg_turn(max(rows[k].pos, 0), i == tid ? freq : qk_ld(a.freqs + f));
        cs[k][f] = c.x;
        sn[k][f] = c.y;
    }
    __syncthreads();
    for (int r = slot; r < end; r += RP) {
        const Head h = head(r);
        const Row w = rows[h.t];
        float x[8], y[8];
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = next[i];
        load(r + RP, next);
        if (w.pos < 0 || (h.which && w.at < 0)) continue;
        const int64_t t = t0 + h.t;
        D *dst = h.which == 0 ? (D *)a.out + t * a.o_token + h.hd * a.o_head
                              : (D *)(h.which == 1 ? a.c.k : a.c.v) + w.at + h.hd * a.c.head_stride;
        const float *nw = h.which == 0 ? a.q_norm : a.k_norm;
        if (h.which < 2 && nw) {
            float wt[8];
#pragma unroll
            for (int i = 0; i < 8; i++) wt[i] = qk_ld(nw + e1 + i);
            float ss = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; i++) ss = fmaf(x[i], x[i], ss);
            ss = qk_group_sum<LP>(on ? ss : 0.0f);
            const float f = 1.0f / sqrtf(ss / (float)HD + a.eps);
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = (x[i] * f) * wt[i];
        }
#pragma unroll
        for (int i = 0; i < 8; i++) y[i] = x[i];
        if (h.which < 2) {
            const float *c = cs[h.t], *s = sn[h.t];
            if (a.inter) {
#pragma unroll
                for (int i = 0; i < 8; i += 2)
                    if (e0 + i < rot) {
                        const int f = (e0 + i) / 2;
                        y[i] = x[i] * c[f] - x[i + 1] * s[f];
                        y[i + 1] = x[i] * s[f] + x[i + 1] * c[f];
                    }
            } else {
                float *b = buf[slot];
                qk_wave_lds_sync();
                if (on) {
                    *(float4 *)(b + e0) = make_float4(x[0], x[1], x[2], x[3]);
                    *(float4 *)(b + e0 + 4) = make_float4(x[4], x[5], x[6], x[7]);
                }
                qk_wave_lds_sync();
                if (a.half % 8 == 0) { /* the lane's partners are another lane's eight */
                    if (e0 < rot) {
                        const bool up = e0 >= a.half;
                        const int f = up ? e0 - a.half : e0;
                        const float4 *p = (const float4 *)(b + (up ? f : f + a.half));
                        const float4 p0 = p[0], p1 = p[1], c0 = *(const float4 *)(c + f), c1 = *(const float4 *)(c + f + 4),
                                     s0 = *(const float4 *)(s + f), s1 = *(const float4 *)(s + f + 4);
                        const float pp[8] = {p0.x, p0.y, p0.z, p0.w, p1.x, p1.y, p1.z, p1.w};
                        const float cc[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
                        const float ss[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
#pragma unroll
                        for (int i = 0; i < 8; i++) y[i] = up ? pp[i] * ss[i] + x[i] * cc[i] : x[i] * cc[i] - pp[i] * ss[i];
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const int e = e0 + i;
                        if (e < a.half) y[i] = x[i] * c[e] - b[e + a.half] * s[e];
                        else if (e < rot) y[i] = b[e - a.half] * s[e - a.half] + x[i] * c[e - a.half];
                    }
                }
            }
        }
        if (on) pg_put8(dst + e0, y);
    }
}

template <typename S, typename D, int TOK>
static int pg_rotary_hd(const PgRotary &a, hipStream_t st) {
    const int64_t lanes = (int64_t)a.per_row.d * pg_head_lanes(a.c.hd); /* of a row: one round of them where 512 threads hold it */
    const dim3 grid((unsigned)(((int64_t)a.n + TOK - 1) / TOK)), wg(TOK > 1 ? 256 : lanes >= 512 ? 512 : (unsigned)(lanes + 63) / 64 * 64);
    switch (a.c.hd) {
    case 64: hipLaunchKernelGGL((k_pg_rotary<S, D, 64, TOK>), grid, wg, 0, st, a); break;
    case 128: hipLaunchKernelGGL((k_pg_rotary<S, D, 128, TOK>), grid, wg, 0, st, a); break;
    case 192: hipLaunchKernelGGL((k_pg_rotary<S, D, 192, TOK>), grid, wg, 0, st, a); break;
    case 256: hipLaunchKernelGGL((k_pg_rotary<S, D, 256, TOK>), grid, wg, 0, st, a); break;
    default: return (int)hipErrorInvalidValue;
    }
    return QK_CHECK_LAUNCH();
}
template <typename S, typename D>
static int pg_rotary_tok(const PgRotary &a, hipStream_t st) {
    return a.n >= PG_ROTARY_MANY ? pg_rotary_hd<S, D, 4>(a, st) : pg_rotary_hd<S, D, 1>(a, st);
}

extern "C" int qk_launch_pg_rotary(const pg_cache *c, const qmoe_paged_rotary *r, const int32_t *starts, const int32_t *slots,
                                   const int32_t *status, const int32_t *depths, int n, int n_seqs, void *stream) {
    hipStream_t st = (hipStream_t)stream;
    PgRotary a;
    a.c = *c;
    a.q = r->q; a.k = r->k; a.v = r->v; a.out = r->out;
    a.q_token = r->q_token_stride; a.q_head = r->q_head_stride;
    a.k_token = r->k_token_stride; a.k_head = r->k_head_stride;
    a.v_token = r->v_token_stride; a.v_head = r->v_head_stride;
    a.o_token = r->out_token_stride; a.o_head = r->out_head_stride;
    a.freqs = r->freqs; a.q_norm = r->q_norm; a.k_norm = r->k_norm;
    a.starts = starts; a.slots = slots; a.status = status; a.depths = depths;
    a.eps = r->eps;
    a.n = n; a.n_seqs = n_seqs;
    a.h = r->n_heads; a.half = r->rot / 2; a.inter = r->interleaved;
    a.per_row = pg_div_make((uint32_t)(r->n_heads + 2 * c->kvh));
    if (c->dtype == QMOE_F32) return pg_rotary_tok<float, float>(a, st);
    return r->src_dtype == QMOE_F32 ? pg_rotary_tok<float, uint16_t>(a, st) : pg_rotary_tok<uint16_t, uint16_t>(a, st);
}

/* ------------------------------------------------------------ trees
 * Depth and ancestors of every drafted row, a workgroup per sequence, a thread
 * per (row, word of 32 of its bits).  A thread walks from its row to the root;
 * a run of rows whose parents are the rows before them is one step, so a
 * chain, however long, is one.  Bound: latency, of the loads of starts and
 * parents and of the walk in LDS: 1.8 us for 8 nodes, 3.1 to 5 for up to 24 of
 * 64 sequences, 5.7 for 256 of 8.  Large trees are bound by the walks, one for
 * each word of a row: 1024 nodes of a star or a chain 24 to 37 us a call, drawn
 * at random 60 to 70, but of two chains row by row, 512 steps each and none of
 * them a run, 1600 (256 nodes 33 to 110). */
#define PG_TREE_ROWS 1024

struct PgTree {
    const int32_t *parents, *starts;
    int n, words;
    int32_t *depths;
    uint32_t *seen;
};

/* rows [start, start + count) of sequence i of the call, brought into [0, n) */
__device__ __forceinline__ int2 pg_rows_of(const int32_t *starts, int n, int i) {
    const int a = min(max(qk_ld(starts + i), 0), n), b = min(qk_ld(starts + i + 1), n);
    return make_int2(a, max(b - a, 0));
}

__global__ __launch_bounds__(1024) void k_pg_tree(PgTree a) {
    __shared__ int up[PG_TREE_ROWS];
    __shared__ uint32_t head[PG_TREE_ROWS / 32]; /* bit t: row t is not the child of row t - 1 */
    const int tid = threadIdx.x;
    const int2 s = pg_rows_of(a.starts, a.n, blockIdx.x);
    const int c = min(s.y, 32 * a.words);
    if (tid < PG_TREE_ROWS / 32) head[tid] = 0;
    __syncthreads();
    for (int t = tid; t < c; t += blockDim.x) {
        const int p = qk_ld(a.parents + s.x + t);
        up[t] = p >= -1 && p < t ? p : -2;
        if (t == 0 || p != t - 1) atomicOr(&head[t >> 5], 1u << (t & 31));
    }
    __syncthreads();
    for (int x = tid; x < c * a.words; x += blockDim.x) {
        const int t = x / a.words, w = x - t * a.words;
        int rows = 0, at = t;
        uint32_t bits = 0;
        while (at >= 0) {
            int k = at >> 5;
            uint32_t m = head[k] & ((2u << (at & 31)) - 1u);
            while (!m) m = head[--k]; /* row 0's bit is set */
            const int b = 32 * k + 31 - __builtin_clz(m); /* the run's first row */
            const int lo = max(b - 32 * w, 0), hi = min(at - 32 * w, 31);
            if (lo <= hi) bits |= (0xFFFFFFFFu << lo) & (0xFFFFFFFFu >> (31 - hi));
            rows += at - b + 1;
            at = up[b];
        }
        a.seen[(int64_t)(s.x + t) * a.words + w] = at == -1 ? bits : 0u;
        if (w == 0) a.depths[s.x + t] = at == -1 ? rows - 1 : -1;
    }
    for (int t = c + tid; t < s.y; t += blockDim.x) { /* past what the words hold: no nodes */
        for (int w = 0; w < a.words; w++) a.seen[(int64_t)(s.x + t) * a.words + w] = 0u;
        a.depths[s.x + t] = -1;
    }
}

extern "C" int qk_launch_pg_tree(const int32_t *parents, const int32_t *starts, int n, int n_seqs, int32_t *depths,
                                 uint32_t *seen, int words, void *stream) {
    const PgTree a = {parents, starts, n, words, depths, seen};
    /* 256 nodes of 8 sequences 10 us with 256 threads, 5 with 1024 */
    hipLaunchKernelGGL(k_pg_tree, dim3(n_seqs), dim3(words > 2 ? 1024 : 256), 0, (hipStream_t)stream, a);
    return QK_CHECK_LAUNCH();
}

/* ------------------------------------------------------------ follow
 * The path that the target's choices take, a workgroup per sequence.  A row
 * is taken where its token is the one chosen after its parent and no lower
 * child of that parent has it too; a row is on the path where it and all its
 * ancestors are taken (row 0 always), so its place is its depth and no walk is
 * needed.  Bound: latency, 2.5 us for 12 nodes, 4.2 for up to 32 of 256
 * sequences. */
struct PgFollow {
    const int32_t *parents, *tokens, *chosen, *starts, *depths;
    const uint32_t *seen;
    int n, words;
    int32_t *rows, *counts, *next;
};

__global__ __launch_bounds__(256) void k_pg_follow(PgFollow a) {
    __shared__ int kid[PG_TREE_ROWS], path[PG_TREE_ROWS];
    __shared__ uint32_t taken[PG_TREE_ROWS / 32];
    __shared__ int deepest;
    const int tid = threadIdx.x;
    const int2 s = pg_rows_of(a.starts, a.n, blockIdx.x);
    const int c = min(s.y, 32 * a.words);
    for (int t = tid; t < c; t += 256) {
        kid[t] = PG_TREE_ROWS;
        path[t] = -1;
    }
    if (tid < PG_TREE_ROWS / 32) taken[tid] = 0;
    if (tid == 0) deepest = -1;
    __syncthreads();
    for (int t = tid; t < c; t += 256) {
        const int p = qk_ld(a.parents + s.x + t);
        if (p >= 0 && p < t && qk_ld(a.tokens + s.x + t) == qk_ld(a.chosen + s.x + p)) atomicMin(&kid[p], t);
    }
    __syncthreads();
    for (int t = tid; t < c; t += 256) {
        const int p = qk_ld(a.parents + s.x + t);
        if (t == 0 || (p >= 0 && p < t && kid[p] == t)) atomicOr(&taken[t >> 5], 1u << (t & 31));
    }
    __syncthreads();
    for (int t = tid; t < c; t += 256) {
        const int d = min(qk_ld(a.depths + s.x + t), t);
        bool on = d >= 0 && (taken[t >> 5] >> (t & 31) & 1u);
        for (int w = 0; on && w <= t >> 5; w++) on = !(qk_ld(a.seen + (int64_t)(s.x + t) * a.words + w) & ~taken[w]);
        /* other roots than row 0 are never taken, so a path has one row of each depth */
        if (on) {
            path[d] = t;
            atomicMax(&deepest, d);
        }
    }
    __syncthreads();
    for (int t = tid; t < s.y; t += 256) a.rows[s.x + t] = t < c ? path[t] : -1;
    if (tid == 0) {
        a.counts[blockIdx.x] = deepest + 1;
        a.next[blockIdx.x] = deepest < 0 || path[deepest] < 0 ? -1 : qk_ld(a.chosen + s.x + path[deepest]);
    }
}

extern "C" int qk_launch_pg_follow(const int32_t *parents, const int32_t *tokens, const int32_t *chosen, const int32_t *starts,
                                   const int32_t *depths, const uint32_t *seen, int words, int n, int n_seqs, int32_t *rows,
                                   int32_t *counts, int32_t *next, void *stream) {
    const PgFollow a = {parents, tokens, chosen, starts, depths, seen, n, words, rows, counts, next};
    hipLaunchKernelGGL(k_pg_follow, dim3(n_seqs), dim3(256), 0, (hipStream_t)stream, a);
    return QK_CHECK_LAUNCH();
}

/* ------------------------------------------------------------ keep
 * Two launches, so that a batch with a sequence that is refused is left as it
 * was: the first finds where every kept row lies and goes to, a workgroup per
 * sequence, the second moves them and cuts the tables.  Small batches take one,
 * of one workgroup.  Kept rows ascend, so row k goes to a place at or before
 * its own and behind those of the rows before it: a thread that moves its 16
 * bytes of every row of a sequence, in order, 8 loads before their stores,
 * never reads what it has written.  Bound: latency, 4.8 and 5.6 us for 256
 * sequences of 12 layers (about two rows of each move, 5.8 MB). */
struct PgKeep {
    pg_cache c;
    const int32_t *starts, *slots, *status, *rows, *counts;
    int n, n_seqs;
    int32_t *result;
    int4 *head;          /* [n_seqs]: refused (1, or the batch's status), slot, rows kept, lens now */
    longlong2 *moves;    /* [n]: element offsets from, to */
    pg_div cols, heads;  /* 16-byte pieces of a row, of a head */
};

/* sequence i: its rows of the call, its slot and what is kept; true where it is refused as far as
 * that shows (the slot named twice, and the rows, are for the caller's lanes) */
struct PgKept {
    int from, count, slot, keep, len;
};
__device__ __forceinline__ bool pg_kept(const PgKeep &a, int i, PgKept &q) {
    const int to = qk_ld(a.starts + i + 1);
    q.from = qk_ld(a.starts + i);
    q.slot = a.slots ? qk_ld(a.slots + i) : i;
    q.keep = qk_ld(a.counts + i);
    q.count = to - q.from;
    q.len = 0;
    if (q.from < 0 || to < q.from || to > a.n || q.slot < 0 || q.slot >= a.c.n_slots || q.keep < 0 || q.keep > q.count) return true;
    q.len = qk_ld(a.c.lens + q.slot);
    return q.len < q.count || q.len > a.c.cap;
}
/* where kept row k moves from and to (equal: it stays); true where it is refused */
__device__ __forceinline__ bool pg_move_of(const PgKeep &a, const PgKept &q, int k, longlong2 &m) {
    const int r = qk_ld(a.rows + q.from + k), before = k ? qk_ld(a.rows + q.from + k - 1) : -1, first = q.len - q.count;
    m.x = m.y = 0;
    if (r <= before || r >= q.count) return true;
    if (r == k) return false;
    const int32_t *row = a.c.table + q.slot * a.c.table_stride;
    m.x = pg_row_at(&a.c, row, first + r);
    m.y = pg_row_at(&a.c, row, first + k);
    return m.x < 0 || m.y < 0 || qk_ld(a.c.refs + qk_ld(row + pg_div_of(a.c.page_rows, (uint32_t)(first + k)))) > 1;
}
/* piece x of all layers' k and v of a sequence's rows; moves(k) is row k's */
template <typename F>
__device__ __forceinline__ void pg_move(const PgKeep &a, int64_t x, int keep, F moves) {
    const int es = a.c.dtype == QMOE_BF16 ? 2 : 4, lv = (int)(x / a.cols.d);
    const uint32_t col = (uint32_t)(x - (int64_t)lv * a.cols.d), hd = pg_div_of(a.heads, col), ch = col - hd * a.heads.d;
    char *base = (char *)(lv & 1 ? a.c.v : a.c.k) + ((lv >> 1) * a.c.layer_stride + hd * a.c.head_stride) * es + 16 * ch;
    for (int k0 = 0; k0 < keep; k0 += 8) {
        float4 y[8];
        longlong2 m[8];
#pragma unroll
        for (int k = 0; k < 8; k++) m[k] = moves(min(k0 + k, keep - 1));
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (k0 + k < keep && m[k].x != m[k].y) y[k] = qk_ld((const float4 *)(base + m[k].x * es));
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (k0 + k < keep && m[k].x != m[k].y) qk_st((float4 *)(base + m[k].y * es), y[k]);
    }
}
/* the slot's length, and the pages behind it, by `threads` */
__device__ __forceinline__ void pg_cut(const PgKeep &a, int slot, int was, int now, int tid, int threads) {
    const int R = (int)a.c.page_rows.d;
    int32_t *row = a.c.table + slot * a.c.table_stride;
    for (int e = (now + R - 1) / R + tid; e < (was + R - 1) / R; e += threads) {
        const int p = qk_ld(row + e);
        if (p >= 0 && p < a.c.n_pages) atomicSub(a.c.refs + p, 1);
        row[e] = -1;
    }
    if (tid == 0) a.c.lens[slot] = now;
}

__global__ __launch_bounds__(256) void k_pg_keep_find(PgKeep a) {
    const int i = blockIdx.x, tid = threadIdx.x;
    const int refused = a.status ? qk_ld(a.status) : 0;
    PgKept q;
    bool bad = pg_kept(a, i, q);
    if (a.slots)
        for (int j = tid; j < a.n_seqs; j += 256) bad |= j != i && qk_ld(a.slots + j) == q.slot;
    for (int k = tid; !bad && k < q.keep; k += 256) {
        longlong2 m;
        bad = pg_move_of(a, q, k, m);
        qk_st((float4 *)(a.moves + q.from + k), __builtin_bit_cast(float4, m));
    }
    bad = __syncthreads_or(bad);
    if (tid == 0) a.head[i] = make_int4(refused ? refused : bad ? -1 : 0, q.slot, q.keep, q.len - q.count + q.keep);
}

__global__ __launch_bounds__(256) void k_pg_keep_move(PgKeep a) {
    const int i = blockIdx.y, tid = threadIdx.x;
    const int from = qk_ld(a.starts + i), count = qk_ld(a.starts + i + 1) - from;
    const int4 h = qk_ld(a.head + i);
    int bad = 0;
    for (int j = tid; j < a.n_seqs; j += 256) bad |= qk_ld((const int *)(a.head + j)) != 0;
    if (__syncthreads_or(bad)) {
        if (i == 0 && blockIdx.x == 0 && tid == 0) {
            const int refused = a.status ? qk_ld(a.status) : 0;
            *a.result = refused ? refused : -1;
        }
        return;
    }
    if (blockIdx.x == 0) {
        pg_cut(a, h.y, h.w - h.z + count, h.w, tid, 256);
        if (i == 0 && tid == 0) *a.result = 0;
    }
    const longlong2 *mv = a.moves + from;
    const int64_t pieces = (int64_t)2 * a.c.n_layers * a.cols.d;
    for (int64_t x = (int64_t)blockIdx.x * 256 + tid; x < pieces; x += (int64_t)gridDim.x * 256)
        pg_move(a, x, h.z, [&](int k) { return __builtin_bit_cast(longlong2, qk_ld((const float4 *)(mv + k))); });
}

/* The same by one workgroup, a wave per sequence up to the moves.  Up to
 * PG_KEEP_SMALL pieces of all sequences' rows: one of one layer 4.9 us in two
 * launches, so 3.7; four of three 7.5 and 5.1. */
#define PG_KEEP_SEQS 16
#define PG_KEEP_ROWS 1024
#define PG_KEEP_SMALL 4096
__global__ __launch_bounds__(1024) void k_pg_keep_small(PgKeep a) {
    __shared__ longlong2 moves[PG_KEEP_ROWS];
    __shared__ PgKept seq[PG_KEEP_SEQS];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int refused = a.status ? qk_ld(a.status) : 0;
    bool bad = refused != 0;
    if (wave < a.n_seqs) {
        PgKept q;
        bad |= pg_kept(a, wave, q);
        if (a.slots) bad |= lane < a.n_seqs && lane != wave && qk_ld(a.slots + min(lane, a.n_seqs - 1)) == q.slot;
        for (int k = lane; !bad && k < q.keep; k += 64) {
            longlong2 m;
            bad = pg_move_of(a, q, k, m);
            moves[q.from + k] = m;
        }
        if (lane == 0) seq[wave] = q;
    }
    if (__syncthreads_or(bad)) {
        if (tid == 0) *a.result = refused ? refused : -1;
        return;
    }
    if (wave < a.n_seqs) pg_cut(a, seq[wave].slot, seq[wave].len, seq[wave].len - seq[wave].count + seq[wave].keep, lane, 64);
    if (tid == 0) *a.result = 0;
    const int pieces = 2 * a.c.n_layers * (int)a.cols.d;
    for (int x = tid; x < pieces * a.n_seqs; x += 1024) {
        const int i = x / pieces;
        pg_move(a, x - i * pieces, seq[i].keep, [&](int k) { return moves[seq[i].from + k]; });
    }
}

static size_t pg_up(size_t v) { return (v + 255) / 256 * 256; }
extern "C" size_t qk_pg_keep_ws(int n, int n_seqs) { return pg_up((size_t)n_seqs * 16) + pg_up((size_t)n * 16); }

/* an empty batch reports too */
__global__ void k_pg_keep_none(const int32_t *status, int32_t *result) { *result = status ? qk_ld(status) : 0; }

extern "C" int qk_launch_pg_keep(const pg_cache *c, const int32_t *starts, const int32_t *slots, const int32_t *status, int n,
                                 int n_seqs, const int32_t *rows, const int32_t *counts, int32_t *result, void *ws, void *stream) {
    hipStream_t st = (hipStream_t)stream;
    PgKeep a;
    const int per_head = c->hd * (c->dtype == QMOE_BF16 ? 2 : 4) / 16;
    a.c = *c;
    a.starts = starts; a.slots = slots; a.status = status; a.rows = rows; a.counts = counts;
    a.n = n; a.n_seqs = n_seqs; a.result = result;
    a.head = (int4 *)ws;
    a.moves = (longlong2 *)((char *)ws + pg_up((size_t)n_seqs * 16));
    a.cols = pg_div_make((uint32_t)(c->kvh * per_head));
    a.heads = pg_div_make((uint32_t)per_head);
    if (n_seqs == 0) {
        hipLaunchKernelGGL(k_pg_keep_none, dim3(1), dim3(1), 0, st, status, result);
        return QK_CHECK_LAUNCH();
    }
    if (n_seqs <= PG_KEEP_SEQS && n <= PG_KEEP_ROWS && (int64_t)2 * c->n_layers * a.cols.d * n_seqs <= PG_KEEP_SMALL) {
        hipLaunchKernelGGL(k_pg_keep_small, dim3(1), dim3(1024), 0, st, a);
        return QK_CHECK_LAUNCH();
    }
    hipLaunchKernelGGL(k_pg_keep_find, dim3(n_seqs), dim3(256), 0, st, a);
    const int rc = QK_CHECK_LAUNCH();
    if (rc) return rc;
    const int64_t blocks = ((int64_t)2 * c->n_layers * a.cols.d + 255) / 256;
    hipLaunchKernelGGL(k_pg_keep_move, dim3((unsigned)(blocks < 1024 ? blocks : 1024), n_seqs), dim3(256), 0, st, a);
    return QK_CHECK_LAUNCH();
}
