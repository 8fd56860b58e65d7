/*
 * paged_attn.hip -- attention of a ragged batch of new tokens over a paged
 * cache: softmax(scale q.k) v over the rows that a token sees (causal, a
 * sliding window, sinks), a group of query heads per kv head.
 *
 * The (token, head) rows of a sequence that read one kv head are one matrix
 * of queries: row r is token r / G, member r % G of the group, so a page is
 * read once for all heads of its group.  Rows are cut into tiles, the keys of
 * a row tile into parts where there are too few tiles to fill the card; a
 * unit of work is (sequence, row tile, part, kv head), numbered on the device
 * from the lengths it finds (pa_find), and a second launch joins the parts.
 *
 * Products are transposed: S^T = K Q^T leaves each lane the scores of one
 * row, for keys 8 a + 4 (lane / 32) + b of a tile of 32, and those registers
 * are the B operand of O^T = V^T P^T as they are, if V^T's operand takes its
 * keys in that order.  Maximum, sum and O stay with the lane (fp32).
 */
#include "qk_device.h"
#include "mfma_parts.h"
#include "paged_parts.h"

typedef float qm_f32x16 __attribute__((ext_vector_type(16)));

#define PM_RT 128 /* rows of a unit of the many-row kernels */

__device__ const uint4 pa_zero[64] = {}; /* a row of zeros, up to 1 KB */

struct PaArgs {
    pg_cache c;   /* k and v of the call's layer */
    pg_attn a;
    int G;        /* query heads per kv head */
    float per_unit; /* kv heads / units that the call is cut into, rounded up */
    int extra;    /* key tiles that a join is worth (pg_share) */
    int one, units; /* the same where no more than `units` units come of it */
    float *po;    /* partial O [slot, RT, HD], unscaled */
    float2 *pml;  /* [slot, RT]: maximum (log2 units), sum */
    int4 *index;  /* [n_seqs], calls of more than PA_INDEX sequences: units, joined tasks
                   * and split units before the sequence's, its parts */
};

/* query head of member g of kv head kh's group: heads kh, kh + kvh, ... (the
 * attention mixer's order) or G in a row */
__device__ __forceinline__ int pa_head(const PaArgs &p, int kh, int g) {
    return p.a.grouped ? kh * p.G + g : kh + g * p.c.kvh;
}

template <typename T>
__device__ __forceinline__ float pa_get(const T *p) {
    if constexpr (sizeof(T) == 2) return qk_bf16(qk_ld((const uint16_t *)p));
    else return qk_ld((const float *)p);
}

/* 8 consecutive elements as f32 */
template <typename T>
__device__ __forceinline__ void pa_get8(const T *p, float x[8]) {
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
/* 4 consecutive elements of the output type */
template <typename T>
__device__ __forceinline__ void pa_put4(T *p, float a, float b, float c, float d) {
    if constexpr (sizeof(T) == 2) {
        qk_u32x2 w = {qk_cvt_pk_bf16(a, b), qk_cvt_pk_bf16(c, d)};
        *(QK_GLOBAL qk_u32x2 *)p = w;
    } else {
        qk_st((float4 *)p, make_float4(a, b, c, d));
    }
}

/* what a row's maximum and sum give: the factor on its sum of p v, NaN for a
 * row whose scores are all -inf (0/0, as the formula), 0 for a row that sees
 * nothing.  A part that sees only scores of -inf has the sum 1 beside the
 * maximum -inf, so that the join tells the two apart. */
__device__ __forceinline__ float pa_sum(float m, float l, bool seen) { return m == -INFINITY && seen ? 1.0f : l; }
__device__ __forceinline__ float pa_norm(float m, float l) {
    return m == -INFINITY ? (l > 0.0f ? NAN : 0.0f) : 1.0f / l;
}

/* ------------------------------------------------------------ units */

struct PaUnit {
    pg_seq s;
    int rtile, part, parts, kh;
    int slot; /* of the part's partial results */
};

/* inclusive prefix sum over the wave */
__device__ __forceinline__ int pa_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false); /* row_shr:1, 2, 4, 8 within 16 lanes */
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, QK_DPP_ROW_BCAST15, 0xA, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, QK_DPP_ROW_BCAST31, 0xC, 0xF, false);
    return v;
}

/* units, tasks that are joined and split units of a sequence */
struct PaCount {
    int parts, units, tasks, split;
};
__device__ __forceinline__ PaCount pa_count(const PaArgs &p, const pg_load &l, int share) {
    PaCount c;
    const int tasks = l.row_tiles * p.c.kvh;
    c.parts = pg_cuts(l.key_tiles, p.extra) ? pg_parts(l.key_tiles, share) : 1;
    c.units = tasks * c.parts;
    c.tasks = c.parts > 1 ? tasks : 0;
    c.split = c.parts > 1 ? c.units : 0;
    return c;
}
__device__ __forceinline__ pg_seq pa_seq(const PaArgs &p, int i) { return pg_seq_at(&p.c, p.a.starts, p.a.slots, p.a.n, i); }

/* Batches of more sequences than a wave has lanes: what precedes each one
 * (units, joined tasks, split units) and its parts, by one workgroup in a
 * launch of its own, which the units then search.  Units that each went over
 * all sequences by themselves took 309 us for single tokens of 1024 sequences
 * of 1000 rows, 198 with the index; of 100 sequences of 200 rows 11.7 and
 * 13.0 (the launch), of 1000 rows 38 and 35.  So the two meet between 64 and some
 * hundred sequences, by their lengths, which the host does not know: the limit
 * is where a lane per sequence ends and the other way would need a loop.  The
 * total is summed in fp32, in a fixed order. */
#define PA_INDEX 64
__global__ __launch_bounds__(1024) void k_pa_index(PaArgs p, int rt, int kt) {
    __shared__ float sum[16];
    __shared__ int before[16][3];
    const int tid = threadIdx.x, wave = tid >> 6, n = p.a.n_seqs, per = (n + 1023) >> 10;
    const int i0 = min(tid * per, n), i1 = min(i0 + per, n);
    auto load = [&](int i) { return pg_load_of(pa_seq(p, i), p.G, rt, p.a.window, p.a.sinks, kt); };
    pg_load last = {0, 0, 0.0f};
    float t = 0.0f;
    for (int i = i0; i < i1; i++) {
        last = load(i);
        t += last.work;
    }
    t = qk_group_sum<64>(t);
    if ((tid & 63) == 0) sum[wave] = t;
    __syncthreads();
    t = 0.0f;
    for (int w = 0; w < 16; w++) t += sum[w];
    int share = pg_share(t, p.per_unit, p.one);
    PaCount all;
    int x[3];
    for (;;) { /* twice at most */
        all = {0, 0, 0, 0};
        for (int i = i0; i < i1; i++) {
            const PaCount c = pa_count(p, per == 1 ? last : load(i), share);
            all.units += c.units;
            all.tasks += c.tasks;
            all.split += c.split;
        }
        x[0] = pa_scan(all.units);
        x[1] = pa_scan(all.tasks);
        x[2] = pa_scan(all.split);
        if ((tid & 63) == 63)
            for (int k = 0; k < 3; k++) before[wave][k] = x[k];
        __syncthreads();
        int units = 0;
        for (int w = 0; w < 16; w++) units += before[w][0];
        const int full = pg_share(t, p.per_unit, p.extra);
        if (units <= p.units || share == full) break;
        share = full;
        __syncthreads();
    }
    for (int k = 0; k < 3; k++)
        for (int w = 0; w < wave; w++) x[k] += before[w][k];
    x[0] -= all.units;
    x[1] -= all.tasks;
    x[2] -= all.split;
    for (int i = i0; i < i1; i++) {
        const PaCount c = pa_count(p, per == 1 ? last : load(i), share);
        qk_st((float4 *)(p.index + i), __builtin_bit_cast(float4, make_int4(x[0], x[1], x[2], c.parts)));
        x[0] += c.units;
        x[1] += c.tasks;
        x[2] += c.split;
    }
}

/* Unit `want` of the call (JOIN: the want-th (sequence, row tile, kv head)
 * that has parts to join); false past the last, and for a refused batch.  Every wave finds it by
 * itself, a lane per sequence (of more: in the index), without LDS or
 * barriers: this stands before the first load of a page, and a decode call is
 * a few microseconds long. */
template <int RT, int KT, bool JOIN>
__device__ __forceinline__ bool pa_find(const PaArgs &p, int want, PaUnit &u) {
    const int lane = threadIdx.x & 63, n = p.a.n_seqs;
    /* in flight beside the lengths; with a branch before them a token took 10.4 us, so 10.1 */
    const int refused = qk_ld(p.a.status ? p.a.status : (const int32_t *)pa_zero);
    int ubase, sbase; /* units and split units before the sequence's */
    if (n <= PA_INDEX) {
        pg_seq s = {-1, 0, 0, 0};
        pg_load l = {0, 0, 0.0f};
        if (lane < n) {
            s = pa_seq(p, lane);
            l = pg_load_of(s, p.G, RT, p.a.window, p.a.sinks, KT);
        }
        const float total = qk_group_sum<64>(l.work);
        PaCount c = pa_count(p, l, pg_share(total, p.per_unit, p.one));
        if (p.one < p.extra && __builtin_amdgcn_readlane(pa_scan(c.units), 63) > p.units)
            c = pa_count(p, l, pg_share(total, p.per_unit, p.extra));
        const int units = JOIN ? c.tasks : c.units;
        int ue, se;
        if (RT == PM_RT) {
            /* the sequences with the longest parts come first, so that the last
             * units to start are short ones */
            const int len = units ? (l.key_tiles + c.parts - 1) / c.parts : 0;
            ue = se = 0;
            for (int k = 0; k < n; k++) {
                const int lk = __builtin_amdgcn_readlane(len, k);
                const bool before = lk > len || (lk == len && k < lane);
                ue += before ? __builtin_amdgcn_readlane(units, k) : 0;
                se += before ? __builtin_amdgcn_readlane(c.split, k) : 0;
            }
        } else {
            ue = pa_scan(units) - units;
            se = pa_scan(c.split) - c.split;
        }
        const uint64_t here = __ballot(want >= ue && want < ue + units);
        if (!here) return false;
        const int at = __builtin_ctzll(here);
        ubase = __builtin_amdgcn_readlane(ue, at);
        sbase = __builtin_amdgcn_readlane(se, at);
        u.parts = __builtin_amdgcn_readlane(c.parts, at);
        u.s.slot = __builtin_amdgcn_readlane(s.slot, at);
        u.s.start = __builtin_amdgcn_readlane(s.start, at);
        u.s.count = __builtin_amdgcn_readlane(s.count, at);
        u.s.len = __builtin_amdgcn_readlane(s.len, at);
    } else {
        /* the last sequence with ubase <= want, 64 of the index at a time */
        int lo = 0, span = n;
        while (span > 1) {
            const int step = (span + 63) >> 6;
            const bool ok = lane * step < span && qk_ld((const int *)(p.index + lo + min(lane * step, span - 1)) + JOIN) <= want;
            const int c = max(__popcll(__ballot(ok)), 1) - 1;
            lo += c * step;
            span = min(step, span - c * step);
        }
        const int4 x = __builtin_bit_cast(int4, qk_ld((const float4 *)(p.index + lo)));
        const pg_seq s = pa_seq(p, lo);
        ubase = __builtin_amdgcn_readfirstlane(JOIN ? x.y : x.x);
        sbase = __builtin_amdgcn_readfirstlane(x.z);
        u.parts = __builtin_amdgcn_readfirstlane(x.w);
        u.s.slot = __builtin_amdgcn_readfirstlane(s.slot);
        u.s.start = __builtin_amdgcn_readfirstlane(s.start);
        u.s.count = __builtin_amdgcn_readfirstlane(s.count);
        u.s.len = __builtin_amdgcn_readfirstlane(s.len);
    }
    const int rtiles = (u.s.count * p.G + RT - 1) / RT, tasks = rtiles * p.c.kvh;
    const int mine = JOIN ? (u.parts > 1 ? tasks : 0) : tasks * u.parts;
    if ((uint32_t)want - (uint32_t)ubase >= (uint32_t)mine || refused) return false; /* past the last */
    const int q = (want - ubase) / p.c.kvh;
    u.kh = want - ubase - q * p.c.kvh;
    const int back = JOIN ? q : q / u.parts;
    u.part = JOIN ? 0 : q - back * u.parts;
    u.rtile = rtiles - 1 - back;
    u.slot = sbase + (back * u.parts + u.part) * p.c.kvh + u.kh;
    return true;
}

/* ------------------------------------------------------------ masks */

/* bits j = 0..31 with base + j <= x */
__device__ __forceinline__ uint32_t pa_upto(int x, int base) {
    const int d = x - base;
    return d >= 31 ? 0xFFFFFFFFu : (d < 0 ? 0u : (2u << d) - 1u);
}
/* the keys base..base+31 that the query at position p sees */
__device__ __forceinline__ uint32_t pa_mask(const PaArgs &p, int pos, int base) {
    uint32_t w = pa_upto(pos, base);
    if (p.a.window > 0) w &= ~pa_upto(pg_lo(pos, p.a.window) - 1, base) | pa_upto(p.a.sinks - 1, base);
    return w;
}
/* all of them are seen at all positions p0..p1 */
__device__ __forceinline__ bool pa_full(const PaArgs &p, int p0, int p1, int base) {
    return base + 31 <= p0 && (p.a.window == 0 || base >= pg_lo(p1, p.a.window) || base + 31 < p.a.sinks);
}

/* ------------------------------------------------- one row at a time
 * fp32 on the vector ALU, keys of the unit's part only, for units whose
 * results are not finite or whose weights vanish (pa_again): a masked key is never multiplied
 * here.  Waves take the unit's rows in turn. */
template <typename T, int HD, int RT, int KT>
__device__ __forceinline__ void pa_slow(const PaArgs &p, const PaUnit &u, int kt0, int kt1, pg_tiles tl, int waves) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const T *kp = (const T *)p.c.k + (int64_t)u.kh * p.c.head_stride, *vp = (const T *)p.c.v + (int64_t)u.kh * p.c.head_stride;
    const int32_t *row = p.c.table + (int64_t)u.s.slot * p.c.table_stride;
    const int rows = u.s.count * p.G;
    for (int r = u.rtile * RT + wave; r < min(u.rtile * RT + RT, rows); r += waves) {
        const int t = r / p.G, hh = pa_head(p, u.kh, r - t * p.G), pos = u.s.len - u.s.count + t;
        const T *q = (const T *)p.a.q + (int64_t)(u.s.start + t) * p.a.q_token + (int64_t)hh * p.a.q_head;
        float m = -INFINITY, l = 0.0f, acc[HD / 16];
        bool seen = false;
#pragma unroll
        for (int e = 0; e < HD / 16; e++) acc[e] = 0.0f;
        for (int b = kt0 * KT; b < kt1 * KT; b += 64) { /* the part's tiles in runs of 64 keys */
            const int i = (b + lane) / KT;
            const int j = i < kt1 ? pg_tile(tl, i) * KT + (b + lane) % KT : 0x7FFFFFFF;
            const int64_t at = pg_sees(pos, j, p.a.window, p.a.sinks) ? pg_row_at(&p.c, row, j) : -1;
            float sc = -INFINITY;
            if (at >= 0) {
                float d = 0.0f;
                for (int c = 0; c < HD; c += 8) {
                    float x[8], y[8];
                    pa_get8(kp + at + c, x);
                    pa_get8(q + c, y);
#pragma unroll
                    for (int k = 0; k < 8; k++) d = fmaf(x[k], y[k], d);
                }
                sc = d * p.a.scale;
            }
            float mx = sc;
            for (int o = 1; o < 64; o <<= 1) mx = fmaxf(mx, __shfl_xor(mx, o, QK_WAVE));
            const float mn = fmaxf(m, mx), f = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
            seen |= __any(at >= 0);
            l *= f;
#pragma unroll
            for (int e = 0; e < HD / 16; e++) acc[e] *= f;
            m = mn;
            const float pr = at < 0 ? 0.0f : __builtin_amdgcn_exp2f(sc - (m == -INFINITY ? 0.0f : m));
            l += pr;
            for (uint64_t todo = __ballot(at >= 0); todo; todo &= todo - 1) {
                const int k = __builtin_ctzll(todo);
                const float pj = __shfl(pr, k, QK_WAVE);
                const int64_t aj = ((int64_t)__shfl((int)(at >> 32), k, QK_WAVE) << 32) | (uint32_t)__shfl((int)at, k, QK_WAVE);
                /* dims 4 (lane % 16) .. of every 64, the four quarters of the wave alike */
#pragma unroll
                for (int e = 0; e < HD / 64; e++)
#pragma unroll
                    for (int x = 0; x < 4; x++)
                        acc[4 * e + x] = fmaf(pj, pa_get(vp + aj + 64 * e + 4 * (lane & 15) + x), acc[4 * e + x]);
            }
        }
        for (int o = 1; o < 64; o <<= 1) l += __shfl_xor(l, o, QK_WAVE);
        l = pa_sum(m, l, seen);
        const float f = pa_norm(m, l);
        if (lane < 16) {
#pragma unroll
            for (int e = 0; e < HD / 64; e++) {
                const int d = 64 * e + 4 * lane;
                const float *o = acc + 4 * e;
                if (u.parts > 1)
                    qk_st((float4 *)(p.po + ((int64_t)u.slot * RT + r - u.rtile * RT) * HD + d), make_float4(o[0], o[1], o[2], o[3]));
                else
                    pa_put4((T *)p.a.out + (int64_t)(u.s.start + t) * p.a.o_token + (int64_t)hh * p.a.o_head + d, o[0] * f, o[1] * f,
                            o[2] * f, o[3] * f);
            }
            if (u.parts > 1 && lane == 0) p.pml[(int64_t)u.slot * RT + r - u.rtile * RT] = make_float2(m, l);
        }
    }
}

/* maximum of three, a NaN passed over; without the canonicalising moves that
 * fmaxf of a matrix result brings */
__device__ __forceinline__ float pa_max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

#define PA_GROW 8.0f
/* running maximum and sum of a row over 32 NS more scores (unscaled, masked
 * ones -inf), held by lanes l and l + 32; leaves the weights in st.  m is in
 * log2 units; the scale is positive (a negative one is in q).  The sums so
 * far are rescaled only when a maximum has grown by more than PA_GROW: weights
 * reach 256 then, which costs no accuracy (fp32 sums, bf16 weights are
 * relative), and most rescalings of a long row are saved. */
template <int NS, int NO>
__device__ __forceinline__ void pa_softmax(qm_f32x16 (&st)[NS], float scale, float &m, float &l, qm_f32x16 (&o)[NO]) {
    float mx = -INFINITY;
#pragma unroll
    for (int t = 0; t < NS; t++)
#pragma unroll
        for (int i = 0; i < 16; i += 2) mx = pa_max3(st[t][i], st[t][i + 1], mx);
    mx = fmaxf(mx, __uint_as_float(qk_xor32_u(__float_as_uint(mx)))) * scale;
    if (__any(mx > m + PA_GROW)) {
        const float mn = fmaxf(m, mx), f = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
        l *= f;
#pragma unroll
        for (int d = 0; d < NO; d++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[d][i] *= f;
        m = mn;
    }
    const float ms = m == -INFINITY ? 0.0f : m; /* no finite score yet */
#pragma unroll
    for (int t = 0; t < NS; t++)
#pragma unroll
        for (int i = 0; i < 16; i++) st[t][i] = __builtin_amdgcn_exp2f(fmaf(st[t][i], scale, -ms));
}

/* Eight weights of a row as a B operand, rounded to bf16: half a step, 2^-8 of
 * each, 0.0015 of the result beside the 0.0017 of its own rounding (relative
 * L2 on normal inputs, 0.0022 together).  A second part, as k_pa_few's, takes
 * that away, but doubles the products with v, which bound a prompt: of 8192
 * 305 and 408 us, of 1000 26 and 30.  l takes the sum of the rounded weights,
 * so that they add up to one again. */
__device__ __forceinline__ qm_bf16x8 pa_pack(const qm_f32x16 &st, int s, float &l) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        w[i] = qk_cvt_pk_bf16(st[8 * s + 2 * i], st[8 * s + 2 * i + 1]);
        l = qk_dot2(w[i], QK_BF16_ONES, l);
    }
    return __builtin_bit_cast(qm_bf16x8, make_uint4(w[0], w[1], w[2], w[3]));
}

/* Where piece pc (16 bytes) of row rr of a tile lies in LDS: the pieces of a
 * row are exchanged by an xor, so that the 16 rows of K that a quarter of a
 * wave reads at once lie on all 64 banks (rows of 128 and 384 bytes start on
 * alternating halves of them), and for V the 4 pieces of each of 4 rows. */
template <int CR>
__device__ __forceinline__ int pa_kswz(int rr) { return CR % 16 == 0 ? rr & 15 : (rr >> 1) & 7; }
template <int CR>
__device__ __forceinline__ int pa_vswz(int rr) { return CR % 16 == 0 ? (rr & 3) << 2 : ((rr >> 1) & 1) << 2; }

/* A row that some query of the unit does not see may hold an infinity or NaN,
 * and weight 0 times that is NaN: such a unit is computed again one row at a
 * time.  It shows in the sums themselves, so the loops need no test: O or the
 * sum of weights is not finite (also where that is the right result), or the
 * sum of a row that sees something is next to nothing.  That is 0 where every
 * score seen was -inf.  Else the largest weight is 2^d, since the weights are
 * exp2 of a product that is not rounded before m is subtracted while m is one
 * that was: |d| is half a step of m, below 1 up to m = 2^24, but -128 at 2^31,
 * where all weights vanish.  From 2^-64 on, what is lost below fp32's range is
 * less than 2^-60 of the sum. */
#define PA_LEAST 0x1p-64f
template <int N, int W, typename V>
__device__ __forceinline__ bool pa_again(const V (&o)[N], float l, bool seen) {
    float x = l == l ? fabsf(l) : INFINITY;
#pragma unroll
    for (int d = 0; d < N; d++)
#pragma unroll
        for (int i = 0; i < W; i++) x = fmaxf(x, o[d][i] == o[d][i] ? fabsf(o[d][i]) : INFINITY);
    return !(x < INFINITY) || (seen && l < PA_LEAST);
}

/* ------------------------------------------------------------ few rows
 * Decode and short calls: a unit is 16 NC rows (a group's heads of one to a
 * few tokens) and a part of the keys; its four waves take the part's tiles of
 * 32 keys in turn and join through LDS at the end.  K and V go straight from
 * the pages to registers in operand order, so the main loop has no barrier and
 * the loads of 8 to 20 waves per CU are in flight; of four where the registers
 * hold one workgroup only (pd_occ 1: f32 past head dim 128, 32 rows of f32 at
 * 128 and of bf16 at 192).  16-wide instructions: lane = (row or key c = lane %
 * 16, quarter g = lane / 16); the scores of a tile leave lane (c, g) the keys 16
 * n + 4 g + b of row c.  K: lane c = key, a quarter has every fourth piece of 16
 * bytes.  V: a lane takes HD / 16 dims of the eight keys its quarter of P^T has;
 * bf16 pairs are turned in registers (two keys' words, one byte permute), and
 * O^T's row x of tile e is dim (HD / 16) x + e.  The weights of bf16 calls are
 * taken in two bf16 parts (16 bits), which leaves the output's rounding alone;
 * the pages' loads hide the second product (64 tokens 172 us with one part, 173
 * with two).  f32 runs on the fp32 matrix instructions, whose operands are single
 * elements.
 * Bound: HBM, the visible pages read once: single tokens of 64 sequences of 64
 * to 65536 rows (841 MB of bf16) 177 us with the join's 10, 4.75 TB/s; of 1024
 * sequences of 1000 rows 204 us, 5.2 TB/s, in f32 405; a kernel that only reads
 * reaches 5.9.  Short calls: latency, f32 under a window of 1024 of 32
 * sequences (68 MB) 25 us, a token on 333 rows 10, a prompt of 64 8. */
#define PD_KT 32
typedef float pa_f32x4 __attribute__((ext_vector_type(4)));

template <typename T, int HD, int NC>
constexpr int pd_occ() { return NC * HD * (int)sizeof(T) <= 512 ? 2 : 1; }

template <typename T, int HD, int NC>
__global__ __launch_bounds__(256, (pd_occ<T, HD, NC>())) void k_pa_few(PaArgs p) {
    constexpr int RT = 16 * NC;
    constexpr int E = HD / 16;  /* dims per lane of V = tiles of O */
    constexpr bool B16 = sizeof(T) == 2;
    constexpr int PE = 16 / (int)sizeof(T);   /* elements of a 16-byte piece */
    constexpr int QN = HD / (4 * PE);         /* pieces of a quarter of a row */
    constexpr int LD = HD + 4;  /* floats per row in LDS: 16-byte pieces of 8 rows on different banks */
    constexpr int VW = E * (int)sizeof(T) / 4; /* words of a lane's dims of one key */
    __shared__ __attribute__((aligned(16))) float sum[RT * LD];
    __shared__ float2 ml[4][RT];
    __shared__ __attribute__((aligned(16))) int64_t where[4][32];
    PaUnit u;
    if (!pa_find<RT, PD_KT, false>(p, blockIdx.x, u)) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = lane & 15, g = lane >> 4;
    const int row0 = u.rtile * RT, nrow = min(RT, u.s.count * p.G - row0);
    const int first = u.s.len - u.s.count;
    const int p0 = first + row0 / p.G, p1 = first + (row0 + nrow - 1) / p.G;
    const pg_tiles tl = pg_tiles_of(p0, p1, p.a.window, p.a.sinks, PD_KT);
    const int kt0 = pg_part(tl.nt, u.part, u.parts), kt1 = pg_part(tl.nt, u.part + 1, u.parts);
    const T *kp = (const T *)p.c.k + (int64_t)u.kh * p.c.head_stride, *vp = (const T *)p.c.v + (int64_t)u.kh * p.c.head_stride;
    const int32_t *row = p.c.table + (int64_t)u.s.slot * p.c.table_stride;

    auto find = [&](int i) { /* key lane % 32 of tile i: row offset or -1 */
        const int j = i < kt1 ? pg_tile(tl, i) * PD_KT + (lane & 31) : -1;
        return j <= p1 ? pg_row_at(&p.c, row, j) : -1;
    };
    int64_t next = find(kt0 + wave);
    /* a negative scale is turned into the sign of q */
    const float scale = fabsf(p.a.scale);
    const uint32_t flip = p.a.scale < 0.0f ? (B16 ? 0x80008000u : 0x80000000u) : 0u;
    uint4 q[NC][QN];
    int pos[NC];
    float m[NC], l[NC];
    bool seen[NC];
    pa_f32x4 o[NC][E];
#pragma unroll
    for (int x = 0; x < NC; x++) {
        const int r = row0 + min(16 * x + c, nrow - 1), t = r / p.G;
        pos[x] = first + t;
        const T *src = (const T *)p.a.q + (int64_t)(u.s.start + t) * p.a.q_token + (int64_t)pa_head(p, u.kh, r - t * p.G) * p.a.q_head + g * PE;
#pragma unroll
        for (int s = 0; s < QN; s++) {
            const uint4 w = qk_ld((const uint4 *)(src + s * 4 * PE));
            q[x][s] = make_uint4(w.x ^ flip, w.y ^ flip, w.z ^ flip, w.w ^ flip);
        }
        m[x] = -INFINITY;
        l[x] = 0.0f;
        seen[x] = false;
#pragma unroll
        for (int e = 0; e < E; e++) o[x][e] = pa_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    for (int i = kt0 + wave; i < kt1; i += 4) {
        const int base = pg_tile(tl, i) * PD_KT;
        const uint32_t valid = (uint32_t)__ballot(next >= 0);
        /* a row without a page reads the pool's first one; its scores are masked, its v zeroed */
        if (lane < 32) where[wave][lane] = next < 0 ? 0 : next;
        __builtin_amdgcn_wave_barrier();
        uint4 kx[2][QN];
#pragma unroll
        for (int n = 0; n < 2; n++) {
            const T *src = kp + where[wave][16 * n + c] + g * PE;
#pragma unroll
            for (int s = 0; s < QN; s++) kx[n][s] = qk_ld((const uint4 *)(src + s * 4 * PE));
        }
        uint32_t vx[8][VW]; /* key 16 (k / 4) + 4 g + k % 4 */
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const uint32_t *src = (const uint32_t *)(vp + where[wave][16 * (k >> 2) + 4 * g + (k & 3)] + c * E);
            if constexpr (VW % 4 == 0) {
#pragma unroll
                for (int x = 0; x < VW; x += 4) {
                    const uint4 w = qk_ld((const uint4 *)(src + x));
                    vx[k][x] = w.x; vx[k][x + 1] = w.y; vx[k][x + 2] = w.z; vx[k][x + 3] = w.w;
                }
            } else {
#pragma unroll
                for (int x = 0; x < VW; x += 2) {
                    const uint2 w = qk_ld((const uint2 *)(src + x));
                    vx[k][x] = w.x; vx[k][x + 1] = w.y;
                }
            }
        }
        next = find(i + 4);

        pa_f32x4 st[NC][2];
#pragma unroll
        for (int x = 0; x < NC; x++)
#pragma unroll
            for (int n = 0; n < 2; n++) {
                pa_f32x4 a = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int s = 0; s < QN; s++) {
                    if constexpr (B16) {
                        a = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(qm_bf16x8, kx[n][s]), __builtin_bit_cast(qm_bf16x8, q[x][s]), a, 0, 0, 0);
                    } else {
                        const float4 kf = __builtin_bit_cast(float4, kx[n][s]), qf = __builtin_bit_cast(float4, q[x][s]);
                        a = __builtin_amdgcn_mfma_f32_16x16x4f32(kf.x, qf.x, a, 0, 0, 0);
                        a = __builtin_amdgcn_mfma_f32_16x16x4f32(kf.y, qf.y, a, 0, 0, 0);
                        a = __builtin_amdgcn_mfma_f32_16x16x4f32(kf.z, qf.z, a, 0, 0, 0);
                        a = __builtin_amdgcn_mfma_f32_16x16x4f32(kf.w, qf.w, a, 0, 0, 0);
                    }
                }
                st[x][n] = a;
            }
        if (valid != 0xFFFFFFFFu || !pa_full(p, p0, p1, base)) {
#pragma unroll
            for (int x = 0; x < NC; x++) {
                uint32_t mw = pa_mask(p, pos[x], base) & valid;
                seen[x] |= mw != 0;
                mw >>= 4 * g;
#pragma unroll
                for (int k = 0; k < 8; k++) st[x][k >> 2][k & 3] = (mw >> (16 * (k >> 2) + (k & 3))) & 1u ? st[x][k >> 2][k & 3] : -INFINITY;
            }
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const bool dead = !((valid >> (16 * (k >> 2) + 4 * g + (k & 3))) & 1u);
#pragma unroll
                for (int x = 0; x < VW; x++) vx[k][x] = dead ? 0u : vx[k][x];
            }
        } else {
#pragma unroll
            for (int x = 0; x < NC; x++) seen[x] = true;
        }
#pragma unroll
        for (int x = 0; x < NC; x++) {
            float mx = pa_max3(st[x][0][0], st[x][0][1], st[x][0][2]);
            mx = pa_max3(st[x][0][3], st[x][1][0], mx);
            mx = pa_max3(st[x][1][1], st[x][1][2], mx);
            mx = fmaxf(mx, st[x][1][3]);
            mx = fmaxf(mx, __uint_as_float(qk_xor16_u(__float_as_uint(mx))));
            mx = fmaxf(mx, __uint_as_float(qk_xor32_u(__float_as_uint(mx)))) * scale;
            if (__any(mx > m[x] + PA_GROW)) { /* as pa_softmax */
                const float mn = fmaxf(m[x], mx), f = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m[x] - mn);
                l[x] *= f;
#pragma unroll
                for (int e = 0; e < E; e++) o[x][e] *= f;
                m[x] = mn;
            }
            const float ms = m[x] == -INFINITY ? 0.0f : m[x];
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const float w = __builtin_amdgcn_exp2f(fmaf(st[x][k >> 2][k & 3], scale, -ms));
                st[x][k >> 2][k & 3] = w;
                l[x] += w;
            }
        }
        if constexpr (B16) {
            qm_bf16x8 pw[NC][2]; /* a weight in two bf16 parts */
#pragma unroll
            for (int x = 0; x < NC; x++) {
                uint32_t w[4], y[4];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const float a = st[x][k >> 1][2 * (k & 1)], b = st[x][k >> 1][2 * (k & 1) + 1];
                    w[k] = qk_cvt_pk_bf16(a, b);
                    y[k] = qk_cvt_pk_bf16(a - qk_bf16_lo(w[k]), b - qk_bf16_hi(w[k]));
                }
                pw[x][0] = __builtin_bit_cast(qm_bf16x8, make_uint4(w[0], w[1], w[2], w[3]));
                pw[x][1] = __builtin_bit_cast(qm_bf16x8, make_uint4(y[0], y[1], y[2], y[3]));
            }
#pragma unroll
            for (int e = 0; e < E; e++) {
                uint32_t w[4];
#pragma unroll
                for (int x = 0; x < 4; x++)
                    w[x] = __builtin_amdgcn_perm(vx[2 * x + 1][e >> 1], vx[2 * x][e >> 1], e & 1 ? 0x07060302u : 0x05040100u);
                const qm_bf16x8 a = __builtin_bit_cast(qm_bf16x8, make_uint4(w[0], w[1], w[2], w[3]));
#pragma unroll
                for (int x = 0; x < NC; x++)
#pragma unroll
                    for (int y = 1; y >= 0; y--) o[x][e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, pw[x][y], o[x][e], 0, 0, 0);
            }
        } else {
#pragma unroll
            for (int k = 0; k < 8; k++)
#pragma unroll
                for (int e = 0; e < E; e++)
#pragma unroll
                    for (int x = 0; x < NC; x++)
                        o[x][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(vx[k][e]), st[x][k >> 2][k & 3], o[x][e], 0, 0, 0);
        }
    }
    bool again = false;
#pragma unroll
    for (int x = 0; x < NC; x++) {
        l[x] += __uint_as_float(qk_xor16_u(__float_as_uint(l[x])));
        l[x] += __uint_as_float(qk_xor32_u(__float_as_uint(l[x])));
        again |= pa_again<E, 4>(o[x], l[x], seen[x]);
        l[x] = pa_sum(m[x], l[x], seen[x]);
        if (g == 0) ml[wave][16 * x + c] = make_float2(m[x], l[x]);
    }
    if (__syncthreads_or(again)) {
        pa_slow<T, HD, RT, PD_KT>(p, u, kt0, kt1, tl, 4);
        return;
    }
    float M[NC], L[NC], f[NC];
#pragma unroll
    for (int x = 0; x < NC; x++) {
        M[x] = -INFINITY;
        L[x] = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; w++) M[x] = fmaxf(M[x], ml[w][16 * x + c].x);
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const float2 y = ml[w][16 * x + c];
            L[x] += y.x == M[x] ? y.y : y.y * __builtin_amdgcn_exp2f(y.x - M[x]);
        }
        f[x] = m[x] == M[x] ? 1.0f : __builtin_amdgcn_exp2f(m[x] - M[x]);
    }
    for (int w = 0; w < 4; w++) { /* in order, so the sum is the same every time */
        if (wave == w)
#pragma unroll
            for (int x = 0; x < NC; x++) {
                if (16 * x + c >= nrow) continue;
                float4 *dst = (float4 *)(sum + (16 * x + c) * LD + 4 * g * E);
#pragma unroll
                for (int k = 0; k < E; k++) { /* dims 4 g E + 4 k ..: element y of tile e at y E + e */
                    float4 y = make_float4(o[x][(4 * k) % E][4 * k / E] * f[x], o[x][(4 * k + 1) % E][(4 * k + 1) / E] * f[x],
                                           o[x][(4 * k + 2) % E][(4 * k + 2) / E] * f[x], o[x][(4 * k + 3) % E][(4 * k + 3) / E] * f[x]);
                    if (w) {
                        const float4 z = dst[k];
                        y = make_float4(z.x + y.x, z.y + y.y, z.z + y.z, z.w + y.w);
                    }
                    dst[k] = y;
                }
            }
        __syncthreads();
    }
    /* rows of the unit, 4 dims per thread */
    if (wave == 0 && g == 0)
#pragma unroll
        for (int x = 0; x < NC; x++) ml[0][16 * x + c] = make_float2(M[x], L[x]);
    __syncthreads();
    for (int i = tid; i < nrow * (HD / 4); i += 256) {
        const int rr = i / (HD / 4), d = 4 * (i - rr * (HD / 4));
        const float4 x = *(const float4 *)(sum + rr * LD + d);
        if (u.parts > 1) {
            qk_st((float4 *)(p.po + ((int64_t)u.slot * RT + rr) * HD + d), x);
        } else {
            const int tt = (row0 + rr) / p.G, oh = pa_head(p, u.kh, row0 + rr - tt * p.G);
            const float n = pa_norm(ml[0][rr].x, ml[0][rr].y);
            pa_put4((T *)p.a.out + (int64_t)(u.s.start + tt) * p.a.o_token + (int64_t)oh * p.a.o_head + d, x.x * n, x.y * n, x.z * n, x.w * n);
        }
    }
    if (u.parts > 1 && tid < nrow) p.pml[(int64_t)u.slot * RT + tid] = ml[0][tid];
}

/* a row of a 32-wide unit, held by lanes l and l + 32: the output, or the
 * part's results */
template <typename T, int HD>
__device__ __forceinline__ void pa_store(const PaArgs &p, const PaUnit &u, const qm_f32x16 (&o)[HD / 32], float m, float l, int rr, int t,
                                         int hh) {
    const int h = (threadIdx.x >> 5) & 1;
    const float f = u.parts > 1 ? 1.0f : pa_norm(m, l);
    T *out = (T *)p.a.out + (int64_t)(u.s.start + t) * p.a.o_token + (int64_t)hh * p.a.o_head + 4 * h;
    float *po = p.po + ((int64_t)u.slot * PM_RT + rr) * HD + 4 * h;
#pragma unroll
    for (int d = 0; d < HD / 32; d++)
#pragma unroll
        for (int g = 0; g < 4; g++) {
            const float4 y = make_float4(o[d][4 * g] * f, o[d][4 * g + 1] * f, o[d][4 * g + 2] * f, o[d][4 * g + 3] * f);
            if (u.parts > 1) qk_st((float4 *)(po + 32 * d + 8 * g), y);
            else pa_put4(out + 32 * d + 8 * g, y.x, y.y, y.z, y.w);
        }
    if (u.parts > 1 && h == 0) p.pml[(int64_t)u.slot * PM_RT + rr] = make_float2(m, l);
}

/* ------------------------------------------------------------ many rows
 * Prompts, bf16: a unit is 128 rows, 32 per wave, and a part of the keys; NG
 * groups of four waves take its tiles in turn and are added at the end
 * (pa_merge).  Tiles of KT keys of K and V are copied straight from the pages
 * to LDS, two buffers, one barrier per step.  The copies' lanes pick the
 * 16-byte pieces, so a tile lies in rows with its pieces exchanged by the
 * row's number (an xor): K's operand reads (a lane per row) and V's transposing
 * reads (a lane per dim, four keys) then meet no bank twice (with the xor made
 * for 32 banks, conflicts were a fifth of the cycles).  Where a tile's rows lie
 * is looked up for 512 keys a group at a time; a row without a page or after
 * the last query is copied from a row of zeros.
 * Bound: a wave's own chain of a step.  A prompt of 8192 (16 heads on 2 of 128)
 * takes 294 to 312 us by the card, 880 to 936 TFLOP/s of 1180 of a large library
 * product.  A step of 5400 clocks was scores 1200, maximum and exponentials
 * 1200, sums of v 1250, issuing the copies 1100 (now between the products) and
 * waiting at the barrier 100 to 970; the matrix cores work 40 % of it.  Without gain: a
 * raised wave priority in either half, two groups half a step apart (360 us),
 * scores of the next tile beside the softmax (337 to 348), three groups (326),
 * units of 64 rows (short prompts 10 % better, long contexts 40 % worse). */
#define PM_CHUNK 1024 /* keys of a look-up of two groups */
typedef short pa_s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) pa_s16x4 *pa_tptr;

/* keys of a tile */
constexpr int pm_kt(int hd, bool f32 = false) { return hd <= 128 && !f32 ? 64 : 32; }

/* the rows' results of the other groups of four waves into the first one's,
 * through `ex` (HD / 8 pieces of 64 float4 per wave) and `ml`, in order; true
 * for the first */
template <int E, int NG>
__device__ __forceinline__ bool pa_merge(qm_f32x16 (&o)[E], float &m, float &l, float4 *ex, float2 *ml) {
    const int tid = threadIdx.x & 255, group = threadIdx.x >> 8;
    float4 *x = ex + (tid >> 6) * (E * 4 * 64) + (tid & 63);
    for (int k = 1; k < NG; k++) {
        if (group == k) {
#pragma unroll
            for (int d = 0; d < E; d++)
#pragma unroll
                for (int g = 0; g < 4; g++) x[(4 * d + g) * 64] = make_float4(o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]);
            ml[tid] = make_float2(m, l);
        }
        __syncthreads();
        if (group == 0) {
            const float2 y = ml[tid];
            const float M = fmaxf(m, y.x);
            const float f0 = m == M ? 1.0f : __builtin_amdgcn_exp2f(m - M), f1 = y.x == M ? 1.0f : __builtin_amdgcn_exp2f(y.x - M);
            l = l * f0 + y.y * f1;
            m = M;
#pragma unroll
            for (int d = 0; d < E; d++)
#pragma unroll
                for (int g = 0; g < 4; g++) {
                    const float4 z = x[(4 * d + g) * 64];
                    o[d][4 * g] = o[d][4 * g] * f0 + z.x * f1;
                    o[d][4 * g + 1] = o[d][4 * g + 1] * f0 + z.y * f1;
                    o[d][4 * g + 2] = o[d][4 * g + 2] * f0 + z.z * f1;
                    o[d][4 * g + 3] = o[d][4 * g + 3] * f0 + z.w * f1;
                }
        }
        if (k + 1 < NG) __syncthreads();
    }
    return group == 0;
}

template <int HD, int NG>
__global__ __launch_bounds__(256 * NG, 2 / NG) void k_pa_many(PaArgs p) {
    typedef uint16_t T;
    constexpr int KT = pm_kt(HD), CR = HD / 8, NB = KT * CR / 256, NS = KT / 32, E = HD / 32, KS = HD / 16;
    constexpr int KEYS = PM_CHUNK / 2 * NG, CH = KEYS / KT / NG; /* steps per look-up */
    __shared__ __attribute__((aligned(16))) uint4 kv[2][NG][2][KT * CR]; /* buffer, group's tile, k / v */
    __shared__ __attribute__((aligned(16))) ulonglong2 where[KEYS]; /* addresses of a key's k and v */
    PaUnit u;
    if (!pa_find<PM_RT, KT, false>(p, blockIdx.x, u)) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane((tid >> 6) & 3), c = lane & 31, h = lane >> 5;
    const int group = __builtin_amdgcn_readfirstlane(tid / 256);
    const int row0 = u.rtile * PM_RT, rows = u.s.count * p.G, nrow = min(PM_RT, rows - row0);
    const int first = u.s.len - u.s.count;
    const int p0 = first + row0 / p.G, p1 = first + (row0 + nrow - 1) / p.G;
    const pg_tiles tl = pg_tiles_of(p0, p1, p.a.window, p.a.sinks, KT);
    const int kt0 = pg_part(tl.nt, u.part, u.parts), kt1 = pg_part(tl.nt, u.part + 1, u.parts), nt = kt1 - kt0;
    /* this wave's rows; a wave past the last row copies and waits only */
    const int w0 = row0 + 32 * wave, wn = min(32, rows - w0);
    const int pw0 = first + w0 / p.G, pw1 = first + (w0 + wn - 1) / p.G;
    const int r = min(w0 + c, rows - 1), t = r / p.G, pos = first + t;
    const int hh = pa_head(p, u.kh, r - t * p.G);
    const T *kp = (const T *)p.c.k + (int64_t)u.kh * p.c.head_stride, *vp = (const T *)p.c.v + (int64_t)u.kh * p.c.head_stride;
    const int32_t *row = p.c.table + (int64_t)u.s.slot * p.c.table_stride;

    const uint64_t zero = (uint64_t)pa_zero;
    /* Addresses of the tiles i0.. of the part, zeros past its last: the steps
     * copy the next step's tiles without asking whether there is one. */
    auto look = [&](int i0) {
        for (int k = tid; k < KEYS; k += 256 * NG) {
            const int i = i0 + k / KT, j = i < nt ? pg_tile(tl, kt0 + i) * KT + k % KT : -1;
            const int64_t at = j <= p1 ? pg_row_at(&p.c, row, j) : -1;
            ulonglong2 w;
            w.x = at < 0 ? zero : (uint64_t)(kp + at);
            w.y = at < 0 ? zero : (uint64_t)(vp + at);
            where[k] = w;
        }
        __syncthreads();
    };
    /* this wave's place in its tile's K; V and the other buffer lie behind */
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(qm_lptr)&kv[0][group][0][0] + 1024 * wave);
    uint64_t vnext = 0;
    auto rows_of = [&](int i) { return where + (NG * (i % CH) + group) * KT; };
    /* this thread's piece x of the group's tile NG i + group, from the row's addresses w */
    auto piece = [&](int i, int x, ulonglong2 w) {
        const int L = x * 256 + wave * 64 + lane, rr = L / CR, pc = L - rr * CR;
        const uint32_t dst = lds0 + (i & 1) * (NG * 2 * KT * CR * 16) + 4096 * x;
        qm_copy<0>((const uint4 *)(w.x + 16 * (pc ^ pa_kswz<CR>(rr))), dst);
        qm_copy<0>((const uint4 *)(w.y + 16 * (pc ^ pa_vswz<CR>(rr))), dst + KT * CR * 16);
    };
    auto row_of = [&](int i, int x) { return rows_of(i)[(x * 256 + wave * 64 + lane) / CR]; };
    auto copy = [&](int i) {
#pragma unroll
        for (int x = 0; x < NB; x++) piece(i, x, row_of(i, x));
    };
    auto pages = [&](int i) { return __ballot(rows_of(i)[lane & (KT - 1)].x != zero); };
    if (nt > 0) {
        look(0);
        copy(0);
        vnext = pages(0);
    }
    const float scale = fabsf(p.a.scale);
    uint4 q[KS];
    {
        const uint32_t flip = p.a.scale < 0.0f ? 0x80008000u : 0u;
        const T *src = (const T *)p.a.q + (int64_t)(u.s.start + t) * p.a.q_token + (int64_t)hh * p.a.q_head + h * 8;
#pragma unroll
        for (int s = 0; s < KS; s++) {
            const uint4 w = qk_ld((const uint4 *)(src + s * 16));
            q[s] = make_uint4(w.x ^ flip, w.y ^ flip, w.z ^ flip, w.w ^ flip);
        }
    }
    float m = -INFINITY, l = 0.0f;
    bool seen = false;
    qm_f32x16 o[E];
#pragma unroll
    for (int d = 0; d < E; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[d][i] = 0.0f;
    /* V: lane j of 16 reads 4 dims of key j / 4 and receives 4 keys of dim j */
    const int j = lane & 15, g16 = (lane >> 4) & 1, fv = pa_vswz<CR>(j >> 2);

    for (int i = 0; i < (nt + NG - 1) / NG; i++) {
        qm_sync<0>(); /* the step's tiles are in LDS; every wave is done with the last step's */
        const uint64_t valid = vnext;
        if (NG * (i + 1) < nt && (i + 1) % CH == 0) look(NG * (i + 1));
        vnext = pages(i + 1);
        const int base = pg_tile(tl, kt0 + NG * i + group) * KT;
        const uint4 *kb = kv[i & 1][group][0], *vb = kv[i & 1][group][1];
        qm_f32x16 st[NS];
        /* The next step's copies go out between the products: all at the start,
         * they filled the address unit and held every wave for a fifth of the
         * step (prompt of 8192: 324 us, so 319).  Past head dim 128 the
         * registers that this takes cost more than it gives (183 and 207 us
         * for a prompt of 8000 at 256). */
        constexpr bool SPREAD = KS <= 8;
        constexpr int PG = NB / (NS * KS / 4); /* pieces per four products */
        if constexpr (!SPREAD) copy(i + 1);
#pragma unroll
        for (int n = 0; n < NS; n++) {
#pragma unroll
            for (int x = 0; x < 16; x++) st[n][x] = 0.0f;
#pragma unroll
            for (int s0 = 0; s0 < KS; s0 += 4) {
                if constexpr (SPREAD) {
#pragma unroll
                    for (int x = (n * KS + s0) / 4 * PG; x < ((n * KS + s0) / 4 + 1) * PG; x++) piece(i + 1, x, row_of(i + 1, x));
                }
#pragma unroll
                for (int s = s0; s < s0 + 4; s++)
                    st[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                        __builtin_bit_cast(qm_bf16x8, kb[(32 * n + c) * CR + ((2 * s + h) ^ pa_kswz<CR>(c))]),
                        __builtin_bit_cast(qm_bf16x8, q[s]), st[n], 0, 0, 0);
            }
        }
        /* a wave that sees nothing of the tile has formed scores in vain */
        if (wn <= 0 || NG * i + group >= nt || base > pw1 || (p.a.window > 0 && base + KT <= pg_lo(pw0, p.a.window) && base >= p.a.sinks)) continue;
#pragma unroll
        for (int n = 0; n < NS; n++) {
            const uint32_t v32 = (uint32_t)(valid >> (32 * n));
            if (v32 == 0xFFFFFFFFu && pa_full(p, pw0, pw1, base + 32 * n)) {
                seen = true;
                continue;
            }
            uint32_t mw = pa_mask(p, pos, base + 32 * n) & v32;
            seen |= mw != 0;
            mw >>= 4 * h;
#pragma unroll
            for (int x = 0; x < 16; x++) st[n][x] = (mw >> (8 * (x >> 2) + (x & 3))) & 1u ? st[n][x] : -INFINITY;
        }
        pa_softmax(st, scale, m, l, o);
#pragma unroll
        for (int n = 0; n < NS; n++)
#pragma unroll
            for (int s = 0; s < 2; s++) {
                const qm_bf16x8 pw = pa_pack(st[n], s, l);
                const int key = 32 * n + 16 * s + 4 * h + (j >> 2);
#pragma unroll
                for (int d = 0; d < E; d++) {
                    const int pc = (4 * d + 2 * g16 + ((j & 3) >> 1)) ^ fv;
                    const pa_s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((pa_tptr)((const short *)(vb + key * CR + pc) + 4 * (j & 1)));
                    const pa_s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((pa_tptr)((const short *)(vb + (key + 8) * CR + pc) + 4 * (j & 1)));
                    const uint2 aw = __builtin_bit_cast(uint2, a), bw = __builtin_bit_cast(uint2, b);
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(qm_bf16x8, make_uint4(aw.x, aw.y, bw.x, bw.y)), pw, o[d], 0, 0, 0);
                }
            }
    }
    qm_sync<0>(); /* the last step's copies, of a step that there is not, are done */
    l += __uint_as_float(qk_xor32_u(__float_as_uint(l)));
    if (__syncthreads_or(wn > 0 && pa_again<E, 16>(o, l, seen))) {
        pa_slow<T, HD, PM_RT, KT>(p, u, kt0, kt1, tl, 4 * NG);
        return;
    }
    if constexpr (NG > 1)
        if (!pa_merge<E, NG>(o, m, l, (float4 *)kv, (float2 *)where)) return;
    if (c < wn) pa_store<T, HD>(p, u, o, m, l, 32 * wave + c, t, hh);
}

/* ------------------------------------------------------------ many rows, f32
 * The same unit at fp32 precision: K, V, Q and the weights as three bf16
 * parts each (hi + mid + lo, 24 bits) and six of the nine partial products
 * (the others are below 2^-24 of them), whose peak is 417 TFLOP/s against 157
 * of the fp32 instructions.  A tile is 32 keys; its rows come through
 * registers, where a group of four waves splits them once, into one LDS buffer
 * for K and one for V: V is written while the scores are formed, the next
 * tile's K while V is multiplied, one barrier after each.  Infinities, NaN and
 * values that round to a bf16 infinity have no parts: their differences are
 * NaN, and the unit is computed again (pa_again).
 * Bound: matrix cores, six products per tile, and the splitting beside them:
 * three prompt chunks and 29 single tokens on up to 6000 rows (25 GFLOP) 203
 * us with the join, 125 TFLOP/s against 154 of a large library product in fp32;
 * fp32 instructions took 631 us. */

/* eight fp32 -> three bf16 parts */
__device__ __forceinline__ void pa_split8(const float x[8], uint4 w[3]) {
    float r[8];
#pragma unroll
    for (int j = 0; j < 8; j++) r[j] = x[j];
#pragma unroll
    for (int i = 0; i < 3; i++) {
        uint32_t v[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            v[j] = qk_cvt_pk_bf16(r[2 * j], r[2 * j + 1]);
            r[2 * j] -= qk_bf16_lo(v[j]);
            r[2 * j + 1] -= qk_bf16_hi(v[j]);
        }
        w[i] = make_uint4(v[0], v[1], v[2], v[3]);
    }
}
/* four fp32 -> three bf16 parts */
__device__ __forceinline__ void pa_split4(float4 x, uint2 w[3]) {
#pragma unroll
    for (int i = 0; i < 3; i++) {
        w[i] = make_uint2(qk_cvt_pk_bf16(x.x, x.y), qk_cvt_pk_bf16(x.z, x.w));
        x = make_float4(x.x - qk_bf16_lo(w[i].x), x.y - qk_bf16_hi(w[i].x), x.z - qk_bf16_lo(w[i].y), x.w - qk_bf16_hi(w[i].y));
    }
}
/* sum of a * b over the parts, the smallest products first */
__device__ __forceinline__ qm_f32x16 pa_mfma6(const uint4 a[3], const uint4 b[3], qm_f32x16 c) {
    constexpr int ia[6] = {2, 1, 0, 1, 0, 0}, ib[6] = {0, 1, 2, 0, 1, 0};
#pragma unroll
    for (int i = 0; i < 6; i++)
        c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(qm_bf16x8, a[ia[i]]), __builtin_bit_cast(qm_bf16x8, b[ib[i]]), c, 0, 0, 0);
    return c;
}

/* head dims past 128: four waves, whose registers and LDS are full */
constexpr int pm_halves32(int hd) { return hd <= 128 ? 2 : 1; }

template <int HD>
__global__ __launch_bounds__(256 * pm_halves32(HD), 1) void k_pa_many32(PaArgs p) {
    typedef float T;
    constexpr int KT = 32, CR = HD / 8, NB = KT * HD / 1024, E = HD / 32, KS = HD / 16, NG = pm_halves32(HD);
    constexpr int CH = PM_CHUNK / KT / NG; /* steps per look-up */
    __shared__ __attribute__((aligned(16))) uint4 kv[NG][2][3][KT * CR]; /* even / odd tile, k / v, part */
    __shared__ __attribute__((aligned(16))) ulonglong2 where[PM_CHUNK]; /* addresses of a key's k and v */
    PaUnit u;
    if (!pa_find<PM_RT, KT, false>(p, blockIdx.x, u)) return;
    const int tid = threadIdx.x & 255, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 31, h = lane >> 5;
    const int odd = NG == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
    const int row0 = u.rtile * PM_RT, rows = u.s.count * p.G, nrow = min(PM_RT, rows - row0);
    const int first = u.s.len - u.s.count;
    const int p0 = first + row0 / p.G, p1 = first + (row0 + nrow - 1) / p.G;
    const pg_tiles tl = pg_tiles_of(p0, p1, p.a.window, p.a.sinks, KT);
    const int kt0 = pg_part(tl.nt, u.part, u.parts), kt1 = pg_part(tl.nt, u.part + 1, u.parts), nt = kt1 - kt0;
    /* this wave's rows; a wave past the last row loads and waits only */
    const int w0 = row0 + 32 * wave, wn = min(32, rows - w0);
    const int pw0 = first + w0 / p.G, pw1 = first + (w0 + wn - 1) / p.G;
    const int r = min(w0 + c, rows - 1), t = r / p.G, pos = first + t;
    const int hh = pa_head(p, u.kh, r - t * p.G);
    const T *kp = (const T *)p.c.k + (int64_t)u.kh * p.c.head_stride, *vp = (const T *)p.c.v + (int64_t)u.kh * p.c.head_stride;
    const int32_t *row = p.c.table + (int64_t)u.s.slot * p.c.table_stride;
    const uint64_t zero = (uint64_t)pa_zero;
    auto look = [&](int i0) { /* as k_pa_many's */
        for (int k = threadIdx.x; k < PM_CHUNK; k += 256 * NG) {
            const int i = i0 + k / KT, j = i < nt ? pg_tile(tl, kt0 + i) * KT + k % KT : -1;
            const int64_t at = j <= p1 ? pg_row_at(&p.c, row, j) : -1;
            ulonglong2 w;
            w.x = at < 0 ? zero : (uint64_t)(kp + at);
            w.y = at < 0 ? zero : (uint64_t)(vp + at);
            where[k] = w;
        }
        __syncthreads();
    };
    float4 kx[NB], vx[NB]; /* this thread's pieces of four of the next step's tile */
    auto rows_of = [&](int i) { return where + (NG * (i % CH) + odd) * KT; };
    auto load_k = [&](int i, int x) {
        const int L = x * 256 + tid, rr = L / (HD / 4);
        kx[x] = qk_ld((const float4 *)rows_of(i)[rr].x + (L - rr * (HD / 4)));
    };
    auto load_v = [&](int i, int x) {
        const int L = x * 256 + tid, rr = L / (HD / 4);
        vx[x] = qk_ld((const float4 *)rows_of(i)[rr].y + (L - rr * (HD / 4)));
    };
    auto pages = [&](int i) { return (uint32_t)__ballot(rows_of(i)[lane & 31].x != zero); };
    auto put = [&](int which, const float4 (&src)[NB]) {
#pragma unroll
        for (int x = 0; x < NB; x++) {
            const int L = x * 256 + tid, rr = L / (HD / 4), q4 = L - rr * (HD / 4), pc = q4 >> 1;
            const int at = 2 * (rr * CR + (pc ^ (which ? pa_vswz<CR>(rr) : pa_kswz<CR>(rr)))) + (q4 & 1);
            uint2 w[3];
            pa_split4(src[x], w);
#pragma unroll
            for (int y = 0; y < 3; y++) ((uint2 *)kv[odd][which][y])[at] = w[y];
        }
    };
    uint32_t vnext = 0;
    if (nt > 0) {
        look(0);
#pragma unroll
        for (int x = 0; x < NB; x++) {
            load_k(0, x);
            load_v(0, x);
        }
        vnext = pages(0);
    }
    const float scale = fabsf(p.a.scale), sign = p.a.scale < 0.0f ? -1.0f : 1.0f;
    uint4 q[KS][3];
    {
        const T *src = (const T *)p.a.q + (int64_t)(u.s.start + t) * p.a.q_token + (int64_t)hh * p.a.q_head + h * 8;
#pragma unroll
        for (int s = 0; s < KS; s++) {
            float x[8];
            pa_get8(src + s * 16, x);
#pragma unroll
            for (int y = 0; y < 8; y++) x[y] *= sign;
            pa_split8(x, q[s]);
        }
    }
    float m = -INFINITY, l = 0.0f;
    bool seen = false;
    qm_f32x16 o[E];
#pragma unroll
    for (int d = 0; d < E; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[d][i] = 0.0f;
    const int j = lane & 15, g16 = (lane >> 4) & 1, fv = pa_vswz<CR>(j >> 2);
    if (nt > 0) put(0, kx);
    qk_lds_barrier();
    for (int i = 0; i < (nt + NG - 1) / NG; i++) {
        const uint32_t valid = vnext;
        /* K of the step is in LDS, and every wave is done with V of the last */
        put(1, vx);
        if (NG * (i + 1) < nt && (i + 1) % CH == 0) look(NG * (i + 1));
        vnext = pages(i + 1);
        const int base = pg_tile(tl, kt0 + NG * i + odd) * KT;
        const bool act = NG * i + odd < nt && wn > 0 && base <= pw1 &&
                         !(p.a.window > 0 && base + KT <= pg_lo(pw0, p.a.window) && base >= p.a.sinks);
        qm_f32x16 st[1];
        const uint4 *kb = kv[odd][0][0];
#pragma unroll
        for (int x = 0; x < 16; x++) st[0][x] = 0.0f;
        /* The next step's loads go out between the products, K's here and V's
         * beside those of the weights (KS = 2 NB of each): all before them, they
         * held every wave for a quarter of the step. */
#pragma unroll
        for (int s = 0; s < KS; s++) {
            if (!(s & 1)) load_k(i + 1, s >> 1);
            uint4 a[3];
#pragma unroll
            for (int y = 0; y < 3; y++) a[y] = kb[y * KT * CR + c * CR + ((2 * s + h) ^ pa_kswz<CR>(c))];
            st[0] = pa_mfma6(a, q[s], st[0]);
            __builtin_amdgcn_sched_barrier(0);
        }
        if (act) {
            if (valid == 0xFFFFFFFFu && pa_full(p, pw0, pw1, base)) {
                seen = true;
            } else {
                uint32_t mw = pa_mask(p, pos, base) & valid;
                seen |= mw != 0;
                mw >>= 4 * h;
#pragma unroll
                for (int x = 0; x < 16; x++) st[0][x] = (mw >> (8 * (x >> 2) + (x & 3))) & 1u ? st[0][x] : -INFINITY;
            }
            pa_softmax(st, scale, m, l, o);
#pragma unroll
            for (int x = 0; x < 16; x++) l += st[0][x];
        }
        qk_lds_barrier(); /* V is in LDS, and every wave has its scores */
        put(0, kx);
        if (act) {
            const uint4 *vb = kv[odd][1][0];
#pragma unroll
            for (int s = 0; s < 2; s++) {
                const float x[8] = {st[0][8 * s], st[0][8 * s + 1], st[0][8 * s + 2], st[0][8 * s + 3],
                                    st[0][8 * s + 4], st[0][8 * s + 5], st[0][8 * s + 6], st[0][8 * s + 7]};
                uint4 pw[3];
                pa_split8(x, pw);
                const int key = 16 * s + 4 * h + (j >> 2);
#pragma unroll
                for (int d = 0; d < E; d++) {
                    const int pc = (4 * d + 2 * g16 + ((j & 3) >> 1)) ^ fv;
                    uint4 a[3];
#pragma unroll
                    for (int y = 0; y < 3; y++) {
                        const pa_s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((pa_tptr)((const short *)(vb + y * KT * CR + key * CR + pc) + 4 * (j & 1)));
                        const pa_s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((pa_tptr)((const short *)(vb + y * KT * CR + (key + 8) * CR + pc) + 4 * (j & 1)));
                        const uint2 aw = __builtin_bit_cast(uint2, lo), bw = __builtin_bit_cast(uint2, hi);
                        a[y] = make_uint4(aw.x, aw.y, bw.x, bw.y);
                    }
                    if (!(d & 1)) load_v(i + 1, s * (E / 2) + (d >> 1));
                    o[d] = pa_mfma6(a, pw, o[d]);
                    if (d & 1) __builtin_amdgcn_sched_barrier(0);
                }
            }
        } else {
#pragma unroll
            for (int x = 0; x < NB; x++) load_v(i + 1, x);
        }
        qk_lds_barrier();
    }
    l += __uint_as_float(qk_xor32_u(__float_as_uint(l)));
    if (__syncthreads_or(wn > 0 && pa_again<E, 16>(o, l, seen))) {
        pa_slow<T, HD, PM_RT, KT>(p, u, kt0, kt1, tl, 4 * NG);
        return;
    }
    if constexpr (NG == 2)
        if (!pa_merge<E, NG>(o, m, l, (float4 *)kv, (float2 *)where)) return;
    if (c < wn) pa_store<T, HD>(p, u, o, m, l, 32 * wave + c, t, hh);
}

/* ------------------------------------------------------------ join
 * Rows of a task whose keys were cut into parts: lane = dims, up to PJ_FEW
 * parts a wave per row, more all W waves on one row, the parts in turn,
 * then a sum in wave order.  Bound: the parts read once, and for few rows the
 * latency of the loads: 5 us where little is cut, 10 us after 64 sequences of up
 * to 65536 rows.  The launch is made wherever the tables are long enough for
 * parts, since only the device knows the lengths. */
#define PJ_FEW 16
template <typename T, int HD>
__device__ __forceinline__ void pa_join_out(const PaArgs &p, const PaUnit &u, int r, int d, float4 y, float f) {
    const int t = r / p.G, hh = pa_head(p, u.kh, r - t * p.G);
    pa_put4((T *)p.a.out + (int64_t)(u.s.start + t) * p.a.o_token + (int64_t)hh * p.a.o_head + d, y.x * f, y.y * f, y.z * f, y.w * f);
}

template <typename T, int HD, int RT, int KT, int W>
__global__ __launch_bounds__(64 * W) void k_pa_join(PaArgs p) {
    constexpr int Q = HD / 4; /* lanes of 4 dims */
    __shared__ __attribute__((aligned(16))) float acc[W][HD];
    __shared__ float lsum[W];
    PaUnit u;
    if (!pa_find<RT, KT, true>(p, blockIdx.x, u)) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const bool few = u.parts <= PJ_FEW;
    const int step = few ? 1 : W, i0 = few ? 0 : wave;
    for (int rr = few ? blockIdx.y * W + wave : blockIdx.y; rr < min(RT, u.s.count * p.G - u.rtile * RT); rr += gridDim.y * (few ? W : 1)) {
        auto at = [&](int i) { return (int64_t)(u.slot + i * p.c.kvh) * RT + rr; };
        float M = -INFINITY;
        for (int i = lane; i < u.parts; i += 64) M = fmaxf(M, qk_ld((const float *)(p.pml + at(i))));
        for (int o = 1; o < 64; o <<= 1) M = fmaxf(M, __shfl_xor(M, o, QK_WAVE));
        float L = 0.0f;
        float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
        for (int i = i0; i < u.parts; i += step) {
            const float pm = qk_ld((const float *)(p.pml + at(i))), pl = qk_ld((const float *)(p.pml + at(i)) + 1);
            const float4 x = qk_ld((const float4 *)(p.po + at(i) * HD + 4 * (lane % Q)));
            const float f = pm == M ? 1.0f : __builtin_amdgcn_exp2f(pm - M);
            L = fmaf(pl, f, L);
            y = make_float4(fmaf(x.x, f, y.x), fmaf(x.y, f, y.y), fmaf(x.z, f, y.z), fmaf(x.w, f, y.w));
        }
        if (few) {
            if (lane < Q) pa_join_out<T, HD>(p, u, u.rtile * RT + rr, 4 * lane, y, pa_norm(M, L));
            continue;
        }
        if (lane < Q) *(float4 *)(acc[wave] + 4 * lane) = y;
        if (lane == 0) lsum[wave] = L;
        __syncthreads();
        if (tid < Q) {
            y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            L = 0.0f;
#pragma unroll
            for (int w = 0; w < W; w++) {
                const float4 z = *(const float4 *)(acc[w] + 4 * tid);
                y = make_float4(y.x + z.x, y.y + z.y, y.z + z.z, y.w + z.w);
                L += lsum[w];
            }
            pa_join_out<T, HD>(p, u, u.rtile * RT + rr, 4 * tid, y, pa_norm(M, L));
        }
        __syncthreads();
    }
}

/* ------------------------------------------------------------ host side */

/* how a call is cut: units asked for, the grid that holds them whatever the
 * lengths, tasks that can need a join, and the slots of partial results */
struct PaPlan {
    int units, extra, one;
    int64_t grid, join, slots;
};

static PaPlan pa_plan(const pg_cache *c, int n, int n_seqs, int h, int rt, int kt, int units, int extra, int one) {
    PaPlan q;
    const int G = h / c->kvh;
    q.units = units;
    q.extra = extra;
    q.one = one;
    /* sum of ceil(rows / rt) over the sequences that have rows */
    const int64_t rows = (int64_t)n * G, seqs = n_seqs < n ? n_seqs : n;
    const int64_t per_head = rows / rt + seqs < rows ? rows / rt + seqs : rows;
    const int64_t tasks = per_head * c->kvh;
    /* parts of the longest task, then the bounds that pg_share gives */
    const int longest = c->cap / kt + 2;
    const int64_t parts = pg_cuts(longest, extra) ? pg_parts(longest, one + 1) : 1, most = tasks * parts;
    q.grid = most < 2 * (int64_t)units + tasks ? most : 2 * (int64_t)units + tasks;
    q.slots = parts == 1 ? 0 : most < 3 * (int64_t)units ? most : 3 * (int64_t)units;
    q.join = parts == 1 ? 0 : tasks < 3 * (int64_t)units / 2 ? tasks : 3 * (int64_t)units / 2; /* two parts at least */
    return q;
}

/* workgroups that share a task's rows: about 2048 in all, where the tasks are
 * few every row has its own */
static unsigned pa_join_rows(int64_t tasks, int rt) {
    const int64_t r = 2048 / tasks;
    return (unsigned)(r < 1 ? 1 : r > rt ? rt : r);
}

/* Rows of a unit: 16 or 32 of the few-row kernel, or PM_RT of the many-row
 * one.  Units of 16 rows read a page once per 16 rows, but start at once and
 * have a short step: they are better as long as the call is short, measured by
 * their number times the rows of a table (or the window): 32 tokens on 1000
 * rows 27 us with 128 rows and 14.5 with 16, on 4000 rows of 4 sequences 30
 * and 39; f32 31 and 20, 52 and 73.  The limits are where the two meet, over 1
 * to 16 sequences, 1000 to 16000 rows and all head dims; f32 kernels past head
 * dim 128 lack registers for more rows (8 tokens of 16 sequences on 4000 rows
 * at 256: 151 and 71), and units of 32 rows take over at half the limit (4
 * tokens of 16 sequences on 4000 rows 29 and 34).  Up to 8 units are 16 rows
 * each whatever the table holds, which may be much more than the sequences
 * have (8 tokens on 1000 rows 23 and 15, on 16000 22 and 23).  Past the limit,
 * by the rows that a sequence has on average; 32 where the registers hold
 * them. */
static bool pa_two(const pg_cache *c) { return c->dtype == QMOE_BF16 ? c->hd <= 192 : c->hd <= 128; }
static int pa_rows_long(const pg_cache *c, int64_t rows, int n_seqs) {
    if (rows <= (int64_t)16 * n_seqs) return 16;
    return rows > (int64_t)32 * n_seqs ? PM_RT : pa_two(c) ? 32 : 16;
}
static int pa_rows(const pg_cache *c, const pg_attn *a) {
    const int64_t rows = (int64_t)a->n * (a->h / c->kvh), units = rows * c->kvh / 16;
    const int later = pa_rows_long(c, rows, a->n_seqs);
    int64_t keys = c->cap, most = c->dtype == QMOE_BF16 || c->hd == 64 ? 1 << 18 : c->hd < 256 ? 1 << 17 : 1 << 19;
    if (a->window > 0 && (int64_t)a->window + a->sinks < keys) keys = (int64_t)a->window + a->sinks;
    if (later == 32) most /= 2;
    return units <= 8 || units * keys <= most ? 16 : later;
}
/* Groups of four waves in a bf16 unit of the many-row kernel.  Two take the
 * unit's tiles in turn and halve its time; where there are units enough for
 * several rounds, two workgroups of one group per CU do better, since one
 * starts and ends under the other's products (two and one: a prompt of 1000 27
 * and 30 us, of 8192 320 and 308, of 16000 1249 and 1151, three of 4000 300 and
 * 264). */
static int pa_groups(const pg_cache *c, int n, int h) {
    return (int64_t)n * (h / c->kvh) / PM_RT * c->kvh >= 1000 && c->hd <= 128 ? 1 : 2;
}
static PaPlan pa_plan_of(const pg_cache *c, int n, int n_seqs, int h, int rt) {
    /* A join costs about 12 bf16 tiles in time, or 2 f32 ones.  Where all units
     * run at once it costs 3, since the others fill CUs that had nothing to do:
     * 64 tokens on 3000 rows 40 us with 12, so 33, on 4000 rows in 16 sequences
     * 81 and 70; but a prompt of 2000 (256 tasks) 46 with 12 and 59 with 3. */
    if (rt == PM_RT && c->dtype == QMOE_BF16) return pa_plan(c, n, n_seqs, h, PM_RT, pm_kt(c->hd), 256, 12, 3);
    if (rt == PM_RT) return pa_plan(c, n, n_seqs, h, PM_RT, pm_kt(c->hd, true), 256, 2, 2);
    /* tables of up to 16 tiles (512 rows) are not cut: the join's launch costs
     * more than the shorter run of tiles gives */
    const int bytes = c->hd * (c->dtype == QMOE_BF16 ? 2 : 4) * (rt / 16); /* of a row's registers, as pd_occ */
    const int wgs = bytes <= 128 ? 4 : bytes <= 256 ? 3 : bytes <= 512 ? 2 : 1; /* workgroups that a CU holds */
    const int extra = c->cap <= 16 * PD_KT ? 17 : 2;
    return pa_plan(c, n, n_seqs, h, rt, PD_KT, 256 * wgs, extra, extra);
}

static size_t pa_up(size_t v) { return (v + 255) / 256 * 256; }
static size_t pa_ws(const pg_cache *c, int n, int n_seqs, int h, int rt) {
    const PaPlan q = pa_plan_of(c, n, n_seqs, h, rt);
    const size_t index = n_seqs > PA_INDEX ? pa_up((size_t)n_seqs * 16) : 0;
    return 256 + index + pa_up((size_t)q.slots * rt * 8) + pa_up((size_t)q.slots * rt * c->hd * 4);
}
static int pa_threads(const pg_cache *c, int n, int h, int rt) {
    if (rt != PM_RT) return 256;
    return 256 * (c->dtype == QMOE_BF16 ? pa_groups(c, n, h) : pm_halves32(c->hd));
}
/* of either choice of rows: the window is not known here.  0 where a launch
 * would have 2^32 threads or more, which HIP does not take; units of 16 rows
 * that are chosen because the call is short (pa_rows) are below 2^24, and more
 * than the longer ones would be. */
extern "C" size_t qk_pg_attn_ws(const pg_cache *c, int n, int n_seqs, int h) {
    const int rt = pa_rows_long(c, (int64_t)n * (h / c->kvh), n_seqs);
    if (pa_plan_of(c, n, n_seqs, h, rt).grid * pa_threads(c, n, h, rt) > 0xFFFFFFFFll) return 0;
    const size_t a = pa_ws(c, n, n_seqs, h, 16), b = pa_ws(c, n, n_seqs, h, rt);
    return a > b ? a : b;
}

template <typename T, int HD, int RT, int KT>
static int pa_launch_rt(PaArgs p, void (*kernel)(PaArgs), void *ws, hipStream_t st) {
    const PaPlan q = pa_plan_of(&p.c, p.a.n, p.a.n_seqs, p.a.h, RT);
    p.per_unit = pg_per_unit(p.c.kvh, q.units);
    p.extra = q.extra;
    p.one = q.one;
    p.units = q.units;
    p.pml = (float2 *)ws;
    p.po = (float *)((char *)ws + pa_up((size_t)q.slots * RT * 8));
    p.index = (int4 *)((char *)p.po + pa_up((size_t)q.slots * RT * HD * 4));
    if (p.a.n_seqs > PA_INDEX) {
        hipLaunchKernelGGL(k_pa_index, dim3(1), dim3(1024), 0, st, p, RT, KT);
        const int rc = QK_CHECK_LAUNCH();
        if (rc) return rc;
    }
    hipLaunchKernelGGL(kernel, dim3((unsigned)q.grid), dim3(pa_threads(&p.c, p.a.n, p.a.h, RT)), 0, st, p);
    const int rc = QK_CHECK_LAUNCH();
    if (rc || q.join == 0) return rc;
    /* few tasks are long sequences on their own, a few rows of a hundred parts:
     * 16 waves a row (one of 64000 rows: 36 us with 4, so 26); else 4 (64 of
     * 1000: 26 us with 16, so 22) */
    const dim3 grid((unsigned)q.join, pa_join_rows(q.join, RT));
    if (q.join <= 16) hipLaunchKernelGGL((k_pa_join<T, HD, RT, KT, 16>), grid, dim3(1024), 0, st, p);
    else hipLaunchKernelGGL((k_pa_join<T, HD, RT, KT, 4>), grid, dim3(256), 0, st, p);
    return QK_CHECK_LAUNCH();
}

template <typename T, int HD>
static int pa_launch(const PaArgs &p, void *ws, hipStream_t st) {
    const int rt = pa_rows(&p.c, &p.a);
    if (rt == PM_RT) {
        if constexpr (sizeof(T) == 2) {
            if constexpr (HD <= 128)
                if (pa_groups(&p.c, p.a.n, p.a.h) == 1) return pa_launch_rt<T, HD, PM_RT, pm_kt(HD)>(p, k_pa_many<HD, 1>, ws, st);
            return pa_launch_rt<T, HD, PM_RT, pm_kt(HD)>(p, k_pa_many<HD, 2>, ws, st);
        } else return pa_launch_rt<T, HD, PM_RT, pm_kt(HD, true)>(p, k_pa_many32<HD>, ws, st);
    }
    if constexpr (HD <= (sizeof(T) == 2 ? 192 : 128)) /* pa_two */
        if (rt == 32) return pa_launch_rt<T, HD, 32, PD_KT>(p, k_pa_few<T, HD, 2>, ws, st);
    return pa_launch_rt<T, HD, 16, PD_KT>(p, k_pa_few<T, HD, 1>, ws, st);
}

template <typename T>
static int pa_launch_hd(const PaArgs &p, void *ws, hipStream_t st) {
    switch (p.c.hd) {
    case 64: return pa_launch<T, 64>(p, ws, st);
    case 128: return pa_launch<T, 128>(p, ws, st);
    case 192: return pa_launch<T, 192>(p, ws, st);
    case 256: return pa_launch<T, 256>(p, ws, st);
    default: return (int)hipErrorInvalidValue;
    }
}

extern "C" int qk_launch_pg_attn(const pg_cache *c, const pg_attn *a, void *ws, void *stream) {
    PaArgs p;
    p.c = *c;
    p.a = *a;
    p.G = a->h / c->kvh;
    p.po = NULL;
    p.pml = NULL;
    p.index = NULL;
    return c->dtype == QMOE_BF16 ? pa_launch_hd<uint16_t>(p, ws, (hipStream_t)stream)
                                 : pa_launch_hd<float>(p, ws, (hipStream_t)stream);
}
