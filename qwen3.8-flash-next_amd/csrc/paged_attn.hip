/*
 * paged_attn.hip -- attention of a ragged batch of new tokens over a paged
 * cache: softmax(scale q.k) v over the rows that a token sees (causal, a
 * sliding window, sinks), a group of query heads per kv head.
 */
#include "qk_device.h"
#include "paged_parts.h"

struct PaArgs {
    pg_cache c; /* k and v of the call's layer */
    pg_attn a;
    int G;      /* query heads per kv head */
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
template <typename T>
__device__ __forceinline__ void pa_put(T *p, float x) {
    if constexpr (sizeof(T) == 2) qk_st((uint16_t *)p, (uint16_t)qk_cvt_pk_bf16(x, x));
    else qk_st((float *)p, x);
}

/* what a row's maximum and sum give: the factor on its sum of p v, NaN for a
 * row whose scores are all -inf (0/0, as the formula), 0 for a row that sees
 * nothing */
__device__ __forceinline__ float pa_norm(float m, float l, bool seen) {
    return m == -INFINITY && !seen ? 0.0f : 1.0f / l;
}

/*
 * One wave per (token, query head): lane = key for the scores, lane = dims
 * for the sum of p v, 64 keys at a time under a running maximum.
 */
template <typename T, int HD>
__global__ __launch_bounds__(256) void k_pa_rows(PaArgs p) {
    const int lane = threadIdx.x & 63;
    const int r = blockIdx.x * 4 + (threadIdx.x >> 6);
    const int t = r / p.a.h, hh = r - t * p.a.h;
    if (t >= p.a.n) return;
    int lo = 0, hi = p.a.n_seqs;
    if (t < qk_ld(p.a.starts) || t >= qk_ld(p.a.starts + hi)) return;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (qk_ld(p.a.starts + mid) <= t) lo = mid;
        else hi = mid;
    }
    const pg_seq s = pg_seq_at(&p.c, p.a.starts, p.a.slots, p.a.n, lo);
    if (t < s.start || t >= s.start + s.count) return;
    const int pos = s.len - s.count + t - s.start;
    const int kh = p.a.grouped ? hh / p.G : hh % p.c.kvh;
    const T *kp = (const T *)p.c.k + (int64_t)kh * p.c.head_stride, *vp = (const T *)p.c.v + (int64_t)kh * p.c.head_stride;
    const T *q = (const T *)p.a.q + t * p.a.q_token + hh * p.a.q_head;
    const int32_t *row = p.c.table + (int64_t)s.slot * p.c.table_stride;
    const pg_tiles tl = pg_tiles_of(pos, pos, p.a.window, p.a.sinks, 64);
    float m = -INFINITY, l = 0.0f, acc[HD / 64];
    bool seen = false;
#pragma unroll
    for (int e = 0; e < HD / 64; e++) acc[e] = 0.0f;
    for (int i = 0; i < tl.nt && s.slot >= 0; i++) {
        const int j = pg_tile(tl, i) * 64 + lane;
        const int64_t at = pg_sees(pos, j, p.a.window, p.a.sinks) ? pg_row_at(&p.c, row, j) : -1;
        float sc = -INFINITY;
        if (at >= 0) {
            float d = 0.0f;
            for (int c = 0; c < HD; c += 8) {
                float x[8], y[8];
                pa_get8(kp + at + c, x);
                pa_get8(q + c, y);
#pragma unroll
                for (int u = 0; u < 8; u++) d = fmaf(x[u], y[u], d);
            }
            sc = d * p.a.scale;
        }
        float mx = sc;
        for (int o = 1; o < 64; o <<= 1) mx = fmaxf(mx, __shfl_xor(mx, o, QK_WAVE));
        const float mn = fmaxf(m, mx), f = mn == -INFINITY ? 1.0f : exp2f(m - mn);
        seen |= __any(at >= 0);
        l *= f;
#pragma unroll
        for (int e = 0; e < HD / 64; e++) acc[e] *= f;
        m = mn;
        const float pr = at < 0 ? 0.0f : exp2f(sc - (m == -INFINITY ? 0.0f : m));
        l += pr;
        for (uint64_t todo = __ballot(at >= 0); todo; todo &= todo - 1) {
            const int b = __builtin_ctzll(todo);
            const float pj = __shfl(pr, b, QK_WAVE);
            const int64_t aj = ((int64_t)__shfl((int)(at >> 32), b, QK_WAVE) << 32) | (uint32_t)__shfl((int)at, b, QK_WAVE);
#pragma unroll
            for (int e = 0; e < HD / 64; e++) acc[e] = fmaf(pj, pa_get(vp + aj + lane + 64 * e), acc[e]);
        }
    }
    for (int o = 1; o < 64; o <<= 1) l += __shfl_xor(l, o, QK_WAVE);
    const float f = pa_norm(m, l, seen);
    T *out = (T *)p.a.out + t * p.a.o_token + hh * p.a.o_head;
#pragma unroll
    for (int e = 0; e < HD / 64; e++) pa_put(out + lane + 64 * e, acc[e] * f);
}

/* ------------------------------------------------------------ host side */

extern "C" size_t qk_pg_attn_ws(const pg_cache *c, int n, int n_seqs, int h) { return 256; }

template <typename T>
static int pa_launch(const PaArgs &p, hipStream_t st) {
    const dim3 grid((unsigned)(((int64_t)p.a.n * p.a.h + 3) / 4));
    switch (p.c.hd) {
    case 64: hipLaunchKernelGGL((k_pa_rows<T, 64>), grid, dim3(256), 0, st, p); break;
    case 128: hipLaunchKernelGGL((k_pa_rows<T, 128>), grid, dim3(256), 0, st, p); break;
    case 192: hipLaunchKernelGGL((k_pa_rows<T, 192>), grid, dim3(256), 0, st, p); break;
    case 256: hipLaunchKernelGGL((k_pa_rows<T, 256>), grid, dim3(256), 0, st, p); break;
    default: return (int)hipErrorInvalidValue;
    }
    return QK_CHECK_LAUNCH();
}

extern "C" int qk_launch_pg_attn(const pg_cache *c, const pg_attn *a, void *ws, void *stream) {
    PaArgs p;
    p.c = *c;
    p.a = *a;
    p.G = a->h / c->kvh;
    return c->dtype == QMOE_BF16 ? pa_launch<uint16_t>(p, (hipStream_t)stream) : pa_launch<float>(p, (hipStream_t)stream);
}
