/*
 * qmoe_paged.c -- C11 host side of the paged cache: argument checks and the
 * launches of paged_pages.hip, paged_attn.hip and paged_tree.hip.  Holds no state: the cache
 * and the workspaces are the caller's.
 */
#include <limits.h>
#include <math.h>
#include <stdarg.h>
#include <stdio.h>
#include <string.h>

#include <hip/hip_runtime_api.h>

#include "paged_parts.h"

static int pg_fail(qmoe_err *err, const char *fmt, ...) {
    if (err) {
        va_list ap;
        va_start(ap, fmt);
        vsnprintf(err->msg, sizeof(err->msg), fmt, ap);
        va_end(ap);
    }
    return -1;
}

static int pg_hip(qmoe_err *err, int rc, const char *what) {
    if (rc == 0) return 0;
    return pg_fail(err, "%s: HIP error %d (%s)", what, rc, hipGetErrorString((hipError_t)rc));
}

static int pg_misaligned(const void *p) { return ((uintptr_t)p & 15) != 0; }

/* elements of the `n` strided dimensions lie apart: each stride, from the
 * smallest, is past what the smaller ones span.  0, or -1 also on overflow */
static int pg_apart(const int64_t *stride, const int64_t *size, int n, int64_t unit) {
    int used[4] = {0, 0, 0, 0};
    int64_t span = unit;
    for (int k = 0; k < n; k++) {
        int best = -1;
        for (int i = 0; i < n; i++)
            if (!used[i] && (best < 0 || stride[i] < stride[best])) best = i;
        used[best] = 1;
        if (size[best] <= 1) continue;
        int64_t ext;
        if (stride[best] < span || __builtin_mul_overflow(stride[best], size[best] - 1, &ext) ||
            __builtin_add_overflow(span, ext, &span) || span > ((int64_t)1 << 46))
            return -1;
    }
    return 0;
}

/* checks a cache and brings it into the kernels' form (k, v of layer 0) */
static int pg_cache_of(const qmoe_paged_cache *q, pg_cache *c, qmoe_err *err) {
    if (err) err->msg[0] = 0;
    if (!q) return pg_fail(err, "cache is NULL");
    if (q->dtype != QMOE_F32 && q->dtype != QMOE_BF16) return pg_fail(err, "dtype %d is not f32 or bf16", q->dtype);
    if (q->head_dim < 64 || q->head_dim > 256 || q->head_dim % 64)
        return pg_fail(err, "head_dim %d is not 64, 128, 192 or 256", q->head_dim);
    if (q->n_kv_heads < 1 || q->n_kv_heads > 1024) return pg_fail(err, "n_kv_heads %d out of range [1, 1024]", q->n_kv_heads);
    if (q->page_rows < 1 || q->page_rows > 4096) return pg_fail(err, "page_rows %d out of range [1, 4096]", q->page_rows);
    if (q->n_layers < 1 || q->n_layers > 65536) return pg_fail(err, "n_layers %d out of range [1, 65536]", q->n_layers);
    if (q->n_pages < 1 || q->n_pages > PG_MAX_PAGES)
        return pg_fail(err, "n_pages %d out of range [1, %d]", q->n_pages, PG_MAX_PAGES);
    if (q->n_slots < 1 || q->max_pages < 1) return pg_fail(err, "n_slots %d and max_pages %d must be >= 1", q->n_slots, q->max_pages);
    if ((int64_t)q->max_pages * q->page_rows > PG_MAX_ROWS)
        return pg_fail(err, "a table of %d pages of %d rows holds more than %d rows", q->max_pages, q->page_rows, PG_MAX_ROWS);
    if (q->table_stride < q->max_pages || q->table_stride > PG_MAX_ROWS)
        return pg_fail(err, "table_stride %lld out of range [max_pages = %d, %d]", (long long)q->table_stride, q->max_pages, PG_MAX_ROWS);
    if (!q->k || !q->v) return pg_fail(err, "%s is NULL", q->k ? "v" : "k");
    if (!q->table || !q->lens || !q->refs) return pg_fail(err, "%s is NULL", !q->table ? "table" : !q->lens ? "lens" : "refs");
    const int es = q->dtype == QMOE_BF16 ? 2 : 4;
    int64_t stride[4] = {q->layer_stride, q->page_stride, q->row_stride, q->head_stride};
    const int64_t size[4] = {q->n_layers, q->n_pages, q->page_rows, q->n_kv_heads};
    for (int i = 0; i < 4; i++)
        if (size[i] == 1) stride[i] = 0; /* the stride of a single element is never taken */
    static const char *const name[4] = {"layer_stride", "page_stride", "row_stride", "head_stride"};
    for (int i = 0; i < 4; i++)
        if (stride[i] < 0 || stride[i] % (16 / es)) return pg_fail(err, "%s %lld is not a multiple of 16 bytes", name[i], (long long)stride[i]);
    if (pg_misaligned(q->k) || pg_misaligned(q->v)) return pg_fail(err, "k and v must be 16-byte aligned");
    if (pg_apart(stride, size, 4, q->head_dim)) return pg_fail(err, "the strides let elements of the pages overlap");
    memset(c, 0, sizeof(*c));
    c->k = q->k;
    c->v = q->v;
    c->layer_stride = stride[0];
    c->page_stride = stride[1];
    c->row_stride = stride[2];
    c->head_stride = stride[3];
    c->table = q->table;
    c->table_stride = q->table_stride;
    c->lens = q->lens;
    c->refs = q->refs;
    c->page_rows = pg_div_make((uint32_t)q->page_rows);
    c->dtype = q->dtype;
    c->n_layers = q->n_layers;
    c->n_pages = q->n_pages;
    c->kvh = q->n_kv_heads;
    c->hd = q->head_dim;
    c->n_slots = q->n_slots;
    c->max_pages = q->max_pages;
    c->cap = q->max_pages * q->page_rows;
    return 0;
}

static int pg_layer(pg_cache *c, int layer, qmoe_err *err) {
    if (layer < 0 || layer >= c->n_layers) return pg_fail(err, "layer %d out of range [0, %d)", layer, c->n_layers);
    const int64_t at = c->layer_stride * layer * (c->dtype == QMOE_BF16 ? 2 : 4);
    c->k = (char *)c->k + at;
    c->v = (char *)c->v + at;
    return 0;
}

static int pg_seqs(const pg_cache *c, const int32_t *slots, int n_seqs, int most, qmoe_err *err) {
    if (n_seqs < 0 || n_seqs > most) return pg_fail(err, "n_seqs = %d out of range [0, %d]", n_seqs, most);
    if (!slots && n_seqs > c->n_slots) return pg_fail(err, "%d sequences without slots, but %d slots", n_seqs, c->n_slots);
    return 0;
}

static int pg_batch(const pg_cache *c, const qmoe_paged_batch *b, qmoe_err *err) {
    if (!b) return pg_fail(err, "batch is NULL");
    if (b->n < 0) return pg_fail(err, "n = %d is negative", b->n);
    if (pg_seqs(c, b->slots, b->n_seqs, PG_MAX_SEQS, err)) return -1;
    if (b->n_seqs > 0 && b->n > 0 && !b->starts) return pg_fail(err, "starts is NULL");
    if ((uintptr_t)b->status & 3) return pg_fail(err, "status must be 4-byte aligned");
    return 0;
}

/* the stride of a dimension of `size`; a single element's is never taken */
static int pg_stride(int64_t s, int64_t size, int es, const char *name, qmoe_err *err) {
    if (size <= 1) return 0;
    if (s < 0 || s % (16 / es) || s > ((int64_t)1 << 40))
        return pg_fail(err, "%s %lld is not a multiple of 16 bytes in range", name, (long long)s);
    return 0;
}

static int pg_work(const void *ws, size_t have, size_t need, qmoe_err *err) {
    if (have < need) return pg_fail(err, "the workspace has %zu bytes, the call needs %zu", have, need);
    if (!ws || pg_misaligned(ws)) return pg_fail(err, "the workspace is NULL or not 16-byte aligned");
    return 0;
}

static int pg_heads(const pg_cache *c, int n, int h, qmoe_err *err) {
    if (h < 1 || h % c->kvh) return pg_fail(err, "n_heads %d is not a multiple of the %d kv heads", h, c->kvh);
    if ((int64_t)n * h > PG_MAX_ROWS) return pg_fail(err, "%d rows of %d heads are more than %d", n, h, PG_MAX_ROWS);
    return 0;
}

size_t qmoe_paged_ws_bytes(const qmoe_paged_cache *q, int call, int n, int n_seqs, int n_heads) {
    pg_cache c;
    if (pg_cache_of(q, &c, NULL) || n_seqs < 0) return 0;
    switch (call) {
    case QMOE_PAGED_ATTN:
        if (n < 0 || n_seqs > PG_MAX_SEQS || pg_heads(&c, n, n_heads, NULL)) return 0;
        return qk_pg_attn_ws(&c, n, n_seqs, n_heads);
    case QMOE_PAGED_ATTN_TREE:
        if (n < 0 || n_seqs > PG_MAX_SEQS || pg_heads(&c, n, n_heads, NULL)) return 0;
        return qk_pg_attn_tree_ws(&c, n, n_seqs, n_heads);
    case QMOE_PAGED_RESERVE: return n_seqs > PG_MAX_BATCH ? 0 : qk_pg_reserve_ws(&c, n_seqs);
    case QMOE_PAGED_FORK: return n_seqs > PG_MAX_BATCH ? 0 : qk_pg_fork_ws(&c, n_seqs);
    case QMOE_PAGED_COMPACT: return qk_pg_compact_ws(&c);
    case QMOE_PAGED_KEEP: return n < 0 || n_seqs > PG_MAX_BATCH ? 0 : qk_pg_keep_ws(n, n_seqs);
    default: return 0;
    }
}

int qmoe_paged_append(const qmoe_paged_cache *q, int layer, const qmoe_paged_batch *b, const void *k, const void *v,
                      int src_dtype, int64_t k_token, int64_t k_head, int64_t v_token, int64_t v_head, void *stream,
                      qmoe_err *err) {
    pg_cache c;
    if (pg_cache_of(q, &c, err) || pg_layer(&c, layer, err) || pg_batch(&c, b, err)) return -1;
    if (src_dtype != c.dtype && src_dtype != QMOE_F32)
        return pg_fail(err, "rows of dtype %d for pages of dtype %d (the pages' type, or f32)", src_dtype, c.dtype);
    const int es = src_dtype == QMOE_BF16 ? 2 : 4;
    if (pg_stride(k_token, b->n, es, "k_token_stride", err) || pg_stride(k_head, c.kvh, es, "k_head_stride", err) ||
        pg_stride(v_token, b->n, es, "v_token_stride", err) || pg_stride(v_head, c.kvh, es, "v_head_stride", err))
        return -1;
    if ((int64_t)b->n * c.kvh * (c.hd / 4) > 0x7FFFFF00) return pg_fail(err, "n = %d rows are too many for one call", b->n);
    if (b->n == 0 || b->n_seqs == 0) return 0;
    if (!k || !v) return pg_fail(err, "%s is NULL", k ? "v" : "k");
    if (pg_misaligned(k) || pg_misaligned(v)) return pg_fail(err, "k and v must be 16-byte aligned");
    return pg_hip(err,
                  qk_launch_pg_append(&c, k, v, src_dtype, k_token, k_head, v_token, v_head, b->starts, b->slots, b->status,
                                      b->n, b->n_seqs, stream),
                  "paged append");
}

/* the tree of a call of n rows */
static int pg_tree_of(const qmoe_paged_tree *t, int n, qmoe_err *err) {
    if (!t) return pg_fail(err, "tree is NULL");
    if (t->words < 1 || t->words > 32) return pg_fail(err, "words %d out of range [1, 32]", t->words);
    if (n > 0 && (!t->depths || !t->seen)) return pg_fail(err, "%s is NULL", t->depths ? "seen" : "depths");
    if (((uintptr_t)t->depths | (uintptr_t)t->seen) & 3) return pg_fail(err, "depths and seen must be 4-byte aligned");
    return 0;
}

/* rows of a call without a cache */
static int pg_call(const int32_t *starts, int n, int n_seqs, qmoe_err *err) {
    if (n < 0 || n > PG_MAX_ROWS) return pg_fail(err, "n = %d out of range [0, %d]", n, PG_MAX_ROWS);
    if (n_seqs < 0 || n_seqs > PG_MAX_SEQS) return pg_fail(err, "n_seqs = %d out of range [0, %d]", n_seqs, PG_MAX_SEQS);
    if (n_seqs > 0 && !starts) return pg_fail(err, "starts is NULL");
    return 0;
}

static int pg_attention(const qmoe_paged_cache *cache, int layer, const qmoe_paged_batch *b, const qmoe_paged_query *q,
                        const qmoe_paged_tree *t, void *ws, size_t ws_bytes, void *stream, qmoe_err *err) {
    pg_cache c;
    if (pg_cache_of(cache, &c, err) || pg_layer(&c, layer, err) || pg_batch(&c, b, err)) return -1;
    if (!q) return pg_fail(err, "query is NULL");
    if (pg_heads(&c, b->n, q->n_heads, err)) return -1;
    if (q->window < 0 || q->sinks < 0) return pg_fail(err, "window %d and sinks %d must be >= 0", q->window, q->sinks);
    if (q->grouped != 0 && q->grouped != 1) return pg_fail(err, "grouped %d is not 0 or 1", q->grouped);
    /* the scores are kept in log2 units */
    const float scale = (float)((q->scale != 0.0f ? (double)q->scale : 1.0 / sqrt((double)c.hd)) * 1.4426950408889634);
    if (!isfinite(scale)) return pg_fail(err, "scale %g or its product with log2(e) is not finite", (double)q->scale);
    const int es = c.dtype == QMOE_BF16 ? 2 : 4;
    if (pg_stride(q->q_token_stride, b->n, es, "q_token_stride", err) || pg_stride(q->q_head_stride, q->n_heads, es, "q_head_stride", err) ||
        pg_stride(q->out_token_stride, b->n, es, "out_token_stride", err) ||
        pg_stride(q->out_head_stride, q->n_heads, es, "out_head_stride", err))
        return -1;
    const int64_t stride[2] = {q->out_token_stride, q->out_head_stride}, size[2] = {b->n, q->n_heads};
    if (pg_apart(stride, size, 2, c.hd)) return pg_fail(err, "the strides let elements of out overlap");
    if (b->n == 0 || b->n_seqs == 0) return 0;
    const size_t need = t ? qk_pg_attn_tree_ws(&c, b->n, b->n_seqs, q->n_heads) : qk_pg_attn_ws(&c, b->n, b->n_seqs, q->n_heads);
    if (!need) return pg_fail(err, "%d rows of %d sequences and %d heads are more work than one launch holds", b->n, b->n_seqs, q->n_heads);
    if (!q->q || !q->out) return pg_fail(err, "%s is NULL", q->q ? "out" : "q");
    if (pg_misaligned(q->q) || pg_misaligned(q->out)) return pg_fail(err, "q and out must be 16-byte aligned");
    if (pg_work(ws, ws_bytes, need, err)) return -1;
    pg_attn a;
    a.q = q->q;
    a.out = q->out;
    a.q_token = q->q_token_stride;
    a.q_head = q->q_head_stride;
    a.o_token = q->out_token_stride;
    a.o_head = q->out_head_stride;
    a.starts = b->starts;
    a.slots = b->slots;
    a.status = b->status;
    a.n = b->n;
    a.n_seqs = b->n_seqs;
    a.h = q->n_heads;
    a.window = q->window;
    a.sinks = q->window > 0 ? q->sinks : 0;
    a.grouped = q->grouped;
    a.scale = scale;
    a.depths = t ? t->depths : NULL;
    a.seen = t ? t->seen : NULL;
    a.words = t ? t->words : 0;
    return pg_hip(err, qk_launch_pg_attn(&c, &a, ws, stream), "paged attention");
}

int qmoe_paged_attn(const qmoe_paged_cache *c, int layer, const qmoe_paged_batch *b, const qmoe_paged_query *q, void *ws,
                    size_t ws_bytes, void *stream, qmoe_err *err) {
    return pg_attention(c, layer, b, q, NULL, ws, ws_bytes, stream, err);
}

int qmoe_paged_attn_tree(const qmoe_paged_cache *c, int layer, const qmoe_paged_batch *b, const qmoe_paged_query *q,
                         const qmoe_paged_tree *t, void *ws, size_t ws_bytes, void *stream, qmoe_err *err) {
    if (err) err->msg[0] = 0;
    if (pg_tree_of(t, b ? b->n : 0, err)) return -1;
    return pg_attention(c, layer, b, q, t, ws, ws_bytes, stream, err);
}

int qmoe_paged_tree_build(const int32_t *parents, const int32_t *starts, int n, int n_seqs, const qmoe_paged_tree *t,
                          void *stream, qmoe_err *err) {
    if (err) err->msg[0] = 0;
    if (pg_tree_of(t, n, err) || pg_call(starts, n, n_seqs, err)) return -1;
    if (n == 0 || n_seqs == 0) return 0;
    if (!parents) return pg_fail(err, "parents is NULL");
    return pg_hip(err, qk_launch_pg_tree(parents, starts, n, n_seqs, t->depths, t->seen, t->words, stream), "paged tree");
}

int qmoe_paged_append_rotary(const qmoe_paged_cache *q, int layer, const qmoe_paged_batch *b, const qmoe_paged_rotary *r,
                             const qmoe_paged_tree *t, void *stream, qmoe_err *err) {
    pg_cache c;
    if (pg_cache_of(q, &c, err) || pg_layer(&c, layer, err) || pg_batch(&c, b, err)) return -1;
    if (!r) return pg_fail(err, "rotary is NULL");
    if (t && pg_tree_of(t, b->n, err)) return -1;
    if (r->src_dtype != c.dtype && r->src_dtype != QMOE_F32)
        return pg_fail(err, "rows of dtype %d for pages of dtype %d (the pages' type, or f32)", r->src_dtype, c.dtype);
    if (r->n_heads < 0 || (int64_t)b->n * r->n_heads > PG_MAX_ROWS)
        return pg_fail(err, "%d rows of %d heads out of range [0, %d]", b->n, r->n_heads, PG_MAX_ROWS);
    if (b->n > PG_MAX_ROTARY) return pg_fail(err, "n = %d rows are too many for one call", b->n);
    if (r->rot < 2 || r->rot > c.hd || r->rot % 2) return pg_fail(err, "rot %d is not even in [2, head_dim = %d]", r->rot, c.hd);
    if (r->interleaved != 0 && r->interleaved != 1) return pg_fail(err, "interleaved %d is not 0 or 1", r->interleaved);
    if (!(r->eps >= 0.0f) || !isfinite(r->eps)) return pg_fail(err, "eps %g is not finite and >= 0", (double)r->eps);
    const int es = r->src_dtype == QMOE_BF16 ? 2 : 4, os = c.dtype == QMOE_BF16 ? 2 : 4;
    if (pg_stride(r->q_token_stride, b->n, es, "q_token_stride", err) || pg_stride(r->q_head_stride, r->n_heads, es, "q_head_stride", err) ||
        pg_stride(r->k_token_stride, b->n, es, "k_token_stride", err) || pg_stride(r->k_head_stride, c.kvh, es, "k_head_stride", err) ||
        pg_stride(r->v_token_stride, b->n, es, "v_token_stride", err) || pg_stride(r->v_head_stride, c.kvh, es, "v_head_stride", err) ||
        pg_stride(r->out_token_stride, b->n, os, "out_token_stride", err) ||
        pg_stride(r->out_head_stride, r->n_heads, os, "out_head_stride", err))
        return -1;
    const int64_t stride[2] = {r->out_token_stride, r->out_head_stride}, size[2] = {b->n, r->n_heads};
    if (r->n_heads > 0 && pg_apart(stride, size, 2, c.hd)) return pg_fail(err, "the strides let elements of out overlap");
    if (b->n == 0 || b->n_seqs == 0) return 0;
    if (!r->k || !r->v || !r->freqs) return pg_fail(err, "%s is NULL", !r->k ? "k" : !r->v ? "v" : "freqs");
    if (r->n_heads > 0 && (!r->q || !r->out)) return pg_fail(err, "%s is NULL", r->q ? "out" : "q");
    if (pg_misaligned(r->k) || pg_misaligned(r->v) || (r->n_heads > 0 && (pg_misaligned(r->q) || pg_misaligned(r->out))))
        return pg_fail(err, "q, k, v and out must be 16-byte aligned");
    if (((uintptr_t)r->freqs | (uintptr_t)r->q_norm | (uintptr_t)r->k_norm) & 3)
        return pg_fail(err, "freqs, q_norm and k_norm must be 4-byte aligned");
    if (r->n_heads > 0 && r->q == r->out &&
        (es != os || (b->n > 1 && r->q_token_stride != r->out_token_stride) ||
         (r->n_heads > 1 && r->q_head_stride != r->out_head_stride)))
        return pg_fail(err, "out is q, but not with the same type and strides");
    return pg_hip(err,
                  qk_launch_pg_rotary(&c, r, b->starts, b->slots, b->status, t ? t->depths : NULL, b->n, b->n_seqs, stream),
                  "paged rotary append");
}

int qmoe_paged_follow(const qmoe_paged_tree *t, const int32_t *parents, const int32_t *tokens, const int32_t *chosen,
                      const int32_t *starts, int n, int n_seqs, int32_t *rows, int32_t *counts, int32_t *next, void *stream,
                      qmoe_err *err) {
    if (err) err->msg[0] = 0;
    if (pg_tree_of(t, n, err) || pg_call(starts, n, n_seqs, err)) return -1;
    if (n_seqs == 0) return 0;
    if (!counts || !next) return pg_fail(err, "%s is NULL", counts ? "next" : "counts");
    if (n > 0 && (!parents || !tokens || !chosen || !rows))
        return pg_fail(err, "%s is NULL", !parents ? "parents" : !tokens ? "tokens" : !chosen ? "chosen" : "rows");
    return pg_hip(err,
                  qk_launch_pg_follow(parents, tokens, chosen, starts, t->depths, t->seen, t->words, n, n_seqs, rows, counts,
                                      next, stream),
                  "paged follow");
}

int qmoe_paged_keep(const qmoe_paged_cache *q, const qmoe_paged_batch *b, const int32_t *rows, const int32_t *counts,
                    int32_t *status, void *ws, size_t ws_bytes, void *stream, qmoe_err *err) {
    pg_cache c;
    if (pg_cache_of(q, &c, err) || pg_batch(&c, b, err) || pg_seqs(&c, b->slots, b->n_seqs, PG_MAX_BATCH, err)) return -1;
    if (!status) return pg_fail(err, "status is NULL");
    if ((uintptr_t)status & 3) return pg_fail(err, "status must be 4-byte aligned");
    if (b->n_seqs > 0 && (!b->starts || !counts)) return pg_fail(err, "%s is NULL", b->starts ? "counts" : "starts");
    if (b->n_seqs > 0 && b->n > 0 && !rows) return pg_fail(err, "rows is NULL");
    if (pg_work(ws, ws_bytes, qk_pg_keep_ws(b->n, b->n_seqs), err)) return -1;
    return pg_hip(err, qk_launch_pg_keep(&c, b->starts, b->slots, b->status, b->n, b->n_seqs, rows, counts, status, ws, stream),
                  "paged keep");
}

int qmoe_paged_reserve(const qmoe_paged_cache *q, const int32_t *slots, const int32_t *n_new, int n_seqs,
                       int32_t *status, void *ws, size_t ws_bytes, void *stream, qmoe_err *err) {
    pg_cache c;
    if (pg_cache_of(q, &c, err) || pg_seqs(&c, slots, n_seqs, PG_MAX_BATCH, err)) return -1;
    if (!status) return pg_fail(err, "status is NULL");
    if (n_seqs > 0 && !n_new) return pg_fail(err, "n_new is NULL");
    if (pg_work(ws, ws_bytes, qk_pg_reserve_ws(&c, n_seqs), err)) return -1;
    return pg_hip(err, qk_launch_pg_reserve(&c, slots, n_new, n_seqs, status, ws, stream), "paged reserve");
}

int qmoe_paged_fork(const qmoe_paged_cache *q, const int32_t *src, const int32_t *dst, const int32_t *rows, int n_seqs,
                    int32_t *status, void *ws, size_t ws_bytes, void *stream, qmoe_err *err) {
    pg_cache c;
    if (pg_cache_of(q, &c, err)) return -1;
    if (n_seqs < 0 || n_seqs > PG_MAX_BATCH) return pg_fail(err, "n_seqs = %d out of range [0, %d]", n_seqs, PG_MAX_BATCH);
    if (!status) return pg_fail(err, "status is NULL");
    if (n_seqs > 0 && (!src || !dst)) return pg_fail(err, "%s is NULL", src ? "dst" : "src");
    if (pg_work(ws, ws_bytes, qk_pg_fork_ws(&c, n_seqs), err)) return -1;
    return pg_hip(err, qk_launch_pg_fork(&c, src, dst, rows, n_seqs, status, ws, stream), "paged fork");
}

int qmoe_paged_evict(const qmoe_paged_cache *q, const int32_t *slots, int n_seqs, int window, int sinks, void *stream,
                     qmoe_err *err) {
    pg_cache c;
    if (pg_cache_of(q, &c, err) || pg_seqs(&c, slots, n_seqs, INT_MAX, err)) return -1;
    if (window < 1 || sinks < 0) return pg_fail(err, "window %d must be >= 1 and sinks %d >= 0", window, sinks);
    if (n_seqs == 0) return 0;
    return pg_hip(err, qk_launch_pg_evict(&c, slots, n_seqs, window, sinks, stream), "paged evict");
}

int qmoe_paged_compact(const qmoe_paged_cache *q, int32_t *used, void *ws, size_t ws_bytes, void *stream,
                       qmoe_err *err) {
    pg_cache c;
    if (pg_cache_of(q, &c, err)) return -1;
    if (!used) return pg_fail(err, "used is NULL");
    if (pg_work(ws, ws_bytes, qk_pg_compact_ws(&c), err)) return -1;
    return pg_hip(err, qk_launch_pg_compact(&c, used, ws, stream), "paged compact");
}
