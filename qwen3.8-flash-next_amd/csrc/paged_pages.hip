/*
 * paged_pages.hip -- rows into the pages of a paged cache, and the pages'
 * bookkeeping on the GPU: appending, forking, reserving (with the copy of a
 * partly filled page that others share), releasing behind a window, and
 * compacting.  Tables, lengths and reference counts stay on the device, so a
 * serving step needs no host round trip and can be captured in a graph.
 *
 * The page counts are changed with atomic adds of whole numbers, whose order
 * does not matter; which page goes to whom follows from ranks (prefix sums),
 * never from arrival, so every result is the same from call to call.
 */
#include "qk_device.h"
#include "paged_parts.h"

/* lanes below this one among the set bits of m */
__device__ __forceinline__ int pg_rank(uint64_t m) {
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
}

/* exclusive prefix sum over the workgroup's 1024 threads; total = the sum */
__device__ __forceinline__ int pg_scan(int v, int *lds, int &total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int x = v;
    for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(x, o, QK_WAVE);
        if (lane >= o) x += y;
    }
    if (lane == 63) lds[wave] = x;
    __syncthreads();
    int before = 0;
    total = 0;
    for (int w = 0; w < 16; w++) {
        const int t = lds[w];
        if (w < wave) before += t;
        total += t;
    }
    __syncthreads();
    return before + x - v;
}

/* ------------------------------------------------------------ append
 * One thread per 16 destination bytes of k or v.  Bound: HBM, each new row
 * read and written once: f32 rows of nine prompts (74 MB) 17.0 us, 4.4 TB/s;
 * 64 single rows 4.1 us, a launch and four dependent loads. */
struct PgAppend {
    pg_cache c;
    const void *src[2];
    int64_t token[2], head[2];
    const int32_t *starts, *slots, *status;
    int n, n_seqs;
    pg_div per_row, per_head; /* 16-byte chunks */
};

/* the sequence that has row t of the call: the last i with starts[i] <= t
 * among those that lie in order; rows of no sequence give n_seqs */
__device__ __forceinline__ int pg_find(const int32_t *starts, int n_seqs, int t) {
    int lo = 0, hi = n_seqs; /* starts[lo] <= t < starts[hi] */
    if (t < qk_ld(starts) || t >= qk_ld(starts + n_seqs)) return n_seqs;
    /* one new row per sequence, the decode step: row t is sequence t's */
    if (t < n_seqs && qk_ld(starts + t) == t && qk_ld(starts + t + 1) == t + 1) return t;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (qk_ld(starts + mid) <= t) lo = mid;
        else hi = mid;
    }
    return lo;
}

template <typename S, typename D>
__global__ __launch_bounds__(256) void k_pg_append(PgAppend a) {
    constexpr int E = 16 / sizeof(D); /* elements per chunk */
    const int refused = a.status ? qk_ld(a.status) : 0;
    const uint32_t i = blockIdx.x * 256u + threadIdx.x;
    const uint32_t t = pg_div_of(a.per_row, i), r = i - t * a.per_row.d;
    if (t >= (uint32_t)a.n) return;
    const uint32_t hd = pg_div_of(a.per_head, r), ch = r - hd * a.per_head.d;
    const int s = pg_find(a.starts, a.n_seqs, (int)t);
    if (s >= a.n_seqs) return;
    const pg_seq q = pg_seq_at(&a.c, a.starts, a.slots, a.n, s);
    const int pos = q.len - q.count + (int)t - q.start;
    if (q.slot < 0 || (int)t < q.start || (int)t >= q.start + q.count) return;
    const int64_t at = pg_row_at(&a.c, a.c.table + q.slot * a.c.table_stride, pos);
    if (at < 0 || refused) return;
    const int which = blockIdx.y;
    const S *src = (const S *)a.src[which] + t * a.token[which] + hd * a.head[which] + ch * E;
    D *dst = (D *)(which ? a.c.v : a.c.k) + at + hd * a.c.head_stride + ch * E;
    if constexpr (sizeof(S) == sizeof(D)) {
        qk_st((float4 *)dst, qk_ld((const float4 *)src));
    } else { /* f32 -> bf16, round to nearest even: the page type's own rounding */
        const float4 x = qk_ld((const float4 *)src), y = qk_ld((const float4 *)src + 1);
        const uint4 w = make_uint4(qk_cvt_pk_bf16(x.x, x.y), qk_cvt_pk_bf16(x.z, x.w), qk_cvt_pk_bf16(y.x, y.y),
                                   qk_cvt_pk_bf16(y.z, y.w));
        qk_st((float4 *)dst, __builtin_bit_cast(float4, w));
    }
}

extern "C" int qk_launch_pg_append(const pg_cache *c, const void *k, const void *v, int src_dtype, int64_t k_token,
                                   int64_t k_head, int64_t v_token, int64_t v_head, const int32_t *starts,
                                   const int32_t *slots, const int32_t *status, int n, int n_seqs, void *stream) {
    hipStream_t st = (hipStream_t)stream;
    PgAppend a;
    const int E = c->dtype == QMOE_BF16 ? 8 : 4;
    a.c = *c;
    a.src[0] = k; a.src[1] = v;
    a.token[0] = k_token; a.token[1] = v_token;
    a.head[0] = k_head; a.head[1] = v_head;
    a.starts = starts; a.slots = slots; a.status = status;
    a.n = n; a.n_seqs = n_seqs;
    a.per_head = pg_div_make((uint32_t)(c->hd / E));
    a.per_row = pg_div_make((uint32_t)(c->kvh * (c->hd / E)));
    const dim3 grid((unsigned)(((int64_t)n * a.per_row.d + 255) / 256), 2);
    if (c->dtype == QMOE_F32) hipLaunchKernelGGL((k_pg_append<float, float>), grid, dim3(256), 0, st, a);
    else if (src_dtype == QMOE_F32) hipLaunchKernelGGL((k_pg_append<float, uint16_t>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((k_pg_append<uint16_t, uint16_t>), grid, dim3(256), 0, st, a);
    return QK_CHECK_LAUNCH();
}

/* ------------------------------------------------------------ page copies
 * Pages (src, dst) of every layer's k and v.  A page is rows x heads x
 * 16-byte chunks with strides; dimensions that lie one after the other are
 * merged on the host, so a dense page is one run.  Bound: memory: 256 copies of
 * 16 pages of 12 layers (101 MB written; the 6 MB of the sources are read from
 * HBM once and 15 times from caches) 18 us, 5.6 TB/s of writes, which stay in
 * the memory-side cache. */
struct PgCopy {
    pg_cache c;
    const int2 *pairs;        /* (-1, -1): none */
    const int32_t *n_pairs;   /* on the device, at most n */
    int n;
    pg_div chunks, inner, mid; /* of a page, of a (row, head) run, runs per row */
    int64_t row, head;         /* strides of the merged dimensions, bytes */
    int64_t page, layer;       /* bytes */
};

static void pg_copy_dims(PgCopy *p, const pg_cache *c) {
    const int es = c->dtype == QMOE_BF16 ? 2 : 4;
    int64_t in = (int64_t)c->hd * es / 16, mid = c->kvh, rows = c->page_rows.d;
    p->c = *c;
    p->head = c->head_stride * es;
    p->row = c->row_stride * es;
    p->page = c->page_stride * es;
    p->layer = c->layer_stride * es;
    if (mid == 1 || p->head == in * 16) {
        in *= mid;
        mid = 1;
    }
    if (mid == 1 && (rows == 1 || p->row == in * 16)) {
        in *= rows;
        rows = 1;
    }
    p->inner = pg_div_make((uint32_t)in);
    p->mid = pg_div_make((uint32_t)mid);
    p->chunks = pg_div_make((uint32_t)(in * mid * rows));
}

/* one workgroup: item = (pair, layer, k or v); all its pages' bytes */
__device__ __forceinline__ void pg_copy_item(const PgCopy &p, int64_t item) {
    const int lv = 2 * p.c.n_layers;
    const int64_t i = item / lv;
    const int r = (int)(item - i * lv), layer = r >> 1;
    const int2 pr = qk_ld(p.pairs + i);
    if (pr.x < 0 || pr.y < 0) return;
    char *base = (char *)(r & 1 ? p.c.v : p.c.k) + layer * p.layer;
    const char *src = base + pr.x * p.page;
    char *dst = base + pr.y * p.page;
    for (uint32_t j = threadIdx.x; j < p.chunks.d; j += blockDim.x) {
        const uint32_t run = pg_div_of(p.inner, j), ch = j - run * p.inner.d;
        const uint32_t row = pg_div_of(p.mid, run), hd = run - row * p.mid.d;
        const int64_t at = row * p.row + hd * p.head + (int64_t)ch * 16;
        qk_st((float4 *)(dst + at), qk_ld((const float4 *)(src + at)));
    }
}

__global__ __launch_bounds__(256) void k_pg_copy(PgCopy p) {
    const int64_t n = (int64_t)min(qk_ld(p.n_pairs), p.n) * 2 * p.c.n_layers;
    for (int64_t i = blockIdx.x; i < n; i += gridDim.x) pg_copy_item(p, i);
}
static unsigned pg_copy_grid(const pg_cache *c, int64_t pairs) {
    const int64_t items = pairs * 2 * c->n_layers;
    return (unsigned)(items < 4096 ? items : 4096);
}

/* ------------------------------------------------------------ reserve
 * One workgroup: the sequences' needs, their prefix sums, and as many free
 * pages, lowest first.  One workgroup, since every page's rank depends on all
 * sequences.  Bound: latency, of its reads of refs (5.3 us for 4 sequences) and
 * of the comparison of every sequence with every other, about 8 of the 13.5 us
 * for 256.  Without gain: several threads
 * per sequence in the scan (12.9, but 7.3 for 4), the free pages counted under
 * the loads of the batch (13.6). */
struct PgReserve {
    pg_cache c;
    const int32_t *slots, *n_new;
    int n;
    int32_t *status, *free_pages, *n_pairs;
    int2 *pairs;
};

/* a refused call: nothing is changed, no page is copied */
__device__ __forceinline__ void pg_refuse(const PgReserve &a, int status) {
    if (threadIdx.x) return;
    *a.status = status;
    *a.n_pairs = 0;
}

__global__ __launch_bounds__(1024) void k_pg_reserve(PgReserve a) {
    __shared__ __attribute__((aligned(16))) int slot_of[PG_MAX_BATCH], part_of[PG_MAX_BATCH];
    __shared__ int base_of[PG_MAX_BATCH], first_of[PG_MAX_BATCH];
    __shared__ int tmp[16];
    __shared__ unsigned long long wanted;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int R = (int)a.c.page_rows.d;
    const bool live = tid < a.n;
    int slot = -1, len = 0, add = 0, part = -1;
    bool bad = false;
    if (live) {
        slot = a.slots ? qk_ld(a.slots + tid) : tid;
        add = qk_ld(a.n_new + tid);
        if (slot < 0 || slot >= a.c.n_slots) bad = true;
        else {
            len = qk_ld(a.c.lens + slot);
            bad = len < 0 || len > a.c.cap || add < 0 || add > a.c.cap - len;
        }
    }
    const int e0 = (int)pg_div_of(a.c.page_rows, (uint32_t)max(len, 0));
    if (live && !bad && add > 0 && len - e0 * R > 0) {
        part = qk_ld(a.c.table + slot * a.c.table_stride + e0);
        if (part < 0 || part >= a.c.n_pages) {
            bad = true;
            part = -1;
        }
    }
    slot_of[tid] = slot;
    part_of[tid] = part;
    if (tid == 0) wanted = 0;
    __syncthreads();
    /* the same slot twice; how many of the batch write to this page, and
     * whether a later one does.  Four of the batch per LDS read, counts in
     * place of truth values: 256 sequences one at a time made the kernel 39 us
     * long instead of 13. */
    int named = 0, writers = 0, last = 0;
    if (live) {
#pragma unroll 4
        for (int j = 0; j < a.n; j += 4) {
            const int4 sl = *(const int4 *)(slot_of + j), pt = *(const int4 *)(part_of + j);
            const int s4[4] = {sl.x, sl.y, sl.z, sl.w}, p4[4] = {pt.x, pt.y, pt.z, pt.w};
#pragma unroll
            for (int k = 0; k < 4; k++) {
                named += s4[k] == slot;
                writers += p4[k] == part;
                last = p4[k] == part ? j + k : last;
            }
        }
        bad |= named != 1;
    }
    const bool later = last > tid;
    if (__syncthreads_or(bad)) {
        pg_refuse(a, -1);
        return;
    }
    bool copy = false;
    if (part >= 0) {
        const int held = qk_ld(a.c.refs + part);
        copy = held > 1 && (later || held > writers);
    }
    const int e1 = len - e0 * R > 0 ? e0 + 1 : e0; /* first entry without a page */
    const int fresh = live ? (int)pg_div_of(a.c.page_rows, (uint32_t)(len + add + R - 1)) - e1 : 0;
    /* one page more than the pool has is past it whatever the others need, and
     * 1024 such needs sum in 32 bits; a refused call sums them whole */
    const int need = min(max(fresh, 0), a.c.n_pages + 1) + copy;
    int total;
    const int base = pg_scan(need, tmp, total);
    base_of[tid] = base;
    first_of[tid] = copy ? e0 : e1;

    /* free pages below rank `total`, in order: wave w counts, then lists, its
     * own run of the pool */
    if (total > 0) {
        const int per = (a.c.n_pages + 16 * 256 - 1) / (16 * 256) * 256, p0 = wave * per, p1 = min(p0 + per, a.c.n_pages);
        int cnt = 0;
        for (int p = p0; p < p1; p += 256)
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const int x = p + 64 * q + lane;
                cnt += __popcll(__ballot(x < p1 && qk_ld(a.c.refs + min(x, a.c.n_pages - 1)) == 0));
            }
        int have, before = pg_scan(lane == 0 ? cnt : 0, tmp, have);
        before = __builtin_amdgcn_readfirstlane(before);
        if (have < total) {
            if (live) atomicAdd(&wanted, (unsigned long long)(max(fresh, 0) + copy));
            __syncthreads();
            pg_refuse(a, (int)min(wanted - (unsigned long long)have, 0x7FFFFFFFull));
            return;
        }
        for (int p = p0; p < p1 && before < total; p += 256)
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const int x = p + 64 * q + lane;
                const bool f = x < p1 && qk_ld(a.c.refs + min(x, a.c.n_pages - 1)) == 0;
                const uint64_t m = __ballot(f);
                const int r = before + pg_rank(m);
                if (f && r < total) a.free_pages[r] = x;
                before += __popcll(m);
            }
    }
    __syncthreads(); /* also makes the list visible to the workgroup */
    /* need k of the batch: its sequence is the last with base <= k */
    for (int k = tid; k < total; k += 1024) {
        int lo = 0, hi = a.n;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (base_of[mid] <= k) lo = mid;
            else hi = mid;
        }
        const int p = a.free_pages[k];
        a.c.table[slot_of[lo] * a.c.table_stride + first_of[lo] + k - base_of[lo]] = p;
        a.c.refs[p] = 1;
    }
    if (live) {
        if (copy) atomicSub(a.c.refs + part, 1);
        a.pairs[tid] = copy ? make_int2(part, a.free_pages[base]) : make_int2(-1, -1);
        a.c.lens[slot] = len + add;
    }
    if (tid == 0) {
        *a.status = 0;
        *a.n_pairs = a.n;
    }
}

static size_t pg_up(size_t v) { return (v + 255) / 256 * 256; }

extern "C" size_t qk_pg_reserve_ws(const pg_cache *c, int n_seqs) {
    return 256 + pg_up((size_t)n_seqs * 8) + pg_up((size_t)c->n_pages * 4);
}

extern "C" int qk_launch_pg_reserve(const pg_cache *c, const int32_t *slots, const int32_t *n_new, int n_seqs,
                                    int32_t *status, void *ws, void *stream) {
    hipStream_t st = (hipStream_t)stream;
    PgReserve a;
    PgCopy p;
    a.c = *c;
    a.slots = slots; a.n_new = n_new; a.n = n_seqs; a.status = status;
    a.n_pairs = (int32_t *)ws;
    a.pairs = (int2 *)((char *)ws + 256);
    a.free_pages = (int32_t *)((char *)a.pairs + pg_up((size_t)n_seqs * 8));
    hipLaunchKernelGGL(k_pg_reserve, dim3(1), dim3(1024), 0, st, a);
    const int rc = QK_CHECK_LAUNCH();
    if (rc || n_seqs == 0) return rc;
    pg_copy_dims(&p, c);
    p.pairs = a.pairs;
    p.n_pairs = a.n_pairs;
    p.n = n_seqs;
    hipLaunchKernelGGL(k_pg_copy, dim3(pg_copy_grid(c, n_seqs)), dim3(256), 0, st, p);
    return QK_CHECK_LAUNCH();
}

/* ------------------------------------------------------------ fork
 * Two launches, so that every source is read before any table is written
 * (beams that take each other's places).  One workgroup per pair.  Bound:
 * latency: 256 pairs of tables of 250 entries 3.9 + 5.3 us. */
struct PgFork {
    pg_cache c;
    const int32_t *src, *dst, *rows;
    int n;
    int32_t *status;
    int32_t *entries; /* [n, max_pages] */
    int2 *head;       /* [n]: (new length, refused) */
};

__global__ __launch_bounds__(256) void k_pg_fork_read(PgFork a) {
    const int i = blockIdx.x, tid = threadIdx.x;
    const int s = qk_ld(a.src + i), d = qk_ld(a.dst + i);
    bool bad = s < 0 || s >= a.c.n_slots || d < 0 || d >= a.c.n_slots;
    for (int j = tid; j < a.n; j += 256) bad |= j != i && qk_ld(a.dst + j) == d;
    bad = __syncthreads_or(bad);
    int len = 0;
    if (!bad) {
        len = min(max(qk_ld(a.c.lens + s), 0), a.c.cap);
        if (a.rows) len = min(max(qk_ld(a.rows + i), 0), len);
        const int keep = (int)pg_div_of(a.c.page_rows, (uint32_t)(len + (int)a.c.page_rows.d - 1));
        const int32_t *row = a.c.table + s * a.c.table_stride;
        for (int e = tid; e < keep; e += 256) a.entries[(int64_t)i * a.c.max_pages + e] = qk_ld(row + e);
    }
    if (tid == 0) a.head[i] = make_int2(len, bad);
}

__global__ __launch_bounds__(256) void k_pg_fork_write(PgFork a) {
    const int i = blockIdx.x, tid = threadIdx.x;
    bool bad = false;
    for (int j = tid; j < a.n; j += 256) bad |= qk_ld(a.head + j).y != 0;
    if (__syncthreads_or(bad)) {
        if (i == 0 && tid == 0) *a.status = -1;
        return;
    }
    if (i == 0 && tid == 0) *a.status = 0;
    const int d = qk_ld(a.dst + i), len = qk_ld(a.head + i).x;
    const int keep = (int)pg_div_of(a.c.page_rows, (uint32_t)(len + (int)a.c.page_rows.d - 1));
    int32_t *row = a.c.table + d * a.c.table_stride;
    for (int e = tid; e < a.c.max_pages; e += 256) {
        const int was = qk_ld(row + e), now = e < keep ? qk_ld(a.entries + (int64_t)i * a.c.max_pages + e) : -1;
        if (was == now) continue;
        if (was >= 0 && was < a.c.n_pages) atomicSub(a.c.refs + was, 1);
        if (now >= 0 && now < a.c.n_pages) atomicAdd(a.c.refs + now, 1);
        row[e] = now;
    }
    if (tid == 0) a.c.lens[d] = len;
}

/* The same in one launch, one workgroup, for batches whose entries fit LDS
 * (empty ones, which report too, among them): four branches of a short prompt
 * 3.1 us. */
#define PG_FORK_SMALL 12288
__global__ __launch_bounds__(1024) void k_pg_fork_small(PgFork a) {
    __shared__ int32_t entries[PG_FORK_SMALL];
    __shared__ int dst[PG_MAX_BATCH], len_of[PG_MAX_BATCH];
    const int tid = threadIdx.x, W = a.c.max_pages, R = (int)a.c.page_rows.d;
    bool bad = false;
    if (tid < a.n) {
        const int s = qk_ld(a.src + tid), d = qk_ld(a.dst + tid);
        bad = s < 0 || s >= a.c.n_slots || d < 0 || d >= a.c.n_slots;
        int len = bad ? 0 : min(max(qk_ld(a.c.lens + s), 0), a.c.cap);
        if (a.rows) len = min(max(qk_ld(a.rows + tid), 0), len);
        dst[tid] = d;
        len_of[tid] = len;
    }
    __syncthreads();
    if (tid < a.n)
        for (int j = 0; j < a.n; j++) bad |= j != tid && dst[j] == dst[tid];
    if (__syncthreads_or(bad)) {
        if (tid == 0) *a.status = -1;
        return;
    }
    for (int x = tid; x < a.n * W; x += 1024) {
        const int i = x / W, e = x - i * W;
        const bool keep = e < (int)pg_div_of(a.c.page_rows, (uint32_t)(len_of[i] + R - 1));
        entries[x] = keep ? qk_ld(a.c.table + qk_ld(a.src + i) * a.c.table_stride + e) : -1;
    }
    __syncthreads();
    for (int x = tid; x < a.n * W; x += 1024) {
        const int i = x / W, e = x - i * W;
        int32_t *at = a.c.table + dst[i] * a.c.table_stride + e;
        const int was = qk_ld(at), now = entries[x];
        if (was == now) continue;
        if (was >= 0 && was < a.c.n_pages) atomicSub(a.c.refs + was, 1);
        if (now >= 0 && now < a.c.n_pages) atomicAdd(a.c.refs + now, 1);
        *at = now;
    }
    if (tid < a.n) a.c.lens[dst[tid]] = len_of[tid];
    if (tid == 0) *a.status = 0;
}

extern "C" size_t qk_pg_fork_ws(const pg_cache *c, int n_seqs) {
    return pg_up((size_t)n_seqs * 8) + pg_up((size_t)n_seqs * c->max_pages * 4);
}

extern "C" int qk_launch_pg_fork(const pg_cache *c, const int32_t *src, const int32_t *dst, const int32_t *rows,
                                 int n_seqs, int32_t *status, void *ws, void *stream) {
    hipStream_t st = (hipStream_t)stream;
    PgFork a;
    a.c = *c;
    a.src = src; a.dst = dst; a.rows = rows; a.n = n_seqs; a.status = status;
    a.head = (int2 *)ws;
    a.entries = (int32_t *)((char *)ws + pg_up((size_t)n_seqs * 8));
    if ((int64_t)n_seqs * c->max_pages <= PG_FORK_SMALL) {
        hipLaunchKernelGGL(k_pg_fork_small, dim3(1), dim3(1024), 0, st, a);
        return QK_CHECK_LAUNCH();
    }
    hipLaunchKernelGGL(k_pg_fork_read, dim3(n_seqs), dim3(256), 0, st, a);
    const int rc = QK_CHECK_LAUNCH();
    if (rc) return rc;
    hipLaunchKernelGGL(k_pg_fork_write, dim3(n_seqs), dim3(256), 0, st, a);
    return QK_CHECK_LAUNCH();
}

/* ------------------------------------------------------------ evict
 * Pages whose rows no later query of the slot can see.  An entry is taken
 * out with an exchange, so a slot that is named twice releases it once.
 * Bound: latency, 4.2 us for 256 slots. */
struct PgEvict {
    pg_cache c;
    const int32_t *slots;
    int n, window, sinks;
};

__global__ __launch_bounds__(256) void k_pg_evict(PgEvict a) {
    const int R = (int)a.c.page_rows.d;
    for (int64_t i = blockIdx.x; i < a.n; i += gridDim.x) {
        const int slot = a.slots ? qk_ld(a.slots + i) : (int)i;
        if (slot < 0 || slot >= a.c.n_slots) continue;
        /* the next query is at position len at the least */
        const int len = min(max(qk_ld(a.c.lens + slot), 0), a.c.cap), lo = pg_lo(len, a.window);
        int32_t *row = a.c.table + slot * a.c.table_stride;
        for (int e = threadIdx.x; (e + 1) * R <= lo; e += 256) {
            if (e * R < a.sinks) continue;
            const int was = atomicExch(row + e, -1);
            if (was >= 0 && was < a.c.n_pages) atomicSub(a.c.refs + was, 1);
        }
    }
}

extern "C" int qk_launch_pg_evict(const pg_cache *c, const int32_t *slots, int n_seqs, int window, int sinks,
                                  void *stream) {
    PgEvict a;
    a.c = *c;
    a.slots = slots; a.n = n_seqs; a.window = window; a.sinks = sinks;
    hipLaunchKernelGGL(k_pg_evict, dim3(n_seqs < 65536 ? n_seqs : 65536), dim3(256), 0, (hipStream_t)stream, a);
    return QK_CHECK_LAUNCH();
}

/* ------------------------------------------------------------ compact
 * U used pages: the used pages from U on, in order, move to the free pages
 * below U, in order (as many of the one as of the other), so no move's
 * destination is another's source.  One workgroup finds the moves, then one
 * launch copies them and rewrites the tables.  Bound: HBM, the moved pages: of
 * 4096 half used pages of 12 layers (405 MB) 7 us for the plan and 81 for the
 * move, 5.0 TB/s; of 256 in one layer 4 + 4.5. */
struct PgCompact {
    PgCopy p;
    int32_t *used, *n_moves, *to; /* to [n_pages]: where a page is afterwards */
    int2 *moves;
};

__global__ __launch_bounds__(1024) void k_pg_compact_plan(PgCompact a) {
    __shared__ int tmp[16];
    const pg_cache &c = a.p.c;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int per = (c.n_pages + 16 * 256 - 1) / (16 * 256) * 256, p0 = wave * per, p1 = min(p0 + per, c.n_pages);
    auto used_at = [&](int x) { return x < p1 && qk_ld(c.refs + min(x, c.n_pages - 1)) > 0; };
    int cnt = 0;
    for (int p = p0; p < p1; p += 256)
#pragma unroll
        for (int q = 0; q < 4; q++) cnt += __popcll(__ballot(used_at(p + 64 * q + lane)));
    int used;
    int before = pg_scan(lane == 0 ? cnt : 0, tmp, used);
    before = __builtin_amdgcn_readfirstlane(before); /* used pages below p0 */
    /* the rank of a hole below `used` is x - (used pages below x); of a used
     * page from there on, (used pages below x) - (used pages below `used`):
     * the second needs that number, the moves */
    int holes = 0;
    for (int p = p0; p < min(p1, used); p += 256)
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const int x = p + 64 * q + lane;
            holes += __popcll(__ballot(x < min(p1, used) && !used_at(x)));
        }
    int moves;
    pg_scan(lane == 0 ? holes : 0, tmp, moves);
    for (int p = p0; p < p1; p += 256)
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const int x = p + 64 * q + lane;
            const bool u = used_at(x);
            const uint64_t m = __ballot(u);
            const int below = before + pg_rank(m); /* used pages below x */
            if (x < p1) {
                if (x < used && !u) a.moves[x - below].y = x;
                if (x >= used && u) a.moves[below - (used - moves)].x = x;
                a.to[x] = x;
            }
            before += __popcll(m);
        }
    __syncthreads();
    for (int i = tid; i < moves; i += 1024) {
        const int2 mv = a.moves[i];
        a.to[mv.x] = mv.y;
        c.refs[mv.y] = c.refs[mv.x];
        c.refs[mv.x] = 0;
    }
    if (tid == 0) {
        *a.used = used;
        *a.n_moves = moves;
    }
}

__global__ __launch_bounds__(256) void k_pg_compact_move(PgCompact a) {
    const pg_cache &c = a.p.c;
    const int n = qk_ld(a.n_moves);
    if (n == 0) return;
    for (int64_t i = blockIdx.x; i < (int64_t)n * 2 * c.n_layers; i += gridDim.x) pg_copy_item(a.p, i);
    for (int s = blockIdx.x; s < c.n_slots; s += gridDim.x) {
        int32_t *row = c.table + s * c.table_stride;
        for (int e = threadIdx.x; e < c.max_pages; e += 256) {
            const int p = qk_ld(row + e);
            if (p >= 0 && p < c.n_pages) row[e] = qk_ld(a.to + p);
        }
    }
}

extern "C" size_t qk_pg_compact_ws(const pg_cache *c) {
    return 256 + pg_up((size_t)c->n_pages * 4) + pg_up((size_t)c->n_pages * 4 + 8);
}

extern "C" int qk_launch_pg_compact(const pg_cache *c, int32_t *used, void *ws, void *stream) {
    hipStream_t st = (hipStream_t)stream;
    PgCompact a;
    pg_copy_dims(&a.p, c);
    a.used = used;
    a.n_moves = (int32_t *)ws;
    a.to = (int32_t *)((char *)ws + 256);
    a.moves = (int2 *)((char *)a.to + pg_up((size_t)c->n_pages * 4)); /* at most n_pages / 2 */
    a.p.pairs = a.moves;
    a.p.n_pairs = a.n_moves;
    a.p.n = c->n_pages / 2;
    hipLaunchKernelGGL(k_pg_compact_plan, dim3(1), dim3(1024), 0, st, a);
    const int rc = QK_CHECK_LAUNCH();
    if (rc) return rc;
    hipLaunchKernelGGL(k_pg_compact_move, dim3(2048), dim3(256), 0, st, a);
    return QK_CHECK_LAUNCH();
}
