/*
 * paged_parts.h -- index arithmetic of the paged cache, shared by the
 * kernels, the host checks and a CPU test (tests/c/paged_index.c): where a
 * cached row lies, which keys a run of query rows sees, and how the work of
 * an attention call is cut into units.  Plain C, no HIP calls.
 */
#ifndef PAGED_PARTS_H
#define PAGED_PARTS_H

#include "qmoe_internal.h"

/* functions that read what the cache holds: device memory for the kernels,
 * host memory for the CPU test */
#ifdef __HIPCC__
#define PG_FN __device__ static inline
#define PG_GET(p) qk_ld(p)
#else
#define PG_FN static inline
#define PG_GET(p) (*(p))
#endif

/* x / d for 0 <= x < 2^31 as one multiply and a shift: with
 * 2^s >= d > 2^(s-1) and mul = ceil(2^(31+s) / d), mul * d - 2^(31+s) < d <=
 * 2^s, so the quotient's excess x * (mul * d - 2^(31+s)) / (d * 2^(31+s)) is
 * below 1/d and never reaches the next integer; mul fits 32 bits. */
QK_HD static inline pg_div pg_div_make(uint32_t d) {
    pg_div r;
    uint32_t s = 0;
    while (((uint64_t)1 << s) < d) s++;
    r.mul = (uint32_t)((((uint64_t)1 << (31 + s)) + d - 1) / d);
    r.shift = 31 + s;
    r.d = d;
    return r;
}
QK_HD static inline uint32_t pg_div_of(pg_div v, uint32_t x) { return (uint32_t)(((uint64_t)x * v.mul) >> v.shift); }

QK_HD static inline int pg_min(int a, int b) { return a < b ? a : b; }
QK_HD static inline int pg_max(int a, int b) { return a > b ? a : b; }

/* element offset of row j of a sequence in the k and v pages of a layer, or
 * -1 when the row has no page: past the table, or an entry that is no page
 * of the pool (-1 where a page was released) */
PG_FN int64_t pg_row_at(const pg_cache *c, const int32_t *row, int j) {
    if (j < 0 || j >= c->cap) return -1;
    const uint32_t e = pg_div_of(c->page_rows, (uint32_t)j);
    const int32_t p = PG_GET(row + e);
    if (p < 0 || p >= c->n_pages) return -1;
    return (int64_t)p * c->page_stride + (int64_t)((uint32_t)j - e * c->page_rows.d) * c->row_stride;
}

/* one sequence of a batch: its rows [start, start + count) of the call, its
 * slot (-1: none, nothing of it is read) and its cached rows with the new
 * ones.  Whatever the device holds is brought into range here: the rows into
 * [0, n), the length into [0, table rows]. */
typedef struct {
    int slot, start, count, len;
} pg_seq;
PG_FN pg_seq pg_seq_at(const pg_cache *c, const int32_t *starts, const int32_t *slots, int n, int i) {
    pg_seq s;
    const int a = PG_GET(starts + i), b = PG_GET(starts + i + 1);
    s.start = pg_min(pg_max(a, 0), n);
    s.count = pg_max(pg_min(b, n) - s.start, 0);
    s.slot = slots ? PG_GET(slots + i) : i;
    if (s.slot < 0 || s.slot >= c->n_slots) s.slot = -1;
    s.len = s.slot < 0 ? 0 : pg_min(pg_max(PG_GET(c->lens + s.slot), 0), c->cap);
    return s;
}

/* keys that the query at position p sees: [lo, p] and [0, sinks) below lo */
QK_HD static inline int pg_lo(int p, int window) { return window > 0 && p >= window ? p - window + 1 : 0; }
QK_HD static inline int pg_sees(int p, int j, int window, int sinks) {
    return j <= p && (j >= pg_lo(p, window) || j < sinks);
}

/* tiles of kt keys that any query at positions p0..p1 sees: tile i of nt is
 * i for i < st (sinks) and ms + i - st after them */
typedef struct {
    int st, ms, nt;
} pg_tiles;
QK_HD static inline pg_tiles pg_tiles_of(int p0, int p1, int window, int sinks, int kt) {
    pg_tiles t;
    t.st = t.ms = t.nt = 0;
    if (p1 < 0) return t;
    const int lo = pg_lo(pg_max(p0, 0), window), s = pg_min(sinks, lo), end = p1 / kt + 1;
    t.ms = lo / kt;
    t.st = s > 0 ? (s - 1) / kt + 1 : 0;
    if (t.st >= t.ms) t.st = t.ms = 0;
    t.nt = t.st + end - t.ms;
    return t;
}
QK_HD static inline int pg_tile(pg_tiles t, int i) { return i < t.st ? i : t.ms + i - t.st; }

/* The work of an attention call: rows (token, head of a kv head's group) of a
 * sequence in tiles of rt, the keys of a row tile in `parts` ranges of about
 * `share` key tiles.  Units are numbered by sequence, then row tile (last
 * first: under a causal mask it has the most keys), part and kv head; tasks =
 * (sequence, row tile, kv head). */
typedef struct {
    int row_tiles, key_tiles; /* key tiles of the last row tile, the longest of the sequence (to one tile) */
    float work;               /* row_tiles times the mean of the first and last row tile's key tiles */
} pg_load;
QK_HD static inline pg_load pg_load_of(pg_seq s, int G, int rt, int window, int sinks, int kt) {
    pg_load l;
    const int rows = s.count * G;
    l.row_tiles = (rows + rt - 1) / rt;
    l.key_tiles = 0;
    l.work = 0.0f;
    if (l.row_tiles > 0) {
        const int p = s.len - s.count, t0 = (l.row_tiles - 1) * rt / G;
        l.key_tiles = pg_tiles_of(p + t0, s.len - 1, window, sinks, kt).nt;
        l.work = (float)l.key_tiles;
        if (l.row_tiles > 1)
            l.work = (float)l.row_tiles * 0.5f *
                     ((float)l.key_tiles + (float)pg_tiles_of(p, p + pg_min((rt - 1) / G, s.count - 1), window, sinks, kt).nt);
    }
    return l;
}
/* Key tiles per part, from the units that fill the card: a run of total / units
 * tiles, and `extra` tiles more, what storing and joining a part costs in
 * time.  total = the sum of `work` over the sequences, per_unit =
 * pg_per_unit(kv heads, units).  total is at least half of the sum of
 * row_tiles * key_tiles, so there are at most 2 units + tasks parts; a task of
 * parts > 1 has 1.5 shares at least, so at most 3 units of them belong to
 * such.  fp32 sums of 64 terms and a tree are off by less than 2^-17, which the
 * factor in per_unit covers. */
QK_HD static inline float pg_per_unit(int kvh, int units) { return 1.0001f * (float)kvh / (float)units; }
QK_HD static inline int pg_share(float total, float per_unit, int extra) {
    const float s = total * per_unit;
    return (s < 1e9f ? (int)s : 1000000000) + 1 + extra;
}
/* a task that is cut at all: into two parts by the smallest share there is */
QK_HD static inline int pg_cuts(int key_tiles, int extra) { return key_tiles + (extra + 1) / 2 >= 2 * (extra + 1); }
/* to the nearest: a task of 1.4 shares is not worth a join.  Key tiles and
 * shares are below 2^30 each. */
QK_HD static inline int pg_parts(int key_tiles, int share) {
    const int n = (int)(((uint32_t)key_tiles + (uint32_t)share / 2) / (uint32_t)share);
    return n < 1 ? 1 : n;
}
/* first of nt key tiles of part i: the first nt % parts parts have one more */
QK_HD static inline int pg_part(int nt, int i, int parts) {
    const uint32_t q = (uint32_t)nt / (uint32_t)parts, r = (uint32_t)nt - q * (uint32_t)parts;
    return (int)(q * (uint32_t)i) + pg_min(i, (int)r);
}

#endif
