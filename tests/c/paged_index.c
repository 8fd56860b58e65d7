/*
 * paged_index.c -- the paged cache's index arithmetic (csrc/paged_parts.h)
 * against plain restatements, on the CPU: division by multiplication, rows
 * and bad table entries, clamped batches, the key tiles that a run of
 * queries sees, and the cut of the tiles into parts.  Prints "ok" or the
 * first difference.
 */
#include <stdio.h>
#include <stdlib.h>

#include "paged_parts.h"

#define CHECK(x, ...)                          \
    do {                                       \
        if (!(x)) {                            \
            printf("line %d: ", __LINE__);     \
            printf(__VA_ARGS__);               \
            printf("\n");                      \
            exit(1);                           \
        }                                      \
    } while (0)

static uint32_t rng_state = 12345;
static uint32_t rnd(void) {
    rng_state = rng_state * 1664525u + 1013904223u;
    return rng_state >> 8 ^ rng_state << 13;
}

static void division(void) {
    for (uint32_t d = 1; d <= 5000; d++) {
        const pg_div v = pg_div_make(d);
        const uint32_t at[] = {0, 1, d - 1, d, d + 1, 2 * d - 1, 2 * d, 0x7FFFFFFF, 0x7FFFFFFF / d * d, 0x7FFFFFFF / d * d - 1};
        for (unsigned i = 0; i < sizeof(at) / sizeof(at[0]); i++)
            CHECK(at[i] > 0x7FFFFFFF || pg_div_of(v, at[i]) == at[i] / d, "%u / %u", at[i], d);
        for (int i = 0; i < 200; i++) {
            const uint32_t x = rnd() & 0x7FFFFFFF;
            CHECK(pg_div_of(v, x) == x / d, "%u / %u", x, d);
        }
    }
    for (int i = 0; i < 200000; i++) { /* chunk counts of large pages */
        const uint32_t d = 1 + (rnd() & 0x0FFFFFFF), x = rnd() & 0x7FFFFFFF;
        CHECK(pg_div_of(pg_div_make(d), x) == x / d, "%u / %u", x, d);
    }
}

static void rows(void) {
    int32_t table[3][7] = {{4, 0, 9, -1, 10, 2147483647, 3}, {-2147483647 - 1, 5, 5, 5, 5, 5, 5}, {1, 2, 3, 4, 5, 6, 7}};
    int32_t lens[3] = {5, -3, 1 << 30}, starts[5] = {-4, 2, 2, 1, 99}, slots[4] = {2, 0, 3, -1};
    pg_cache c = {0};
    c.n_pages = 10;
    c.max_pages = 7;
    c.page_rows = pg_div_make(5);
    c.cap = 35;
    c.page_stride = (int64_t)1 << 33;
    c.row_stride = 192;
    c.table = &table[0][0];
    c.table_stride = 7;
    c.n_slots = 3;
    c.lens = lens;
    for (int s = 0; s < 3; s++)
        for (int j = -70; j < 80; j++) {
            const int64_t got = pg_row_at(&c, table[s], j);
            int64_t want = -1;
            if (j >= 0 && j < 35 && table[s][j / 5] >= 0 && table[s][j / 5] < 10)
                want = table[s][j / 5] * ((int64_t)1 << 33) + j % 5 * 192;
            CHECK(got == want, "row %d of slot %d: %lld, not %lld", j, s, (long long)got, (long long)want);
        }
    for (int n = 0; n < 8; n++)
        for (int i = 0; i < 4; i++) {
            const pg_seq a = pg_seq_at(&c, starts, slots, n, i);
            CHECK(a.start >= 0 && a.count >= 0 && a.start + a.count <= n, "sequence %d of %d rows: %d + %d", i, n, a.start, a.count);
            CHECK(a.len >= 0 && a.len <= 35 && (a.slot >= 0 || a.len == 0) && a.slot < 3, "slot %d length %d", a.slot, a.len);
        }
    CHECK(pg_seq_at(&c, starts, NULL, 2, 1).slot == 1 && pg_seq_at(&c, starts, NULL, 2, 1).len == 0, "slot 1");
    CHECK(pg_seq_at(&c, starts, NULL, 2, 3).slot == -1, "slot 3");
}

static void tiles(void) {
    for (int it = 0; it < 60000; it++) {
        const int kt = 32 << (rnd() % 3), len = rnd() % 700, count = 1 + rnd() % 40;
        const int window = rnd() % 3 ? 1 + (int)(rnd() % 300) : 0, sinks = window ? (int)(rnd() % 2 ? rnd() % 200 : 0) : 0;
        const int p1 = len - 1 - (int)(rnd() % count), p0 = p1 - (int)(rnd() % count);
        const pg_tiles t = pg_tiles_of(p0, p1, window, sinks, kt);
        int last = -1, i = 0;
        CHECK(t.nt >= 0, "count");
        for (; i < t.nt; i++) {
            const int k = pg_tile(t, i);
            CHECK(k > last && k * kt <= (p1 > 0 ? p1 : 0), "tile %d after %d", k, last);
            last = k;
        }
        for (int j = 0; j < len; j++) {
            int seen = 0, in = 0;
            for (int p = p0; p <= p1; p++) {
                const int vis = j <= p && (window == 0 || p - j < window || j < sinks);
                CHECK(pg_sees(p, j, window, sinks) == vis, "p %d j %d window %d sinks %d", p, j, window, sinks);
                seen |= p >= 0 && vis;
            }
            if (!seen) continue;
            for (i = 0; i < t.nt; i++) in += pg_tile(t, i) == j / kt;
            CHECK(in == 1, "key %d of p %d..%d window %d sinks %d: in %d tiles", j, p0, p1, window, sinks, in);
        }
    }
    /* the largest arguments stay in range */
    const pg_tiles t = pg_tiles_of((1 << 30) - 2, (1 << 30) - 1, 2147483647, 2147483647, 32);
    CHECK(t.nt == 1 << 25 && t.st == 0, "%d", t.nt);
    const pg_tiles u = pg_tiles_of((1 << 30) - 2, (1 << 30) - 1, 1, 2147483647, 32);
    CHECK(u.nt == 1 << 25, "%d", u.nt);
}

/* every unit of a batch is numbered once, parts cover the tiles in order */
static void units(void) {
    for (int it = 0; it < 3000; it++) {
        const int G = 1 + rnd() % 12, rt = rnd() % 2 ? 32 : 128, kt = 64, window = rnd() % 2 ? 100 : 0, sinks = rnd() % 20;
        const int n_seqs = 1 + rnd() % 6, want = 1 + rnd() % 600;
        pg_seq s[6];
        float total = 0.0f;
        int64_t most = 0, n_units = 0, tasks = 0, split = 0, rows = 0;
        for (int i = 0; i < n_seqs; i++) {
            s[i].slot = s[i].start = 0;
            s[i].count = rnd() % 300;
            s[i].len = rnd() % 5000;
            rows += s[i].count;
            const pg_load l = pg_load_of(s[i], G, rt, window, sinks, kt);
            CHECK(l.row_tiles == (s[i].count * G + rt - 1) / rt, "row tiles");
            total += l.work;
            most += (int64_t)l.row_tiles * l.key_tiles;
        }
        const int share = pg_share(total, pg_per_unit(1, want), 1 + rnd() % 8);
        for (int i = 0; i < n_seqs; i++) {
            const pg_load l = pg_load_of(s[i], G, rt, window, sinks, kt);
            const int parts = pg_parts(l.key_tiles, share);
            n_units += (int64_t)l.row_tiles * parts;
            tasks += l.row_tiles;
            if (parts > 1) split += (int64_t)l.row_tiles * parts;
            for (int nt = 0; nt < 40; nt += 7) {
                CHECK(pg_part(nt, 0, parts) == 0 && pg_part(nt, parts, parts) == nt, "parts");
                for (int p = 0; p < parts; p++) CHECK(pg_part(nt, p, parts) <= pg_part(nt, p + 1, parts), "order");
            }
            for (int r = 0; r < l.row_tiles; r++) { /* no row tile has many more tiles than the last */
                const int t0 = r * rt / G, t1 = pg_min((r * rt + rt - 1) / G, s[i].count - 1);
                CHECK(pg_tiles_of(s[i].len - s[i].count + t0, s[i].len - s[i].count + t1, window, sinks, kt).nt <=
                          l.key_tiles + 2 + rt / kt, "row tile %d", r);
            }
        }
        CHECK(2 * (double)total >= (double)most, "%g of %lld", (double)total, (long long)most);
        CHECK(n_units <= 2 * (int64_t)want + tasks, "%lld units of %d + %lld", (long long)n_units, want, (long long)tasks);
        CHECK(split <= 3 * (int64_t)want, "%lld split units of %d", (long long)split, want);
        CHECK(tasks <= rows * G / rt + n_seqs, "tasks");
    }
}

int main(void) {
    division();
    rows();
    tiles();
    units();
    printf("ok\n");
    return 0;
}
