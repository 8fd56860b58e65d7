/*
 * paged_plan.cpp -- the workspace of a paged attention call (csrc/paged_plan.h)
 * against what its launch takes of it, on the CPU: over types, head shapes,
 * tables, windows, sequences around the index's limit and rows a sequence, the
 * places of the units that are chosen lie apart from each other, each as large
 * as its plan says, and end inside the size that a caller is told, which knows
 * no window.  Prints "ok" or the first difference.
 */
#include <stdio.h>
#include <stdlib.h>

#include "paged_plan.h"

static long calls, on[3][2]; /* launches of 16, 32, PM_RT rows; causal, trees */

static void one(int dtype, int hd, int kvh, int G, int cap, int window, int sinks, int n_seqs, int n, bool tree) {
    pg_cache c = {};
    c.dtype = dtype;
    c.hd = hd;
    c.kvh = kvh;
    c.cap = cap;
    const int h = kvh * G;
    const size_t size = pa_ws(&c, n, n_seqs, h, tree);
    if (!size) return; /* refused */
    const int rt = pa_rows(&c, n, n_seqs, h, window, sinks, tree);
    const PaLayout l = pa_layout(&c, n, n_seqs, h, rt, tree);
    size_t slots, records, entries = n_seqs > PA_INDEX ? (size_t)n_seqs : 0;
    int64_t grid;
    if (tree && rt == PM_RT) {
        const PaTreePlan q = pa_tree_plan(&c, n, n_seqs, h);
        slots = (size_t)q.slots;
        records = (size_t)q.joins;
        if (entries) entries++; /* what they come to */
        grid = q.grid * 256 * (dtype == QMOE_BF16 ? pa_tree_groups(&c) : pm_halves32(hd));
    } else {
        const PaPlan q = pa_plan_of(&c, n, n_seqs, h, rt);
        slots = (size_t)q.slots;
        records = 0;
        grid = q.grid * pa_threads(&c, n, h, rt);
    }
    const size_t rows = slots * (size_t)rt;
    const bool fits = l.po >= l.pml + rows * 8 && l.split >= l.po + rows * (size_t)hd * 4 && l.index >= l.split + records * 32 &&
                      l.end >= l.index + entries * 16 && l.end <= size;
    const bool even = !((l.pml | l.po | l.split | l.index) & 15);
    if (!fits || !even || grid > 0xFFFFFFFFll) {
        printf("%s dtype %d, %d heads on %d of %d, table %d, window %d + %d, %d rows of %d sequences: units of %d, %zu slots, "
               "places %zu %zu %zu %zu %zu of %zu, %lld threads\n", tree ? "tree" : "causal", dtype, h, kvh, hd, cap, window, sinks,
               n, n_seqs, rt, slots, l.pml, l.po, l.split, l.index, l.end, size, (long long)grid);
        exit(1);
    }
    calls++;
    on[rt == 16 ? 0 : rt == 32 ? 1 : 2][tree]++;
}

int main() {
    const int types[] = {QMOE_BF16, QMOE_F32};
    const int hds[] = {64, 128, 192, 256};
    const int heads[][2] = {{1, 1}, {2, 1}, {2, 2}, {1, 4}, {2, 8}, {8, 1}, {8, 8}, {1, 40}, {3, 5}, {512, 1}, {64, 4}};
    const int caps[] = {1, 16, 500, 512, 513, 528, 544, 560, 575, 576, 577, 640, 688, 703, 704, 705, 1000, 2048, 4000, 12848, 30000, 1 << 20, 1 << 30};
    const int windows[][2] = {{0, 0}, {1, 0}, {64, 4}, {500, 3}, {512, 0}, {512, 16}, {700, 3}, {700, 4}, {704, 0}, {2000, 0}, {0x7FFFFFFF, 9}};
    const int seqs[] = {1, 2, 3, 8, 16, 48, 63, 64, 65, 66, 100, 128, 500, 1000, 1025, 65536};
    const int nodes[] = {1, 2, 3, 4, 5, 7, 8, 9, 12, 15, 16, 17, 20, 24, 31, 32, 33, 40, 64, 100, 129, 256, 257, 1024, 9000};
    for (int dtype : types)
        for (int hd : hds)
            for (const auto &x : heads)
                for (int cap : caps)
                    for (const auto &w : windows)
                        for (int m : seqs)
                            for (int k : nodes)
                                for (int tree = 0; tree < 2; tree++)
                                    for (int part = 0; part < 2; part++) { /* as many rows each; some sequences without */
                                        const int64_t n = part ? (int64_t)m * k * 3 / 4 + 1 : (int64_t)m * k;
                                        if (n * x[0] * x[1] > PG_MAX_ROWS) continue;
                                        one(dtype, hd, x[0], x[1], cap, w[0], w[1], m, (int)n, tree);
                                    }
    for (int i = 0; i < 3; i++)
        for (int t = 0; t < 2; t++)
            if (!on[i][t]) {
                printf("no %s call on units of %d rows\n", t ? "tree" : "causal", i == 0 ? 16 : i == 1 ? 32 : PM_RT);
                return 1;
            }
    if (calls < 1000000) {
        printf("%ld calls only\n", calls);
        return 1;
    }
    printf("ok\n");
    return 0;
}
