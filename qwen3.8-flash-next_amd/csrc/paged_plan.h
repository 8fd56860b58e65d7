/*
 * paged_plan.h -- how a paged attention call is cut and launched: the rows of
 * a unit, the grid that holds the units whatever the lengths on the device, and
 * where partial results, records and the index lie in the workspace.  Host
 * code without HIP calls, shared by the launches (paged_attn.hip) and a CPU test
 * (tests/c/paged_plan.cpp).
 */
#ifndef PAGED_PLAN_H
#define PAGED_PLAN_H

#include "paged_parts.h"

#define PM_RT 128   /* rows of a unit of the many-row kernels */
#define PD_KT 32    /* keys of a tile of the few-row kernels */
#define PA_INDEX 64 /* sequences up to which a unit is found without an index (k_pa_index) */
#define PA_JOIN 10  /* tiles that a part of a tree's task has to save (pa_length) */

/* keys of a tile of the many-row kernels */
constexpr int pm_kt(int hd, bool f32 = false) { return hd <= 128 && !f32 ? 64 : 32; }
/* groups of four waves in a unit of k_pa_many32: head dims past 128 fill four waves' registers and LDS */
constexpr int pm_halves32(int hd) { return hd <= 128 ? 2 : 1; }

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
/* The same for trees, whose units of PM_RT rows start sooner and are joined
 * sooner: those of bf16 take over wherever the table's keys (or the window's)
 * are enough to be cut (with fewer rows, and with more: 8 nodes of a sequence
 * of 300 rows 13.6 us and 17.8, of 1000 17.8 and 14.9, of 32000 38 and 26; 4 of
 * 16 of 4000 33 and 26; one of 64 of 6000 89 and 84), at head dim 192 from 17
 * rows of a sequence on (24 of 16 of 4000 41 and 38; 6 of 64 85 and 86), at 256
 * from 33 rows and 40 units of 16 (32 of 48 of 2000 49 and 59, 64 of 16 of 4000
 * 103 and 67; 96 of 4 of 3000 43 and 45).  With fewer keys, and in f32, they come
 * after units of 16 or 32 rows, in f32 at a quarter of a prompt's limit (16 nodes
 * of a sequence of 8000 41 and 35, 4 of 64 of 2000 94 and 104); at f32's head dim
 * 256, whose many rows spill, later up to 256 rows a sequence (20 nodes of 16 of
 * 2000 88 and 123, 60 of 4 of 3000 82 and 102, 150 of 4 of 2000 190 and 145). */
#define PA_TREE_KEYS ((PA_JOIN + 1) * 64)
static bool pa_tree_many(const pg_cache *c, int64_t rows, int n_seqs) {
    if (c->dtype != QMOE_BF16) return false;
    return c->hd <= 128 || (c->hd == 192 ? rows > (int64_t)16 * n_seqs : rows > (int64_t)32 * n_seqs && rows * c->kvh > 640);
}
/* keys that a row sees at the most */
static int64_t pa_keys(const pg_cache *c, int window, int sinks) {
    return window > 0 && (int64_t)window + sinks < c->cap ? (int64_t)window + sinks : c->cap;
}
/* The units that a call of n rows may run on, whatever its window: `early`
 * while it is short, `later` past that, `many` where it is a tree whose keys
 * are enough to be cut (0: never).  The launch takes one of them (pa_rows) and
 * the workspace holds each (pa_ws). */
struct PaChoice {
    int early, later, many;
};
static PaChoice pa_choice(const pg_cache *c, int n, int n_seqs, int h, bool tree) {
    const int64_t rows = (int64_t)n * (h / c->kvh);
    const PaChoice q = {16, pa_rows_long(c, rows, n_seqs), tree && pa_tree_many(c, rows, n_seqs) ? PM_RT : 0};
    return q;
}
static int pa_rows(const pg_cache *c, int n, int n_seqs, int h, int window, int sinks, bool tree) {
    const PaChoice q = pa_choice(c, n, n_seqs, h, tree);
    const int64_t rows = (int64_t)n * (h / c->kvh), units = rows * c->kvh / 16, keys = pa_keys(c, window, sinks);
    if (q.many && keys >= PA_TREE_KEYS) return q.many;
    int64_t most = c->dtype == QMOE_BF16 || c->hd == 64 ? 1 << 18 : c->hd < 256 ? 1 << 17 : 1 << 19;
    if (tree && c->dtype == QMOE_F32) most = c->hd == 64 ? 1 << 16 : c->hd < 256 ? 1 << 15 : rows <= (int64_t)256 * n_seqs ? 1 << 21 : 1 << 17;
    if (q.later == 32) most /= 2;
    return units <= 8 || units * keys <= most ? q.early : q.later;
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
static int pa_threads(const pg_cache *c, int n, int h, int rt) {
    if (rt != PM_RT) return 256;
    return 256 * (c->dtype == QMOE_BF16 ? pa_groups(c, n, h) : pm_halves32(c->hd));
}

/* Trees on units of PM_RT rows: as many units as run at once, two to a CU
 * where a unit is one group of four waves; the grid that holds the call's, the
 * slots of partial results and the tasks that may be cut. */
struct PaTreePlan {
    int units, slots, joins, twice;
    int64_t tasks, grid;
};
static int pa_tree_groups(const pg_cache *c) { return c->dtype == QMOE_BF16 && c->hd <= 128 ? 1 : 2; }
static PaTreePlan pa_tree_plan(const pg_cache *c, int n, int n_seqs, int h) {
    PaTreePlan q;
    q.units = pa_tree_groups(c) == 1 ? 512 : 256;
    const int64_t rows = (int64_t)n * (h / c->kvh), seqs = n_seqs < n ? n_seqs : n;
    const int64_t per_head = rows / PM_RT + seqs < rows ? rows / PM_RT + seqs : rows, tasks = per_head * c->kvh;
    const int64_t longest = c->cap / pm_kt(c->hd, c->dtype == QMOE_F32) + 2; /* tiles of a task */
    const bool cut = longest >= PA_JOIN + 1, even = tasks <= q.units;
    /* with 1024 units they may begin one after the other, 64 tiles each in the mean */
    q.twice = even && q.units == 512 && tasks * longest >= 64 * q.units;
    q.grid = even ? (q.twice ? 2 : 1) * q.units : tasks + q.units;
    if (q.grid > tasks * longest) q.grid = tasks * longest;
    q.tasks = tasks;
    q.slots = !cut ? 0 : (even && !q.twice ? 1 : 2) * q.units;
    q.joins = !cut ? 0 : (int)(even ? tasks : q.units);
    return q;
}

/* Where a call on units of rt rows has what, in bytes from the workspace's
 * start: maxima and sums, partial O, records of tasks that are cut (trees on
 * units of PM_RT rows), the index (more than PA_INDEX sequences), its end. */
struct PaLayout {
    size_t pml, po, split, index, end;
};
static size_t pa_up(size_t v) { return (v + 255) / 256 * 256; }
static PaLayout pa_layout(const pg_cache *c, int n, int n_seqs, int h, int rt, bool tree) {
    const bool cut = tree && rt == PM_RT; /* pa_tree_plan's */
    const PaTreePlan t = cut ? pa_tree_plan(c, n, n_seqs, h) : PaTreePlan();
    const size_t rows = (size_t)rt * (size_t)(cut ? t.slots : pa_plan_of(c, n, n_seqs, h, rt).slots);
    PaLayout l;
    l.pml = 0;
    l.po = pa_up(rows * 8);
    l.split = l.po + pa_up(rows * c->hd * 4);
    l.index = l.split + (cut ? pa_up((size_t)t.joins * 32) : 0);
    l.end = l.index + (n_seqs > PA_INDEX ? pa_up(((size_t)n_seqs + (cut ? 1 : 0)) * 16) : 0);
    return l;
}

/* threads of a launch, which HIP takes below 2^32.  Units of 16 rows that are
 * chosen because the call is short (pa_rows) are below 2^22, and more than the
 * longer ones would be. */
static bool pa_fits(const pg_cache *c, int n, int n_seqs, int h, int rt, bool tree) {
    if (tree && rt == PM_RT) return pa_tree_plan(c, n, n_seqs, h).grid * 512 <= 0xFFFFFFFFll;
    return pa_plan_of(c, n, n_seqs, h, rt).grid * pa_threads(c, n, h, rt) <= 0xFFFFFFFFll;
}
/* workspace of a call, of any window: the largest of what pa_rows may choose;
 * 0 where a launch does not fit */
static size_t pa_ws(const pg_cache *c, int n, int n_seqs, int h, bool tree) {
    const PaChoice q = pa_choice(c, n, n_seqs, h, tree);
    const int rt[3] = {q.early, q.later, q.many};
    size_t most = 0;
    for (int i = 0; i < 3; i++) {
        if (!rt[i]) continue;
        if (i > 0 && !pa_fits(c, n, n_seqs, h, rt[i], tree)) return 0;
        const size_t end = pa_layout(c, n, n_seqs, h, rt[i], tree).end;
        most = end > most ? end : most;
    }
    return 256 + most;
}

#endif
