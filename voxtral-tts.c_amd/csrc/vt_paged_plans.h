/*
 * vt_paged_plans.h - a batch of sequences over a paged cache (vt_paged.hip): what is refused, and the attention's work items from shapes and the number of
 * CUs.  Host code without HIP, so that a host test can walk it.
 */
#ifndef VT_PAGED_PLANS_H
#define VT_PAGED_PLANS_H

#include <limits.h>
#include <math.h>
#include <stdint.h>
#include <stdlib.h>

#define PAGED_MAX_POS (1 << 30)            /* rows of a sequence */
#define PAGED_MAX_ROWS (1 << 22)           /* new rows of a batch */
#define PAGED_MAX_GROUP 4096               /* heads on a kv head */
#define PAGED_COUNTERS 16384               /* heads times tiles of columns that several workgroups share */

/* Columns are a sequence's new rows times the heads that share a kv head: column c is row c / group, head c % group of the group. Few columns: 16 or 32 to
 * a workgroup, whose waves take 32 rows of the cache each in turn.  Many: 128 to a workgroup, 64 rows at a time. */
#define PAGED_FEW_ROWS 32
#define PAGED_FEW_WAVES 4
#define PAGED_MANY_COLS 128
#define PAGED_MANY_ROWS 64
#define PAGED_MAX_PARTS 64
#define PAGED_CACHED 32e6                  /* bytes: all L2s */
#define PAGED_SPLIT_ITEMS 4096             /* items that a launch may have beyond one for each tile of columns */

/* What a workgroup does for every kv head: columns c0 .. of a sequence whose new rows are `row` .. of the batch and lie behind `past` rows, over the
 * cache's rows lo .. end - 1; `parts` of them make up the columns' result, in slots `slot` .. */
struct vt_paged_item { int row, past, cols, table, c0, lo, end, slot, part, parts, counter, many; };

struct vt_paged_shape { int n_pages, page_rows, n_heads, n_kv_heads, head_dim, window; };

/* NULL, or why the shape is none */
static inline const char *vt_paged_shape_bad(const vt_paged_shape &s) {
    if (s.page_rows < 16 || s.page_rows > 1 << 20 || (s.page_rows & (s.page_rows - 1))) return "page_rows is a power of two from 16 to 2^20";
    if (s.n_pages < 1) return "no pages";
    if (s.head_dim < 64 || s.head_dim > 256 || s.head_dim % 64) return "head_dim is 64, 128, 192 or 256";
    if (s.n_kv_heads < 1 || s.n_kv_heads > 65535 || s.n_heads < 1 || s.n_heads % s.n_kv_heads) return "n_heads is a multiple of n_kv_heads, which are at most 65535";
    if (s.n_heads / s.n_kv_heads > PAGED_MAX_GROUP) return "more than 4096 heads on a kv head";
    if ((long long)s.n_heads * s.head_dim > INT_MAX / 4) return "rows of more values than 2^29";
    if (s.window < 0) return "a negative window";
    return NULL;
}

/* rows of the cache that the new rows q0 .. q1 of a sequence see: from first on, up to past + q1 */
static inline int vt_paged_first(int window, int past, int q0) { return window && past + q0 >= window ? past + q0 - window + 1 : 0; }

static int vt_paged_by_value(const void *a, const void *b) {
    const int x = *(const int *)a, y = *(const int *)b;
    return x < y ? -1 : x > y;
}

/* The batch as the kernels read it: of each new row its position, page and row in the page, of each sequence its pages' numbers one behind the other from
 * `starts` on. */
struct vt_paged_rows { int *pos, *place, *tables, *starts, *written; };

enum { PAGED_OK, PAGED_COUNT, PAGED_SEQUENCE, PAGED_TOO_MANY_ROWS, PAGED_TABLE, PAGED_PAGE, PAGED_WRITTEN };
struct vt_paged_fault { int what, seq, at, value; };

/* Checks a batch and lays it out; `tables` [n_seqs, stride].  Entries of pages that no new row sees are not looked at. */
static inline vt_paged_fault vt_paged_lay_out(const vt_paged_shape &s, int max_seqs, int max_rows, int max_table, int n_seqs, const int *past, const int *rows,
                                              const int *tables, int stride, const vt_paged_rows &to, int *n_rows, int *n_table) {
    int at = 0, entry = 0, written = 0, log = 0;
    while (1 << log < s.page_rows) log++;
    if (n_seqs < 0 || n_seqs > max_seqs || stride < 0) return vt_paged_fault{PAGED_COUNT, 0, 0, 0};
    for (int i = 0; i < n_seqs; i++) {
        if (past[i] < 0 || rows[i] < 0 || (long long)past[i] + rows[i] > PAGED_MAX_POS) return vt_paged_fault{PAGED_SEQUENCE, i, 0, 0};
        if (rows[i] > max_rows - at) return vt_paged_fault{PAGED_TOO_MANY_ROWS, i, 0, 0};
        to.starts[i] = entry;
        if (rows[i] == 0) continue;
        const int pages = ((past[i] + rows[i] - 1) >> log) + 1, seen = vt_paged_first(s.window, past[i], 0) >> log, fresh = past[i] >> log;
        if (pages > stride || pages > max_table - entry) return vt_paged_fault{PAGED_TABLE, i, pages, 0};
        const int *from = tables + (size_t)i * stride;
        for (int p = 0; p < pages; p++) {
            if (p >= seen && (from[p] < 0 || from[p] >= s.n_pages)) return vt_paged_fault{PAGED_PAGE, i, p, from[p]};
            to.tables[entry + p] = p >= seen ? from[p] : 0;
            if (p >= fresh) to.written[written++] = from[p];
        }
        for (int r = 0; r < rows[i]; r++, at++) {
            const int pos = past[i] + r;
            to.pos[at] = pos;
            to.place[2 * at] = from[pos >> log];
            to.place[2 * at + 1] = pos & (s.page_rows - 1);
        }
        entry += pages;
    }
    /* a page that two sequences write to, or one twice, would hold whichever came last */
    qsort(to.written, written, sizeof(int), vt_paged_by_value);
    for (int i = 1; i < written; i++)
        if (to.written[i] == to.written[i - 1]) return vt_paged_fault{PAGED_WRITTEN, 0, 0, to.written[i]};
    *n_rows = at;
    *n_table = entry;
    return vt_paged_fault{PAGED_OK, 0, 0, 0};
}

/* ---- work items --- */

/* items of either kernel (the few's first), parts that they leave; wide: the few's columns go by 32; once: their rows are read by one workgroup each, but for
 * pages that sequences share (vt_paged_once), more of them than a cache holds */
struct vt_paged_plan { int few, many, few_slots, many_slot, many_slots, wide, once, both; };

/* Which kernels a batch goes to: `any`, whether there are sequences for the one for many columns; columns of a workgroup of the other, whether one workgroup
 * reads a sequence's rows, and their bytes */
struct vt_paged_kinds { bool any; int few_cols; bool once; double bytes; };

static inline long long vt_paged_max_items(int max_seqs, int max_rows, int group) {
    return (long long)max_rows * group / 16 + max_seqs + 2 * PAGED_SPLIT_ITEMS;
}

/* Which sequences go to the kernel for many columns: those of more than 64, where there is enough for it to do, as columns times the rows that they see on
 * average times kv heads times values, over all of them.  It does more with what it reads, but by few workgroups.  Measured, us with the kernel for few
 * columns, 32 at a time, and for many (fp32 / bf16), 32 heads on 8 of 128: 450 rows behind 200 (0.8e9) 18 / 16 and 26 / 20, 700 behind none (1.0e9) 25 / 21
 * and 27 / 20, 200 behind 2000 (1.7e9) 33 / 25 and 35 / 26, 50 behind 16000 (3.3e9) 61 / 48 and 64 / 47, 100 behind 500 sixteen times (3.6e9) 60 / 46 and
 * 51 / 34, 512 behind 1500 (3.7e9) 46 / 39 and 50 / 36; 16 heads of 64: 512 behind 1500 (0.9e9) 21 / 17 and 25 / 20.  One figure serves both types: fp32
 * calls of one sequence would do better by 5 to 10 % from 3e9 on with the other kernel up to about 4e9, several sequences of the same figure worse by 18.
 * Heads of 256 values leave it registers if they are bf16: 12 on 4, 300 behind 1000 (1.1e9) 28 and 34, 1000 behind none (1.5e9) 38 and 33, 200 behind 3000
 * (1.9e9) 50 and 45, 512 behind 1500 (2.8e9) 69 and 42, 3000 behind none (14e9) 245 and 130; fp32 it keeps some in memory and 3000 take 250 and 344.  Heads
 * of 192 do not lie as it reads them.
 *
 * Else 32 columns to a workgroup, not 16, where there is enough for that, as columns / 16 times rows times kv heads times values (less where every CU has
 * one of 16); 16 and 32 at a time: 37 rows behind 300 (3e6) 7.0 / 6.4 and 9.9 / 8.2, 100 behind 1000 (27e6) 13 / 13 and 19 / 15, 37 behind 4000 (41e6) 21 /
 * 21 and 23 / 20, 16 behind 300 32 times (40e6) 22 / 22 and 17 / 14, 200 behind 2000 (107e6) 42 / 41 and 32 / 24; 16 heads of 64: 37 behind 4000 (12e6) 14
 * / 13 and 17 / 16, 512 behind 1500 (57e6) 24 / 23 and 21 / 17. */
#define PAGED_MANY_FROM 2.5e9
#define PAGED_MANY_FROM_256 1.3e9
#define PAGED_WIDE_FROM 45e6
#define PAGED_WIDE_FULL 30e6
static inline bool vt_paged_may_be_many(int hp, long long cols) { return hp != 3 && cols > 64; }
/* .. and both kernels be one launch's */
static inline bool vt_paged_may_be_both(const vt_paged_shape &s, const vt_paged_kinds &kinds) { return s.head_dim <= 128 && kinds.few_cols == 16; }
static inline vt_paged_kinds vt_paged_kinds_of(const vt_paged_shape &s, bool bf16, int n_cu, int n_seqs, const int *past, const int *rows) {
    const int group = s.n_heads / s.n_kv_heads, hp = s.head_dim / 64;
    double many = 0, wide = 0, wgs = 0;
    long long most = 0;
    for (int i = 0; i < n_seqs; i++) {
        const long long cols = (long long)rows[i] * group;
        const double seen = past[i] + 0.5 * rows[i], each = (s.window && seen > s.window ? s.window : seen) * s.n_kv_heads * s.head_dim;
        if (vt_paged_may_be_many(hp, cols)) many += (double)cols * each;
    }
    vt_paged_kinds k = {hp <= 2 ? many >= PAGED_MANY_FROM : bf16 && many >= PAGED_MANY_FROM_256, 16, false, 0};
    for (int i = 0; i < n_seqs; i++) {
        const long long cols = (long long)rows[i] * group;
        const double seen = past[i] + 0.5 * rows[i], each = (s.window && seen > s.window ? s.window : seen) * s.n_kv_heads * s.head_dim;
        if (k.any && vt_paged_may_be_many(hp, cols)) continue;
        most = cols > most ? cols : most;
        k.bytes += ((double)past[i] + rows[i] - vt_paged_first(s.window, past[i], 0)) * 4 * s.n_kv_heads * s.head_dim;
        if (cols > 16) {
            wide += (double)((cols + 15) / 16) * each;
            wgs += (double)((cols + 15) / 16) * s.n_kv_heads;
        }
    }
    if (hp <= 2 && most > 16 && wide >= (wgs >= n_cu ? PAGED_WIDE_FULL : PAGED_WIDE_FROM)) k.few_cols = 32;
    k.once = most <= 16;
    return k;
}

/* A kernel's part of a batch.  Calls f(sequence, c0, first row, end) for every tile of columns. */
template <class F>
static inline void vt_paged_tiles(const vt_paged_shape &s, const vt_paged_kinds &kinds, bool many, int n_seqs, const int *past, const int *rows, F f) {
    const int group = s.n_heads / s.n_kv_heads, wide = many ? PAGED_MANY_COLS : kinds.few_cols, hp = s.head_dim / 64;
    for (int i = 0; i < n_seqs; i++) {
        const long long cols = (long long)rows[i] * group;
        if ((kinds.any && vt_paged_may_be_many(hp, cols)) != many) continue;
        for (long long c0 = 0; c0 < cols; c0 += wide) {
            const long long last = (c0 + wide < cols ? c0 + wide : cols) - 1;
            f(i, (int)c0, vt_paged_first(s.window, past[i], (int)(c0 / group)), past[i] + (int)(last / group) + 1);
        }
    }
}

/* rows of the cache that a part has: `run` steps of `unit` */
static inline int vt_paged_parts(int first, int end, int unit, int run) {
    const long long units = ((long long)end + unit - 1) / unit - first / unit;
    return (int)((units + run - 1) / run);
}

/* What a workgroup takes: `fixed` us, `step` for a unit of its rows, alone on its CU and with `beside` of them on it, `part` more where it leaves a part,
 * and `merge` for each of the parts that the last one adds; `tail`: the share of the longest that a launch of more than fit at once ends with.  By head_dim
 * / 64; fitted to 25 to 30 batches at every run.  The run that these choose is behind the best one by 1 to 2 % on average, 10 at the worst.  us at some of
 * them: 1531 rows behind none, many columns, in runs of 4 / 8 / 12 / 16 / whole (fp32) 76 / 67 / 61 / 65 / 72, 4000 of them 502 / 381 / 350 / 343 / 310,
 * 512 behind 1500 62 / 50 / 54 / 51 / 83; few columns: one row behind 1999 in runs of 1 / 2 / 4 / 8 / 16 7.8 / 8.0 / 9.3 / 13 / 20, behind 65535 of 8 / 16
 * / 32 / 64 47 / 45 / 53 / 96; 200 rows behind 2000, 32 columns, of 4 / 8 / 16 / whole 51 / 44 / 45 / 32. */
struct vt_paged_cost { int beside; float fixed, alone, step, part, merge, tail; };
static const vt_paged_cost vt_paged_few_cost[4] = {{4, 1.1f, 0.8f, 2.55f, 2.85f, 0.35f, 0.37f}, {3, 2.7f, 0.95f, 3.2f, 2.6f, 0.12f, 0.11f},
                                                   {2, 1.2f, 1.04f, 1.93f, 1.9f, 0.08f, 0.31f}, {2, 5.1f, 1.2f, 2.8f, 3.9f, 0.07f, 0.29f}};
static const vt_paged_cost vt_paged_wide_cost[2] = {{3, 1.4f, 0.32f, 0.7f, 2.5f, 0.16f, 0.39f}, {2, 0.85f, 0.42f, 1.09f, 4.85f, 0.07f, 0.08f}};
static const vt_paged_cost vt_paged_many_cost[4] = {{2, 7.9f, 1.9f, 3.0f, 5.0f, 1.0f, 0.45f}, {2, 9.25f, 2.2f, 3.8f, 3.6f, 2.2f, 0.24f}, {},
                                                    {1, 8.5f, 2.57f, 2.57f, 5.0f, 1.0f, 0.24f}};

static const vt_paged_cost &vt_paged_cost_of(const vt_paged_shape &s, const vt_paged_kinds &kinds, bool many) {
    return (many ? vt_paged_many_cost : kinds.few_cols == 32 ? vt_paged_wide_cost : vt_paged_few_cost)[s.head_dim / 64 - 1];
}

/* A kernel's part of a batch in runs of `run` units at most: its workgroups and their units, us of all of them; the longest one's units, whether it leaves
 * a part; us of the merge */
struct vt_paged_try { int run; double wgs, units, all, most, late, merge; };
#define PAGED_TRIES 40
static inline int vt_paged_tries(const vt_paged_shape &s, const vt_paged_kinds &kinds, bool many, int n_seqs, const int *past, const int *rows, vt_paged_try *to) {
    const int unit = many ? PAGED_MANY_ROWS : PAGED_FEW_ROWS * PAGED_FEW_WAVES;
    const vt_paged_cost &c = vt_paged_cost_of(s, kinds, many);
    long long longest = 0;
    if (!many || kinds.any)
        vt_paged_tiles(s, kinds, many, n_seqs, past, rows, [&](int, int, int first, int end) {
            const long long n = vt_paged_parts(first, end, unit, 1);
            longest = n > longest ? n : longest;
        });
    int tries = 0;
    for (int parts = 1; longest && parts <= PAGED_MAX_PARTS; parts += parts < 16 ? 1 : parts / 8) {
        const int run = (int)((longest + parts - 1) / parts);
        if (tries && to[tries - 1].run == run) continue;
        long long items = 0, extra = 0, split = 0, most = 0, all = 0;
        int late = 0;
        vt_paged_tiles(s, kinds, many, n_seqs, past, rows, [&](int, int, int first, int end) {
            const int n = vt_paged_parts(first, end, unit, 1), p = (n + run - 1) / run, each = (n + p - 1) / p;
            items += p;
            all += n;
            if (p > 1) { extra += p; split++; }
            if (each > most || (each == most && p > 1)) { late = p > 1; most = each; }
        });
        if (extra > PAGED_SPLIT_ITEMS || split > PAGED_COUNTERS / 2 / s.n_kv_heads) break;
        const double heads = s.n_kv_heads, us = (double)items * c.fixed + (double)all * c.step + (double)extra * c.part;
        to[tries++] = vt_paged_try{run, items * heads, all * heads, us * heads, (double)most, (double)late, split ? c.merge * parts : 0.0};
        if (run == 1) break;
    }
    return tries;
}
/* us of the longest one, by the share of the CU that has most of them; `slow`: a unit's time by what else is there */
static inline double vt_paged_one(const vt_paged_cost &c, const vt_paged_try &t, int n_cu, double slow) {
    const double full = ceil(t.wgs / n_cu) - 1, share = full < c.beside - 1 ? full / (c.beside - 1) : 1.0;
    return c.fixed + t.most * slow * (c.alone + (c.step - c.alone) * share) + t.late * c.part;
}

/* The runs of both kernels.  In one launch they share the CUs: a workgroup of many columns runs better beside one of few than beside another, and fewer of
 * them that leave no parts do best.  The factors are fitted to 30 pairs of runs of nine batches; the pair that they choose is behind the best one by 1 % on
 * average. */
static inline void vt_paged_runs(const vt_paged_shape &s, const vt_paged_kinds &kinds, int n_cu, int n_seqs, const int *past, const int *rows, int *runs) {
    vt_paged_try t[2][PAGED_TRIES];
    int n[2];
    for (int k = 0; k < 2; k++) {
        n[k] = vt_paged_tries(s, kinds, k, n_seqs, past, rows, t[k]);
        const vt_paged_cost &c = vt_paged_cost_of(s, kinds, k && kinds.any);
        double least = 1e300;
        runs[k] = 1;
        for (int i = 0; i < n[k]; i++) {
            const double room = (double)n_cu * c.beside, one = vt_paged_one(c, t[k][i], n_cu, 1);
            const double sum = t[k][i].all / room + (t[k][i].wgs > room ? c.tail * one : 0.0), us = (one > sum ? one : sum) + t[k][i].merge;
            if (us < least) { least = us; runs[k] = t[k][i].run; }
        }
    }
    if (!n[0] || !n[1] || !vt_paged_may_be_both(s, kinds)) return;
    const vt_paged_cost &c = vt_paged_cost_of(s, kinds, false), &d = vt_paged_cost_of(s, kinds, true);
    double least = 1e300;
    for (int i = 0; i < n[0]; i++)
        for (int j = 0; j < n[1]; j++) {
            const vt_paged_try &x = t[0][i], &y = t[1][j];
            const double a = c.fixed + 0.8 * x.most * c.step + x.late * c.part, b = vt_paged_one(d, y, n_cu, 0.65), one = a > b ? a : b;
            const double sum = (0.9 * x.all + y.all - 0.45 * y.units * d.step) / (2 * n_cu) + (x.wgs + y.wgs > 2 * n_cu ? 0.1 * (a < b ? a : b) : 0.0);
            const double us = (one > sum ? one : sum) + 0.15 * a + (x.merge > y.merge ? x.merge : y.merge);
            if (us < least) { least = us; runs[0] = x.run; runs[1] = y.run; }
        }
}

static int vt_paged_longest(const void *a, const void *b) {
    const vt_paged_item *x = (const vt_paged_item *)a, *y = (const vt_paged_item *)b;
    const int n = x->end - x->lo, m = y->end - y->lo;
    if (n != m) return n > m ? -1 : 1;
    if (x->row != y->row) return x->row < y->row ? -1 : 1;
    if (x->c0 != y->c0) return x->c0 < y->c0 ? -1 : 1;
    return x->part < y->part ? -1 : x->part > y->part;
}

/* .. of both kernels: the few's units, of 128 rows, take about as long as the many's, of 64 */
static int vt_paged_slowest(const void *a, const void *b) {
    const vt_paged_item *x = (const vt_paged_item *)a, *y = (const vt_paged_item *)b;
    const long long n = (long long)(x->end - x->lo) << x->many, m = (long long)(y->end - y->lo) << y->many;
    if (n != m) return n > m ? -1 : 1;
    return x->many != y->many ? (x->many ? -1 : 1) : vt_paged_longest(a, b);
}

/* Items of one kernel into `to`, the longest first; -> how many, and their slots */
static inline int vt_paged_items(const vt_paged_shape &s, const vt_paged_kinds &kinds, bool many, int run, int n_seqs, const int *past, const int *rows,
                                 const int *starts, vt_paged_item *to, int slot, int *n_slots) {
    const int unit = many ? PAGED_MANY_ROWS : PAGED_FEW_ROWS * PAGED_FEW_WAVES, group = s.n_heads / s.n_kv_heads;
    *n_slots = 0;
    if (many && !kinds.any) return 0;
    int n = 0, slots = slot, counters = many ? PAGED_COUNTERS / 2 / s.n_kv_heads : 0, row = 0, seq = 0;
    vt_paged_tiles(s, kinds, many, n_seqs, past, rows, [&](int i, int c0, int first, int end) {
        while (seq < i) row += rows[seq++];
        const int units = vt_paged_parts(first, end, unit, 1), parts = (units + run - 1) / run, u0 = first / unit;
        for (int p = 0; p < parts; p++) {
            const int from = (int)((long long)units * p / parts), till = (int)((long long)units * (p + 1) / parts);
            to[n++] = vt_paged_item{row, past[i], rows[i] * group, starts[i], c0, p ? (u0 + from) * unit : first, p + 1 < parts ? (u0 + till) * unit : end,
                                    slots, p, parts, counters, many};
        }
        if (parts > 1) { slots += parts; counters++; }
    });
    qsort(to, n, sizeof *to, vt_paged_longest);
    *n_slots = slots - slot;
    return n;
}

/* bytes of a part of one head */
static inline long long vt_paged_few_part(const vt_paged_shape &s, int cols) { return (long long)cols * (s.head_dim + 4) * 4; }
static inline long long vt_paged_many_part(const vt_paged_shape &s) { return 4ll * (s.head_dim / 8 + 1) * 1024; }

/* bf16: the queries' type, which a batch does not know: two plans where it matters */
static inline bool vt_paged_type_matters(const vt_paged_shape &s) { return s.head_dim == 256; }
static inline vt_paged_plan vt_paged_plan_of(const vt_paged_shape &s, bool bf16, int n_cu, int n_seqs, const int *past, const int *rows, const int *starts,
                                             vt_paged_item *to) {
    vt_paged_plan p = {0, 0, 0, 0, 0, 0, 0, 0};
    const vt_paged_kinds kinds = vt_paged_kinds_of(s, bf16, n_cu, n_seqs, past, rows);
    int runs[2];
    vt_paged_runs(s, kinds, n_cu, n_seqs, past, rows, runs);
    p.few = vt_paged_items(s, kinds, false, runs[0], n_seqs, past, rows, starts, to, 0, &p.few_slots);
    const long long part = vt_paged_few_part(s, kinds.few_cols) * p.few_slots, each = vt_paged_many_part(s);
    p.many_slot = (int)((part + each - 1) / each);
    p.many = vt_paged_items(s, kinds, true, runs[1], n_seqs, past, rows, starts, to + p.few, p.many_slot, &p.many_slots);
    p.both = p.few && p.many && p.few + p.many <= 65535 && vt_paged_may_be_both(s, kinds);
    if (p.both) qsort(to, p.few + p.many, sizeof *to, vt_paged_slowest);
    p.wide = kinds.few_cols > 16;
    p.once = kinds.once && kinds.bytes >= PAGED_CACHED;
    return p;
}

/* Requests that leave nothing behind in the caches, for rows that nobody reads again and that the caches (32 MB of L2) do not keep for the next call: 65535 rows of
 * 8 x 128 53.6 -> 48.2 us, 64 sequences of 118000 91.6 -> 83.4; but 300 rows 6.8 -> 7.2.  Beside a prompt as well: 31 sequences 43.4 -> 41.3, three of 10000 to
 * 30000 76 -> 72.  Sequences may share pages that they read, a common beginning, and with such requests each fetches these for itself.  us without and with
 * them, steps of 64 sequences on c common rows and r of their own, share of the rows read that another one has read before: c 4000, r 1 (98 %) 73.6 / 83.1,
 * c 4000, r 1000 (79 %) 114 / 124, c 1000, r 1000 (49 %) 61.6 / 61.5, c 1000, r 4000 (20 %) 189 / 179, none 90 / 82; 16 sequences c 8000, r 4000 (62 %) 79 /
 * 92; 256 sequences c 512, r 512 (50 %) 118 / 125. */
#define PAGED_AGAIN 0.33
/* What is left of `once` in n plans of a batch that vt_paged_lay_out has laid out.  `seen`: a bit for each page of the pool, all 0 before and after. */
static inline void vt_paged_once(vt_paged_plan *plans, int n, const vt_paged_shape &s, int n_seqs, const int *past, const int *rows, const int *starts,
                                 const int *tables, unsigned long long *seen) {
    int once = 0, log = 0;
    for (int i = 0; i < n; i++) once |= plans[i].once;
    if (!once) return;
    while (1 << log < s.page_rows) log++;
    long long all = 0, again = 0;
    for (int clear = 0; clear < 2; clear++)
        for (int i = 0; i < n_seqs; i++) {
            if (rows[i] == 0) continue;
            const int first = vt_paged_first(s.window, past[i], 0) >> log, last = (past[i] + rows[i] - 1) >> log;
            for (int p = first; p <= last; p++) {
                const int page = tables[starts[i] + p];
                unsigned long long *word = seen + page / 64, bit = 1ull << (page & 63);
                if (clear) { *word = 0; continue; }
                all++;
                again += (*word & bit) != 0;
                *word |= bit;
            }
        }
    const double bytes = (double)(all - again) * s.page_rows * 4 * s.n_kv_heads * s.head_dim;
    if ((double)again <= PAGED_AGAIN * (double)all && bytes >= PAGED_CACHED) return;
    for (int i = 0; i < n; i++) plans[i].once = 0;
}

#endif /* VT_PAGED_PLANS_H */
