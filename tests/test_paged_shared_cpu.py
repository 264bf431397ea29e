"""Sequences that share pages of a paged cache (vt_paged_plans.h), on the CPU: whose rows are asked for as rows that nobody reads again."""
import plansupport as P

SHARED = r"""
#include <stdio.h>
#include <vector>
#include "vt_paged_plans.h"
struct batch { std::vector<int> past, rows, tables; int stride; };
/* n steps behind `prefix` common pages and `own` of their own, of 16 rows */
static batch steps(int n, int prefix, int own) {
    batch b;
    b.stride = prefix + own;
    for (int i = 0; i < n; i++) {
        b.past.push_back(16 * b.stride - 1);
        b.rows.push_back(1);
        for (int p = 0; p < b.stride; p++) b.tables.push_back(p < prefix ? p : prefix + i * own + p - prefix);
    }
    return b;
}
static int once(const batch &b, int window, std::vector<unsigned long long> &seen) {
    const int n = (int)b.past.size();
    const vt_paged_shape s = {(int)seen.size() * 64 - 5, 16, 32, 8, 128, window};
    std::vector<int> pos(n), place(2 * n), tables(b.tables.size()), starts(n), written(n);
    int n_rows, n_table;
    const vt_paged_fault f = vt_paged_lay_out(s, n, n, (int)tables.size(), n, b.past.data(), b.rows.data(), b.tables.data(), b.stride,
                                              vt_paged_rows{pos.data(), place.data(), tables.data(), starts.data(), written.data()}, &n_rows, &n_table);
    if (f.what) return -f.what;
    std::vector<vt_paged_item> items(vt_paged_max_items(n, n, 4));
    vt_paged_plan p = vt_paged_plan_of(s, true, 256, n, b.past.data(), b.rows.data(), starts.data(), items.data());
    vt_paged_once(&p, 1, s, n, b.past.data(), b.rows.data(), starts.data(), tables.data(), seen.data());
    for (unsigned long long w : seen) if (w) return -100;                          /* as it was */
    return p.once;
}
int main(void) {
    std::vector<unsigned long long> seen(1 << 12);
    const struct { int n, prefix, own, window, once; } c[] = {
        {64, 0, 125, 0, 1},              /* 64 steps behind 2000 rows each: 524 MB, nobody's twice */
        {64, 0, 5, 0, 0},                /* what a cache holds */
        {64, 63, 1, 0, 0}, {64, 63, 7, 0, 0}, {64, 250, 1, 0, 0}, {64, 250, 63, 0, 0}, {16, 500, 250, 0, 0}, {256, 32, 32, 0, 0},
        {64, 63, 250, 0, 1},             /* a fifth of the reads are others' too */
        {2, 2000, 1, 0, 0}, {1, 2000, 1, 0, 1}, {2, 100, 4000, 0, 1},
        {64, 500, 125, 2000, 1},         /* the common pages are out of the window */
        {64, 500, 125, 0, 0},
    };
    int bad = 0;
    for (const auto &k : c) {
        const int got = once(steps(k.n, k.prefix, k.own), k.window, seen);
        if (got != k.once) { bad++; printf("%d steps, %d common pages, %d of each, window %d: %d\n", k.n, k.prefix, k.own, k.window, got); }
    }
    printf("%d\n", bad);
    return 0;
}
"""


def test_rows_that_others_read_too():
    out = P.run(SHARED)
    assert out.splitlines()[-1] == "0", out


LONGEST = r"""
#include <stdio.h>
#include "vt_paged_plans.h"
int main(void) {
    /* row, past, cols, table, c0, lo, end, slot, part, parts, counter, many */
    vt_paged_item it[] = {{0, 100, 16, 0, 0, 0, 101, 0, 0, 1, 0, 0}, {1, (1 << 30) - 1, 128, 0, 0, 0, 1 << 30, 0, 0, 1, 0, 1},
                          {2, (1 << 30) - 2, 16, 0, 0, 0, (1 << 30) - 1, 0, 0, 1, 0, 0}, {3, 700, 128, 0, 0, 0, 701, 0, 0, 1, 0, 1}};
    qsort(it, 4, sizeof *it, vt_paged_slowest);
    for (const auto &x : it) printf("%d ", x.row);
    return 0;
}
"""


def test_the_longest_comes_first_at_any_length():
    assert P.run(LONGEST).split() == ["1", "2", "3", "0"]
