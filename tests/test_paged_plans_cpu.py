"""The batch over a paged cache (vt_paged_plans.h), walked on the CPU: the header compiled with g++, 256 CUs."""
import plansupport as P

WALK = r"""
#include <stdio.h>
#include <vector>
#include "vt_paged_plans.h"
static unsigned long long seed = 1;
static int below(int n) { seed = seed * 6364136223846793005ull + 1442695040888963407ull; return (int)((seed >> 33) % (unsigned long long)n); }
static int spread(int most) { int n = 1; while (n < most && below(4)) n *= 2; return 1 + below(n < most ? n : most); }
int main(void) {
    long long checked = 0, split = 0, wide = 0, both = 0, bad = 0;
    const int layouts[][3] = {{32, 8, 128}, {16, 16, 64}, {8, 1, 128}, {12, 4, 256}, {14, 2, 64}, {6, 2, 192}, {20, 1, 64}, {4096, 1, 64}, {1, 1, 256}};
    for (int round = 0; round < 1500; round++) {
        const int *lay = layouts[below(round % 5 ? 9 : 3)], n_seqs = 1 + below(round % 3 ? 5 : 70), page_rows = 16 << below(6), group = lay[0] / lay[1];
        vt_paged_shape s = {1 << 20, page_rows, lay[0], lay[1], lay[2], below(2) ? 0 : spread(5000)};
        std::vector<int> past(n_seqs), rows(n_seqs), starts(n_seqs);
        int max_rows = 0, pages = 1;
        for (int i = 0; i < n_seqs; i++) {
            rows[i] = below(3) == 0 ? below(3) : spread(n_seqs > 8 ? 40 : 1600);
            if (round % 5 == 0) rows[i] = i % 8 ? 1 + below(16 / group < 1 ? 1 : 16 / group) : 600 + below(1500);          /* prompts and steps */
            past[i] = below(4) ? spread(70000) : 0;
            max_rows += rows[i];
            const int p = (past[i] + rows[i] + page_rows - 1) / page_rows;
            pages = p > pages ? p : pages;
        }
        max_rows += !max_rows;
        std::vector<int> tables((size_t)n_seqs * pages), pos(max_rows), place(2 * max_rows), out((size_t)n_seqs * pages), written(max_rows);
        for (size_t i = 0; i < tables.size(); i++) tables[i] = (int)i % s.n_pages;
        int n_rows = 0, n_table = 0;
        vt_paged_rows to = {pos.data(), place.data(), out.data(), starts.data(), written.data()};
        const vt_paged_fault f = vt_paged_lay_out(s, n_seqs, max_rows, n_seqs * pages, n_seqs, past.data(), rows.data(), tables.data(), pages, to, &n_rows,
                                                  &n_table);
        if (vt_paged_shape_bad(s) || f.what) { bad++; printf("refused %d\n", f.what); continue; }
        std::vector<vt_paged_item> items(vt_paged_max_items(n_seqs, max_rows, group));
        const vt_paged_plan plan = vt_paged_plan_of(s, round & 1, 256, n_seqs, past.data(), rows.data(), starts.data(), items.data());
        const vt_paged_kinds kinds = vt_paged_kinds_of(s, round & 1, 256, n_seqs, past.data(), rows.data());
        if (plan.wide != (kinds.few_cols == 32) || (plan.once && plan.wide)) { bad++; printf("wide %d once %d\n", plan.wide, plan.once); }
        if (plan.both != (plan.few && plan.many && !plan.wide && lay[2] <= 128 && plan.few + plan.many <= 65535)) { bad++; printf("both %d\n", plan.both); }
        both += plan.both;
        if (plan.few + plan.many > (int)items.size()) { bad++; printf("items %d %d\n", plan.few, plan.many); }
        /* every column's rows are read once, by the parts of one group, in slots of its own */
        std::vector<long long> want(n_seqs), got(n_seqs);
        std::vector<int> left(PAGED_COUNTERS);           /* one launch may have both kinds */
        if (plan.many_slot * vt_paged_many_part(s) < plan.few_slots * vt_paged_few_part(s, kinds.few_cols)) { bad++; printf("parts\n"); }
        for (int k = 0; k < 2; k++) {
            const int n = k ? plan.many : plan.few, cols = k ? PAGED_MANY_COLS : kinds.few_cols;
            const int unit = k ? 64 : 32, n_slots = k ? plan.many_slots : plan.few_slots, slot0 = k ? plan.many_slot : 0;
            std::vector<char> slot(n_slots);
            int found = 0, longest = 1 << 30;
            for (int j = 0; j < plan.few + plan.many; j++) {
                const vt_paged_item &it = items[j];
                if (it.many != k) { if (!plan.both && (j >= plan.few) == k) { bad++; printf("order\n"); } continue; }
                found++;
                int i = 0, row = 0;
                while (i < n_seqs && !(row == it.row && rows[i] && past[i] == it.past)) row += rows[i++];
                if (i == n_seqs || it.cols != rows[i] * group || it.table != starts[i]) { bad++; printf("no sequence\n"); break; }
                const int c1 = it.c0 + cols < it.cols ? it.c0 + cols : it.cols, q0 = it.c0 / group, q1 = (c1 - 1) / group;
                const int first = s.window && past[i] + q0 >= s.window ? past[i] + q0 - s.window + 1 : 0, end = past[i] + q1 + 1;
                const bool off = it.c0 % cols || it.c0 >= it.cols || it.lo < first || it.end > end || it.lo >= it.end;
                const bool torn = (it.lo % unit && it.lo != first) || (it.end % unit && it.end != end);
                const bool unshared = it.parts < 1 || it.parts > PAGED_MAX_PARTS || it.part < 0 || it.part >= it.parts ||
                                      (it.part == 0 && it.lo != first) || (it.part == it.parts - 1 && it.end != end);
                const bool unknown = it.end - 1 >= past[i] + rows[i] || (it.end - 1) / page_rows + it.table >= n_table;
                const bool wrong = off || torn || unshared || unknown || it.end - it.lo > longest;
                longest = it.end - it.lo;
                if (wrong && bad++ < 5) printf("item %d of %d: columns %d of %d, rows %d .. %d of %d .. %d, part %d of %d\n", j, n, it.c0, it.cols, it.lo, it.end,
                                               first, end, it.part, it.parts);
                got[i] += (long long)(c1 - it.c0) * (it.end - it.lo);
                if (it.part == 0) want[i] += (long long)(c1 - it.c0) * (end - first);
                if (it.parts > 1) {
                    const int at = it.slot - slot0 + it.part;
                    if (at < 0 || at >= n_slots || slot[at] || (long long)(it.counter + 1) * lay[1] > PAGED_COUNTERS) { bad++; printf("slot\n"); } else slot[at] = 1;
                    if (left[it.counter] == 0) left[it.counter] = it.parts;
                    left[it.counter]--;
                    split++;
                }
                wide += k;
                checked++;
            }
            for (char v : slot) bad += !v;
            bad += found != n;
        }
        for (int v : left) bad += v != 0;
        for (int i = 0; i < n_seqs; i++) {
            long long all = 0;
            const bool many = kinds.any && vt_paged_may_be_many(lay[2] / 64, (long long)rows[i] * group);
            const int cols = many ? PAGED_MANY_COLS : kinds.few_cols;
            for (int c = 0; c < rows[i] * group; c += cols) all++;
            if (got[i] != want[i] || (rows[i] && !got[i])) { bad++; printf("sequence %d of %d: %lld of %lld\n", i, n_seqs, got[i], want[i]); }
        }
        for (int i = 0, r = 0; i < n_seqs; i++)
            for (int k = 0; k < rows[i]; k++, r++)
                if (pos[r] != past[i] + k || place[2 * r] != tables[(size_t)i * pages + pos[r] / page_rows] || place[2 * r + 1] != pos[r] % page_rows) bad++;
    }
    printf("%lld %lld %lld %lld %lld\n", checked, split, wide, both, bad);
    return 0;
}
"""


def test_every_row_that_a_column_sees_is_one_parts():
    """Items cover every tile of columns, a tile's parts its rows, each once; slots and counters are a group's own; a table is read within its sequence's entries."""
    out = P.run(WALK)
    checked, split, wide, both, bad = map(int, out.splitlines()[-1].split())
    assert bad == 0 and checked > 50000 and split > 5000 and wide > 2000 and both > 50, out


REFUSED = r"""
#include <stdio.h>
#include "vt_paged_plans.h"
int main(void) {
    const vt_paged_shape s = {10, 16, 32, 8, 128, 0}, w = {10, 16, 32, 8, 128, 20};
    int pos[64], place[128], out[64], starts[4], written[64], n, m;
    const vt_paged_rows to = {pos, place, out, starts, written};
    struct { vt_paged_shape s; int n_seqs, past[3], rows[3], tables[3][4], what; } const c[] = {
        {s, 2, {16, 0}, {1, 3}, {{1, 2}, {3}}, PAGED_OK},
        {s, 0, {0}, {0}, {{0}}, PAGED_OK},
        {s, 2, {16, 0}, {1, 0}, {{1, 2}, {-1}}, PAGED_OK},                /* no new rows: nothing looked at */
        {s, 2, {16, 20}, {1, 1}, {{1, 2}, {1, 3}}, PAGED_OK},             /* a page that both read */
        {s, 2, {17, 20}, {1, 1}, {{1, 2}, {1, 2}}, PAGED_WRITTEN},
        {s, 1, {0}, {33}, {{1, 2, 1}}, PAGED_WRITTEN},
        {s, 1, {16}, {1}, {{1, 10}}, PAGED_PAGE},
        {s, 1, {16}, {1}, {{-1, 2}}, PAGED_PAGE},
        {w, 1, {34}, {1}, {{-1, 2, 3}}, PAGED_PAGE},                      /* row 15 is the first that it sees */
        {w, 1, {35}, {1}, {{-1, 2, 3}}, PAGED_OK},                        /* row 16 */
        {w, 1, {36}, {1}, {{1, 77, 3}}, PAGED_PAGE},
        {s, 4, {0}, {0}, {{0}}, PAGED_COUNT},
        {s, -1, {0}, {0}, {{0}}, PAGED_COUNT},
        {s, 1, {-1}, {1}, {{1}}, PAGED_SEQUENCE},
        {s, 1, {1}, {-1}, {{1}}, PAGED_SEQUENCE},
        {s, 1, {1 << 30}, {1}, {{1}}, PAGED_SEQUENCE},
        {s, 1, {0x7fffffff}, {0x7fffffff}, {{1}}, PAGED_SEQUENCE},
        {s, 2, {0, 0}, {30, 35}, {{1, 2}, {3, 4, 5}}, PAGED_TOO_MANY_ROWS},
        {s, 1, {0}, {0x7fffffff >> 2}, {{1}}, PAGED_TOO_MANY_ROWS},
        {s, 1, {63}, {2}, {{1, 2, 3, 4}}, PAGED_TABLE},
        {s, 3, {63, 63, 63}, {1, 1, 1}, {{1, 2, 3, 4}, {1, 2, 3, 5}, {1, 2, 3, 6}}, PAGED_TABLE},
    };
    int bad = 0;
    for (const auto &k : c) {
        const vt_paged_fault f = vt_paged_lay_out(k.s, 3, 64, 10, k.n_seqs, k.past, k.rows, k.tables[0], 4, to, &n, &m);
        if (f.what != k.what) { bad++; printf("case %d: %d instead of %d\n", (int)(&k - c), f.what, k.what); }
    }
    const vt_paged_shape shapes[] = {{0, 16, 32, 8, 128, 0}, {1, 8, 32, 8, 128, 0}, {1, 24, 32, 8, 128, 0}, {1, 1 << 21, 32, 8, 128, 0}, {1, 16, 32, 8, 96, 0},
                                     {1, 16, 32, 8, 320, 0}, {1, 16, 32, 0, 128, 0},
                                     {1, 16, 33, 8, 128, 0}, {1, 16, 0, 8, 128, 0}, {1, 16, 32, 8, 128, -1}, {1, 16, 4097, 1, 128, 0},
                                     {1, 16, 65536, 65536, 64, 0}, {1, -16, 32, 8, 128, 0}};
    for (const auto &x : shapes) if (!vt_paged_shape_bad(x)) { bad++; printf("shape %d\n", (int)(&x - shapes)); }
    printf("%d\n", bad);
    return 0;
}
"""


def test_batches_that_are_refused():
    out = P.run(REFUSED)
    assert out.splitlines()[-1] == "0", out
