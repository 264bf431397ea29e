"""The 4-bit operators' launches (vt_mx4_plans.h), walked on the CPU: the header compiled with g++, 256 CUs."""
import plansupport as P
import test_gpu_kv4
import test_gpu_kv4_many
import test_gpu_mx4

LANES = r"""
#include <stdio.h>
#include "vt_mx4_plans.h"
int main(void) {
    long long checked = 0, many = 0, bad = 0;
    const int rows[] = {1, 2, 15, 16, 17, 300, 9216, 1 << 20, (1 << 27) - 9, (1 << 27) - 8, (1 << 27) - 7, (1 << 28) - 16, (1 << 28) - 15, (1 << 28) + 3, (1 << 30) - 1, 1 << 30};
    for (long long cols = 1; cols <= 1 << 27; cols += 1 + cols / 9)
        for (int r : rows)
            for (int values = 4; values <= 8; values += 4) {
                long long done = 0, launches = 0;
                for (; done < r; launches++) {
                    const vt_mx4_lanes l = vt_mx4_lanes_of((int)(r - done), (int)cols, values);
                    const long long tall = l.grid / l.chunks * (256ll >> l.wide_log);       /* rows that the launch has lanes for */
                    const int wrong = l.grid < 1 || 256ll * l.grid >= 1ll << 32 || l.grid % l.chunks || ((long long)l.chunks << l.wide_log) < l.units ||
                                      (long long)l.units * values < cols || l.units % (128 / values) || l.rows < 1 || l.rows > r - done || tall < l.rows;
                    if (wrong && bad++ < 5) printf("%d x %lld by %d, from %lld: %d rows, grid %d, chunks %d, lanes 2^%d, units %d\n", r, cols, values, done, l.rows, l.grid, l.chunks, l.wide_log, l.units);
                    if (l.rows < 1) break;
                    done += l.rows;
                    checked++;
                    if (launches > 100) { r = 1; done = 1; }       /* far enough: a matrix that no memory holds */
                }
                many += launches > 1;
            }
    printf("%lld %lld %lld\n", checked, many, bad);
    return 0;
}
"""


def test_every_row_is_converted_by_launches_that_the_device_takes():
    """Fewer than 2^32 threads a launch, and every row of a matrix in one of them."""
    out = P.run(LANES)
    checked, many, bad = map(int, out.splitlines()[-1].split())
    assert checked > 5000 and many > 200 and bad == 0, out


TILES = r"""
#include <stdio.h>
#include "vt_mx4_plans.h"
int main(void) {
    long long checked = 0, halved = 0, bad = 0;
    for (long long n = 1; n <= 1 << 30; n += 1 + n / 7)
        for (long long k = 1; k <= 1 << 23; k += 1 + k / 5) {
            const int panels = vt_mx4_panels((int)k), most = vt_mxt_rows((int)n, panels);
            halved += most < VT_MXT_ROWS;
            for (int m = 1; m <= most; m += 1 + m / 2) {
                const int at[2] = {m, most};
                for (int s : at) {
                    const vt_mxt_plan p = vt_mxt_plan_of(256, s, (int)n, panels);
                    const vt_mxt_tile &t = vt_mxt_tiles[p.tile];
                    const long long split = ((s + 31) / 32 * 2ll * panels + 3) / 4 * 256;
                    const int wrong = most < 32 || p.grid < 1 || p.grid * t.threads >= 1ll << 32 || split >= 1ll << 32 || p.cuts < 1 || p.cuts > panels ||
                                      p.grid != (n + t.bm - 1) / t.bm * ((s + t.bn - 1) / t.bn) * p.cuts || p.m_tiles != (n + t.bm - 1) / t.bm;
                    checked++;
                    if (wrong && bad++ < 5) printf("%d x %lld x %lld: tile %d, %d cuts, grid %lld\n", s, n, k, p.tile, p.cuts, p.grid);
                }
            }
        }
    printf("%lld %lld %lld\n", checked, halved, bad);
    return 0;
}
"""


def test_tiles_in_launches_that_the_device_takes():
    out = P.run(TILES)
    checked, halved, bad = map(int, out.splitlines()[-1].split())
    assert checked > 100000 and halved > 100 and bad == 0, out


ASK = r"""
#include <stdio.h>
#include "vt_mx4_plans.h"
int main(void) {
    int m, n, k;
    while (scanf("%d %d %d", &m, &n, &k) == 3) {
        const vt_mxt_plan p = vt_mxt_plan_of(256, m, n, vt_mx4_panels(k));
        printf("%dx%d %d\n", vt_mxt_tiles[p.tile].bm, vt_mxt_tiles[p.tile].bn, p.cuts);
    }
    return 0;
}
"""


def test_the_tiles_that_the_device_tests_are_there_for():
    cases = test_gpu_mx4.TILES
    got = [(t, int(c)) for t, c in (line.split() for line in P.run(ASK, "\n".join("%d %d %d" % c for c in cases)).splitlines())]
    assert got == list(cases.values())


ATTENTION = r"""
#include <stdio.h>
#include "vt_mx4_plans.h"
int main(void) {
    long long checked = 0, many = 0, shared = 0, bad = 0;
    for (int hp = 1; hp <= 4; hp++)
        for (long long heads = 1; heads <= 65535; heads += 1 + heads / 2)
            for (long long group = 1; group <= 1 << 19; group += 1 + group / 2)
                for (long long rows = 1; rows * group <= 1 << 19; rows += 1 + rows / 2)
                    for (long long start = 0; start + rows <= 1 << 24; start += 1 + start) {
                        const int cols = (int)(rows * group), end = (int)(start + rows);
                        const vt_kv4_plan p = vt_kv4_plan_of(256, hp, (int)heads, (int)group, cols, (int)start, end);
                        const int wide = p.many ? KV4_TILE : KV4_COLS, tall = p.many ? 64 : 32 * vt_kv4_waves(hp);
                        const long long covered = (long long)p.parts * p.run * tall, row = 32 * hp;
                        /* a wave's (many: a workgroup's) codes through one descriptor, and where its requests for the two tiles behind end */
                        const long long bytes = ((long long)p.run * (p.many ? 64 : 32) + 128) * row;
                        const int wrong = p.tiles != (cols + wide - 1) / wide || p.run < 1 || p.parts < 1 || p.parts > (p.many ? KV4_MAX_PARTS : KV4_MAX_CHUNKS) || covered < end ||
                                          covered - (long long)p.run * tall >= end || covered > 0x7fffffff || (p.parts > 1 && heads * p.tiles > VT_MX4_COUNTERS) || bytes > 0x7fffffff ||
                                          p.tiles > 65535 || p.parts > 65535 || (p.many && hp > 2);
                        checked++;
                        many += p.many;
                        shared += p.parts > 1;
                        if (wrong && bad++ < 5)
                            printf("hp %d, %lld heads, group %lld, %lld rows behind %lld: %s, %d tiles, run %d, %d parts\n", hp, heads, group, rows, start, p.many ? "many" : "few", p.tiles, p.run, p.parts);
                    }
    printf("%lld %lld %lld %lld\n", checked, many, shared, bad);
    return 0;
}
"""


def test_every_row_of_an_attention_in_a_part_and_a_counter_for_every_shared_tile():
    out = P.run(ATTENTION)
    checked, many, shared, bad = map(int, out.splitlines()[-1].split())
    assert checked > 100000 and many > 10000 and shared > 10000 and bad == 0, out


ASK_ATTENTION = r"""
#include <stdio.h>
#include "vt_mx4_plans.h"
int main(void) {
    int heads, kv, hd, rows, pos;
    while (scanf("%d %d %d %d %d", &heads, &kv, &hd, &rows, &pos) == 5) {
        const vt_kv4_plan p = vt_kv4_plan_of(256, hd / 64, kv, heads / kv, heads / kv * rows, pos, pos + rows);
        printf("%d %d\n", p.many, p.parts);
    }
    return 0;
}
"""


def attention(cases):
    return [tuple(map(int, line.split())) for line in P.run(ASK_ATTENTION, "\n".join("%d %d %d %d %d" % c for c in cases)).splitlines()]


def test_the_kernels_that_the_device_tests_are_there_for():
    many = test_gpu_kv4_many.CASES
    assert attention(many) == [(1, parts) for parts in many.values()]
    assert [m for m, _ in attention(test_gpu_kv4.BOTH)] == [0, 0, 0, 0, 1, 1, 1]
