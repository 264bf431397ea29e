"""The 4-bit operators' launches (vt_mx4_plans.h), walked on the CPU: the header compiled with g++, 256 CUs."""
import plansupport as P

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
