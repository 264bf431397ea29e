/*
 * vt_mx4_plans.h - the 4-bit operators' launches (vt_mx4.hip, vt_kv4.hip) from shapes and the number of CUs: lanes of a conversion,
 * tiles and K cuts of a product, workgroups of an attention.  Host code without HIP, so that a host test can walk it.
 */
#ifndef VT_MX4_PLANS_H
#define VT_MX4_PLANS_H

#include <math.h>
#include <stddef.h>

#define VT_MX4_COUNTERS 16384     /* tiles, or heads times tiles of columns, that several workgroups share */

/* A launch has fewer than 2^32 threads in a dimension; workgroups of `threads` of it */
static inline long long vt_launch_most(int threads) { return 0xffffffffll / threads; }

static inline int vt_mx4_panels(int cols) { return cols / 128 + (cols % 128 != 0); }

/* ---- conversions: a lane has `values` of a row, 2^wide_log lanes lie along a row and the rest of a workgroup's 256 on the rows below,
 * whichever width leaves the fewest lanes behind the row's end; `chunks` workgroups along a row, `rows` of the rows in one launch --- */
struct vt_mx4_lanes { int units, wide_log, chunks, rows, grid; };

static inline vt_mx4_lanes vt_mx4_lanes_of(int rows, int cols, int values) {
    vt_mx4_lanes s;
    s.units = 128 / values * vt_mx4_panels(cols);
    s.wide_log = 8;
    long long lanes = 0;
    for (int w = 8; w >= 4; w--) {
        const long long n = ((long long)s.units + (1 << w) - 1) >> w << w;
        if (lanes == 0 || n < lanes) { s.wide_log = w; lanes = n; }
    }
    s.chunks = (int)(lanes >> s.wide_log);
    const int per = 256 >> s.wide_log;
    const long long tall = ((long long)rows + per - 1) / per, most = vt_launch_most(256) / s.chunks;
    s.rows = tall <= most ? rows : (int)(most * per);
    s.grid = (int)((tall <= most ? tall : most) * s.chunks);
    return s;
}

/* ---- linear layers of more than a few rows --- */

/* Tiles: weight rows, rows of x, threads, workgroups that a CU holds, and us per panel with one, two, three of them on it.  These, what
 * cuts cost and the rate of their sums are the numbers that choose best, fitted to 4000 runs of every tile and cut count on 190 shapes
 * of 9 to 1531 rows. */
struct vt_mxt_tile { int bm, bn, threads, per_cu; float panel_us[3]; };
static const vt_mxt_tile vt_mxt_tiles[] = {{256, 128, 512, 1, {1.4f}}, {128, 64, 256, 2, {0.95f, 1.35f}}, {128, 32, 256, 3, {0.65f, 0.78f, 1.45f}}};
#define VT_MXT_MAX_CUTS 16
#define VT_MXT_ROWS (1 << 14)

/* Rows of x at a time: so many that the work area stays small beside the operands, and no more than a launch has threads for, the one
 * that splits x (a wave per 32 rows and 64 columns, four a workgroup) and the product's. */
static inline int vt_mxt_rows(int out_dim, int panels) {
    const long long most = vt_launch_most(256), tall = ((long long)out_dim + 127) / 128;
    int rows = VT_MXT_ROWS;
    while (rows > 32 && (tall * (rows / 32) > most || ((long long)rows / 32 * 2 * panels + 3) / 4 > most)) rows /= 2;
    return rows;
}

/* The tile and the cuts of K with the least time by these figures (which leave out the split of x and, where there are few rows of x for
 * many weights, the weights' way from memory: alike for all).  Over those shapes the plan taken is 1.6 % behind the fastest on average,
 * at worst 12 % (512 x 1024 x 3072).  us a call, with the best of other tiles or cuts: 1531 x 9216 x 3072 123 (256 x 128 whole; 147 on
 * 128 x 64), 512 of them 52 (the same; 64 on 128 x 32), 400 49 (128 x 64 whole; 52 on 256 x 128), 128 25 (128 x 32 whole; 28 on 128 x
 * 64), 64 20 (128 x 32 in 3; 21 on 128 x 64), 1000 x 3072 x 4096 54 (256 x 128 in 2; 56 on 128 x 64), 226 x 3072 x 9216 39 (256 x 128 in
 * 8; 40 on 128 x 64 in 5, 43 on 128 x 32), 16 x 131072 x 3072 78 (128 x 32 whole; 81 on 128 x 64). */
struct vt_mxt_plan { int tile, cuts, m_tiles; long long grid; double us; };
static inline vt_mxt_plan vt_mxt_plan_of(int n_cu, int seq_len, int out_dim, int panels) {
    vt_mxt_plan best = {0, 1, 0, 0, 1e30};
    for (int t = 0; t < 3; t++) {
        const vt_mxt_tile &k = vt_mxt_tiles[t];
        const long long m_tiles = ((long long)out_dim + k.bm - 1) / k.bm, tiles = m_tiles * ((seq_len + k.bn - 1) / k.bn);
        for (int cuts = 1; cuts <= VT_MXT_MAX_CUTS && cuts <= panels && tiles * cuts <= vt_launch_most(k.threads); cuts++) {
            const double wgs = (double)tiles * cuts, full = floor(wgs / ((double)n_cu * k.per_cu)), rest = wgs - full * n_cu * k.per_cu;
            const int each = (panels + cuts - 1) / cuts, beside = (int)ceil(rest / n_cu);
            const double us = each * (full * k.panel_us[k.per_cu - 1] + (beside ? k.panel_us[beside - 1] : 0.0)) + full +
                              (cuts > 1 ? 4.2 + (double)seq_len * out_dim * 4.0 * (2 * cuts + 1) / 3.9e6 : 0.0);
            if (us < best.us) best = vt_mxt_plan{t, cuts, (int)m_tiles, tiles * cuts, us};
        }
    }
    return best;
}

/* ---- attention over a 4-bit cache: columns are queries times heads per kv head --- */

#define KV4_COLS 16                        /* of a workgroup of the kernel for few columns */
#define KV4_MAX_CHUNKS 64
#define KV4_TILE_WAVES 4                   /* of the kernel for many, 32 columns a wave */
#define KV4_TILE (32 * KV4_TILE_WAVES)
#define KV4_MAX_PARTS 32

/* tiles of columns; tiles of 32 (many: 64) rows to a wave (many: a workgroup), and the workgroups that share a head's rows for a tile of columns */
struct vt_kv4_plan { int many, tiles, run, parts; };

static constexpr int vt_kv4_waves(int hp) { return hp <= 2 ? 8 : 4; }

/* hp: head_dim / 64; the rows of the columns that see most end at `end` */
static inline vt_kv4_plan vt_kv4_few(int n_cu, int hp, int heads, int cols, int end) {
    const int waves = vt_kv4_waves(hp), col_tiles = (cols + KV4_COLS - 1) / KV4_COLS;
    const long long wgs = (long long)col_tiles * heads, tiles = ((long long)end + 31) / 32, slots = (long long)n_cu * (hp == 1 ? 2 : 1);
    /* Workgroups per head and tile of columns: the number that takes the least time at 3.5 us a round of workgroups, 1.2 us a tile of
     * 128 values a row and 2.8 us for adding parts. (us at 1 / 2 / 4 / 8 / 32 of them: 1 query behind 300 rows 7.4 / 8.5 / 8.5 / 8.5 /
     * 8.5, behind 1999 13.4 / 11.8 / 9.8 / 9.1 / 9.0, behind 65535 264 / 137 / 73 / 41 / 20, 37 queries behind 4000, ten tiles of
     * columns, 24 / 20 / 27 / 35 and at 3 18.) */
    long long best = 1;
    float least = 1e30f;
    for (long long chunks = 1; chunks <= KV4_MAX_CHUNKS && (chunks == 1 || (wgs <= VT_MX4_COUNTERS && chunks <= (tiles + waves - 1) / waves)); chunks++) {
        const float each = (float)((tiles + chunks * waves - 1) / (chunks * waves)), rounds = (float)((wgs * chunks + slots - 1) / slots);
        const float us = rounds * (3.5f + 0.6f * hp * each) + (chunks > 1 ? 2.8f : 0.f);
        if (us < least) { least = us; best = chunks; }
    }
    const int run = (int)((tiles + best * waves - 1) / (best * waves));
    return vt_kv4_plan{0, col_tiles, run, (int)((tiles + (long long)run * waves - 1) / ((long long)run * waves))};
}

/* us that a launch takes when its columns' rows, first .. last tiles of them, are cut into runs: 1.75 a tile for a workgroup that has a
 * CU to itself and 2.9 for each of two on one, 3.1 a tile and 12 a part over all of them, 7 and 1 a part to make one of a column's
 * parts.  Measured and (expected), at runs of 4 / 8 / 12 / 16 / whole: 1531 queries 68 / 53 / 54 / 59 / 55 to 60 (69 / 55 / 51 / 61 /
 * 61), 2000 of them 104 / 80 / 78 / 68 / 75 (112 / 88 / 79 / 75 / 84), 1000 35 / 36 / 39 / - / 37 (36 / 35 / 40 / - / 37), 1531 behind
 * 2000 207 / 148 / 136 / 136 / 136 (215 / 167 / 153 / 147 / 153), 300 behind 1000 31 / 30 / 33 / 40 / 43 (30 / 31 / 37 / 44 / 46), 300
 * behind 8000 - / 96 / 95 / 92, in runs of 22 and of 32 82 and 102, 4000 425 / 291 / 262 / 241 / 220 (400 / 306 / 275 / 259 / 218). */
static inline float vt_kv4_tiles_us(float run, float first, float last, float wgs, float n_cu) {
    const float all = 0.5f * (first + last) * wgs;
    if (run >= last) {                                   /* whole: the longest, and what shares its CU with it */
        if (wgs > 2.f * n_cu) return 9.f + (3.1f * all + 8.f * wgs) / (2.f * n_cu);
        const float second = wgs > n_cu ? last - (last - first) * n_cu / wgs : 0.f;
        return 9.f + 2.9f * second + 1.75f * (last - second);
    }
    const float parts = wgs * (0.5f * (first + last) / run + 0.5f), shared = fminf(fmaxf(parts / n_cu - 1.f, 0.f), 1.f);
    /* parts of one length in more than one round: half a part on average that has a CU to itself */
    const float behind = parts > 2.f * n_cu ? 0.5f * 1.75f * run * first / last : 0.f;
    return 7.f + fmaxf(run * (1.75f + 1.15f * shared) + 7.f + ceilf(last / run), (3.1f * all + 12.f * parts) / (2.f * n_cu) + behind);
}

static inline vt_kv4_plan vt_kv4_many(int n_cu, int heads, int group, int cols, int start, int end) {
    const int col_tiles = (cols + KV4_TILE - 1) / KV4_TILE, last = (end + 63) / 64, first = (start + (cols < KV4_TILE ? cols - 1 : KV4_TILE - 1) / group + 64) / 64;
    const long long wgs = (long long)heads * col_tiles;
    int best = last;
    float least = 1e30f;
    for (int parts = 1; parts <= KV4_MAX_PARTS && (parts == 1 || (wgs <= VT_MX4_COUNTERS && last > 4 * (parts - 1))); parts++) {
        const int run = (last + parts - 1) / parts;
        const float us = vt_kv4_tiles_us((float)run, (float)first, (float)last, (float)wgs, (float)n_cu);
        if (us < least) { least = us; best = run; }
    }
    return vt_kv4_plan{1, col_tiles, best, (last + best - 1) / best};
}

/* Many columns: from two rounds of the other kernel's workgroups on (us for 32 heads on 8 of 128 values, few columns' kernel and many
 * columns': 100 queries behind 300 rows 9.5 and 21, 200 of them 17 and 23, 250 behind none 14.2 and 16.5, 300 21 and 18, 500 behind 500
 * 41 and 30; of 64 values 200 behind 300 12.9 and 17.9, 300 behind none 15.2 and 13.8), and for heads of up to 128 values, whose results
 * and queries leave two waves of a SIMD their registers.  With 192 and 256 the kernel for many columns would keep 227 and 117 registers
 * in memory: 500 queries behind 500 rows 73 and 108, 77 and 91; 1000 behind none 130 and 152, 140 and 104; 3000 806 and 808, 881 and
 * 464.  (Prompts of 1000 and more with 256 would gain by one made for them.) */
static inline vt_kv4_plan vt_kv4_plan_of(int n_cu, int hp, int heads, int group, int cols, int start, int end) {
    if (hp <= 2 && (long long)((cols + KV4_COLS - 1) / KV4_COLS) * heads > 2ll * n_cu) return vt_kv4_many(n_cu, heads, group, cols, start, end);
    return vt_kv4_few(n_cu, hp, heads, cols, end);
}

#endif /* VT_MX4_PLANS_H */
