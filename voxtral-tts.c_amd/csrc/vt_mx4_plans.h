/*
 * vt_mx4_plans.h - the 4-bit operators' launches (vt_mx4.hip, vt_kv4.hip) from shapes and the number of CUs: lanes of a conversion,
 * tiles and K cuts of a product.  Host code without HIP, so that a host test can walk it.
 */
#ifndef VT_MX4_PLANS_H
#define VT_MX4_PLANS_H

#include <math.h>
#include <stddef.h>

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

/* Tiles: weight rows, rows of x, threads, workgroups that a CU holds, and us per panel with one, two, three of them on it (from runs of one cut on
 * part of the chip and on all of it: 226 x 3072 x 9216, 1531 x 9216 x 3072). */
struct vt_mxt_tile { int bm, bn, threads, per_cu; float panel_us[3]; };
static const vt_mxt_tile vt_mxt_tiles[] = {{256, 128, 512, 1, {1.8f}}, {128, 64, 256, 2, {0.72f, 1.2f}}, {128, 32, 256, 3, {0.56f, 0.85f, 1.25f}}};
#define VT_MXT_MAX_CUTS 16
#define VT_MXT_ROWS (1 << 14)

/* Rows of x at a time: so many that the work area stays small beside the operands, and no more than a launch has threads for, the one that splits x (a
 * wave per 32 rows and 64 columns, four a workgroup) and the product's. */
static inline int vt_mxt_rows(int out_dim, int panels) {
    int rows = VT_MXT_ROWS;
    while (rows > 32 && (((long long)out_dim + 127) / 128 * (rows / 32) > vt_launch_most(256) || ((long long)rows / 32 * 2 * panels + 3) / 4 > vt_launch_most(256))) rows /= 2;
    return rows;
}

/* The tile and the cuts of K with the least time by these figures.  us a call, with the best of the others: 1531 x 9216 x 3072 107 (256 x 128 whole; 131 on 128 x 64), 512 of them 48 (the same;
 * 57), 400 41 (128 x 64 whole; 47 on 256 x 128), 1000 x 3072 x 4096 47 (128 x 64; 48), 300 x 3072 x 9216 38 (128 x 64 in 4 cuts; 41 in 3), 226 x 3072 x 9216 36, 64 x 9216 x 3072 20 (128 x 32 in 3). */
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
                              (cuts > 1 ? 2.0 + (double)seq_len * out_dim * 4.0 * (2 * cuts + 1) / 5.0e6 : 0.0);
            if (us < best.us) best = vt_mxt_plan{t, cuts, (int)m_tiles, tiles * cuts, us};
        }
    }
    return best;
}

#endif /* VT_MX4_PLANS_H */
