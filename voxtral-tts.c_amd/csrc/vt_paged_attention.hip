/*
 * vt_paged_attention.hip - attention of a batch's new rows over a paged cache of bf16 keys and values (vt_paged.h).
 *
 * The queries of the heads that share a kv head are columns (vt_paged_plans.h).  Scores are S^T[row][column] = K Q^T and results O^T[value][column] = V^T P^T
 * on the bf16 matrix instructions: keys and values as they lie, queries and weights as planes that each hold 8 bits of what the one before leaves, smallest
 * first: three make fp32 of fp32, one is a bf16 query itself, whose weights are two: 16 bits, so that its result's rounding is what is seen of them.  A lane
 * holds the same column of S^T and of O^T, and the order of the rows inside an instruction is free, so that weights go from one product to the next in their
 * registers.  Maximum, sum and results of a column are fp32, one pass over the rows with the running maximum.
 *
 * What a column does not see: a hidden score is -infinity whatever the key holds.  A hidden value's weight is 0, but 0 times an infinity or NaN would be NaN,
 * so that where rows at hand are hidden from some column and a value among them is not finite, the value counts as 0, and a product of its own, with ones as
 * the weights of what a column sees, tells which results are NaN.  Rows behind a sequence's last are never read: requests have the size of the rows that are
 * there, and the rest is zeros.
 */
#include "vt_paged.h"
#include "vt_device.h"
#include "vt_requests.h"
#include "vt_mx4_plans.h"

#include <math.h>

typedef __bf16 pa_bf16x8 __attribute__((ext_vector_type(8)));
typedef float pa_f32x16 __attribute__((ext_vector_type(16)));

/* 104 bytes at most: a launch with more takes the host 0.9 us longer */
struct pa_job {
    const uint16_t *K, *V;
    const void *Q;
    void *out;
    float *part;
    unsigned *cnt;
    const vt_paged_item *items;
    const int *tables;
    int q_stride, n_heads, page_log, window;
    vt_divisor group;
    float scale;                                         /* times log2 e */
};
static_assert(sizeof(pa_job) <= 104, "arguments");
static_assert(PAGED_COUNTERS <= VT_MX4_COUNTERS, "counters");

static __device__ __forceinline__ pa_bf16x8 pa_operand(const u32x4 &w) { return __builtin_bit_cast(pa_bf16x8, w); }

/* two values -> N planes of bf16 pairs; what a plane leaves is exact in fp32 */
template <int N>
static __device__ __forceinline__ void pa_planes2(float a, float b, unsigned (&w)[N]) {
#pragma unroll
    for (int p = 0; p < N; p++) {
        w[p] = __builtin_bit_cast(unsigned, __builtin_convertvector((f32x2{a, b}), vt_bf16x2));
        if (p + 1 < N) {
            a = __fsub_rn(a, __uint_as_float(w[p] << 16));
            b = __fsub_rn(b, __uint_as_float(w[p] & 0xffff0000u));
        }
    }
}

/* 8 values of a query as they lie, and as operands, one for each plane.  fp32 ones are scaled first; bf16 ones are the operand, and their scores are scaled. */
template <bool F32>
static __device__ __forceinline__ void pa_query_load(const void *Q, size_t at, u32x4 (&raw)[2]) {
    if constexpr (F32) {
        const u32x4 *p = reinterpret_cast<const u32x4 *>((const float *)Q + at);
        raw[0] = p[0];
        raw[1] = p[1];
    } else raw[0] = *reinterpret_cast<const u32x4 *>((const uint16_t *)Q + at);
}
template <bool F32, int NQ>
static __device__ __forceinline__ void pa_query_planes(const u32x4 (&raw)[2], float scale, u32x4 (&to)[NQ]) {
    if constexpr (F32) {
        const f32x4 a = __builtin_bit_cast(f32x4, raw[0]) * scale, b = __builtin_bit_cast(f32x4, raw[1]) * scale;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            unsigned w[NQ];
            pa_planes2<NQ>(e < 2 ? a[2 * e] : b[2 * e - 4], e < 2 ? a[2 * e + 1] : b[2 * e - 3], w);
#pragma unroll
            for (int k = 0; k < NQ; k++) to[k][e] = w[k];
        }
    } else to[0] = raw[0];
}

template <bool F32>
static __device__ __forceinline__ void pa_store4(void *out, size_t at, const f32x4 &v) {
    if constexpr (F32) *reinterpret_cast<f32x4 *>((float *)out + at) = v;
    else {
        unsigned w0[1], w1[1];
        pa_planes2<1>(v.x, v.y, w0);
        pa_planes2<1>(v.z, v.w, w1);
        *reinterpret_cast<u32x2 *>((uint16_t *)out + at) = u32x2{w0[0], w1[0]};
    }
}

/* pairs of bf16 of which one is not finite */
typedef unsigned short pa_u16x2 __attribute__((ext_vector_type(2)));
static __device__ __forceinline__ pa_u16x2 pa_larger(pa_u16x2 most, unsigned w) {
    return __builtin_elementwise_max(most, __builtin_bit_cast(pa_u16x2, w & 0x7fff7fffu));
}
static __device__ __forceinline__ bool pa_not_finite(pa_u16x2 most) { return max((int)most.x, (int)most.y) >= 0x7f80; }
/* such values as ones, others as zeros; and the other way round, they as zeros */
static __device__ __forceinline__ unsigned pa_marks(unsigned w) {
    return ((w & 0x7f80u) == 0x7f80u ? 0x3f80u : 0u) | ((w & 0x7f800000u) == 0x7f800000u ? 0x3f800000u : 0u);
}
static __device__ __forceinline__ unsigned pa_finite(unsigned w) {
    return ((w & 0x7f80u) == 0x7f80u ? 0u : w & 0xffffu) | ((w & 0x7f800000u) == 0x7f800000u ? 0u : w & 0xffff0000u);
}

static __device__ __forceinline__ float pa_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

/* A column's weights are relative to m, which follows the largest score only where that is further above than this: weights up to 2^8 are as exact as ones
 * below 1, and what was summed so far is scaled anew in the first tile and hardly ever after it (with 32 columns to a wave one of them has a new largest
 * score in nearly every tile).  The wave goes there together, but a column's m stays unless its own score is far above: what another column sees is none of
 * its business. */
#define PA_SLACK 8.f
static __device__ __forceinline__ bool pa_far(float top, float m) { return __any(!(top <= m + PA_SLACK)); }
/* -> what the column's sums are scaled by; a NaN stays one */
static __device__ __forceinline__ float pa_follow(float top, float &m) {
    if (top <= m + PA_SLACK) return 1.f;
    const float before = m;
    m = __builtin_elementwise_maximum(top, before);
    return pa_exp2(before - m);
}
template <bool F32>
static __device__ __forceinline__ float pa_weight(float s, float m, float scale) { return pa_exp2(F32 ? s - m : fmaf(s, scale, -m)); }

/* Sums that leave fp32 although their mean does not: a column's weights are relative to its m, up to 2^8 each and as many as there are rows, so that values
 * above 2^120 over the number of rows may do that.  A column whose results are not finite is summed once more with an m so much further up that all its
 * weights come to less than 1; its neighbours' m stays, and with it every bit of theirs.  (Not everybody's from the start: a product of such a weight with
 * a value is lost below 2^-126, and a score's difference to m loses bits.  A column that answers NaN or infinity anyway is summed twice.)  The look and what
 * the second copy of the loop does to the first's registers: one query behind 1999 rows 7.94 -> 8.06 us, 1531 behind none bf16 40.4 -> 40.5, heads of 256
 * 3000 rows 128 -> 134. */
static __device__ __forceinline__ float pa_largest(float so_far, const f32x4 &v) {       /* a NaN stays one */
    so_far = __builtin_elementwise_maximum(__builtin_elementwise_maximum(so_far, fabsf(v.x)), fabsf(v.y));
    return __builtin_elementwise_maximum(__builtin_elementwise_maximum(so_far, fabsf(v.z)), fabsf(v.w));
}
template <int COLS> static __device__ __forceinline__ unsigned long long pa_same_columns(unsigned long long lanes) {      /* all lanes of a column that one is of */
    lanes |= lanes >> 32 | lanes << 32;
    return COLS == 16 ? lanes | lanes >> 16 | lanes << 48 : lanes;
}
static __device__ __forceinline__ float pa_lift(unsigned long long over, int rows) {
    return over >> __lane_id() & 1 ? (float)(9 + 32 - __clz(rows)) : 0.f;
}

/* What the batch's description holds is the same for a whole workgroup: scalar loads, which the kernel's own stores cannot touch */
typedef __attribute__((address_space(4))) const int pa_const_int;
static __device__ __forceinline__ vt_paged_item pa_item(const vt_paged_item *items, int at) {
    static_assert(sizeof(vt_paged_item) == 48, "words");
    const pa_const_int *w = (const pa_const_int *)(uintptr_t)(items + at);
    return vt_paged_item{w[0], w[1], w[2], w[3], w[4], w[5], w[6], w[7], w[8], w[9], w[10], w[11]};
}

/* 16 rows from `at` on, a multiple of 16, of those lo .. end - 1: where they lie, and the bytes of them that are there */
struct pa_rows { size_t row; int bytes; };
static __device__ __forceinline__ int pa_entry(int at, int lo, int end, int page_log) { return max(min(at, end - 1), lo) >> page_log; }
static __device__ __forceinline__ pa_rows pa_rows_of(int page, int at, int lo, int end, int page_log, int heads, int head, int row_bytes) {
    const int n = at + 16 > lo ? min(max(end - at, 0), 16) : 0;
    return pa_rows{((((size_t)(unsigned)page * heads + head) << page_log) + (at & ((1 << page_log) - 1))), n * row_bytes};
}
static __device__ __forceinline__ pa_rows pa_place(const pa_const_int *table, int at, int lo, int end, int page_log, int heads, int head, int row_bytes) {
    return pa_rows_of(table[pa_entry(at, lo, end, page_log)], at, lo, end, page_log, heads, head, row_bytes);
}

/* ---- few columns ----
 * A wave has 32 rows of K and V in registers at a time, asks for the next as soon as these are used, and waits for nobody; the waves of a workgroup, and then
 * the workgroups that share the columns' rows, add their parts in a fixed order, the last workgroup to arrive those of all.  K is the A operand of 16 x 16 x
 * 32, a lane's 16 bytes from its own row.  V's rows are its columns: a lane loads CD values each of the eight rows that it has weights of, 16 lanes a whole
 * row, and pairs of rows are put together two values at a time.  Queries, the same for all waves, wait in LDS as operands.  ONCE: other workgroups
 * read few of these rows, and there are more than a cache holds.
 *
 * Rows are read as they lie and once for 16 or 32 columns, so that memory bounds a long cache: one query behind 65535 rows of 8 x 128, 268 MB, 44 us
 * (6.1 TB/s), steps of 64 sequences of 118000 rows, 483 MB, 83 us (5.8 TB/s).  A short one is bound by what follows on each other in a workgroup - its
 * item, its table, queries and rows, a part's store, counter and merge: one query behind 1999 rows 8 us a call with 4 for the launch. */
template <int HP, bool F32, int CT>
struct pa_few_sizes {
    static constexpr int OD = 64 * HP + 4, COLS = 16 * CT, QUERIES = 2 * HP * (F32 ? 3 : 1) * CT * 1024, AREA = COLS * OD * 4, ML = PAGED_FEW_WAVES * COLS * 8,
                         WT = COLS * PAGED_MAX_PARTS * 4;
};
/* LDS: `queries`, and after the last product area(k), wave k's part; ml beside both, wt where nothing is once the parts have left */
template <int HP, bool F32, bool ONCE, int CT, class AREA>
static __device__ __forceinline__ void pa_few(const pa_job &a, int item, u32x4 *queries, AREA area, float (*ml)[16 * CT][2],
                                              float (*wt)[PAGED_MAX_PARTS], int &last) {
    constexpr int HD = 64 * HP, ROW = 2 * HD, KS = 2 * HP, CD = HP % 2 ? 4 : 8, CHUNKS = HD / (16 * CD), OD = HD + 4, WAVES = PAGED_FEW_WAVES;
    constexpr int NQ = F32 ? 3 : 1, NP = F32 ? 3 : 2, COLS = 16 * CT, HOW = ONCE ? 2 /* nt */ : 0;
    const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
    const int h = (int)blockIdx.x, heads = (int)gridDim.x;
    const vt_paged_item it = pa_item(a.items, item);
    const pa_const_int *table = (const pa_const_int *)(uintptr_t)(a.tables + it.table);
    const int base = it.lo & ~(PAGED_FEW_ROWS - 1), tiles = (it.end - base + PAGED_FEW_ROWS - 1) / PAGED_FEW_ROWS;
    u32x4 k[2][KS];
    u32x4 v[8][CHUNKS];                                  /* CD == 4: the first half of each */
    pa_rows at[2];
    auto place = [&](int t) __attribute__((always_inline)) {
#pragma unroll
        for (int kt = 0; kt < 2; kt++) at[kt] = pa_place(table, base + PAGED_FEW_ROWS * t + 16 * kt, it.lo, t < tiles ? it.end : 0, a.page_log, heads, h, ROW);
    };
    auto ask_k = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int kt = 0; kt < 2; kt++) {
            const __amdgpu_buffer_rsrc_t d = vt_buffer(a.K + at[kt].row * HD, at[kt].bytes);
#pragma unroll
            for (int ks = 0; ks < KS; ks++) k[kt][ks] = __builtin_amdgcn_raw_buffer_load_b128(d, n * ROW + 64 * ks + 16 * g, 0, HOW);
        }
    };
    auto ask_v = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int kt = 0; kt < 2; kt++) {
            const __amdgpu_buffer_rsrc_t d = vt_buffer(a.V + at[kt].row * HD, at[kt].bytes);
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int ch = 0; ch < CHUNKS; ch++) {
                    const int in = (4 * g + j) * ROW + ch * 32 * CD + n * 2 * CD;
                    if constexpr (CD == 8) v[4 * kt + j][ch] = __builtin_amdgcn_raw_buffer_load_b128(d, in, 0, HOW);
                    else {
                        const u32x2 w = __builtin_amdgcn_raw_buffer_load_b64(d, in, 0, HOW);
                        v[4 * kt + j][ch] = u32x4{w.x, w.y, 0u, 0u};
                    }
                }
        }
    };
    const int nc = min(COLS, it.cols - it.c0);
    const bool two = CT == 2 && nc > 16;
    int qi[2], see_lo[2], see_hi[2];                     /* CT of them */
    size_t q_at[2];
#pragma unroll
    for (int c = 0; c < CT; c++) {
        const int cc = min(it.c0 + 16 * c + n, it.cols - 1);
        qi[c] = vt_div(cc, a.group);
        const int pos = it.past + qi[c];
        see_lo[c] = max(a.window && pos >= a.window ? pos - a.window + 1 : 0, it.lo);
        see_hi[c] = min(pos + 1, it.end);
        q_at[c] = (size_t)(it.row + qi[c]) * a.q_stride + ((size_t)h * a.group.d + (cc - qi[c] * a.group.d)) * HD;
    }
    /* queries first: loads return in order */
    constexpr int MINE = (KS * CT + WAVES - 1) / WAVES;  /* operands of queries that a wave brings: step x / CT of the product, columns 16 (x % CT) .. */
    u32x4 raw[MINE][2];
#pragma unroll
    for (int x = 0; x < MINE; x++) {
        const int y = min(wave + WAVES * x, KS * CT - 1);
        pa_query_load<F32>(a.Q, (CT == 2 && y % CT ? q_at[1] : q_at[0]) + 32 * (y / CT) + 8 * g, raw[x]);
    }
    place(wave);
    ask_k();
    ask_v();
#pragma unroll
    for (int x = 0; x < MINE; x++) {
        const int y = wave + WAVES * x;
        if (KS * CT % WAVES && y >= KS * CT) break;
        u32x4 q[NQ];
        pa_query_planes<F32, NQ>(raw[x], a.scale, q);
#pragma unroll
        for (int p = 0; p < NQ; p++) queries[(y * NQ + p) * 64 + lane] = q[p];
    }
    const int q_first = it.past + vt_div(it.c0, a.group), q_last = it.past + vt_div(it.c0 + nc - 1, a.group);
    const int all_lo = max(a.window && q_last >= a.window ? q_last - a.window + 1 : 0, it.lo), all_hi = min(q_first + 1, it.end);      /* that every column sees */
    float m[2], l[2];
    f32x4 o[CT][CHUNKS * CD];
    __syncthreads();
    auto sums = [&](const unsigned long long (&over)[2]) __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < CT; c++) {
            m[c] = -3.402823466e38f;                         /* finite: with nothing seen yet a hidden score's weight is exp2(-inf) all the same */
            l[c] = 0.f;
#pragma unroll
            for (int i = 0; i < CHUNKS * CD; i++) o[c][i] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
#pragma unroll 1
        for (int t = wave; t < tiles; t += WAVES) {
            const int first = base + PAGED_FEW_ROWS * t;
            const bool hidden = first < all_lo || first + PAGED_FEW_ROWS > all_hi;
            place(t + WAVES);
            int own = lane;                                  /* (through an empty asm: else the queries are kept in registers after all) */
            asm volatile("" : "+v"(own));
            f32x4 s[CT][2];
#pragma unroll
            for (int c = 0; c < CT; c++) {
                s[c][0] = s[c][1] = f32x4{0.f, 0.f, 0.f, 0.f};
                if (c && !two) break;
#pragma unroll
                for (int ks = 0; ks < KS; ks++)
#pragma unroll
                    for (int p = NQ - 1; p >= 0; p--) {
                        const pa_bf16x8 q = pa_operand(queries[((ks * CT + c) * NQ + p) * 64 + own]);
#pragma unroll
                        for (int kt = 0; kt < 2; kt++) s[c][kt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pa_operand(k[kt][ks]), q, s[c][kt], 0, 0, 0);
                    }
            }
            ask_k();
            auto sees = [&](int c, int kt, int v) { const int key = first + 16 * kt + 4 * g + v; return key >= see_lo[c] && key < see_hi[c]; };
            bool bad = false;
            if (hidden) {
#pragma unroll
                for (int c = 0; c < CT; c++)
#pragma unroll
                    for (int kt = 0; kt < 2; kt++)
#pragma unroll
                        for (int v = 0; v < 4; v++) s[c][kt][v] = sees(c, kt, v) ? s[c][kt][v] : -INFINITY;
                pa_u16x2 most = {0, 0};
#pragma unroll
                for (int j = 0; j < 8; j++)
#pragma unroll
                    for (int ch = 0; ch < CHUNKS; ch++)
#pragma unroll
                        for (int e = 0; e < CD / 2; e++) most = pa_larger(most, v[j][ch][e]);
                bad = __any(pa_not_finite(most));
            }
            u32x4 w4[CT][NP];
#pragma unroll
            for (int c = 0; c < CT; c++) {
                if (c && !two) break;
                float top = __builtin_elementwise_maximum(s[c][0][0], s[c][1][0]);                /* a NaN stays one: who sees it answers NaN */
#pragma unroll
                for (int v = 1; v < 4; v++) top = __builtin_elementwise_maximum(__builtin_elementwise_maximum(top, s[c][0][v]), s[c][1][v]);
                {
                    f32x2 r = vt_swap16(top, top);
                    top = __builtin_elementwise_maximum(r.x, r.y);
                    r = vt_swap32(top, top);
                    top = __builtin_elementwise_maximum(r.x, r.y);
                }
                if constexpr (!F32) top = top * a.scale;
                if (over[c]) top += pa_lift(over[c], it.end - it.lo);
                if (pa_far(top, m[c])) {
                    const float less = pa_follow(top, m[c]);
                    l[c] *= less;
#pragma unroll
                    for (int i = 0; i < CHUNKS * CD; i++) o[c][i] = o[c][i] * less;
                }
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float p0 = pa_weight<F32>(s[c][e >> 1][2 * (e & 1)], m[c], a.scale), p1 = pa_weight<F32>(s[c][e >> 1][2 * (e & 1) + 1], m[c], a.scale);
                    l[c] += p0 + p1;
                    unsigned w[NP];
                    pa_planes2<NP>(p0, p1, w);
#pragma unroll
                    for (int p = 0; p < NP; p++) w4[c][p][e] = w[p];
                }
            }
            if (bad) {                                       /* rare */
#pragma unroll
                for (int c = 0; c < CT; c++) {
                    u32x4 ones;
#pragma unroll
                    for (int e = 0; e < 4; e++) ones[e] = (sees(c, e >> 1, 2 * (e & 1)) ? 0x3f80u : 0u) | (sees(c, e >> 1, 2 * (e & 1) + 1) ? 0x3f800000u : 0u);
#pragma unroll
                    for (int ch = 0; ch < CHUNKS; ch++)
#pragma unroll
                        for (int i = 0; i < CD; i++) {
                            u32x4 v4;
#pragma unroll
                            for (int e = 0; e < 4; e++)
                                v4[e] = pa_marks(__builtin_amdgcn_perm(v[2 * e + 1][ch][i / 2], v[2 * e][ch][i / 2], i & 1 ? 0x07060302u : 0x05040100u));
                            const f32x4 hit = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pa_operand(v4), pa_operand(ones), (f32x4{0.f, 0.f, 0.f, 0.f}), 0, 0, 0);
#pragma unroll
                            for (int e = 0; e < 4; e++) o[c][ch * CD + i][e] = hit[e] > 0.f ? NAN : o[c][ch * CD + i][e];
                        }
                }
#pragma unroll
                for (int j = 0; j < 8; j++)
#pragma unroll
                    for (int ch = 0; ch < CHUNKS; ch++)
#pragma unroll
                        for (int e = 0; e < CD / 2; e++) v[j][ch][e] = pa_finite(v[j][ch][e]);
            }
#pragma unroll
            for (int ch = 0; ch < CHUNKS; ch++)
#pragma unroll
                for (int i = 0; i < CD; i++) {
                    u32x4 v4;
#pragma unroll
                    for (int e = 0; e < 4; e++) v4[e] = __builtin_amdgcn_perm(v[2 * e + 1][ch][i / 2], v[2 * e][ch][i / 2], i & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
                    for (int p = NP - 1; p >= 0; p--)
                        o[0][ch * CD + i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pa_operand(v4), pa_operand(w4[0][p]), o[0][ch * CD + i], 0, 0, 0);
                    if constexpr (CT == 2) {                 /* (also where there is no second: a branch for each would cost more) */
#pragma unroll
                        for (int p = NP - 1; p >= 0; p--)
                            o[CT - 1][ch * CD + i] =
                                __builtin_amdgcn_mfma_f32_16x16x32_bf16(pa_operand(v4), pa_operand(w4[CT - 1][p]), o[CT - 1][ch * CD + i], 0, 0, 0);
                    }
                }
            ask_v();
        }
    };
    unsigned long long over[2] = {0, 0};
    sums({0, 0});
#pragma unroll
    for (int c = 0; c < CT; c++) {
        if (c && !two) break;
        float most = 0.f;
#pragma unroll
        for (int i = 0; i < CHUNKS * CD; i++) most = pa_largest(most, o[c][i]);
        over[c] = pa_same_columns<16>(__ballot(!(most < INFINITY)));
    }
    if (__builtin_expect((over[0] | over[1]) != 0, 0)) { /* rare */
        place(wave);
        ask_k();
        ask_v();
        sums(over);
    }
    /* The waves' parts, each times its share of the sum of weights: a mean of values */
#pragma unroll
    for (int c = 0; c < CT; c++) {
        l[c] = vt_rows_sum(l[c]);
        ml[wave][16 * c + n][0] = m[c];                  /* four lanes the same */
        ml[wave][16 * c + n][1] = l[c];
    }
    __syncthreads();
    float M[2], L[2];
#pragma unroll
    for (int c = 0; c < CT; c++) {
        const int col = 16 * c + n;
        M[c] = m[c];
        L[c] = 0.f;
#pragma unroll
        for (int k = 0; k < WAVES; k++) M[c] = fmaxf(M[c], ml[k][col][0]);
#pragma unroll
        for (int k = 0; k < WAVES; k++) L[c] = fmaf(ml[k][col][1], pa_exp2(ml[k][col][0] - M[c]), L[c]);
        const float f = L[c] == 0.f && it.parts > 1 ? 0.f : pa_exp2(m[c] - M[c]) / L[c];
        float *to = area(wave) + col * OD + 4 * g * CD;
#pragma unroll
        for (int ch = 0; ch < CHUNKS; ch++)
#pragma unroll
            for (int v = 0; v < 4; v++)
#pragma unroll
                for (int i = 0; i < CD; i++) to[16 * CD * ch + CD * v + i] = o[c][ch * CD + i][v] * f;
    }
    __syncthreads();
    const __amdgpu_buffer_rsrc_t pd = vt_buffer(a.part + (size_t)(it.slot * heads + h * it.parts) * COLS * OD, it.parts * COLS * OD * 4);
    auto result = [&](int col, int d, const f32x4 &v) {
        const int k = it.c0 + col, i = vt_div(k, a.group);
        const size_t to = ((size_t)(it.row + i) * a.n_heads + (size_t)h * a.group.d + (k - i * a.group.d)) * HD + d;
        pa_store4<F32>(a.out, to, v);
    };
    for (int e = (int)threadIdx.x; e < nc * (HD / 4); e += 64 * WAVES) {
        const int col = e / (HD / 4), d = 4 * (e - col * (HD / 4));
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < WAVES; k++) v = v + *reinterpret_cast<const f32x4 *>(area(k) + col * OD + d);
        if (it.parts == 1) result(col, d, v);
        else {
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), pd, ((it.part * COLS + col) * OD + 4 + d) * 4, 0, 16 /* sc1 */);
        }
    }
    if (it.parts == 1) return;
    if (wave == 0 && g < CT && 16 * g + n < nc) {
        const float most = CT == 2 && g ? M[CT - 1] : M[0], sum = CT == 2 && g ? L[CT - 1] : L[0];
        __builtin_amdgcn_raw_buffer_store_b64(u32x2{__float_as_uint(most), __float_as_uint(sum)}, pd, (it.part * COLS + lane) * OD * 4, 0, 16);
    }
    __builtin_amdgcn_s_waitcnt(0x0f70);                  /* the part's stores are acknowledged */
    __syncthreads();
    unsigned *cnt = a.cnt + it.counter * heads + h;
    if (threadIdx.x == 0) last = __hip_atomic_fetch_add(cnt, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)(it.parts - 1);
    __syncthreads();
    if (!last) return;
    if (threadIdx.x == 0) vt_stc_u32(cnt, 0u);           /* ready for the next launch */
    /* a wave per column: lane k has part k's largest score and sum of weights */
    for (int col = wave; col < nc; col += WAVES) {
        const u32x2 v = __builtin_amdgcn_raw_buffer_load_b64(pd, (min(lane, it.parts - 1) * COLS + col) * OD * 4, 0, 16 /* sc1 */);
        const float pm = __uint_as_float(v.x), pl = lane < it.parts ? __uint_as_float(v.y) : 0.f;
        const float w = pl * pa_exp2(pm - vt_wave_max(pm)), all = vt_wave_sum(w);
        wt[col][lane] = w / all;
    }
    __syncthreads();
    for (int e = (int)threadIdx.x; e < nc * (HD / 4); e += 64 * WAVES) {
        const int col = e / (HD / 4), d = 4 * (e - col * (HD / 4)), from = (col * OD + 4 + d) * 4;
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
        for (int k0 = 0; k0 < it.parts; k0 += 16) {      /* parts past the last: the last again, times 0 */
            f32x4 p[16];
#pragma unroll
            for (int k = 0; k < 16; k++)
                p[k] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(pd, from + min(k0 + k, it.parts - 1) * (COLS * OD * 4), 0, 16));
#pragma unroll
            for (int k = 0; k < 16; k++) v = v + p[k] * wt[col][k0 + k];
        }
        result(col, d, v);
    }
}

/* ---- many columns ----
 * A workgroup has 128 columns, a wave 32, and goes through its rows 64 at a time, 16 of them each wave's to ask for, by requests that write LDS.  K's rows
 * are the A operand of 32 x 32 x 16 as they lie; of V, whose rows are that operand's columns, the transposing reads of LDS give a lane four rows' values of
 * one column.
 *
 * A unit is 32 rows.  While unit u's weights are made and multiplied, the matrix cores make unit u + 1's scores, so that K's tiles lie half a tile behind
 * V's: beside V's rows 64 t .. 64 t + 63 stand K's 64 t + 32 .. 64 t + 95.
 *
 * Matrix instructions bound it, and for bf16 the vector unit beside them, which has two values' weights to make for each: with two waves to a SIMD they overlap
 * little (busy 49 and 39 % of the time; 62 and 35 in fp32).  4000 rows behind none of 32 heads of 128 fp32 (three planes of queries and of weights, 393 G
 * multiplications and additions) 316 us, the rate of a large matrix product, bf16 (two planes of weights, 197 G) 193 us; 1531 rows fp32 61 us, of which the
 * first tiles' way and the parts' end are 15; four prompts of 226 to 2000 rows in a window of 2048 bf16 137 us.  Heads of 256 bf16 values have one workgroup
 * to a CU, for its LDS and registers: 3000 rows of 12 on 4 behind none 134 us (83 G).  With weights of one plane these three take 153, 107 and 115 us, and a
 * result is off by 2.1e-3 of its norm instead of the 1.6e-3 that its own rounding leaves. */
typedef short pa_s16x4 __attribute__((ext_vector_type(4)));

/* fp32: the compiler keeps to the order that is written, in which an instruction's operands are asked for just ahead of it and no more of them wait in
 * registers than there are; bf16 has registers for its own order (four prompts in a window 142.0 us as written, 140.4 so, 138.6 with the weights held
 * ahead of the branch) */
template <bool F32> static __device__ __forceinline__ void pa_here() { if constexpr (F32) __builtin_amdgcn_sched_barrier(0); }

/* Tiles with rows that some column does not see: at most 3 where the columns' rows begin to be seen and 3 where they end (fewer queries than 128 apart), or 5
 * with a window of less.  `marks`: of such a tile the values that are not finite, 32 of a row's to a word; `odd`: where there are any. */
#define PA_EDGES 6
template <int HP, bool F32>
static __device__ __forceinline__ void pa_many(const pa_job &a, int item, unsigned char *k0, unsigned char *k1, unsigned char *v0, unsigned char *v1,
                                               unsigned (*marks)[64][2 * HP], int (*odd)[4], int &last) {
    constexpr int HD = 64 * HP, ROW = 2 * HD, WAVES = 4, DT = 2 * HP, KS = 4 * HP, PIECES = HD / 8, EDGES = PA_EDGES;
    constexpr int NQ = F32 ? 3 : 1, NP = F32 ? 3 : 2;
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 31, g = lane >> 5;
    const int h = (int)blockIdx.x, heads = (int)gridDim.x;
    const vt_paged_item it = pa_item(a.items, item);
    const pa_const_int *table = (const pa_const_int *)(uintptr_t)(a.tables + it.table);
    const int w0 = it.c0 + 32 * wave, wc = min(w0 + 32, it.cols) - w0;                   /* this wave's columns: none, perhaps */
    const int cc = min(w0 + n, it.cols - 1), qi = vt_div(cc, a.group), pos = it.past + qi;
    const int see_lo = max(a.window && pos >= a.window ? pos - a.window + 1 : 0, it.lo), see_hi = min(pos + 1, it.end);
    const int q_first = it.past + vt_div(min(w0, it.cols - 1), a.group), q_last = it.past + vt_div(min(w0 + 31, it.cols - 1), a.group);
    const int all_lo = max(a.window && q_last >= a.window ? q_last - a.window + 1 : 0, it.lo);          /* rows that every column of the wave sees */
    const int all_hi = min(q_first + 1, it.end);
    const int any_lo = a.window && q_first >= a.window ? q_first - a.window + 1 : 0, any_hi = wc > 0 ? min(q_last + 1, it.end) : 0;   /* .. that any does */
    const int wg_last = it.past + vt_div(min(it.c0 + PAGED_MANY_COLS, it.cols) - 1, a.group);
    const int wg_lo = max(a.window && wg_last >= a.window ? wg_last - a.window + 1 : 0, it.lo);             /* rows that every column sees */
    const int wg_hi = min(it.past + vt_div(it.c0, a.group) + 1, it.end);
    const int base = it.lo & ~(PAGED_MANY_ROWS - 1), tiles = (it.end - base + PAGED_MANY_ROWS - 1) / PAGED_MANY_ROWS;
    const size_t head_at = (size_t)h * a.group.d + (cc - qi * a.group.d);
    u32x4 raw[KS][2];
#pragma unroll
    for (int ks = 0; ks < KS; ks++) pa_query_load<F32>(a.Q, (size_t)(it.row + qi) * a.q_stride + head_at * HD + 16 * ks + 8 * g, raw[ks]);
    /* Pieces of 16 bytes change places within a row, so that what is read at once lies in different banks: K's with the row's last bits, so that 16 (8)
     * rows' same piece do; V's fours of them, so that four rows' same 64 bytes do. */
    constexpr int SWAP = PIECES < 16 ? PIECES - 1 : 15;
    auto v_swap = [](int r) { return HP == 1 ? 4 * ((r >> 1) & 1) : 4 * (r & 3); };
    int k_at[8], v_at[8];                                /* DT of them (with that size the host pass drops the kernel) */
#pragma unroll
    for (int d = 0; d < DT; d++) {
        const int u = d * 64 + lane, r = u / PIECES;
        k_at[d] = r * ROW + ((u - r * PIECES) ^ (r & SWAP)) * 16;
        v_at[d] = r * ROW + ((u - r * PIECES) ^ v_swap(r)) * 16;
    }
    /* The wave's pages of the next 64 tiles, a lane each: scalar loads on their way would turn every wait for LDS into one for all of LDS and for them. */
    int k_page, v_page;
    auto pages = [&](int t) __attribute__((always_inline)) {
        const int own = base + 64 * (t + lane) + 16 * wave;
        k_page = table[pa_entry(own + 32, it.lo, it.end, a.page_log)];
        v_page = table[pa_entry(own, it.lo, it.end, a.page_log)];
    };
    auto k_place = [&](int t) __attribute__((always_inline)) {
        return pa_rows_of(__builtin_amdgcn_readlane(k_page, t & 63), base + 64 * t + 32 + 16 * wave, it.lo, it.end, a.page_log, heads, h, ROW);
    };
    auto v_place = [&](int t) __attribute__((always_inline)) {
        return pa_rows_of(__builtin_amdgcn_readlane(v_page, t & 63), base + 64 * t + 16 * wave, it.lo, it.end, a.page_log, heads, h, ROW);
    };
    auto load = [&](const uint16_t *pool, const pa_rows &at, const int (&from)[8], unsigned char *to) __attribute__((always_inline)) {
        const __amdgpu_buffer_rsrc_t d = vt_buffer(pool + at.row * HD, at.bytes);
#pragma unroll
        for (int i = 0; i < DT; i++)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(d, (__attribute__((address_space(3))) void *)(to + wave * 16 * ROW + i * 1024), 16, from[i], 0, 0, 0);
    };
    auto first_tiles = [&]() __attribute__((always_inline)) {
        pages(0);
        load(a.K, pa_place(table, base - 32 + 16 * wave, it.lo, it.end, a.page_log, heads, h, ROW), k_at, k1);
        load(a.V, v_place(0), v_at, v0);
        load(a.K, k_place(0), k_at, k0);
    };
    first_tiles();
    u32x4 q[KS][NQ];                                     /* (made while the first tiles are on their way) */
#pragma unroll
    for (int ks = 0; ks < KS; ks++) pa_query_planes<F32, NQ>(raw[ks], a.scale, q[ks]);
    float m, l;
    pa_f32x16 o[DT];
    unsigned long long over = 0;
    /* addresses in LDS: one for all of K's pieces and one for all of V's, which differ from them in bits of their own.  (fp32: through an empty asm in each
     * unit, else each piece's, for each buffer, is kept in a register.) */
    const int k_base = n * ROW + (g ^ (n & SWAP)) * 16, r4 = (n & 15) >> 2;
    const int v_base = (4 * g + r4) * ROW + (v_swap(r4) + 2 * (n >> 4) + ((n & 3) >> 1)) * 16 + (n & 1) * 8;
    auto read_k = [&](const unsigned char *kb, int half, int ks, int from) __attribute__((always_inline)) {
        return pa_operand(*reinterpret_cast<const u32x4 *>(kb + 32 * half * ROW + (from ^ (32 * ks))));
    };
    /* values 32 i + n of rows 16 st + 8 (j / 4) + 4 g + j % 4 */
    auto read_v = [&](const unsigned char *vb, int st, int i, int from) __attribute__((always_inline)) {
        const unsigned char *p = vb + 16 * st * ROW + (from ^ (64 * i));
        const pa_s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) pa_s16x4 *)p);
        const pa_s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) pa_s16x4 *)(p + 8 * ROW));
        return __builtin_bit_cast(u32x4, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    auto visible = [&](int u) { const int from = base + 32 * u; return from < any_hi && from + 32 > any_lo; };
    auto hidden = [&](int u) { const int from = base + 32 * u; return from < all_lo || from + 32 > all_hi; };          /* from some column */
    auto sees = [&](int u, int v) { const int key = base + 32 * u + 8 * (v >> 2) + 4 * g + (v & 3); return key >= see_lo && key < see_hi; };
    auto hide = [&](int u, pa_f32x16 &s) __attribute__((always_inline)) {
        if (hidden(u)) {
#pragma unroll
            for (int v = 0; v < 16; v++) s[v] = sees(u, v) ? s[v] : -INFINITY;
        }
    };
    auto follow = [&](float top) __attribute__((always_inline)) {         /* the running maximum; a NaN stays one: who sees it answers NaN */
        { const f32x2 r = vt_swap32(top, top); top = __builtin_elementwise_maximum(r.x, r.y); }
        if constexpr (!F32) top = top * a.scale;
        if (over) top += pa_lift(over, it.end - it.lo);
        if (pa_far(top, m)) {
            const float less = pa_follow(top, m);
            l *= less;
#pragma unroll
            for (int i = 0; i < DT; i++) o[i] = o[i] * less;
        }
    };
    /* Where rows of a V tile are hidden from some column, values that are not finite become 0, and are remembered.  All waves come here or none. */
    int edges;                                           /* tiles that were looked at: the first ones up to the rows that all columns see, and the last ones */
    auto look = [&](int t, unsigned char *vb) __attribute__((always_inline)) {
        if ((base + 64 * t >= wg_lo && base + 64 * t + 64 <= wg_hi) || edges == EDGES) return;
        pa_u16x2 most = {0, 0};
        unsigned char *mine = vb + 16 * wave * ROW;
#pragma unroll
        for (int i = 0; i < DT; i++) {
            const u32x4 w = *reinterpret_cast<const u32x4 *>(mine + (i * 64 + lane) * 16);
#pragma unroll
            for (int e = 0; e < 4; e++) most = pa_larger(most, w[e]);
        }
        const int bad = __any(pa_not_finite(most));
        if (lane == 0) odd[edges][wave] = bad;
        if (bad) {                                       /* rare; what it derives from the lane is not kept in registers for it */
            int own = lane;
            asm volatile("" : "+v"(own));
#pragma unroll
            for (int i = 0; i < DT; i++) {
                const int u = i * 64 + own, r = u / PIECES, piece = (u - r * PIECES) ^ v_swap(r);
                u32x4 w = *reinterpret_cast<const u32x4 *>(mine + u * 16);
                unsigned bits = 0;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const unsigned x = pa_marks(w[e]);
                    bits |= (x & 0x3f80u ? 1u : 0u) << (2 * e) | (x & 0x3f800000u ? 2u : 0u) << (2 * e);
                    w[e] = pa_finite(w[e]);
                }
                *reinterpret_cast<u32x4 *>(mine + u * 16) = w;
                reinterpret_cast<unsigned char *>(&marks[edges][16 * wave + r][0])[piece] = (unsigned char)bits;
            }
        }
        __syncthreads();
        edges++;
    };
    /* pairs of weights that are made beside the scores; the others beside the first products with values.  An instruction takes the matrix cores 32 cycles,
     * a pair 70 (fp32, with twice the instructions: 90) of the vector unit. */
    constexpr int EARLY = F32 ? 8 : HP == 1 ? 6 : 5, AHEAD = F32 ? 1 : 3, BEFORE = F32 ? 1 : 2;
    /* (AHEAD: operands that are asked for ahead of their instruction; BEFORE: those in front of what depends on the maximum) */
    float top;                                           /* the largest score of the unit at hand, in a lane's rows */
    auto unit = [&](int u, const unsigned char *kb, int khalf, pa_f32x16 &next, pa_f32x16 &s, const unsigned char *vb, int vhalf) __attribute__((always_inline)) {
        if (!visible(u)) {
            if (!visible(u + 1)) return;
#pragma unroll
            for (int v = 0; v < 16; v++) s[v] = -INFINITY;
            top = -INFINITY;
        }
        int k_from = k_base, v_from = v_base;
        if constexpr (F32) asm volatile("" : "+v"(k_from), "+v"(v_from));
        u32x4 w4[2][NP];
        auto weigh = [&](int e) __attribute__((always_inline)) {
            const float p0 = pa_weight<F32>(s[2 * e], m, a.scale), p1 = pa_weight<F32>(s[2 * e + 1], m, a.scale);
            l += p0 + p1;
            unsigned w[NP];
            pa_planes2<NP>(p0, p1, w);
#pragma unroll
            for (int p = 0; p < NP; p++) w4[e >> 2][p][e & 3] = w[p];
        };
        next = pa_f32x16{};
        pa_bf16x8 k[KS];
        u32x4 v[2 * DT];
#pragma unroll
        for (int ks = 0; ks < AHEAD; ks++) k[ks] = read_k(kb, khalf, ks, k_from);
        pa_here<F32>();
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            const int then = ks + AHEAD;
            if (then < KS) k[then] = read_k(kb, khalf, then, k_from);
            else v[then - KS] = read_v(vb, 2 * vhalf + (then - KS) / DT, (then - KS) % DT, v_from);
#pragma unroll
            for (int p = NQ - 1; p >= 0; p--) next = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k[ks], pa_operand(q[ks][p]), next, 0, 0, 0);
            if (ks == BEFORE - 1) follow(top);
            if (ks >= BEFORE) {
#pragma unroll
                for (int e = EARLY * (ks - BEFORE) / (KS - BEFORE); e < EARLY * (ks - BEFORE + 1) / (KS - BEFORE); e++) weigh(e);
            }
            pa_here<F32>();
        }
        if constexpr (!F32) {                            /* else the compiler moves them behind hide's branch, where no scores are made */
#pragma unroll
            for (int e = 0; e < EARLY; e++)
#pragma unroll
                for (int p = 0; p < NP; p++) asm volatile("" : "+v"(w4[e >> 2][p][e & 3]));
            asm volatile("" : "+v"(l));
        }
        hide(u + 1, next);
        top = next[0];
        pa_here<F32>();
#pragma unroll
        for (int x = 0; x < 2 * DT; x++) {               /* 16 rows a step: elements 8 st .. of the scores */
            const int st = x / DT, i = x % DT;
            const int then = x + AHEAD;
            if (then < 2 * DT) v[then] = read_v(vb, 2 * vhalf + then / DT, then % DT, v_from);
#pragma unroll
            for (int p = NP - 1; p >= 0; p--) o[i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(pa_operand(v[x]), pa_operand(w4[st][p]), o[i], 0, 0, 0);
            if (st == 0) {
#pragma unroll
                for (int e = EARLY + (8 - EARLY) * i / DT; e < EARLY + (8 - EARLY) * (i + 1) / DT; e++) weigh(e);
            } else {
#pragma unroll
                for (int e = 16 * i / DT; e < 16 * (i + 1) / DT; e += 2)
                    top = __builtin_elementwise_maximum(__builtin_elementwise_maximum(top, next[e]), next[e + 1]);
            }
            pa_here<F32>();
        }
    };
    pa_f32x16 sa, sb;
    auto step = [&](int t, const unsigned char *kb, unsigned char *vb, unsigned char *k_to, unsigned char *v_to) __attribute__((always_inline)) {
        if (t + 1 < tiles) {
            if (((t + 1) & 63) == 0) pages(t + 1);
            load(a.K, k_place(t + 1), k_at, k_to);
            load(a.V, v_place(t + 1), v_at, v_to);
        }
        look(t, vb);
        unit(2 * t, kb, 0, sb, sa, vb, 0);
        unit(2 * t + 1, kb, 1, sa, sb, vb, 1);
        __builtin_amdgcn_s_waitcnt(0x0f70);              /* the next tiles have arrived */
        __syncthreads();
    };
    auto sums = [&]() __attribute__((always_inline)) {
        m = -3.402823466e38f;
        l = 0.f;
        top = -INFINITY;
        edges = 0;
#pragma unroll
        for (int i = 0; i < DT; i++) o[i] = pa_f32x16{};
        __builtin_amdgcn_s_waitcnt(0x0f70);
        __syncthreads();
        if (visible(0)) {                                /* the first unit's scores */
            sa = pa_f32x16{};
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                const pa_bf16x8 k = read_k(k1, 1, ks, k_base);
#pragma unroll
                for (int p = NQ - 1; p >= 0; p--) sa = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k, pa_operand(q[ks][p]), sa, 0, 0, 0);
            }
            hide(0, sa);
#pragma unroll
            for (int v = 0; v < 16; v++) top = __builtin_elementwise_maximum(top, sa[v]);
        }
        __syncthreads();
#pragma unroll 1
        for (int t = 0; t < tiles; t += 2) {
            step(t, k0, v0, k1, v1);
            if (t + 1 >= tiles) break;
            step(t + 1, k1, v1, k0, v0);
        }
    };
    if (tid == 0) last = 0;
    sums();
    {
        float most = 0.f;
#pragma unroll
        for (int i = 0; i < DT; i++)
#pragma unroll
            for (int v = 0; v < 16; v += 4) most = pa_largest(most, f32x4{o[i][v], o[i][v + 1], o[i][v + 2], o[i][v + 3]});
        over = pa_same_columns<32>(__ballot(!(most < INFINITY)));
        if (over && lane == 0) last = 1;
        __syncthreads();
    }
    if (__builtin_expect(last, 0)) {                     /* rare; all waves go, for their requests and barriers */
        first_tiles();
        sums();
    }
    { const f32x2 r = vt_swap32(l, l); l = r.x + r.y; }
    {
        const float f = l == 0.f && it.parts > 1 ? 0.f : 1.f / l;
#pragma unroll
        for (int i = 0; i < DT; i++) o[i] = o[i] * f;
    }
    /* results of who sees a value that is not finite */
#pragma unroll 1
    for (int x = 0, t = 0; x < edges; x++, t++) {
        while (base + 64 * t >= wg_lo && base + 64 * t + 64 <= wg_hi) t++;         /* the x-th tile that was looked at */
#pragma unroll 1
        for (int r = 0; r < 64; r++) {
            if (!odd[x][r / 16]) { r += 15; continue; }
            const int key = base + 64 * t + r;
            const bool see = key >= see_lo && key < see_hi;
#pragma unroll
            for (int i = 0; i < DT; i++) {
                const unsigned w = see ? marks[x][r][i] >> (4 * g) : 0u;
                if (__any(w)) {
#pragma unroll
                    for (int v = 0; v < 16; v++) o[i][v] = w >> (8 * (v >> 2) + (v & 3)) & 1u ? NAN : o[i][v];
                }
            }
        }
    }
    if (it.parts > 1) {
        /* a part lies as the lanes hold it: [part][wave][4 DT vectors of four, then largest score and sum of weights][lane] */
        constexpr int WAVE_PART = (DT * 4 + 1) * 1024, PART = WAVES * WAVE_PART;
        const __amdgpu_buffer_rsrc_t pd = vt_buffer((unsigned char *)a.part + (size_t)(it.slot * heads + h * it.parts) * PART, it.parts * PART);
        const int mine = wave * WAVE_PART + lane * 16;
#pragma unroll
        for (int i = 0; i < DT; i++)
#pragma unroll
            for (int v = 0; v < 4; v++)
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, (f32x4{o[i][4 * v], o[i][4 * v + 1], o[i][4 * v + 2], o[i][4 * v + 3]})), pd,
                                                       mine + it.part * PART + (4 * i + v) * 1024, 0, 16 /* sc1 */);
        __builtin_amdgcn_raw_buffer_store_b64(u32x2{__float_as_uint(m), __float_as_uint(l)}, pd, mine + it.part * PART + DT * 4 * 1024, 0, 16);
        __builtin_amdgcn_s_waitcnt(0x0f70);              /* acknowledged */
        __syncthreads();
        unsigned *cnt = a.cnt + it.counter * heads + h;
        if (tid == 0) last = __hip_atomic_fetch_add(cnt, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)(it.parts - 1);
        __syncthreads();
        if (!last) return;
        if (tid == 0) vt_stc_u32(cnt, 0u);
        if (wc <= 0) return;
        float M = -3.402823466e38f, L = 0.f;
#pragma unroll 4
        for (int k = 0; k < it.parts; k++) {
            const u32x2 v = __builtin_amdgcn_raw_buffer_load_b64(pd, mine + k * PART + DT * 4 * 1024, 0, 16);
            const float pm = __uint_as_float(v.x), top = fmaxf(M, pm);
            L = fmaf(L, pa_exp2(M - top), __uint_as_float(v.y) * pa_exp2(pm - top));
            M = top;
        }
#pragma unroll
        for (int i = 0; i < DT; i++) o[i] = pa_f32x16{};
#pragma unroll 1
        for (int k = 0; k < it.parts; k++) {
            const u32x2 one = __builtin_amdgcn_raw_buffer_load_b64(pd, mine + k * PART + DT * 4 * 1024, 0, 16);
            f32x4 p[DT * 4];
#pragma unroll
            for (int x = 0; x < DT * 4; x++) p[x] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(pd, mine + k * PART + x * 1024, 0, 16));
            const float w = __uint_as_float(one.y) * pa_exp2(__uint_as_float(one.x) - M) / L;
#pragma unroll
            for (int x = 0; x < DT * 4; x++)
#pragma unroll
                for (int e = 0; e < 4; e++) o[x / 4][4 * (x % 4) + e] = fmaf(p[x][e], w, o[x / 4][4 * (x % 4) + e]);
        }
    }
    /* element v of lane l in o[i] is value 32 i + 8 (v / 4) + 4 (l / 32) + v % 4 */
    if (n < wc) {
        const size_t to = ((size_t)(it.row + qi) * a.n_heads + head_at) * HD;
#pragma unroll
        for (int i = 0; i < DT; i++)
#pragma unroll
            for (int v = 0; v < 16; v += 4) pa_store4<F32>(a.out, to + 32 * i + 2 * v + 4 * g, f32x4{o[i][v], o[i][v + 1], o[i][v + 2], o[i][v + 3]});
    }
}

template <int HP, bool F32, bool ONCE, int CT>
__global__ void __launch_bounds__(64 * PAGED_FEW_WAVES, 2) vt_paged_few_kernel(pa_job a) {
    typedef pa_few_sizes<HP, F32, CT> S;
    __shared__ __attribute__((aligned(16))) float area[PAGED_FEW_WAVES][S::COLS][S::OD];
    __shared__ float ml[PAGED_FEW_WAVES][S::COLS][2], wt[S::COLS][PAGED_MAX_PARTS];
    __shared__ int last;
    static_assert(sizeof area >= S::QUERIES, "operands");
    pa_few<HP, F32, ONCE, CT>(a, (int)blockIdx.y, reinterpret_cast<u32x4 *>(area), [&](int k) { return &area[k][0][0]; }, ml, wt, last);
}

/* objects of their own: a read waits for the requests that write the same one */
#define PA_MANY_LDS(HP)                                                                                                               \
    __shared__ __attribute__((aligned(16))) unsigned char k0[64 * 128 * HP], k1[64 * 128 * HP], v0[64 * 128 * HP], v1[64 * 128 * HP]; \
    __shared__ __attribute__((aligned(16))) unsigned marks[PA_EDGES][64][2 * HP];                                                     \
    __shared__ int odd[PA_EDGES][4], last;

template <int HP, bool F32>
__global__ void __launch_bounds__(256, HP <= 2 ? 2 : 1) vt_paged_many_kernel(pa_job a) {
    PA_MANY_LDS(HP)
    pa_many<HP, F32>(a, (int)blockIdx.y, k0, k1, v0, v1, marks, odd, last);
}

/* Prompts and steps in one launch, an item either kernel's work: what reads memory and what multiplies share the CUs.  One behind the other / so: 512 rows
 * behind 1500 with 31 steps behind up to 1999 bf16 59 / 42 us, with steps behind 60 to 9000 71 / 53 (fp32 88 / 72), 300 behind 6000 with three behind 10000
 * to 30000 90 / 72. */
template <int HP, bool F32, bool ONCE>
__global__ void __launch_bounds__(256, 2) vt_paged_both_kernel(pa_job a) {
    typedef pa_few_sizes<HP, F32, 1> S;
    PA_MANY_LDS(HP)
    static_assert(S::QUERIES <= sizeof k0 && S::AREA <= sizeof k0 && S::ML <= sizeof marks && S::WT <= sizeof k0, "LDS");
    const int y = (int)blockIdx.y;
    if (pa_item(a.items, y).many) pa_many<HP, F32>(a, y, k0, k1, v0, v1, marks, odd, last);
    else
        pa_few<HP, F32, ONCE, 1>(a, y, reinterpret_cast<u32x4 *>(k0),
                                 [&](int k) { return reinterpret_cast<float *>(k == 0 ? k0 : k == 1 ? k1 : k == 2 ? v0 : v1); },
                                 reinterpret_cast<float (*)[16][2]>(marks),
                                 reinterpret_cast<float (*)[PAGED_MAX_PARTS]>(k0), last);
}

/* items are the grid's second dimension, of at most 65535 */
template <class F>
static void pa_items(const pa_job &job, int from, int n, int heads, F launch) {
    for (int at = 0; at < n; at += 65535) {
        pa_job part = job;
        part.items = job.items + from + at;
        launch(part, dim3((unsigned)heads, (unsigned)(n - at < 65535 ? n - at : 65535)));
    }
}

template <int HP, bool F32>
static void pa_launch(const pa_job &job, const vt_paged_plan &p, int heads) {
    if constexpr (HP <= 2) {
        if (p.both) {
            const dim3 grid((unsigned)heads, (unsigned)(p.few + p.many));
            if (p.once) hipLaunchKernelGGL((vt_paged_both_kernel<HP, F32, true>), grid, dim3(256), 0, g_vt.stream, job);
            else hipLaunchKernelGGL((vt_paged_both_kernel<HP, F32, false>), grid, dim3(256), 0, g_vt.stream, job);
            return;
        }
    }
    pa_items(job, 0, p.few, heads, [&](const pa_job &a, const dim3 &grid) {
        const dim3 threads(64 * PAGED_FEW_WAVES);
        if constexpr (HP <= 2) {
            if (p.wide) { hipLaunchKernelGGL((vt_paged_few_kernel<HP, F32, false, 2>), grid, threads, 0, g_vt.stream, a); return; }
        }
        if (p.once) hipLaunchKernelGGL((vt_paged_few_kernel<HP, F32, true, 1>), grid, threads, 0, g_vt.stream, a);
        else hipLaunchKernelGGL((vt_paged_few_kernel<HP, F32, false, 1>), grid, threads, 0, g_vt.stream, a);
    });
    if constexpr (HP <= 2 || (HP == 4 && !F32))
        pa_items(job, p.few, p.many, heads,
                 [](const pa_job &a, const dim3 &grid) { hipLaunchKernelGGL((vt_paged_many_kernel<HP, F32>), grid, dim3(256), 0, g_vt.stream, a); });
}

extern "C" int tts_hip_paged_attention(void *d_out, const void *d_Q, int x_bf16, int q_stride, const tts_hip_paged_t *b, const void *d_k_pages,
                                       const void *d_v_pages, float scale) {
    static const char who[] = "tts_hip_paged_attention";
    if (!b) { vt_set_error("%s: no batch", who); return -1; }
    if (!d_out || !d_Q || !d_k_pages || !d_v_pages || (((uintptr_t)d_out | (uintptr_t)d_Q | (uintptr_t)d_k_pages | (uintptr_t)d_v_pages) & 15)) {
        vt_set_error("%s: queries, results and pages lie on 16 bytes", who);
        return -1;
    }
    const vt_paged_shape &s = b->shape;
    const int width = s.n_heads * s.head_dim, HP = s.head_dim / 64;
    if (q_stride == 0) q_stride = width;
    if (q_stride < width || q_stride % 8) { vt_set_error("%s: rows of %d values %d apart (a multiple of 8)", who, width, q_stride); return -1; }
    if (!(scale > 0) || isinf(scale)) { vt_set_error("%s: scale %g", who, scale); return -1; }
    if (!vt_paged_ready(who, b)) return -1;
    if (b->n_rows == 0) return 0;
    const int group = s.n_heads / s.n_kv_heads;
    int page_log = 4;
    while (1 << page_log < s.page_rows) page_log++;
    const vt_paged_plan &p = b->plan[x_bf16 != 0];
    const long long few = p.few_slots * vt_paged_few_part(s, p.wide ? 32 : 16), many = p.many_slots ? (p.many_slot + p.many_slots) * vt_paged_many_part(s) : 0;
    pa_job job = {(const uint16_t *)d_k_pages, (const uint16_t *)d_v_pages, d_Q, d_out, NULL, g_vt.d_mx4_cnt,
                  (const vt_paged_item *)(b->dev + b->at_items) + (x_bf16 ? b->bf16_items : 0), (const int *)(b->dev + b->at_tables),
                  q_stride, s.n_heads, page_log, s.window, vt_divisor_of(group, (long long)b->max_rows * group),
                  scale * 1.44269504f};
    if ((few || many) && !(job.part = (float *)vt_scratch((size_t)(few > many ? few : many) * s.n_kv_heads))) return -1;
#define ATTEND(H) (x_bf16 ? pa_launch<H, false>(job, p, s.n_kv_heads) : pa_launch<H, true>(job, p, s.n_kv_heads))
    switch (HP) {
    case 1: ATTEND(1); break;
    case 2: ATTEND(2); break;
    case 3: ATTEND(3); break;
    default: ATTEND(4);
    }
#undef ATTEND
    return vt_check(hipGetLastError(), who) ? -1 : 0;
}
