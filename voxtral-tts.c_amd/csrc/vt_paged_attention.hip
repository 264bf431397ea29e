/*
 * vt_paged_attention.hip - attention of a batch's new rows over a paged cache of bf16 keys and values (vt_paged.h).
 *
 * The queries of the heads that share a kv head are columns (vt_paged_plans.h).  Scores are S^T[row][column] = K Q^T and results O^T[value][column] = V^T P^T on
 * the bf16 matrix instructions: keys and values as they lie, queries and weights as planes that each hold 8 bits of what the one before leaves, smallest
 * first: three make fp32 of fp32, one is a bf16 query itself.  A lane holds the same column of S^T and of O^T, and the order of the rows inside an
 * instruction is free, so that weights go from one product to the next in their registers.  Maximum, sum and results of a column are fp32, one pass over the rows with
 * the running maximum.
 *
 * What a column does not see: a hidden score is -infinity whatever the key holds.  A hidden value's weight is 0, but 0 times an infinity or NaN would be NaN,
 * so that where rows at hand are hidden from some column and a value among them is not finite, the value counts as 0, and a product of its own, with ones as the
 * weights of what a column sees, tells which results are NaN.  Rows behind a sequence's last are never read: requests have the size of the rows
 * that are there, and the rest is zeros.
 */
#include "vt_paged.h"
#include "vt_device.h"
#include "vt_requests.h"

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

/* 8 values of a query -> operands, one for each plane.  fp32 ones are scaled first; bf16 ones are the operand, and their scores are scaled. */
template <bool F32, int NQ>
static __device__ __forceinline__ void pa_query(const void *Q, size_t at, float scale, u32x4 (&to)[NQ]) {
    if constexpr (F32) {
        const f32x4 *p = reinterpret_cast<const f32x4 *>((const float *)Q + at);
        const f32x4 a = p[0] * scale, b = p[1] * scale;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            unsigned w[NQ];
            pa_planes2<NQ>(e < 2 ? a[2 * e] : b[2 * e - 4], e < 2 ? a[2 * e + 1] : b[2 * e - 3], w);
#pragma unroll
            for (int k = 0; k < NQ; k++) to[k][e] = w[k];
        }
    } else to[0] = *reinterpret_cast<const u32x4 *>((const uint16_t *)Q + at);
}

/* pairs of bf16 of which one is not finite */
typedef unsigned short pa_u16x2 __attribute__((ext_vector_type(2)));
static __device__ __forceinline__ pa_u16x2 pa_larger(pa_u16x2 most, unsigned w) { return __builtin_elementwise_max(most, __builtin_bit_cast(pa_u16x2, w & 0x7fff7fffu)); }
static __device__ __forceinline__ bool pa_not_finite(pa_u16x2 most) { return max((int)most.x, (int)most.y) >= 0x7f80; }
/* such values as ones, others as zeros; and the other way round, they as zeros */
static __device__ __forceinline__ unsigned pa_marks(unsigned w) { return ((w & 0x7f80u) == 0x7f80u ? 0x3f80u : 0u) | ((w & 0x7f800000u) == 0x7f800000u ? 0x3f800000u : 0u); }
static __device__ __forceinline__ unsigned pa_finite(unsigned w) { return ((w & 0x7f80u) == 0x7f80u ? 0u : w & 0xffffu) | ((w & 0x7f800000u) == 0x7f800000u ? 0u : w & 0xffff0000u); }

static __device__ __forceinline__ float pa_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

/* 16 rows from `at` on, a multiple of 16, of those lo .. end - 1: where they lie, and the bytes of them that are there */
struct pa_rows { size_t row; int bytes; };
static __device__ __forceinline__ pa_rows pa_place(const int *table, int at, int lo, int end, int page_log, int heads, int head, int row_bytes) {
    const int seen = min(at, end - 1), n = at + 16 > lo ? min(max(end - at, 0), 16) : 0;
    const int page = __builtin_amdgcn_readfirstlane(table[max(seen, lo) >> page_log]);
    return pa_rows{((((size_t)(unsigned)page * heads + head) << page_log) + (at & ((1 << page_log) - 1))), n * row_bytes};
}

/* ---- few columns -------------------------------------------------------------------------------------------------
 * A wave has 32 rows of K and V in registers at a time, asks for the next as soon as these are used, and waits for nobody; the waves of a workgroup, and then the
 * workgroups that share the columns' rows, add their parts in a fixed order, the last workgroup to arrive those of all.  K is the A operand of 16 x 16 x 32, a lane's 16
 * bytes from its own row.  V's rows are its columns: a lane loads CD values each of the eight rows that it has weights of, 16 lanes a whole row, and pairs of rows are
 * put together two values at a time. */
template <int HP, bool F32>
__global__ void __launch_bounds__(64 * PAGED_FEW_WAVES, 2) vt_paged_few_kernel(pa_job a) {
    constexpr int HD = 64 * HP, ROW = 2 * HD, KS = 2 * HP, CD = HP % 2 ? 4 : 8, CHUNKS = HD / (16 * CD), OD = HD + 4, WAVES = PAGED_FEW_WAVES;
    constexpr int NQ = F32 ? 3 : 1, NP = F32 ? 3 : 2, COLS = PAGED_FEW_COLS;
    __shared__ __attribute__((aligned(16))) float area[WAVES][COLS][OD];
    __shared__ float ml[WAVES][COLS][2], wt[COLS][PAGED_MAX_PARTS];
    __shared__ int last;
    const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), n = lane & 15, g = lane >> 4, h = (int)blockIdx.x, heads = (int)gridDim.x;
    const vt_paged_item it = a.items[blockIdx.y];
    const int nc = min(COLS, it.cols - it.c0), *table = a.tables + it.table;
    const int cc = min(it.c0 + n, it.cols - 1), qi = vt_div(cc, a.group), pos = it.past + qi;
    const int see_lo = a.window && pos >= a.window ? pos - a.window + 1 : 0, see_hi = pos + 1;
    const int q_first = it.past + vt_div(it.c0, a.group), q_last = it.past + vt_div(it.c0 + nc - 1, a.group);
    const int all_lo = a.window && q_last >= a.window ? q_last - a.window + 1 : 0, all_hi = q_first + 1;       /* rows that every column sees */
    const int base = it.lo & ~(PAGED_FEW_ROWS - 1), tiles = (it.end - base + PAGED_FEW_ROWS - 1) / PAGED_FEW_ROWS;
    const size_t head_at = (size_t)h * a.group.d + (cc - qi * a.group.d);
    u32x4 q[KS][NQ];
#pragma unroll
    for (int ks = 0; ks < KS; ks++) pa_query<F32, NQ>(a.Q, (size_t)(it.row + qi) * a.q_stride + head_at * HD + 32 * ks + 8 * g, a.scale, q[ks]);
    u32x4 kr[2][KS];
    u32x4 vr[8][CHUNKS];                                 /* CD == 4: the first half of each */
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
            for (int ks = 0; ks < KS; ks++) kr[kt][ks] = __builtin_amdgcn_raw_buffer_load_b128(d, n * ROW + 64 * ks + 16 * g, 0, 0);
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
                    const int from = (4 * g + j) * ROW + ch * 32 * CD + n * 2 * CD;
                    if constexpr (CD == 8) vr[4 * kt + j][ch] = __builtin_amdgcn_raw_buffer_load_b128(d, from, 0, 0);
                    else {
                        const u32x2 w = __builtin_amdgcn_raw_buffer_load_b64(d, from, 0, 0);
                        vr[4 * kt + j][ch] = u32x4{w.x, w.y, 0u, 0u};
                    }
                }
        }
    };
    place(wave);
    ask_k();
    ask_v();
    float m = -3.402823466e38f, l = 0.f;                 /* finite: with nothing seen yet a hidden score's weight is exp2(-inf) all the same */
    f32x4 o[CHUNKS * CD];
#pragma unroll
    for (int i = 0; i < CHUNKS * CD; i++) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int t = wave; t < tiles; t += WAVES) {
        const int first = base + PAGED_FEW_ROWS * t;
        const bool hidden = first < all_lo || first + PAGED_FEW_ROWS > all_hi || first < it.lo || first + PAGED_FEW_ROWS > it.end;
        f32x4 s[2];
#pragma unroll
        for (int kt = 0; kt < 2; kt++) {
            s[kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int p = NQ - 1; p >= 0; p--)
#pragma unroll
                for (int ks = 0; ks < KS; ks++) s[kt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pa_operand(kr[kt][ks]), pa_operand(q[ks][p]), s[kt], 0, 0, 0);
            if constexpr (!F32) s[kt] = s[kt] * a.scale;
        }
        place(t + WAVES);
        ask_k();
        auto sees = [&](int kt, int v) { const int key = first + 16 * kt + 4 * g + v; return key >= max(see_lo, it.lo) && key < min(see_hi, it.end); };
        bool bad = false;
        if (hidden) {
#pragma unroll
            for (int kt = 0; kt < 2; kt++)
#pragma unroll
                for (int v = 0; v < 4; v++) s[kt][v] = sees(kt, v) ? s[kt][v] : -INFINITY;
            pa_u16x2 most = {0, 0};
#pragma unroll
            for (int j = 0; j < 8; j++)
#pragma unroll
                for (int ch = 0; ch < CHUNKS; ch++)
#pragma unroll
                    for (int e = 0; e < CD / 2; e++) most = pa_larger(most, vr[j][ch][e]);
            bad = __any(pa_not_finite(most));
        }
        float top = m;                                   /* a NaN stays one: who sees it answers NaN */
#pragma unroll
        for (int v = 0; v < 4; v++) top = __builtin_elementwise_maximum(__builtin_elementwise_maximum(top, s[0][v]), s[1][v]);
        {
            f32x2 r = vt_swap16(top, top);
            top = __builtin_elementwise_maximum(r.x, r.y);
            r = vt_swap32(top, top);
            top = __builtin_elementwise_maximum(r.x, r.y);
        }
        if (__any(top != m)) {
            const float less = pa_exp2(m - top);
            l *= less;
#pragma unroll
            for (int i = 0; i < CHUNKS * CD; i++) o[i] = o[i] * less;
            m = top;
        }
        u32x4 w4[NP];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float p0 = pa_exp2(s[e >> 1][2 * (e & 1)] - m), p1 = pa_exp2(s[e >> 1][2 * (e & 1) + 1] - m);
            l += p0 + p1;
            unsigned w[NP];
            pa_planes2<NP>(p0, p1, w);
#pragma unroll
            for (int p = 0; p < NP; p++) w4[p][e] = w[p];
        }
        if (bad) {                                       /* rare */
            u32x4 ones;
#pragma unroll
            for (int e = 0; e < 4; e++) ones[e] = (sees(e >> 1, 2 * (e & 1)) ? 0x3f80u : 0u) | (sees(e >> 1, 2 * (e & 1) + 1) ? 0x3f800000u : 0u);
#pragma unroll
            for (int ch = 0; ch < CHUNKS; ch++)
#pragma unroll
                for (int i = 0; i < CD; i++) {
                    u32x4 v4;
#pragma unroll
                    for (int e = 0; e < 4; e++) v4[e] = pa_marks(__builtin_amdgcn_perm(vr[2 * e + 1][ch][i / 2], vr[2 * e][ch][i / 2], i & 1 ? 0x07060302u : 0x05040100u));
                    const f32x4 hit = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pa_operand(v4), pa_operand(ones), (f32x4{0.f, 0.f, 0.f, 0.f}), 0, 0, 0);
#pragma unroll
                    for (int v = 0; v < 4; v++) o[ch * CD + i][v] = hit[v] > 0.f ? NAN : o[ch * CD + i][v];
                }
#pragma unroll
            for (int j = 0; j < 8; j++)
#pragma unroll
                for (int ch = 0; ch < CHUNKS; ch++)
#pragma unroll
                    for (int e = 0; e < CD / 2; e++) vr[j][ch][e] = pa_finite(vr[j][ch][e]);
        }
#pragma unroll
        for (int ch = 0; ch < CHUNKS; ch++)
#pragma unroll
            for (int i = 0; i < CD; i++) {
                u32x4 v4;
#pragma unroll
                for (int e = 0; e < 4; e++) v4[e] = __builtin_amdgcn_perm(vr[2 * e + 1][ch][i / 2], vr[2 * e][ch][i / 2], i & 1 ? 0x07060302u : 0x05040100u);
                f32x4 &acc = o[ch * CD + i];
#pragma unroll
                for (int p = NP - 1; p >= 0; p--) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pa_operand(v4), pa_operand(w4[p]), acc, 0, 0, 0);
            }
        ask_v();
    }
    l = vt_rows_sum(l);
    /* The waves' parts, each times its share of the sum of weights: a mean of values */
    ml[wave][n][0] = m;                                  /* four lanes the same */
    ml[wave][n][1] = l;
    __syncthreads();
    float M = m, L = 0.f;
#pragma unroll
    for (int k = 0; k < WAVES; k++) M = fmaxf(M, ml[k][n][0]);
#pragma unroll
    for (int k = 0; k < WAVES; k++) L = fmaf(ml[k][n][1], pa_exp2(ml[k][n][0] - M), L);
    {
        const float f = L == 0.f && it.parts > 1 ? 0.f : pa_exp2(m - M) / L;
        float *to = &area[wave][n][4 * g * CD];
#pragma unroll
        for (int ch = 0; ch < CHUNKS; ch++)
#pragma unroll
            for (int v = 0; v < 4; v++)
#pragma unroll
                for (int i = 0; i < CD; i++) to[16 * CD * ch + CD * v + i] = o[ch * CD + i][v] * f;
    }
    __syncthreads();
    float *part = a.part + (size_t)(it.slot * heads + h * it.parts) * COLS * OD;
    auto result = [&](int col, int d, const f32x4 &v) {
        const int k = it.c0 + col, i = vt_div(k, a.group);
        const size_t to = ((size_t)(it.row + i) * a.n_heads + (size_t)h * a.group.d + (k - i * a.group.d)) * HD + d;
        if constexpr (F32) *reinterpret_cast<f32x4 *>((float *)a.out + to) = v;
        else {
            unsigned w0[1], w1[1];
            pa_planes2<1>(v.x, v.y, w0);
            pa_planes2<1>(v.z, v.w, w1);
            *reinterpret_cast<u32x2 *>((uint16_t *)a.out + to) = u32x2{w0[0], w1[0]};
        }
    };
    for (int e = (int)threadIdx.x; e < nc * (HD / 4); e += 64 * WAVES) {
        const int col = e / (HD / 4), d = 4 * (e - col * (HD / 4));
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < WAVES; k++) v = v + *reinterpret_cast<const f32x4 *>(&area[k][col][d]);
        if (it.parts == 1) result(col, d, v);
        else {
            float *to = part + ((size_t)it.part * COLS + col) * OD + 4 + d;
#pragma unroll
            for (int i = 0; i < 4; i++) vt_stc(to + i, v[i]);
        }
    }
    if (it.parts == 1) return;
    if (wave == 0 && lane < nc) {
        float *to = part + ((size_t)it.part * COLS + lane) * OD;
        vt_stc(to, M);
        vt_stc(to + 1, L);
    }
    __builtin_amdgcn_s_waitcnt(0x0f70);                  /* the part's stores are acknowledged */
    __syncthreads();
    unsigned *cnt = a.cnt + it.counter * heads + h;
    if (threadIdx.x == 0) last = __hip_atomic_fetch_add(cnt, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)(it.parts - 1);
    __syncthreads();
    if (!last) return;
    if (threadIdx.x == 0) vt_stc_u32(cnt, 0u);           /* ready for the next launch */
    /* a wave per column: lane k has part k's largest score and sum of weights */
    const __amdgpu_buffer_rsrc_t pd = vt_buffer(part, it.parts * COLS * OD * 4);
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
            for (int k = 0; k < 16; k++) p[k] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(pd, from + min(k0 + k, it.parts - 1) * (COLS * OD * 4), 0, 16));
#pragma unroll
            for (int k = 0; k < 16; k++) v = v + p[k] * wt[col][k0 + k];
        }
        result(col, d, v);
    }
}

/* ---- many columns ------------------------------------------------------------------------------------------------
 * A workgroup has 128 columns, a wave 32, and goes through its rows 64 at a time, 16 of them each wave's to bring: K through requests that write LDS, V as the matrix
 * instruction's operand (A of 32 x 32 x 16, value 2 HP r + i in row r of instruction i; four rows of a value are 8 bytes), put together in registers while the rows before are multiplied. */
template <int HP, bool F32>
__global__ void __launch_bounds__(256, 2) vt_paged_many_kernel(pa_job a) {
    constexpr int HD = 64 * HP, ROW = 2 * HD, WAVES = 4, DT = 2 * HP, KS = 4 * HP, PIECES = HD / 8, VD = 4 * HP, VW = VD / 2;
    constexpr int NQ = F32 ? 3 : 1, NP = F32 ? 3 : 1, KB = 64 * ROW;
    constexpr int SUB = 2;                               /* 32 rows: tiles of scores that are worked on together */
    __shared__ __attribute__((aligned(16))) unsigned char buf[2][2 * KB];
    __shared__ int odd[2][WAVES];                        /* values at hand that are not finite */
    __shared__ int last;
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 31, g = lane >> 5, h = (int)blockIdx.x, heads = (int)gridDim.x;
    const vt_paged_item it = a.items[blockIdx.y];
    const int *table = a.tables + it.table;
    const int w0 = it.c0 + 32 * wave, wc = min(w0 + 32, it.cols) - w0;                   /* this wave's columns: none, perhaps */
    const int cc = min(w0 + n, it.cols - 1), qi = vt_div(cc, a.group), pos = it.past + qi;
    const int see_lo = max(a.window && pos >= a.window ? pos - a.window + 1 : 0, it.lo), see_hi = min(pos + 1, it.end);
    const int q_first = it.past + vt_div(min(w0, it.cols - 1), a.group), q_last = it.past + vt_div(min(w0 + 31, it.cols - 1), a.group);
    const int all_lo = max(a.window && q_last >= a.window ? q_last - a.window + 1 : 0, it.lo), all_hi = min(q_first + 1, it.end);     /* rows that every column of the wave sees */
    const int any_lo = a.window && q_first >= a.window ? q_first - a.window + 1 : 0, any_hi = wc > 0 ? q_last + 1 : 0;                 /* .. that any does */
    const int base = it.lo & ~(PAGED_MANY_ROWS - 1), tiles = (it.end - base + PAGED_MANY_ROWS - 1) / PAGED_MANY_ROWS;
    const size_t head_at = (size_t)h * a.group.d + (cc - qi * a.group.d);
    u32x4 q[KS][NQ];
#pragma unroll
    for (int ks = 0; ks < KS; ks++) pa_query<F32, NQ>(a.Q, (size_t)(it.row + qi) * a.q_stride + head_at * HD + 16 * ks + 8 * g, a.scale, q[ks]);
    /* K's pieces of 16 bytes are exchanged within a row, so that 16 (8) rows' same piece lie in different banks */
    constexpr int SWAP = PIECES % 16 ? 7 : 15;
    int k_at[4];                                         /* DT of them (with that size the host pass drops the kernel) */
#pragma unroll
    for (int d = 0; d < DT; d++) {
        const int u = d * 64 + lane, r = u / PIECES;
        k_at[d] = r * ROW + ((u - r * PIECES) ^ (r & SWAP)) * 16;
    }
    const int v_at = 4 * (lane >> 4) * ROW + (lane & 15) * 2 * VD;
    unsigned vr[4][4];                                   /* VW of each */
    pa_rows at = pa_place(table, base + 16 * wave, it.lo, it.end, a.page_log, heads, h, ROW);
    auto load = [&](unsigned char *b) __attribute__((always_inline)) {
        const __amdgpu_buffer_rsrc_t kd = vt_buffer(a.K + at.row * HD, at.bytes), vd = vt_buffer(a.V + at.row * HD, at.bytes);
#pragma unroll
        for (int k = 0; k < 4; k++) {
#pragma unroll
            for (int e = 0; e < VW; e += VW % 4 ? 2 : 4) {
                if constexpr (VW % 4) {
                    const u32x2 w = __builtin_amdgcn_raw_buffer_load_b64(vd, v_at + k * ROW + 4 * e, 0, 0);
                    vr[k][e] = w.x; vr[k][e + 1] = w.y;
                } else {
                    const u32x4 w = __builtin_amdgcn_raw_buffer_load_b128(vd, v_at + k * ROW + 4 * e, 0, 0);
                    vr[k][e] = w.x; vr[k][e + 1] = w.y; vr[k][e + 2] = w.z; vr[k][e + 3] = w.w;
                }
            }
        }
#pragma unroll
        for (int d = 0; d < DT; d++)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(kd, (__attribute__((address_space(3))) void *)(b + wave * 16 * ROW + d * 1024), 16, k_at[d], 0, 0, 0);
    };
    /* value d's four rows (kg = 4 wave + lane / 16 of the tile's 16 fours) go to row r = d / DT of instruction i = d % DT, step kg / 4, group of lanes kg % 2, half kg / 2 % 2 */
    const int v_to = KB + ((wave * 64 + ((lane >> 4) & 1) * 32 + 2 * (lane & 15)) * 2 + (lane >> 5)) * 8;
    auto put = [&](int which) __attribute__((always_inline)) {
        pa_u16x2 most = {0, 0};
#pragma unroll
        for (int k = 0; k < 4; k++)
#pragma unroll
            for (int e = 0; e < VW; e++) most = pa_larger(most, vr[k][e]);
        const int bad = __any(pa_not_finite(most));
        if (lane == 0) odd[which][wave] = bad;
#pragma unroll
        for (int d = 0; d < VD; d++) {
            const unsigned pick = d & 1 ? 0x07060302u : 0x05040100u;
            *reinterpret_cast<u32x2 *>(buf[which] + v_to + (d % DT) * 4096 + (d / DT) * 16) =
                u32x2{__builtin_amdgcn_perm(vr[1][d / 2], vr[0][d / 2], pick), __builtin_amdgcn_perm(vr[3][d / 2], vr[2][d / 2], pick)};
        }
    };
    float m = -3.402823466e38f, l = 0.f;
    pa_f32x16 o[DT];
#pragma unroll
    for (int i = 0; i < DT; i++) o[i] = pa_f32x16{};
    load(buf[0]);
    put(0);
    __builtin_amdgcn_s_waitcnt(0x0f70);                  /* K has arrived */
    __syncthreads();
#pragma unroll 1
    for (int t = 0; t < tiles; t++) {
        const unsigned char *b = buf[t & 1];
        const int first = base + PAGED_MANY_ROWS * t;
        at = pa_place(table, first + PAGED_MANY_ROWS + 16 * wave, it.lo, it.end, a.page_log, heads, h, ROW);
        if (t + 1 < tiles) load(buf[(t + 1) & 1]);
#pragma unroll 1
        for (int sub = 0; sub < 2; sub += SUB) {
            const int from = first + 32 * sub;
            if (from >= any_hi || from + 32 * SUB <= any_lo) continue;               /* nobody of this wave sees these rows */
            pa_f32x16 s[SUB];
#pragma unroll
            for (int kt = 0; kt < SUB; kt++) {
                const int row = 32 * (sub + kt) + n;
                s[kt] = pa_f32x16{};
#pragma unroll
                for (int ks = 0; ks < KS; ks++) {
                    const u32x4 k = *reinterpret_cast<const u32x4 *>(b + row * ROW + ((2 * ks + g) ^ (row & SWAP)) * 16);
#pragma unroll
                    for (int p = NQ - 1; p >= 0; p--) s[kt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(pa_operand(k), pa_operand(q[ks][p]), s[kt], 0, 0, 0);
                }
                if constexpr (!F32) s[kt] = s[kt] * a.scale;
            }
            auto sees = [&](int kt, int v) { const int key = from + 32 * kt + 8 * (v >> 2) + 4 * g + (v & 3); return key >= see_lo && key < see_hi; };
            bool bad = false;
            if (from < all_lo || from + 32 * SUB > all_hi) {
#pragma unroll
                for (int kt = 0; kt < SUB; kt++)
#pragma unroll
                    for (int v = 0; v < 16; v++) s[kt][v] = sees(kt, v) ? s[kt][v] : -INFINITY;
                bad = __any(odd[t & 1][lane & 3]);
            }
            float top = m;                                /* a NaN stays one: who sees it answers NaN */
#pragma unroll
            for (int kt = 0; kt < SUB; kt++)
#pragma unroll
                for (int v = 0; v < 16; v++) top = __builtin_elementwise_maximum(top, s[kt][v]);
            { const f32x2 r = vt_swap32(top, top); top = __builtin_elementwise_maximum(r.x, r.y); }
            if (__any(top != m)) {
                const float less = pa_exp2(m - top);
                l *= less;
#pragma unroll
                for (int i = 0; i < DT; i++) o[i] = o[i] * less;
                m = top;
            }
            if (bad) {                                   /* rare */
#pragma unroll 1
                for (int st = 0; st < 2 * SUB; st++) {
                    u32x4 ones;
#pragma unroll
                    for (int e = 0; e < 4; e++) ones[e] = (sees(st >> 1, 8 * (st & 1) + 2 * e) ? 0x3f80u : 0u) | (sees(st >> 1, 8 * (st & 1) + 2 * e + 1) ? 0x3f800000u : 0u);
#pragma unroll
                    for (int i = 0; i < DT; i++) {
                        u32x4 v4 = *reinterpret_cast<const u32x4 *>(b + KB + ((i * 4 + 2 * sub + st) * 64 + lane) * 16);
#pragma unroll
                        for (int e = 0; e < 4; e++) v4[e] = pa_marks(v4[e]);
                        const pa_f32x16 hit = __builtin_amdgcn_mfma_f32_32x32x16_bf16(pa_operand(v4), pa_operand(ones), pa_f32x16{}, 0, 0, 0);
#pragma unroll
                        for (int v = 0; v < 16; v++) o[i][v] = hit[v] > 0.f ? NAN : o[i][v];
                    }
                }
            }
#pragma unroll
            for (int st = 0; st < 2 * SUB; st++) {       /* 16 rows a step: elements 8 (st % 2) .. of scores st / 2 */
                u32x4 w4[NP];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float p0 = pa_exp2(s[st >> 1][8 * (st & 1) + 2 * e] - m), p1 = pa_exp2(s[st >> 1][8 * (st & 1) + 2 * e + 1] - m);
                    l += p0 + p1;
                    unsigned w[NP];
                    pa_planes2<NP>(p0, p1, w);
#pragma unroll
                    for (int p = 0; p < NP; p++) w4[p][e] = w[p];
                }
#pragma unroll
                for (int i = 0; i < DT; i++) {
                    u32x4 v4 = *reinterpret_cast<const u32x4 *>(b + KB + ((i * 4 + 2 * sub + st) * 64 + lane) * 16);
                    if (bad) {
#pragma unroll
                        for (int e = 0; e < 4; e++) v4[e] = pa_finite(v4[e]);
                    }
#pragma unroll
                    for (int p = NP - 1; p >= 0; p--) o[i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(pa_operand(v4), pa_operand(w4[p]), o[i], 0, 0, 0);
                }
            }
        }
        if (t + 1 < tiles) {
            put((t + 1) & 1);
            __builtin_amdgcn_s_waitcnt(0x0f70);
        }
        __syncthreads();
    }
    { const f32x2 r = vt_swap32(l, l); l = r.x + r.y; }
    {
        const float f = l == 0.f && it.parts > 1 ? 0.f : 1.f / l;
#pragma unroll
        for (int i = 0; i < DT; i++) o[i] = o[i] * f;
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
    /* element v of lane l is value DT (8 (v / 4) + 4 (l / 32) + v % 4) + i */
    if (n < wc) {
        const size_t to = ((size_t)(it.row + qi) * a.n_heads + head_at) * HD;
#pragma unroll
        for (int v = 0; v < 16; v++)
#pragma unroll
            for (int i = 0; i < DT; i += 2) {
                const size_t x = to + DT * (8 * (v >> 2) + 4 * g + (v & 3)) + i;
                if constexpr (F32) *reinterpret_cast<f32x2 *>((float *)a.out + x) = f32x2{o[i][v], o[i + 1][v]};
                else {
                    unsigned w[1];
                    pa_planes2<1>(o[i][v], o[i + 1][v], w);
                    *reinterpret_cast<unsigned *>((uint16_t *)a.out + x) = w[0];
                }
            }
    }
}

template <int HP>
static void pa_launch(const pa_job &job, const vt_paged_plan &p, int heads, bool f32) {
    if (p.few) {
        const dim3 grid((unsigned)heads, (unsigned)p.few);
        if (f32) hipLaunchKernelGGL((vt_paged_few_kernel<HP, true>), grid, dim3(64 * PAGED_FEW_WAVES), 0, g_vt.stream, job);
        else hipLaunchKernelGGL((vt_paged_few_kernel<HP, false>), grid, dim3(64 * PAGED_FEW_WAVES), 0, g_vt.stream, job);
    }
    if constexpr (HP <= 2) {
        if (p.many) {
            pa_job many = job;
            many.items += p.few;
            const dim3 grid((unsigned)heads, (unsigned)p.many);
            if (f32) hipLaunchKernelGGL((vt_paged_many_kernel<HP, true>), grid, dim3(256), 0, g_vt.stream, many);
            else hipLaunchKernelGGL((vt_paged_many_kernel<HP, false>), grid, dim3(256), 0, g_vt.stream, many);
        }
    }
}

extern "C" int tts_hip_paged_attention(void *d_out, const void *d_Q, int x_bf16, int q_stride, const tts_hip_paged_t *b, const void *d_k_pages, const void *d_v_pages, float scale) {
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
    const size_t few = (size_t)b->plan.few_slots * s.n_kv_heads * PAGED_FEW_COLS * (s.head_dim + 4) * 4, many = (size_t)b->plan.many_slots * s.n_kv_heads * 4 * (8 * HP + 1) * 1024;
    pa_job job = {(const uint16_t *)d_k_pages, (const uint16_t *)d_v_pages, d_Q, d_out, NULL, g_vt.d_mx4_cnt, (const vt_paged_item *)(b->dev + b->at_items),
                  (const int *)(b->dev + b->at_tables), q_stride, s.n_heads, page_log, s.window, vt_divisor_of(group, (long long)b->max_rows * group), scale * 1.44269504f};
    if ((few || many) && !(job.part = (float *)vt_scratch(few > many ? few : many))) return -1;
    switch (HP) {
    case 1: pa_launch<1>(job, b->plan, s.n_kv_heads, !x_bf16); break;
    case 2: pa_launch<2>(job, b->plan, s.n_kv_heads, !x_bf16); break;
    case 3: pa_launch<3>(job, b->plan, s.n_kv_heads, !x_bf16); break;
    default: pa_launch<4>(job, b->plan, s.n_kv_heads, !x_bf16);
    }
    return vt_check(hipGetLastError(), who) ? -1 : 0;
}
