/*
 * vt_kv4.hip - a key/value cache in microscaled 4-bit floats (vt_mx4.h) and the attention that reads it.  Per kv head the
 * rows lie one behind the other, codes [kv heads, max_rows, head_dim / 2] and scales [kv heads, max_rows, head_dim / 32], for K
 * and for V: what one head's attention reads is one piece of memory.
 */
#include "vt_state.h"
#include "vt_mx4.h"
#include "vt_mx4_plans.h"
#include "vt_requests.h"

#include <math.h>

static int cache_ok(const char *who, const tts_hip_kv4_t *c, long long first, long long n) {
    if (!c || !c->k_codes || !c->k_scales || !c->v_codes || !c->v_scales) { vt_set_error("%s: no cache, or a NULL pointer in it", who); return 0; }
    if (c->max_rows < 1 || c->n_kv_heads < 1 || c->head_dim < 64 || c->head_dim > 256 || c->head_dim % 64) {
        vt_set_error("%s: a cache of %d rows, %d heads of %d (head_dim: 64, 128, 192 or 256)", who, c->max_rows, c->n_kv_heads, c->head_dim);
        return 0;
    }
    if (((uintptr_t)c->k_codes | (uintptr_t)c->v_codes) & 15 || ((uintptr_t)c->k_scales | (uintptr_t)c->v_scales) & 3) {
        vt_set_error("%s: codes lie on 16 bytes, scales on 4", who);
        return 0;
    }
    if (first < 0 || n < 1 || first + n > c->max_rows) {
        vt_set_error("%s: rows %lld .. %lld of a cache of %d", who, first, first + n - 1, c->max_rows);
        return 0;
    }
    return 1;
}

/* ---- rows into the cache (a lane per eight values) and back (four); K in blockIdx.y = 0 and V in 1 -----------------------
 * Bound by the launch: a row of 8 x 128 takes 1.7 us on the device and 1.5 back, of 4 that a call takes; 1531 rows 4.4 (14 MB, 3.2 TB/s) and 5.3. */
struct kv4_rows { int n, pos, max_rows, stride, whole; vt_divisor per_row, per_head; };      /* lanes of a row, of a row of one head */

static __device__ __forceinline__ bool kv4_place(const kv4_rows &r, int values, long long &from, size_t &at) {
    const int i = (int)(blockIdx.x * 256 + threadIdx.x);
    if (i >= r.n * r.per_row.d) return false;
    const int row = vt_div(i, r.per_row), u = i - row * r.per_row.d, h = vt_div(u, r.per_head), d = u - h * r.per_head.d;
    from = (long long)row * r.stride + values * u;
    at = ((size_t)h * r.max_rows + r.pos + row) * r.per_head.d + d;
    return true;
}

__global__ void __launch_bounds__(256) vt_kv4_append_kernel(tts_hip_kv4_t c, const float *K, const float *V, kv4_rows r) {
    long long from;
    size_t at;
    if (!kv4_place(r, 8, from, at)) return;
    f32x4 a, b;
    vt_mx4_load8((blockIdx.y ? V : K) + from, 8, r.whole, a, b);
    unsigned scale;
    const unsigned code = vt_mx4_encode8(a, b, scale);
    ((unsigned *)(blockIdx.y ? c.v_codes : c.k_codes))[at] = code;
    if ((at & 3) == 0) (blockIdx.y ? c.v_scales : c.k_scales)[at >> 2] = (uint8_t)scale;
}

__global__ void __launch_bounds__(256) vt_kv4_read_kernel(float *K, float *V, tts_hip_kv4_t c, kv4_rows r) {
    long long to;
    size_t at;
    if (!kv4_place(r, 4, to, at)) return;
    const uint16_t *codes = (const uint16_t *)(blockIdx.y ? c.v_codes : c.k_codes);
    const uint8_t *scales = blockIdx.y ? c.v_scales : c.k_scales;
    vt_mx4_store4((blockIdx.y ? V : K) + to, 4, r.whole, vt_mx4_decode4(codes[at], scales[at >> 3]));
}

static int kv4_rows_ok(const char *who, kv4_rows *r, const tts_hip_kv4_t *c, const float *K, const float *V, int n, int pos, int stride, int values) {
    if (!cache_ok(who, c, pos, n)) return 0;
    const long long width = (long long)c->n_kv_heads * c->head_dim;
    if (stride == 0) stride = (int)(width > 0x7fffffff ? 0x7fffffff : width);
    if (!K || !V || (((uintptr_t)K | (uintptr_t)V) & 3) || stride < width || width / values * n > 0x7fffff00ll) {
        vt_set_error("%s: %d rows of %lld values %d apart", who, n, width, stride);
        return 0;
    }
    *r = kv4_rows{n, pos, c->max_rows, stride, (((uintptr_t)K | (uintptr_t)V) & 15) == 0 && stride % 4 == 0,
                  vt_divisor_of((int)(width / values), width / values * n), vt_divisor_of(c->head_dim / values, width / values)};
    return vt_mx4_ready(who);
}

extern "C" int tts_hip_kv4_append(const tts_hip_kv4_t *cache, const float *d_K, const float *d_V, int n_rows, int pos, int stride) {
    static const char who[] = "tts_hip_kv4_append";
    kv4_rows r;
    if (!kv4_rows_ok(who, &r, cache, d_K, d_V, n_rows, pos, stride, 8)) return -1;
    hipLaunchKernelGGL(vt_kv4_append_kernel, dim3((r.n * r.per_row.d + 255) / 256, 2), dim3(256), 0, g_vt.stream, *cache, d_K, d_V, r);
    return vt_check(hipGetLastError(), who) ? -1 : 0;
}

extern "C" int tts_hip_kv4_read(float *d_K, float *d_V, const tts_hip_kv4_t *cache, int n_rows, int pos, int stride) {
    static const char who[] = "tts_hip_kv4_read";
    kv4_rows r;
    if (!kv4_rows_ok(who, &r, cache, d_K, d_V, n_rows, pos, stride, 4)) return -1;
    hipLaunchKernelGGL(vt_kv4_read_kernel, dim3((r.n * r.per_row.d + 255) / 256, 2), dim3(256), 0, g_vt.stream, d_K, d_V, *cache, r);
    return vt_check(hipGetLastError(), who) ? -1 : 0;
}

/* ---- attention -------------------------------------------------------------------------------------------------------
 * The queries of the heads that share a kv head are columns: column c is query c / group, head c % group of the group.  Scores are
 * S^T[row][column] = K Q^T on the scaled matrix instruction, keys in 4 bits as they lie, queries as five e2m3 planes (vt_mx4.h), the
 * smallest plane first: the accumulators are cut and not rounded at 2^-23, and so only the last sum meets that.  Results are
 * O^T[value][column] = V^T P^T in fp16: 4-bit values are exact in fp16 once they are scaled by the largest scale E of the rows at hand,
 * to 2^13 of it, and a weight p 2^14 goes in as two planes of 22 bits in all.  Maximum, sum and results of a column are fp32, one pass
 * over the rows with the running maximum.  A lane holds the same column of S^T and of O^T, and the order of keys inside an instruction
 * is free, so that weights go from one product to the next in their registers.  Rows at hand with scales further apart than fp16 reaches
 * (36 binades) go another way (kv4_column): fp32 all through, rare, and slow: 1 query of 32 heads behind 1999 rows 44 us with the call
 * and the wait for it, 1531 behind none 3.4 ms where one row of each head is so.  A score beyond fp32 meets the planes one by one, with
 * signs of their own: what comes out may be an infinity of the wrong sign, and so it counts as NaN.  NaN: a key's shows in the scores of
 * who sees it.  A value's scale of 255 is taken for a finite one in the product (a hidden row's weight is 0, and 0 times NaN would reach
 * who does not see it), and behind the last row NaN goes to the columns that see such a row. */
typedef _Float16 vt_f16x8 __attribute__((ext_vector_type(8)));
#define KV4_PLANES 5
#define KV4_P_EXP 14                       /* weights times 2^14 .. */
#define KV4_V_EXP 13                       /* .. and values up to 6 times 2^13 are fp16 */

/* 104 bytes: a launch with 112 and more, or one that asks for the size of its grid, takes the host 0.9 us longer (of 2.7) */
struct kv4_job {
    const uint8_t *k_codes, *k_scales, *v_codes, *v_scales;
    float *out;
    const float *Q;
    unsigned char *part;
    unsigned *cnt;
    /* cols, tiles: columns and tiles of them; run: tiles of 32 rows a wave, of 64 a workgroup; parts: workgroups per head and tile of columns */
    int max_rows, start, n_heads, cols, run, parts, tiles;
    vt_divisor group;
    float scale;                                         /* times log2 e */
};

/* column / heads per kv head, for fewer than 2^20 columns: (c + 1/2) / d is no nearer to a whole number than 1 / 2 d, and c 2^-22 / d off */
static __device__ __forceinline__ int kv4_query(int col, float inv) { return (int)(((float)col + 0.5f) * inv); }

/* What the scales of the values at hand span: bytes s as t = s + 1 mod 256, pairs of them.  255 is t = 0 and the block of zeros 1; neither counts. */
typedef unsigned short kv4_u16x2 __attribute__((ext_vector_type(2)));
struct kv4_span {
    kv4_u16x2 top = {1, 1}, low = {1, 1}, least = {65535, 65535};         /* largest t, 0 if there is one, smallest t - 2 */
    __device__ __forceinline__ void add4(unsigned w) {
#pragma unroll
        for (int b = 0; b < 2; b++) {
            const kv4_u16x2 t = __builtin_bit_cast(kv4_u16x2, (((w >> (8 * b)) & 0x00ff00ffu) + 0x00010001u) & 0x00ff00ffu);
            top = __builtin_elementwise_max(top, t);
            low = __builtin_elementwise_min(low, t);
            least = __builtin_elementwise_min(least, (kv4_u16x2)(t - (kv4_u16x2){2, 2}));
        }
    }
    __device__ __forceinline__ int most() const { return max((int)top.x, (int)top.y) - 1; }
    __device__ __forceinline__ int smallest() const { return min((int)least.x, (int)least.y) + 1; }
    __device__ __forceinline__ bool nan() const { return min((int)low.x, (int)low.y) == 0; }
};
#define KV4_SPAN 36                        /* 2^13 2^-36 times half a code is fp16's smallest step */

/* From this largest score m on rounding 14 - m, what a score has added in front of its exponential, would show in the factor 2^14 of all
 * weights (behind 2^25 it is off by up to 4), which the sums' rescaling and joins take for constant: the maximum is taken off first,
 * whose difference to a near score is exact. */
#define KV4_FAR 0x1p10f

/* Scores are below 2^128 where neither the queries' planes nor the keys at hand have a larger scale than this: head_dim 256 times 7.75
 * times 6, times 2^(184 - 127) twice, and the smaller planes' sixteenths.  Else an infinity is one that the sum made: NaN.  (Both of
 * these looked at where a wave has a branch anyway: with a branch of their own 8.99 us for one query behind 1999 rows, so 8.84.) */
#define KV4_FINITE 184
static __device__ __forceinline__ float kv4_seen(float s, bool see) { return !see ? -INFINITY : fabsf(s) == INFINITY ? NAN : s; }

/* K's pieces of 16 bytes are exchanged within a row in LDS, so that eight rows' same piece lie in different banks */
template <int HP> static __device__ __forceinline__ int kv4_swizzle(int row, int piece) {
    return HP == 2 ? piece ^ ((row >> 1) & 3) : HP == 4 ? piece ^ (row & 7) : piece ^ ((row >> 2) & 1);
}

/* One column over `rows` rows, all of which it sees, by a wave in fp32: a lane per row for the scores, per value for the results; -> the
 * largest score, the sum of weights times 2^14, and the mean of values, value 64 k + lane of it to at[64 k + lane].  The mean is kept as
 * one, row after row: a sum of values near the end of the range would leave it, and scaled down small ones would lose bits. */
template <int HP>
static __device__ __forceinline__ void kv4_column(const kv4_job &a, const float *q, size_t row0, int rows, int lane, float *at, float &m, float &l) {
    constexpr int ROW = 32 * HP;
    float o[HP];
    m = -3.402823466e38f;
    l = 0.f;
#pragma unroll
    for (int k = 0; k < HP; k++) o[k] = 0.f;
#pragma unroll 1
    for (int first = 0; first < rows; first += 64) {
        const size_t row = row0 + min(first + lane, rows - 1);
        float s = 0.f;
#pragma unroll 1
        for (int u = 0; u < 8 * HP; u++) {               /* eight values */
            const unsigned w = reinterpret_cast<const unsigned *>(a.k_codes + row * ROW)[u], sc = a.k_scales[row * 2 * HP + u / 4];
            const f32x4 k0 = vt_mx4_decode4(w & 0xffffu, sc), k1 = vt_mx4_decode4(w >> 16, sc);
#pragma unroll
            for (int i = 0; i < 4; i++) s = fmaf(k1[i], q[8 * u + 4 + i] * a.scale, fmaf(k0[i], q[8 * u + i] * a.scale, s));
        }
        s = kv4_seen(s, first + lane < rows);
        const float top = __any(s != s) ? NAN : fmaxf(m, vt_wave_max(s)), less = __builtin_amdgcn_exp2f(m - top), p = __builtin_amdgcn_exp2f(s - top);
        const float before = l * less, share = p / (l = before + vt_wave_sum(p));
        m = m != m ? m : top;
#pragma unroll
        for (int k = 0; k < HP; k++) o[k] *= before / l;
#pragma unroll 8
        for (int j = 0; j < 64; j++) {                   /* past the last row: the last again, times 0 */
            const float w = __shfl(share, j);
            const size_t r = row0 + min(first + j, rows - 1);
#pragma unroll
            for (int k = 0; k < HP; k++) {
                const int d = 64 * k + lane;
                const f32x4 v = vt_mx4_decode4((unsigned)a.v_codes[r * ROW + d / 2] >> (4 * (d & 1)), a.v_scales[r * 2 * HP + d / 32]);
                o[k] = fmaf(w, v.x, o[k]);
            }
        }
    }
#pragma unroll
    for (int k = 0; k < HP; k++) at[64 * k + lane] = o[k];
    l = __builtin_amdgcn_ldexpf(l, KV4_P_EXP);
}

/* Few columns: a wave streams 32 rows of K and V at a time into LDS of its own, two such tiles on their way while one is multiplied, and
 * waits for nobody else; the waves of a workgroup, and then the workgroups of a head, add their parts in a fixed order, the last
 * workgroup to arrive those of all.  K is the A operand of 16 x 16 x 128, V of 16 x 16 x 32: lane l has the values of column n = l % 16,
 * CD of each 16 CD, for the eight keys that its group of 16 lanes has weights of.  Most of a short call is instructions that run once,
 * from a cold instruction cache: the code in front of the loop and behind it is kept short.  Bound: one query of 32 heads on 8 with 128
 * values behind 65535 rows 19.5 us, 71 MB at 3.6 TB/s, of which 7 us do not depend on the rows; behind 1999 8.8 us, nothing but those. */
template <int HP, int WAVES>
__global__ void __launch_bounds__(64 * WAVES) vt_kv4_stream_kernel(kv4_job a) {
    constexpr int HD = 64 * HP, ROW = 32 * HP, KS = (HP + 1) / 2, CD = HP % 2 ? 4 : 8, CHUNKS = HD / (16 * CD), OD = HD + 4;
    constexpr int SC = 32 * ROW * 2, STAGE = SC + 512;    /* K rows, V rows, their scales in 256 bytes each */
    __shared__ __attribute__((aligned(16))) unsigned char buf0[WAVES * STAGE], buf1[WAVES * STAGE], buf2[WAVES * STAGE];
    __shared__ float ml[WAVES][KV4_COLS][2], wt[KV4_COLS][KV4_MAX_CHUNKS];
    __shared__ int last;
    const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
    const int chunk = (int)blockIdx.y, ct = (int)blockIdx.z, h = (int)blockIdx.x, group = a.group.d;
    const float inv_group = 1.f / (float)group;
    const int c0 = ct * KV4_COLS, nc = min(KV4_COLS, a.cols - c0);
    /* queries (lane's column, values 32 g .. of each 128) are asked for first: loads return in order.  Columns past the last repeat it; the
     * half of 128 values that a head_dim of 64 or 192 leaves empty repeats the other, against codes of 0. */
    const int cc = min(c0 + n, a.cols - 1), qi = kv4_query(cc, inv_group), see = a.start + qi + 1;
    const int seen_first = a.start + kv4_query(c0, inv_group) + 1, seen_last = a.start + kv4_query(c0 + nc - 1, inv_group) + 1;
    f32x4 q4[KS][8];
    {
        const float *src = a.Q + ((size_t)qi * a.n_heads + (size_t)(h * group + cc - qi * group)) * HD;
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            const float *from = src + 128 * ks + 32 * (HP % 2 && ks == KS - 1 ? g & 1 : g);
#pragma unroll
            for (int i = 0; i < 8; i++) q4[ks][i] = *reinterpret_cast<const f32x4 *>(from + 4 * i);
        }
    }
    const int lo = (chunk * WAVES + wave) * a.run * 32, rows = max(min(a.run * 32, seen_last - lo), 0), tiles = (rows + 31) / 32;
    const size_t row0 = (size_t)h * a.max_rows + lo;
    /* scales come in words; where a row has 2 or 6 bytes of them (HP odd) its first may start in the middle of one, whose other half is
     * memory that a word of the cache's reaches anyway */
    const int sub = HP % 2 ? (int)((uintptr_t)(a.v_scales + row0 * 2 * HP) & 3) : 0, words = rows ? (rows * 2 * HP + sub + 3) / 4 : 0;
    /* what lies past the wave's rows reads as zeros */
    const __amdgpu_buffer_rsrc_t kd = vt_buffer(a.k_codes + row0 * ROW, rows * ROW), vd = vt_buffer(a.v_codes + row0 * ROW, rows * ROW);
    const __amdgpu_buffer_rsrc_t ksd = vt_buffer(a.k_scales + row0 * 2 * HP - sub, words * 4), vsd = vt_buffer(a.v_scales + row0 * 2 * HP - sub, words * 4);
    u32x4 scan = __builtin_bit_cast(u32x4, vt_buffer_ld4(vsd, lane * 16));
    /* a tile's requests: unit u of 16 bytes is row u / 2 HP, piece u % 2 HP of it */
    int k_at[4];                                         /* HP of them (with that size the host pass drops the kernel) */
#pragma unroll
    for (int d = 0; d < HP; d++) {
        const int u = d * 64 + lane, r = u / (2 * HP);
        k_at[d] = r * ROW + kv4_swizzle<HP>(r, u - r * 2 * HP) * 16;
    }
    auto ask = [&](unsigned char *buf, int t) __attribute__((always_inline)) {
        unsigned char *b = buf + wave * STAGE;
#define LDS(at) (__attribute__((address_space(3))) void *)(b + (at))
#pragma unroll
        for (int d = 0; d < HP; d++) __builtin_amdgcn_raw_ptr_buffer_load_lds(kd, LDS(d * 1024), 16, k_at[d] + t * 32 * ROW, 0, 0, 0);
#pragma unroll
        for (int d = 0; d < HP; d++) __builtin_amdgcn_raw_ptr_buffer_load_lds(vd, LDS(32 * ROW + d * 1024), 16, d * 1024 + lane * 16 + t * 32 * ROW, 0, 0, 0);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(ksd, LDS(SC), 4, lane * 4 + t * 64 * HP, 0, 0, 0);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(vsd, LDS(SC + 256), 4, lane * 4 + t * 64 * HP, 0, 0, 0);
#undef LDS
    };
    ask(buf0, 0);
    ask(buf1, 1);
    vt_u32x6 q[KS][KV4_PLANES];
    unsigned qs[KS][KV4_PLANES];
#pragma unroll
    for (int ks = 0; ks < KS; ks++) {
        vt_f32x16 even, odd;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const f32x4 v = q4[ks][i] * a.scale;
            even[2 * i] = v.x; odd[2 * i] = v.y; even[2 * i + 1] = v.z; odd[2 * i + 1] = v.w;
        }
        vt_mx4_planes<KV4_PLANES>(even, odd, q[ks], qs[ks]);
#pragma unroll
        for (int p = 0; p < KV4_PLANES; p++) asm volatile("" : "+v"(q[ks][p]));       /* here, while the first tiles are on their way, and not behind the loop below */
    }
    unsigned q_scale = 0;
#pragma unroll
    for (int ks = 0; ks < KS; ks++) q_scale = max(q_scale, qs[ks][0]);
    const int k_most = __any(q_scale > KV4_FINITE) ? -1 : KV4_FINITE;
    kv4_span span;                                       /* of the wave's values */
    auto look = [&](int i) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if (HP % 2) {                                 /* halves of a word that are not this wave's rows */
                if (i + e == 0 && sub) scan[e] &= 0xffff0000u;
                if (i + e == words - 1 && ((rows * 2 * HP + sub) & 3)) scan[e] &= 0xffffu;
            }
            span.add4(scan[e]);
        }
    };
    look(lane * 4);
    for (int i = 256; i < words; i += 256) {
        scan = __builtin_bit_cast(u32x4, vt_buffer_ld4(vsd, (i + lane * 4) * 4));
        look(i + lane * 4);
    }
    const int most = (int)vt_wave_max((float)span.most());
    const bool nan = __any(span.nan()), wide = __any(most - span.smallest() > KV4_SPAN);
    const int shift = 127 + KV4_V_EXP - most;
    float minus = -1.f;                                   /* a number that the compiler does not know: fp16 to fp32 and the difference are one instruction */
    asm("" : "+v"(minus));
    bool far = false;
    float m = -3.402823466e38f, l = 0.f;                  /* finite: with nothing seen yet a hidden score's weight is exp2(-inf) all the same */
    f32x4 o[CHUNKS * CD];
#pragma unroll
    for (int i = 0; i < CHUNKS * CD; i++) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int k_row = wave * STAGE + n * ROW, v_row = wave * STAGE + 32 * ROW + 4 * g * ROW + n * (CD / 2);
    const int ks_row = wave * STAGE + SC + sub + n * 2 * HP, vs_row = wave * STAGE + SC + 256 + sub + 4 * g * 2 * HP + n * CD / 32;
    auto tile = [&](const unsigned char *buf, int t) __attribute__((always_inline)) {
        f32x4 s[2];
        int k_scale = 0;
#pragma unroll
        for (int kt = 0; kt < 2; kt++) {
            u32x4 k[KS];
            int ksc[KS];
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                const bool half = HP % 2 && ks == KS - 1;        /* 64 values behind the last 128: the other two groups of lanes have zeros */
                const int p = 4 * ks + (half ? g & 1 : g);
                k[ks] = *reinterpret_cast<const u32x4 *>(buf + k_row + 16 * kt * ROW + kv4_swizzle<HP>(n, p) * 16);      /* the exchange is the same 16 rows on */
                ksc[ks] = buf[ks_row + 16 * kt * 2 * HP + p];
                if (half && g >= 2) { k[ks] = u32x4{0u, 0u, 0u, 0u}; ksc[ks] = 0; }
                k_scale = max(k_scale, ksc[ks]);
            }
            s[kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int p = KV4_PLANES - 1; p >= 0; p--)
#pragma unroll
                for (int ks = 0; ks < KS; ks++)
                    s[kt] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(vt_mfma_e2m1(k[ks]), vt_mfma_e2m3(q[ks][p]), s[kt], VT_MFMA_E2M1, VT_MFMA_E2M3, 0,
                                                                            ksc[ks], 0, (int)qs[ks][p]);
        }
        const int first = lo + 32 * t;
        if (first + 32 > seen_first || __any(k_scale > k_most)) {
#pragma unroll
            for (int kt = 0; kt < 2; kt++)
#pragma unroll
                for (int v = 0; v < 4; v++) s[kt][v] = kv4_seen(s[kt][v], first + 16 * kt + 4 * g + v < see);
        }
        float top = m;                                    /* a NaN stays one: who sees it answers NaN */
#pragma unroll
        for (int v = 0; v < 4; v++) top = __builtin_elementwise_maximum(__builtin_elementwise_maximum(top, s[0][v]), s[1][v]);
        {
            f32x2 r = vt_swap16(top, top);
            top = __builtin_elementwise_maximum(r.x, r.y);
            r = vt_swap32(top, top);
            top = __builtin_elementwise_maximum(r.x, r.y);
        }
        if (__any(top != m)) {
            const float less = __builtin_amdgcn_exp2f(m - top);
            l *= less;
#pragma unroll
            for (int i = 0; i < CHUNKS * CD; i++) o[i] = o[i] * less;
            m = top;
            far = __any(fabsf(m) >= KV4_FAR);
        }
        float base = (float)KV4_P_EXP - m;
        if (far) {
            s[0] = s[0] - m;
            s[1] = s[1] - m;
            base = (float)KV4_P_EXP;
        }
        u32x4 hi4, lo4;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float p0 = __builtin_amdgcn_exp2f(s[e >> 1][2 * (e & 1)] + base), p1 = __builtin_amdgcn_exp2f(s[e >> 1][2 * (e & 1) + 1] + base);
            l += p0 + p1;
            const vt_f16x2 hi2 = __builtin_convertvector((f32x2{p0, p1}), vt_f16x2);
            hi4[e] = __builtin_bit_cast(unsigned, hi2);
            lo4[e] = __builtin_bit_cast(unsigned, __builtin_convertvector((f32x2{fmaf((float)hi2.x, minus, p0), fmaf((float)hi2.y, minus, p1)}), vt_f16x2));
        }
        const vt_f16x8 ph = __builtin_bit_cast(vt_f16x8, hi4), pl = __builtin_bit_cast(vt_f16x8, lo4);
#pragma unroll
        for (int ch = 0; ch < CHUNKS; ch++) {
            unsigned two[8][CD / 2];                           /* key j's values 2 i, 2 i + 1 */
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int row = (j >> 2) * 16 + (j & 3);       /* and 4 g more */
                const unsigned char *at = buf + v_row + row * ROW + ch * 8 * CD;
                const unsigned w = CD == 8 ? *reinterpret_cast<const unsigned *>(at) : (unsigned)*reinterpret_cast<const uint16_t *>(at);
                /* a byte of 255 makes the sum wrap or meet the upper end: finite either way */
                const int e = (int)((unsigned)(buf[vs_row + row * 2 * HP + CD / 2 * ch] + shift) << 23);
                const float f = __int_as_float(min(max(e, 64 << 23), (127 + KV4_V_EXP) << 23));
                two[j][0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, f, 0));
                two[j][1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, f, 1));
                if constexpr (CD == 8) {
                    two[j][2] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, f, 2));
                    two[j][3] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, f, 3));
                }
            }
#pragma unroll
            for (int i = 0; i < CD; i++) {
                u32x4 v4;
#pragma unroll
                for (int e = 0; e < 4; e++) v4[e] = __builtin_amdgcn_perm(two[2 * e + 1][i / 2], two[2 * e][i / 2], i & 1 ? 0x07060302u : 0x05040100u);
                const vt_f16x8 v = __builtin_bit_cast(vt_f16x8, v4);
                f32x4 &acc = o[ch * CD + i];
                acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pl, acc, 0, 0, 0);
                acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, ph, acc, 0, 0, 0);
            }
        }
    };
    auto item = [&](int t, const unsigned char *here, unsigned char *later) __attribute__((always_inline)) {
        asm volatile("" ::: "memory");
        /* vmcnt: the next tile may be on its way; lgkmcnt(0): what is asked for below overwrites what the last tile read */
        __builtin_amdgcn_s_waitcnt(0x0070 | (2 * HP + 2));
        asm volatile("" ::: "memory");
        ask(later, t + 2);
        asm volatile("" ::: "memory");
        tile(here, t);
    };
    for (int t = wide ? tiles : 0; t < tiles; t += 3) {
        item(t, buf0, buf2);
        if (t + 1 >= tiles) break;
        item(t + 1, buf1, buf0);
        if (t + 2 >= tiles) break;
        item(t + 2, buf2, buf1);
    }
    l = vt_rows_sum(l);
    if (wide) {                                          /* o: means of values */
        __builtin_amdgcn_s_waitcnt(0x0f70);              /* nothing arrives in the buffer any more */
        float *at = reinterpret_cast<float *>(buf0 + wave * STAGE);
#pragma unroll 1
        for (int col = 0; col < nc; col++) {
            const int c = c0 + col, i = kv4_query(c, inv_group);
            float cm, cl;
            kv4_column<HP>(a, a.Q + ((size_t)i * a.n_heads + (size_t)(h * group + c - i * group)) * HD, row0, max(min(rows, a.start + i + 1 - lo), 0), lane, at, cm, cl);
            __builtin_amdgcn_wave_barrier();             /* the wave's own LDS, in order */
            if (n == col) {
                m = cm;
                l = cl;
#pragma unroll
                for (int ch = 0; ch < CHUNKS; ch++)
#pragma unroll
                    for (int i = 0; i < CD; i++)
#pragma unroll
                        for (int v = 0; v < 4; v++) o[ch * CD + i][v] = at[16 * CD * ch + CD * (4 * g + v) + i];
            }
            __builtin_amdgcn_wave_barrier();
        }
    } else if (nan) {
        /* rare: the first row of the wave's with a NaN in a block of 32 values reaches the columns that see it */
#pragma unroll 1
        for (int blk = 0; blk < 2 * HP; blk++) {
            int at = 0x7fffffff;
            for (int r = lane; r < rows; r += 64)
                if (a.v_scales[(row0 + r) * 2 * HP + blk] == 255) { at = lo + r; break; }
#pragma unroll
            for (int w = 32; w > 0; w /= 2) at = min(at, __shfl_xor(at, w));
#pragma unroll
            for (int ch = 0; ch < CHUNKS; ch++)
#pragma unroll
                for (int i = 0; i < CD; i++)
#pragma unroll
                    for (int v = 0; v < 4; v++)
                        if ((16 * CD * ch + CD * (4 * g + v)) / 32 == blk && see > at) o[ch * CD + i][v] = NAN;
        }
    }
    /* The waves' parts, each times its share of the sum of weights, which is a mean of values: a sum of values near the end of the range would
     * leave it. */
    ml[wave][n][0] = m;                                          /* four lanes the same */
    ml[wave][n][1] = l;
    __builtin_amdgcn_s_waitcnt(0x0f70);                          /* nothing arrives in the buffers any more */
    __syncthreads();
    float M = m, L = 0.f;
#pragma unroll
    for (int k = 0; k < WAVES; k++) M = fmaxf(M, ml[k][n][0]);
#pragma unroll
    for (int k = 0; k < WAVES; k++) L = fmaf(ml[k][n][1], __builtin_amdgcn_exp2f(ml[k][n][0] - M), L);
    const auto area = [&](int w, int col) { return reinterpret_cast<float *>((col < 8 ? buf0 : buf1) + w * STAGE) + (col & 7) * OD; };
    {
        const float f = L == 0.f && a.parts > 1 ? 0.f : __builtin_amdgcn_exp2f(m - M) / L * (wide ? l : 1.f);
        float *to = area(wave, n) + 4 * g * CD;
#pragma unroll
        for (int ch = 0; ch < CHUNKS; ch++)
#pragma unroll
            for (int v = 0; v < 4; v++)
#pragma unroll
                for (int i = 0; i < CD; i++) to[16 * CD * ch + CD * v + i] = __builtin_amdgcn_ldexpf(o[ch * CD + i][v] * f, wide ? 0 : -shift);
    }
    __syncthreads();
    const int per = a.parts;
    float *part = reinterpret_cast<float *>(a.part) + ((size_t)h * a.tiles + ct) * per * KV4_COLS * OD;
    auto result = [&](int col) {
        const int k = c0 + col, i = kv4_query(k, inv_group);
        return a.out + ((size_t)i * a.n_heads + (size_t)(h * group + k - i * group)) * HD;
    };
    for (int e = (int)threadIdx.x; e < nc * (HD / 4); e += 64 * WAVES) {
        const int col = e / (HD / 4), d = 4 * (e - col * (HD / 4));
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < WAVES; k++) v = v + *reinterpret_cast<const f32x4 *>(area(k, col) + d);
        if (per == 1) *reinterpret_cast<f32x4 *>(result(col) + d) = v;
        else {
            float *to = part + ((size_t)chunk * KV4_COLS + col) * OD + 4 + d;
#pragma unroll
            for (int i = 0; i < 4; i++) vt_stc(to + i, v[i]);
        }
    }
    if (per == 1) return;
    if (wave == 0 && lane < nc) {
        float *to = part + ((size_t)chunk * KV4_COLS + lane) * OD;
        vt_stc(to, M);
        vt_stc(to + 1, L);
    }
    __builtin_amdgcn_s_waitcnt(0x0f70);                          /* the part's stores are acknowledged */
    __syncthreads();
    unsigned *cnt = a.cnt + h * a.tiles + ct;
    if (threadIdx.x == 0) last = __hip_atomic_fetch_add(cnt, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)(per - 1);
    __syncthreads();
    if (!last) return;
    if (threadIdx.x == 0) vt_stc_u32(cnt, 0u);                   /* ready for the next launch */
    /* a wave per column: lane k has part k's largest score and sum of weights */
    const __amdgpu_buffer_rsrc_t pd = vt_buffer(part, per * KV4_COLS * OD * 4);
    for (int col = wave; col < nc; col += WAVES) {
        const u32x2 v = __builtin_amdgcn_raw_buffer_load_b64(pd, (min(lane, per - 1) * KV4_COLS + col) * OD * 4, 0, 16 /* sc1 */);
        const float pm = __uint_as_float(v.x), pl = lane < per ? __uint_as_float(v.y) : 0.f;
        const float w = pl * __builtin_amdgcn_exp2f(pm - vt_wave_max(pm)), all = vt_wave_sum(w);
        wt[col][lane] = w / all;
    }
    __syncthreads();
    for (int e = (int)threadIdx.x; e < nc * (HD / 4); e += 64 * WAVES) {
        const int col = e / (HD / 4), d = 4 * (e - col * (HD / 4)), at = (col * OD + 4 + d) * 4;
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
        for (int k0 = 0; k0 < per; k0 += 16) {                   /* parts past the last: the last again, times 0 */
            f32x4 p[16];
#pragma unroll
            for (int k = 0; k < 16; k++) p[k] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(pd, at + min(k0 + k, per - 1) * (KV4_COLS * OD * 4), 0, 16));
#pragma unroll
            for (int k = 0; k < 16; k++) v = v + p[k] * wt[col][k0 + k];
        }
        *reinterpret_cast<f32x4 *>(result(col) + d) = v;
    }
}

/* Many columns: a workgroup has KV4_TILE of them, a wave 32, and goes through its rows 64 at a time.  K comes as it lies, V as fp16 in
 * the order of the matrix instruction's operand (A of 32 x 32 x 16, value 2 HP r + i in row r of instruction i; four keys of a value are
 * 8 bytes): the workgroup converts the next rows while it multiplies these, each lane four keys of eight values, so that a conversion
 * serves all columns.  Scores are 32 x 32 x 64. Where there are few columns for the chip, or a prompt's last ones would be behind
 * everybody, several workgroups share a head's rows, `run` tiles each; the last to arrive adds their parts.  Bound: 4000 queries of 32
 * heads on 8 with 128 values, 220 us, are 64 tiles for each of 512 workgroups that are there at once, 5000 cycles for the two of a SIMD,
 * of which 3300 are matrix instructions (20 for scores, 32 for results) and 3600 vector ones, at the clock that their power allows.
 * Reads of what is multiplied next, and the next weights' arithmetic, stand between the products, and work is handed out head by head,
 * the longest first: neither 283 us, the one 264, the other 231. */

template <int HP>
__global__ void __launch_bounds__(64 * KV4_TILE_WAVES, 2) vt_kv4_tile_kernel(kv4_job a) {
    constexpr int HD = 64 * HP, ROW = 32 * HP, THREADS = 64 * KV4_TILE_WAVES, UNITS = 128 * HP, UN = (UNITS + THREADS - 1) / THREADS, DT = 2 * HP;
    constexpr int KB = 64 * ROW, SB = KB + UNITS, VB = SB;      /* K rows, their scales, V's operands */
    __shared__ __attribute__((aligned(16))) unsigned char buf[2][VB + 64 * HD * 2];
    __shared__ int scan[KV4_TILE_WAVES][3];
    __shared__ int last;
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 31, g = lane >> 5, h = (int)blockIdx.x;
    /* Work is handed out head by head, the columns that see most first, and their last parts, which others do not have, before these. */
    const int part = a.parts - 1 - (int)blockIdx.z, ct = a.tiles - 1 - (int)blockIdx.y;
    const int c0 = ct * KV4_TILE, nc = min(KV4_TILE, a.cols - c0);
    const int end = a.start + vt_div(c0 + nc - 1, a.group) + 1, parts = ((end + 63) / 64 + a.run - 1) / a.run;
    if (part >= parts) return;
    const int lo = part * a.run * 64, rows = min(a.run * 64, end - lo), tiles = (rows + 63) / 64;
    const int w0 = c0 + 32 * wave, wc = min(w0 + 32, a.cols) - w0;               /* this wave's columns: none, perhaps */
    const int cc = min(w0 + n, a.cols - 1), qi = vt_div(cc, a.group), see = a.start + qi + 1;
    const int seen_first = a.start + vt_div(min(w0, a.cols - 1), a.group) + 1, seen_last = wc > 0 ? a.start + vt_div(w0 + wc - 1, a.group) + 1 : 0;
    const size_t row0 = (size_t)h * a.max_rows + lo;
    const __amdgpu_buffer_rsrc_t kd = vt_buffer(a.k_codes + row0 * ROW, rows * ROW), vd = vt_buffer(a.v_codes + row0 * ROW, rows * ROW);
    const __amdgpu_buffer_rsrc_t ksd = vt_buffer(a.k_scales + row0 * DT, rows * DT), vsd = vt_buffer(a.v_scales + row0 * DT, rows * DT);
    /* unit u: 16 bytes of K, row u / 2 HP; a scale of K; V's keys 4 (u / 8 HP) .. + 3, values 8 (u % 8 HP) .. + 7 */
    u32x4 kr[UN];
    unsigned vr[UN][4];
    unsigned char ksr[UN], vsr[UN][4];
    auto load = [&](int t) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < UN; i++) {
            const int u = tid + THREADS * i;
            if (UNITS % THREADS && u >= UNITS) break;
            kr[i] = __builtin_bit_cast(u32x4, vt_buffer_ld4(kd, t * 64 * ROW + u * 16));
            ksr[i] = __builtin_amdgcn_raw_buffer_load_b8(ksd, t * 64 * DT + u, 0, 0);
            const int kg = u / (8 * HP), dg = u - kg * 8 * HP;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                vr[i][k] = __builtin_amdgcn_raw_buffer_load_b32(vd, (t * 64 + 4 * kg + k) * ROW + dg * 4, 0, 0);
                vsr[i][k] = __builtin_amdgcn_raw_buffer_load_b8(vsd, (t * 64 + 4 * kg + k) * DT + dg / 4, 0, 0);
            }
        }
    };
    /* queries and the first scales of values are asked for in front of the first rows: loads return in order */
    f32x4 q4[HP][8];
    {
        const float *src = a.Q + ((size_t)qi * a.n_heads + (size_t)h * a.group.d + (cc - qi * a.group.d)) * HD + 32 * g;
#pragma unroll
        for (int k = 0; k < HP; k++)
#pragma unroll
            for (int i = 0; i < 8; i++) q4[k][i] = *reinterpret_cast<const f32x4 *>(src + 64 * k + 4 * i);
    }
    unsigned char seen[8];
    auto ask_scales = [&](int i) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < 8; e++) seen[e] = __builtin_amdgcn_raw_buffer_load_b8(vsd, i + e * THREADS, 0, 0);      /* zeros past the last */
    };
    ask_scales(tid);
    load(0);
    vt_u32x6 q[HP][KV4_PLANES];
    unsigned qs[HP][KV4_PLANES];
#pragma unroll
    for (int k = 0; k < HP; k++) {
        vt_f32x16 even, odd;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const f32x4 v = q4[k][i] * a.scale;
            even[2 * i] = v.x; odd[2 * i] = v.y; even[2 * i + 1] = v.z; odd[2 * i + 1] = v.w;
        }
        vt_mx4_planes<KV4_PLANES>(even, odd, q[k], qs[k]);
    }
    unsigned q_scale = 0;
#pragma unroll
    for (int k = 0; k < HP; k++) q_scale = max(q_scale, qs[k][0]);
    const int k_most = __any(q_scale > KV4_FINITE) ? -1 : KV4_FINITE;
    unsigned top = 1, low = 1, least = 0xffffffffu;       /* as in kv4_span */
    for (int i = tid;;) {
#pragma unroll
        for (int e = 0; e < 8; e++) { const unsigned t = (unsigned char)(seen[e] + 1); top = max(top, t); low = min(low, t); least = min(least, t - 2); }
        if ((i += THREADS * 8) - tid >= rows * DT) break;
        ask_scales(i);
    }
    int most = (int)vt_wave_max((float)top) - 1, small = 1 - (int)vt_wave_max(-(float)(int)min(least, 65535u));
    int nan = __any(low == 0);
    if (lane == 0) { scan[wave][0] = most; scan[wave][1] = small; scan[wave][2] = nan; }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < KV4_TILE_WAVES; w++) { most = max(most, scan[w][0]); small = min(small, scan[w][1]); nan |= scan[w][2]; }
    const bool wide = __builtin_amdgcn_readfirstlane(most - small > KV4_SPAN);
    const int shift = __builtin_amdgcn_readfirstlane(127 + KV4_V_EXP - most);
    /* where value d's four keys go: row r = d / 2 HP of instruction i = d % 2 HP, step t of 16 keys, half h of the lane's eight (step and half by the
     * unit: its keys are 4 (kg % 4) .. of step kg / 4, i.e. group of lanes kg % 2, half kg / 2 % 2) */
    int v_to[2][8];                                       /* UN of them (with that size the host pass drops the kernel) */
#pragma unroll
    for (int i = 0; i < UN; i++) {
        const int u = tid + THREADS * i, kg = u / (8 * HP), dg = u - kg * 8 * HP;
#pragma unroll
        for (int d = 0; d < 8; d++) {
            const int r = (8 * dg + d) / DT, in = (8 * dg + d) - r * DT;
            v_to[i][d] = VB + (((in * 4 + (kg >> 2)) * 64 + (kg & 1) * 32 + r) * 2 + ((kg >> 1) & 1)) * 8;
        }
    }
    auto put = [&](unsigned char *b) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < UN; i++) {
            const int u = tid + THREADS * i;
            if (UNITS % THREADS && u >= UNITS) break;
            const int r = u / DT;
            *reinterpret_cast<u32x4 *>(b + r * ROW + kv4_swizzle<HP>(r, u - r * DT) * 16) = kr[i];
            b[KB + u] = ksr[i];
            unsigned two[4][4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int e = (int)((unsigned)(vsr[i][k] + shift) << 23);
                const float f = __int_as_float(min(max(e, 64 << 23), (127 + KV4_V_EXP) << 23));
                two[k][0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(vr[i][k], f, 0));
                two[k][1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(vr[i][k], f, 1));
                two[k][2] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(vr[i][k], f, 2));
                two[k][3] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(vr[i][k], f, 3));
            }
#pragma unroll
            for (int d = 0; d < 8; d++) {
                const unsigned pick = d & 1 ? 0x07060302u : 0x05040100u;
                *reinterpret_cast<u32x2 *>(b + v_to[i][d]) = u32x2{__builtin_amdgcn_perm(two[1][d / 2], two[0][d / 2], pick),
                                                                  __builtin_amdgcn_perm(two[3][d / 2], two[2][d / 2], pick)};
            }
        }
    };
    float minus = -1.f;
    asm("" : "+v"(minus));
    bool far = false;
    float m = -3.402823466e38f, l = 0.f;
    vt_f32x16 o[DT];
#pragma unroll
    for (int i = 0; i < DT; i++) o[i] = vt_f32x16{};
    put(buf[0]);
    __syncthreads();
#pragma unroll 1
    for (int t = wide ? tiles : 0; t < tiles; t++) {
        const unsigned char *b = buf[t & 1];
        if (t + 1 < tiles) load(t + 1);
        const int first = lo + 64 * t;
        if (first < seen_last) {                          /* else nobody of this wave sees these rows */
            vt_f32x16 s[2];
            int k_scale = 0;
#pragma unroll
            for (int kt = 0; kt < 2; kt++) {
                const int row = 32 * kt + n;
                u32x4 k[HP];
                int ksc[HP];
#pragma unroll
                for (int kk = 0; kk < HP; kk++) {
                    k[kk] = *reinterpret_cast<const u32x4 *>(b + row * ROW + kv4_swizzle<HP>(row, 2 * kk + g) * 16);
                    ksc[kk] = b[KB + row * DT + 2 * kk + g];
                    k_scale = max(k_scale, ksc[kk]);
                }
                s[kt] = vt_f32x16{};
#pragma unroll
                for (int p = KV4_PLANES - 1; p >= 0; p--)
#pragma unroll
                    for (int kk = 0; kk < HP; kk++)
                        s[kt] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(vt_mfma_e2m1(k[kk]), vt_mfma_e2m3(q[kk][p]), s[kt], VT_MFMA_E2M1, VT_MFMA_E2M3,
                                                                                0, ksc[kk], 0, (int)qs[kk][p]);
            }
            if (first + 64 > seen_first || __any(k_scale > k_most)) {
#pragma unroll
                for (int kt = 0; kt < 2; kt++)
#pragma unroll
                    for (int v = 0; v < 16; v++) s[kt][v] = kv4_seen(s[kt][v], first + 32 * kt + 8 * (v >> 2) + 4 * g + (v & 3) < see);
            }
            float top = m;                                /* a NaN stays one: who sees it answers NaN */
#pragma unroll
            for (int v = 0; v < 16; v++) top = __builtin_elementwise_maximum(__builtin_elementwise_maximum(top, s[0][v]), s[1][v]);
            { const f32x2 r = vt_swap32(top, top); top = __builtin_elementwise_maximum(r.x, r.y); }
            if (__any(top != m)) {
                const float less = __builtin_amdgcn_exp2f(m - top);
                l *= less;
#pragma unroll
                for (int i = 0; i < DT; i++) o[i] = o[i] * less;
                m = top;
                far = __any(fabsf(m) >= KV4_FAR);
            }
            float base = (float)KV4_P_EXP - m;
            if (far) {
                s[0] = s[0] - m;
                s[1] = s[1] - m;
                base = (float)KV4_P_EXP;
            }
            /* 16 keys a step: elements 8 (st % 2) .. of scores st / 2.  The next step's weights are made, and its values read, between
             * this one's products. */
            u32x4 hi4, lo4;
            vt_f16x8 v[DT];
            auto weight = [&](int st, int e) __attribute__((always_inline)) {
                const float p0 = __builtin_amdgcn_exp2f(s[st >> 1][8 * (st & 1) + 2 * e] + base), p1 = __builtin_amdgcn_exp2f(s[st >> 1][8 * (st & 1) + 2 * e + 1] + base);
                l += p0 + p1;
                const vt_f16x2 hi2 = __builtin_convertvector((f32x2{p0, p1}), vt_f16x2);
                hi4[e] = __builtin_bit_cast(unsigned, hi2);
                lo4[e] = __builtin_bit_cast(unsigned, __builtin_convertvector((f32x2{fmaf((float)hi2.x, minus, p0), fmaf((float)hi2.y, minus, p1)}), vt_f16x2));
            };
            auto value = [&](int st, int i) __attribute__((always_inline)) {
                v[i] = __builtin_bit_cast(vt_f16x8, *reinterpret_cast<const u32x4 *>(b + VB + ((i * 4 + st) * 64 + lane) * 16));
            };
#pragma unroll
            for (int i = 0; i < DT; i++) value(0, i);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int e = 0; e < 4; e++) weight(0, e);
#pragma unroll
            for (int st = 0; st < 4; st++) {
                const vt_f16x8 ph = __builtin_bit_cast(vt_f16x8, hi4), pl = __builtin_bit_cast(vt_f16x8, lo4);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < DT; i++) {
                    o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[i], pl, o[i], 0, 0, 0);
                    if (st < 3) {
#pragma unroll
                        for (int e = 4 * i / DT; e < 4 * (i + 1) / DT; e++) weight(st + 1, e);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                    o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[i], ph, o[i], 0, 0, 0);
                    if (st < 3) value(st + 1, i);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
        if (t + 1 < tiles) put(buf[(t + 1) & 1]);
        __syncthreads();
    }
    { const f32x2 r = vt_swap32(l, l); l = r.x + r.y; }
    if (wide) {                                          /* o: means of values */
        float *at = reinterpret_cast<float *>(buf[0]) + wave * HD;
#pragma unroll 1
        for (int col = 0; col < wc; col++) {
            const int c = w0 + col, i = vt_div(c, a.group);
            float cm, cl;
            kv4_column<HP>(a, a.Q + ((size_t)i * a.n_heads + (size_t)h * a.group.d + (c - i * a.group.d)) * HD, row0, max(min(rows, a.start + i + 1 - lo), 0), lane, at, cm, cl);
            __builtin_amdgcn_wave_barrier();
            if (n == col) {
                m = cm;
                l = cl;
#pragma unroll
                for (int i = 0; i < DT; i++)
#pragma unroll
                    for (int v = 0; v < 16; v++) o[i][v] = at[DT * (8 * (v >> 2) + 4 * g + (v & 3)) + i];
            }
            __builtin_amdgcn_wave_barrier();
        }
    } else if (nan) {
#pragma unroll 1
        for (int blk = 0; blk < DT; blk++) {
            int at = 0x7fffffff;
            for (int r = lane; r < rows; r += 64)
                if (a.v_scales[(row0 + r) * DT + blk] == 255) { at = lo + r; break; }
#pragma unroll
            for (int w = 32; w > 0; w /= 2) at = min(at, __shfl_xor(at, w));
#pragma unroll
            for (int i = 0; i < DT; i++)
#pragma unroll
                for (int v = 0; v < 16; v++)
                    if ((DT * (8 * (v >> 2) + 4 * g + (v & 3)) + i) / 32 == blk && see > at) o[i][v] = NAN;
        }
    }
    if (!wide) {                                         /* the part's mean of values */
        const float f = l == 0.f && parts > 1 ? 0.f : 1.f / l;
#pragma unroll
        for (int i = 0; i < DT; i++)
#pragma unroll
            for (int v = 0; v < 16; v++) o[i][v] = __builtin_amdgcn_ldexpf(o[i][v] * f, -shift);
    }
    if (parts > 1) {
        /* a part lies as the lanes hold it: [part][wave][4 HD / 32 vectors of four, then largest score and sum of weights][lane] */
        constexpr int WAVE_PART = (DT * 4 + 1) * 1024, PART = KV4_TILE_WAVES * WAVE_PART;
        const __amdgpu_buffer_rsrc_t pd = vt_buffer(a.part + ((size_t)h * a.tiles + ct) * a.parts * PART, parts * PART);
        const int mine = wave * WAVE_PART + lane * 16;
#pragma unroll
        for (int i = 0; i < DT; i++)
#pragma unroll
            for (int v = 0; v < 4; v++)
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, (f32x4{o[i][4 * v], o[i][4 * v + 1], o[i][4 * v + 2], o[i][4 * v + 3]})), pd,
                                                       mine + part * PART + (4 * i + v) * 1024, 0, 16 /* sc1 */);
        __builtin_amdgcn_raw_buffer_store_b64(u32x2{__float_as_uint(m), __float_as_uint(l)}, pd, mine + part * PART + DT * 4 * 1024, 0, 16);
        __builtin_amdgcn_s_waitcnt(0x0f70);              /* acknowledged */
        __syncthreads();
        unsigned *cnt = a.cnt + h * a.tiles + ct;
        if (tid == 0) last = __hip_atomic_fetch_add(cnt, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)(parts - 1);
        __syncthreads();
        if (!last) return;
        if (tid == 0) vt_stc_u32(cnt, 0u);
        if (wc <= 0) return;
        float M = -3.402823466e38f, L = 0.f;
#pragma unroll 4
        for (int k = 0; k < parts; k++) {
            const u32x2 v = __builtin_amdgcn_raw_buffer_load_b64(pd, mine + k * PART + DT * 4 * 1024, 0, 16);
            const float pm = __uint_as_float(v.x), top = fmaxf(M, pm);
            L = fmaf(L, __builtin_amdgcn_exp2f(M - top), __uint_as_float(v.y) * __builtin_amdgcn_exp2f(pm - top));
            M = top;
        }
#pragma unroll
        for (int i = 0; i < DT; i++) o[i] = vt_f32x16{};
#pragma unroll 1
        for (int k = 0; k < parts; k++) {
            const u32x2 ml = __builtin_amdgcn_raw_buffer_load_b64(pd, mine + k * PART + DT * 4 * 1024, 0, 16);
            f32x4 p[DT * 4];
#pragma unroll
            for (int x = 0; x < DT * 4; x++) p[x] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(pd, mine + k * PART + x * 1024, 0, 16));
            const float w = __uint_as_float(ml.y) * __builtin_amdgcn_exp2f(__uint_as_float(ml.x) - M) / L;
#pragma unroll
            for (int x = 0; x < DT * 4; x++)
#pragma unroll
                for (int e = 0; e < 4; e++) o[x / 4][4 * (x % 4) + e] = fmaf(p[x][e], w, o[x / 4][4 * (x % 4) + e]);
        }
    }
    /* element v of lane l is value 2 HP (8 (v / 4) + 4 (l / 32) + v % 4) + i */
    if (n < wc) {
        float *to = a.out + ((size_t)qi * a.n_heads + (size_t)h * a.group.d + (cc - qi * a.group.d)) * HD;
#pragma unroll
        for (int v = 0; v < 16; v++)
#pragma unroll
            for (int i = 0; i < DT; i += 2) *reinterpret_cast<f32x2 *>(to + DT * (8 * (v >> 2) + 4 * g + (v & 3)) + i) = f32x2{o[i][v], o[i + 1][v]};
    }
}

static_assert(sizeof(kv4_job) <= 104, "arguments");

template <int HP, int WAVES>
static int kv4_stream(const kv4_job &a, int heads, long long wgs) {
    static_assert(WAVES == vt_kv4_waves(HP), "the plan's");
    kv4_job job = a;
    if (a.parts > 1 && !(job.part = (unsigned char *)vt_scratch(sizeof(float) * (size_t)wgs * a.parts * KV4_COLS * (64 * HP + 4)))) return -1;
    hipLaunchKernelGGL((vt_kv4_stream_kernel<HP, WAVES>), dim3((unsigned)heads, (unsigned)a.parts, (unsigned)a.tiles), dim3(64 * WAVES), 0, g_vt.stream, job);
    return 0;
}

template <int HP>
static int kv4_tiles(const kv4_job &a, int heads, long long wgs) {
    kv4_job job = a;
    if (a.parts > 1 && !(job.part = (unsigned char *)vt_scratch((size_t)wgs * a.parts * KV4_TILE_WAVES * (8 * HP + 1) * 1024))) return -1;
    hipLaunchKernelGGL(vt_kv4_tile_kernel<HP>, dim3((unsigned)heads, (unsigned)a.tiles, (unsigned)a.parts), dim3(64 * KV4_TILE_WAVES), 0, g_vt.stream, job);
    return 0;
}

extern "C" int tts_hip_kv4_attention(float *d_out, const float *d_Q, const tts_hip_kv4_t *cache, int seq_len, int start_pos, int n_heads, float scale) {
    static const char who[] = "tts_hip_kv4_attention";
    if (!d_out || !d_Q || (((uintptr_t)d_out | (uintptr_t)d_Q) & 15)) { vt_set_error("%s: queries and results lie on 16 bytes", who); return -1; }
    if (seq_len < 1 || start_pos < 0) { vt_set_error("%s: %d queries behind %d rows", who, seq_len, start_pos); return -1; }
    if (!cache_ok(who, cache, 0, (long long)start_pos + seq_len)) return -1;
    if (n_heads < 1 || n_heads % cache->n_kv_heads) { vt_set_error("%s: %d heads on %d kv heads", who, n_heads, cache->n_kv_heads); return -1; }
    const int group = n_heads / cache->n_kv_heads, HP = cache->head_dim / 64;
    if (cache->n_kv_heads > 65535 || group > 1 << 19 || (long long)start_pos + seq_len > 1 << 24) {
        vt_set_error("%s: %d queries of %d heads on %d behind %d rows are too many", who, seq_len, n_heads, cache->n_kv_heads, start_pos);
        return -1;
    }
    if (!vt_mx4_ready(who)) return -1;
    const int n_cu = g_vt.n_cu > 0 ? g_vt.n_cu : 256, most = (1 << 19) / group;        /* queries of a launch: their tiles of columns are a dimension of the grid */
    for (int s = 0; s < seq_len; s += most) {
        const int n = seq_len - s < most ? seq_len - s : most, cols = n * group;
        const size_t at = (size_t)s * n_heads * cache->head_dim;
        const int heads = cache->n_kv_heads;
        const vt_kv4_plan p = vt_kv4_plan_of(n_cu, HP, heads, group, cols, start_pos + s, start_pos + s + n);
        const kv4_job a = {cache->k_codes, cache->k_scales, cache->v_codes, cache->v_scales, d_out + at, d_Q + at, NULL, g_vt.d_mx4_cnt,
                           cache->max_rows, start_pos + s, n_heads, cols, p.run, p.parts, p.tiles, vt_divisor_of(group, cols), scale * 1.44269504f};
        const long long wgs = (long long)heads * p.tiles;
        int bad;
        if (p.many) bad = HP == 1 ? kv4_tiles<1>(a, heads, wgs) : kv4_tiles<2>(a, heads, wgs);
        else if (HP <= 2) bad = HP == 1 ? kv4_stream<1, 8>(a, heads, wgs) : kv4_stream<2, 8>(a, heads, wgs);
        else bad = HP == 3 ? kv4_stream<3, 4>(a, heads, wgs) : kv4_stream<4, 4>(a, heads, wgs);
        if (bad) return -1;
    }
    return vt_check(hipGetLastError(), who) ? -1 : 0;
}
