/*
 * vt_paged.hip - several sequences over one paged key/value cache: the batch's handle, rotary positions (with the norm of each head in the same pass), and
 * keys and values into pages.  The attention is in vt_paged_attention.hip.
 *
 * A pool is [n_pages, n_kv_heads, page_rows, head_dim] bf16, one for K and one for V: what one head's attention reads of a page is one piece of memory.
 */
#include "vt_paged.h"
#include "vt_device.h"
#include "vt_requests.h"

#include <math.h>
#include <new>
#include <string.h>

/* ---- the handle ----------------------------------------------------------------------------------------------- */

static size_t paged_up(size_t n) { return (n + 255) & ~(size_t)255; }

extern "C" tts_hip_paged_t *tts_hip_paged_create(const tts_hip_paged_shape_t *shape, int max_seqs, int max_rows, int max_table) {
    static const char who[] = "tts_hip_paged_create";
    if (!shape) { vt_set_error("%s: no shape", who); return NULL; }
    const vt_paged_shape s = {shape->n_pages, shape->page_rows, shape->n_heads, shape->n_kv_heads, shape->head_dim, shape->window};
    if (const char *why = vt_paged_shape_bad(s)) {
        vt_set_error("%s: %d pages of %d rows, %d heads on %d of %d, window %d: %s", who, s.n_pages, s.page_rows, s.n_heads, s.n_kv_heads, s.head_dim, s.window,
                     why);
        return NULL;
    }
    const int group = s.n_heads / s.n_kv_heads;
    if (max_seqs < 1 || max_rows < 1 || max_table < 1 || max_seqs > PAGED_MAX_ROWS || max_rows > PAGED_MAX_ROWS || max_table > 1 << 28 ||
        (long long)max_rows * group > INT_MAX / 4) {
        vt_set_error("%s: batches of up to %d sequences, %d rows of %d heads on each kv head, %d table entries", who, max_seqs, max_rows, group, max_table);
        return NULL;
    }
    tts_hip_paged *b = new (std::nothrow) tts_hip_paged();
    int *own = (int *)malloc(sizeof(int) * ((size_t)max_seqs + max_rows));
    unsigned long long *seen = (unsigned long long *)calloc((size_t)s.n_pages / 64 + 1, sizeof *seen);
    if (!b || !own || !seen) {
        vt_set_error("%s: out of host memory", who);
        delete b;
        free(own);
        free(seen);
        return NULL;
    }
    b->shape = s;
    b->max_seqs = max_seqs;
    b->max_rows = max_rows;
    b->max_table = max_table;
    b->max_items = (int)vt_paged_max_items(max_seqs, max_rows, group) << vt_paged_type_matters(s);
    b->device = b->n_seqs = -1;
    b->described = paged_up(sizeof(int) * (size_t)max_rows) + paged_up(2 * sizeof(int) * (size_t)max_rows) + paged_up(sizeof(int) * (size_t)max_table);
    b->bytes = b->described + sizeof(vt_paged_item) * (size_t)b->max_items;
    b->starts = own;
    b->written = own + max_seqs;
    b->seen = seen;
    return b;
}

extern "C" void tts_hip_paged_free(tts_hip_paged_t *b) {
    if (!b) return;
    if (b->device >= 0) {
        int before = b->device;
        (void)hipGetDevice(&before);
        if (before != b->device) (void)hipSetDevice(b->device);
        (void)hipDeviceSynchronize();                    /* launches that read it */
        (void)hipFree(b->dev);
        (void)hipHostFree(b->host);
        (void)hipEventDestroy(b->copied);
        if (before != b->device) (void)hipSetDevice(before);
    }
    free(b->starts);
    free(b->seen);
    delete b;
}

/* memory for a batch, on the first one; all of it or none */
static int paged_memory(const char *who, tts_hip_paged *b) {
    if (b->device == g_vt.device) return 0;
    if (b->device >= 0) { vt_set_error("%s: the batch is on device %d, the context on %d", who, b->device, g_vt.device); return -1; }
    if (!(b->dev = (unsigned char *)vt_dev_alloc(b->bytes))) return -1;
    if (vt_check(hipHostMalloc((void **)&b->host, b->bytes, hipHostMallocDefault), "hipHostMalloc")) { (void)hipFree(b->dev); return -1; }
    if (vt_check(hipEventCreateWithFlags(&b->copied, hipEventDisableTiming), "hipEventCreateWithFlags")) {
        (void)hipFree(b->dev);
        (void)hipHostFree(b->host);
        return -1;
    }
    b->device = g_vt.device;
    return 0;
}

static void paged_say(const char *who, const tts_hip_paged *b, const vt_paged_fault &f, const int *past, const int *rows, int n_seqs, int stride) {
    switch (f.what) {
    case PAGED_COUNT: vt_set_error("%s: %d sequences of at most %d, tables %d entries apart", who, n_seqs, b->max_seqs, stride); break;
    case PAGED_SEQUENCE: vt_set_error("%s: sequence %d has %d rows behind %d", who, f.seq, rows[f.seq], past[f.seq]); break;
    case PAGED_TOO_MANY_ROWS: vt_set_error("%s: more than %d new rows with sequence %d", who, b->max_rows, f.seq); break;
    case PAGED_TABLE: vt_set_error("%s: %d pages of sequence %d, tables %d entries apart, at most %d entries in all", who, f.at, f.seq, stride, b->max_table); break;
    case PAGED_PAGE: vt_set_error("%s: page %d of sequence %d is %d, of %d", who, f.at, f.seq, f.value, b->shape.n_pages); break;
    default: vt_set_error("%s: new rows go into page %d twice", who, f.value);
    }
}

extern "C" int tts_hip_paged_set(tts_hip_paged_t *b, int n_seqs, const int *past, const int *rows, const int *tables, int table_stride) {
    static const char who[] = "tts_hip_paged_set";
    if (!b) { vt_set_error("%s: no batch", who); return -1; }
    b->n_seqs = -1;                                      /* refused: none */
    if (n_seqs > 0 && (!past || !rows || !tables)) { vt_set_error("%s: a NULL pointer", who); return -1; }
    const bool first = b->device < 0;
    unsigned char *host = b->host;
    if (first && !(host = (unsigned char *)malloc(b->described))) { vt_set_error("%s: out of host memory", who); return -1; }
    /* `host` may still be on its way from the last call */
    if (!first && vt_check(hipEventSynchronize(b->copied), who)) return -1;
    /* one piece of memory, one copy: what comes first is as long as these rows need */
    long long some = 0;
    for (int i = 0; i < n_seqs && i < b->max_seqs && some < b->max_rows; i++) some += rows[i] > 0 ? rows[i] : 0;
    if (some > b->max_rows) some = b->max_rows;
    b->at_place = paged_up(sizeof(int) * (size_t)some);
    b->at_tables = b->at_place + paged_up(2 * sizeof(int) * (size_t)some);
    vt_paged_rows to = {(int *)host, (int *)(host + b->at_place), (int *)(host + b->at_tables), b->starts, b->written};
    int n_rows = 0, n_table = 0;
    const vt_paged_fault f = vt_paged_lay_out(b->shape, b->max_seqs, b->max_rows, b->max_table, n_seqs, past, rows, tables, table_stride, to, &n_rows, &n_table);
    b->at_items = b->at_tables + paged_up(sizeof(int) * (size_t)n_table);
    int bad = f.what != PAGED_OK;
    if (bad) paged_say(who, b, f, past, rows, n_seqs, table_stride);
    bad = bad || !vt_mx4_ready(who) || paged_memory(who, b);
    if (first) {
        if (!bad) memcpy(b->host, host, b->at_items);
        free(host);
    }
    if (bad) return -1;
    vt_paged_item *items = (vt_paged_item *)(b->host + b->at_items);
    const int n_cu = g_vt.n_cu > 0 ? g_vt.n_cu : 256;
    b->plan[0] = b->plan[1] = vt_paged_plan_of(b->shape, false, n_cu, n_seqs, past, rows, b->starts, items);
    int n_items = b->plan[0].few + b->plan[0].many;
    b->bf16_items = 0;
    if (vt_paged_type_matters(b->shape)) {
        b->bf16_items = n_items;
        b->plan[1] = vt_paged_plan_of(b->shape, true, n_cu, n_seqs, past, rows, b->starts, items + n_items);
        n_items += b->plan[1].few + b->plan[1].many;
    }
    vt_paged_once(b->plan, 2, b->shape, n_seqs, past, rows, b->starts, (const int *)(b->host + b->at_tables), b->seen);
    const size_t all = b->at_items + sizeof(vt_paged_item) * (size_t)n_items;
    if (n_rows && vt_check(hipMemcpyAsync(b->dev, b->host, all, hipMemcpyHostToDevice, g_vt.stream), who)) return -1;
    if (vt_check(hipEventRecord(b->copied, g_vt.stream), who)) return -1;
    b->n_rows = n_rows;
    b->n_seqs = n_seqs;
    return 0;
}

int vt_paged_ready(const char *who, const tts_hip_paged *b) {
    if (!b || b->n_seqs < 0) { vt_set_error("%s: no batch", who); return 0; }
    if (!vt_mx4_ready(who)) return 0;
    if (b->device == g_vt.device) return 1;
    vt_set_error("%s: the batch is on device %d, the context on %d", who, b->device, g_vt.device);
    return 0;
}

extern "C" const int *tts_hip_paged_positions(const tts_hip_paged_t *b) {
    static const char who[] = "tts_hip_paged_positions";
    return vt_paged_ready(who, b) ? (const int *)b->dev : NULL;
}

/* ---- positions ----
 * Pair i of a head turns by 2 pi position turns[i].  The product is made in 64 bits, with what that rounds away, and only what is left of it below one turn
 * goes on in fp32, in two parts: the angle is that of these turns to 2^-24 or so however far the position (in fp32 it would be off by 0.03 at position 10^6).
 * The turns themselves are made here to some 2^-52: what is left of the formula's angle is off by that times the position, 2^-24 at 2^28, 2^-21 at 2^31. */
__global__ void __launch_bounds__(256) vt_rotary_turns_kernel(double *turns, int pairs, double theta, double factor, double original, double low, double high) {
    const int i = (int)(blockIdx.x * 256 + threadIdx.x);
    if (i >= pairs) return;
    const double f = pow(theta, -(double)i / (double)pairs) * 0.15915494309189533577;
    const double keep = fmin(fmax((f * original - low) / (high - low), 0.0), 1.0);
    turns[i] = factor == 1.0 ? f : f * (keep + (1.0 - keep) / factor);
}

extern "C" int tts_hip_rotary_turns(double *d_turns, int rot_dim, double theta, double factor, int original_rows, double low_turns, double high_turns) {
    static const char who[] = "tts_hip_rotary_turns";
    if (!d_turns || ((uintptr_t)d_turns & 7) || rot_dim < 2 || rot_dim > 512 || rot_dim % 2) {
        vt_set_error("%s: %d values that turn (2 .. 512, even)", who, rot_dim);
        return -1;
    }
    if (!(theta > 0) || !(factor > 0) || isinf(theta) || isinf(factor) || original_rows < 0 || !(low_turns < high_turns) || isinf(low_turns) || isinf(high_turns)) {
        vt_set_error("%s: theta %g, factor %g, %d rows, between %g and %g turns", who, theta, factor, original_rows, low_turns, high_turns);
        return -1;
    }
    if (!vt_mx4_ready(who)) return -1;
    hipLaunchKernelGGL(vt_rotary_turns_kernel, dim3(1), dim3(256), 0, g_vt.stream, d_turns, rot_dim / 2, theta, factor, (double)original_rows, low_turns,
                       high_turns);
    return vt_check(hipGetLastError(), who) ? -1 : 0;
}

/* ---- heads: norm, turn, store ----
 * A lane has a unit of four pairs of a head, 2^log lanes a head, and makes the angles once for the HEADS heads that it walks: angles are more than half of
 * the instructions that a unit takes.  (2 p, 2 p + 1) is pair p in both layouts where p does not turn.  Bound by the launch for a few rows (1 to 226 rows of
 * 32 heads 3.8 to 4.3 us a call, 2.5 to 3.8 of them the kernel's); 1531 rows of 32 heads 7.5 us, 25 MB at 3.3 TB/s. */
struct turn_job {
    const void *x, *x2;                                  /* K and V for pages */
    void *out, *out2;
    const int *pos, *place;
    const double *turns;
    const float *gain;
    float magnitude, eps, inv_hd;
    int n, heads, hd, x_stride, out_stride, rot_half;    /* n: rows times sets of heads; rot_half: 2 rot + half */
    int lanes_log;
    vt_divisor sets;                                     /* sets of heads of a row */
};

typedef unsigned short turn_u16x4 __attribute__((ext_vector_type(4)));

template <bool BF16, bool WIDE>
static __device__ __forceinline__ void turn_load(const void *x, long long at, int hd, int u, int rot, int half, float a[4], float b[4]) {
    const bool apart = half && 8 * u < rot;
    if constexpr (WIDE) {
        const int first = apart ? 4 * u : 8 * u, second = apart ? first + rot / 2 : first + 4;
        float v[8];
        if constexpr (BF16) {
            const uint16_t *p = (const uint16_t *)x + at;
            const u32x2 w0 = *reinterpret_cast<const u32x2 *>(p + first), w1 = *reinterpret_cast<const u32x2 *>(p + second);
            v[0] = vt_bf16_lo(w0.x); v[1] = vt_bf16_hi(w0.x); v[2] = vt_bf16_lo(w0.y); v[3] = vt_bf16_hi(w0.y);
            v[4] = vt_bf16_lo(w1.x); v[5] = vt_bf16_hi(w1.x); v[6] = vt_bf16_lo(w1.y); v[7] = vt_bf16_hi(w1.y);
        } else {
            const float *p = (const float *)x + at;
            const f32x4 w0 = *reinterpret_cast<const f32x4 *>(p + first), w1 = *reinterpret_cast<const f32x4 *>(p + second);
#pragma unroll
            for (int i = 0; i < 4; i++) { v[i] = w0[i]; v[4 + i] = w1[i]; }
        }
#pragma unroll
        for (int e = 0; e < 4; e++) {
            a[e] = apart ? v[e] : v[2 * e];
            b[e] = apart ? v[4 + e] : v[2 * e + 1];
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int p = 4 * u + e;
            const bool far = half && 2 * p < rot, there = 2 * p < hd;
            const int i = !there ? 0 : far ? p : 2 * p, j = !there ? 0 : far ? p + rot / 2 : 2 * p + 1;
            const float vi = BF16 ? __uint_as_float((unsigned)((const uint16_t *)x)[at + i] << 16) : ((const float *)x)[at + i];
            const float vj = BF16 ? __uint_as_float((unsigned)((const uint16_t *)x)[at + j] << 16) : ((const float *)x)[at + j];
            a[e] = there ? vi : 0.f;
            b[e] = there ? vj : 0.f;
        }
    }
}

static __device__ __forceinline__ unsigned turn_pack(float a, float b) {
    return __builtin_bit_cast(unsigned, __builtin_convertvector((f32x2{a, b}), vt_bf16x2));
}

template <bool BF16, bool WIDE>
static __device__ __forceinline__ void turn_store(void *out, long long at, int hd, int u, int rot, int half, const float a[4], const float b[4]) {
    const bool apart = half && 8 * u < rot;
    if constexpr (WIDE) {
        const int first = apart ? 4 * u : 8 * u, second = apart ? first + rot / 2 : first + 4;
        float v[8];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            v[e] = apart ? a[e] : e & 1 ? b[e >> 1] : a[e >> 1];
            v[4 + e] = apart ? b[e] : e & 1 ? b[2 + (e >> 1)] : a[2 + (e >> 1)];
        }
        if constexpr (BF16) {
            uint16_t *p = (uint16_t *)out + at;
            *reinterpret_cast<u32x2 *>(p + first) = u32x2{turn_pack(v[0], v[1]), turn_pack(v[2], v[3])};
            *reinterpret_cast<u32x2 *>(p + second) = u32x2{turn_pack(v[4], v[5]), turn_pack(v[6], v[7])};
        } else {
            float *p = (float *)out + at;
            *reinterpret_cast<f32x4 *>(p + first) = f32x4{v[0], v[1], v[2], v[3]};
            *reinterpret_cast<f32x4 *>(p + second) = f32x4{v[4], v[5], v[6], v[7]};
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int p = 4 * u + e;
            if (2 * p >= hd) break;
            const bool far = half && 2 * p < rot;
            const int i = far ? p : 2 * p, j = far ? p + rot / 2 : 2 * p + 1;
            if constexpr (BF16) {
                const unsigned w = turn_pack(a[e], b[e]);
                ((uint16_t *)out)[at + i] = (uint16_t)w;
                ((uint16_t *)out)[at + j] = (uint16_t)(w >> 16);
            } else {
                ((float *)out)[at + i] = a[e];
                ((float *)out)[at + j] = b[e];
            }
        }
    }
}

/* sum over 2^log lanes that lie together, the same in each of them */
static __device__ __forceinline__ float turn_sum(float v, int log) {
    if (log > 0) v += vt_dpp<0xB1>(v);
    if (log > 1) v += vt_dpp<0x4E>(v);
    if (log > 2) v += vt_dpp<0x141>(v);
    if (log > 3) v += vt_dpp<0x140>(v);
    if (log > 4) { const f32x2 r = vt_swap16(v, v); v = r.x + r.y; }
    if (log > 5) { const f32x2 r = vt_swap32(v, v); v = r.x + r.y; }
    return v;
}

/* PAGES: blockIdx.y 0 turns K into its pages, 1 takes V into its own as it is */
template <bool BF16, bool WIDE, bool PAGES, int HEADS>
__global__ void __launch_bounds__(256) vt_turn_kernel(turn_job a) {
    constexpr bool OUT16 = BF16 || PAGES;
    const int i = (int)(blockIdx.x * 256 + threadIdx.x), G = 1 << a.lanes_log, at = i >> a.lanes_log, u = i & (G - 1);
    if (at >= a.n) return;                               /* whole groups of lanes */
    const bool values = PAGES && blockIdx.y;
    const int row = vt_div(at, a.sets), h0 = (at - row * a.sets.d) * HEADS, rot = values ? 0 : a.rot_half >> 1, half = a.rot_half & 1;
    const bool mine = 8 * u < a.hd;
    const void *x = values ? a.x2 : a.x;
    float p[HEADS][4], q[HEADS][4];
#pragma unroll
    for (int k = 0; k < HEADS; k++) {
        const int h = min(h0 + k, a.heads - 1);
        turn_load<BF16, WIDE>(x, (long long)row * a.x_stride + h * a.hd, a.hd, mine ? u : 0, rot, half, p[k], q[k]);
    }
    float c[4], s[4];
    const bool turns = 8 * u < rot;
    if (turns) {
        const double pos = (double)a.pos[row];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const double f = a.turns[min(4 * u + e, rot / 2 - 1)], t = pos * f, left = t - rint(t) + fma(pos, f, -t);
            const float near = (float)left, more = (float)(left - (double)near) * 6.28318531f;
            float sn, cs;
            sincospif(2.f * near, &sn, &cs);
            c[e] = fmaf(-sn, more, cs) * a.magnitude;
            s[e] = fmaf(cs, more, sn) * a.magnitude;
        }
    }
    float g[4], gb[4];
    const bool norm = a.gain && !values;
    if (norm) {
        turn_load<false, WIDE>(a.gain, 0, a.hd, mine ? u : 0, rot, half, g, gb);
    }
    long long to = 0;
    if constexpr (PAGES) {
        const int page = a.place[2 * row], r = a.place[2 * row + 1];
        to = ((long long)page * a.heads * a.out_stride + r) * a.hd;              /* out_stride: a page's rows */
    }
#pragma unroll
    for (int k = 0; k < HEADS; k++) {
        if (norm) {
            float sum = 0.f;
            if (mine) {
#pragma unroll
                for (int e = 0; e < 4; e++) sum = fmaf(q[k][e], q[k][e], fmaf(p[k][e], p[k][e], sum));
            }
            sum = turn_sum(sum, a.lanes_log);
            const float f = rsqrtf(fmaf(sum, a.inv_hd, a.eps));
#pragma unroll
            for (int e = 0; e < 4; e++) { p[k][e] = p[k][e] * f * g[e]; q[k][e] = q[k][e] * f * gb[e]; }
        }
        if (turns) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float v = p[k][e], w = q[k][e];
                const bool turn = 8 * u + 2 * e < rot;           /* what does not is passed on as it is */
                p[k][e] = turn ? fmaf(v, c[e], -(w * s[e])) : v;
                q[k][e] = turn ? fmaf(v, s[e], w * c[e]) : w;
            }
        }
        const int h = h0 + k;
        if (mine && h < a.heads)
            turn_store<OUT16, WIDE>(values ? a.out2 : a.out, PAGES ? to + (long long)h * a.out_stride * a.hd : (long long)row * a.out_stride + h * a.hd, a.hd, u,
                                    rot, half, p[k], q[k]);
    }
}

static int turn_ok(const char *who, const tts_hip_rotary_t *how, int head_dim) {
    if (how->rot_dim < 0 || how->rot_dim > head_dim || how->rot_dim % 2 || (how->half != 0 && how->half != 1)) {
        vt_set_error("%s: %d of %d values turn, half %d", who, how->rot_dim, head_dim, how->half);
        return 0;
    }
    if (how->rot_dim && (!how->d_turns || ((uintptr_t)how->d_turns & 7) || !isfinite(how->magnitude))) {
        vt_set_error("%s: no turns, or a magnitude that is no number", who);
        return 0;
    }
    if (how->d_gain && (((uintptr_t)how->d_gain & 3) || !(how->eps >= 0) || isinf(how->eps))) {
        vt_set_error("%s: gains of a norm, eps %g", who, how->eps);
        return 0;
    }
    return 1;
}

/* Heads that a lane walks: two from where every CU has 16 waves of units on (us at one / two / four of them: 1531 rows of 32 heads of 128 bf16 values,
 * normed, 8.8 / 7.5 / 7.6, into pages 1531 rows of 8 fp32 ones 5.1 / 5.4 / 5.9 and 4000 bf16 ones 8.7 / 7.8 / 7.9). */
template <bool PAGES>
static void turn_launch(turn_job &a, int rows, int bf16, int aligned) {
    int log = 0;
    while (8 << log < a.hd) log++;
    a.lanes_log = log;
    const int rot = a.rot_half >> 1, half = a.rot_half & 1;
    const bool wide = aligned && a.hd % 8 == 0 && (!half || rot % 8 == 0);
    const int n_cu = g_vt.n_cu > 0 ? g_vt.n_cu : 256;
    const bool two = a.heads >= 2 && (((long long)rows * a.heads) << log) > 1024ll * n_cu;
    const int each = two ? 2 : 1, sets = (a.heads + each - 1) / each, most = (int)((0x7fffffffll >> log) / sets);
    const int all = rows;
    const turn_job whole = a;
    for (int at = 0; at < all; at += most) {             /* rows of a launch: their lanes are counted in 31 bits */
        const int n = all - at < most ? all - at : most;
        const size_t in = (size_t)at * whole.x_stride * (bf16 ? 2 : 4), out = PAGES ? 0 : (size_t)at * whole.out_stride * (bf16 ? 2 : 4);
        a.x = (const char *)whole.x + in;
        if (PAGES) a.x2 = (const char *)whole.x2 + in;
        a.out = (char *)whole.out + out;
        a.pos = whole.pos ? whole.pos + at : NULL;
        a.place = PAGES ? whole.place + 2 * (size_t)at : NULL;
        a.n = n * sets;
        a.sets = vt_divisor_of(sets, (long long)n * sets);
        const dim3 grid((unsigned)((((long long)a.n << log) + 255) / 256), PAGES ? 2 : 1);
#define TURN(B, W, H) hipLaunchKernelGGL((vt_turn_kernel<B, W, PAGES, H>), grid, dim3(256), 0, g_vt.stream, a)
        if (bf16) { if (wide) { if (two) TURN(true, true, 2); else TURN(true, true, 1); } else { if (two) TURN(true, false, 2); else TURN(true, false, 1); } }
        else { if (wide) { if (two) TURN(false, true, 2); else TURN(false, true, 1); } else { if (two) TURN(false, false, 2); else TURN(false, false, 1); } }
#undef TURN
    }
}

extern "C" int tts_hip_rotary(void *d_out, const void *d_x, int x_bf16, int rows, int n_heads, int head_dim, int out_stride, int x_stride, const int *d_positions,
                              const tts_hip_rotary_t *how) {
    static const char who[] = "tts_hip_rotary";
    const int size = x_bf16 ? 2 : 4;
    if (!how || !d_out || !d_x || (((uintptr_t)d_out | (uintptr_t)d_x) & (size - 1))) {
        vt_set_error("%s: a NULL pointer, or values that do not lie on %d bytes", who, size);
        return -1;
    }
    if (head_dim < 2 || head_dim > 512 || head_dim % 2 || n_heads < 1 || rows < 0 || rows > 1 << 30 || (long long)n_heads * head_dim > 1 << 29) {
        vt_set_error("%s: %d rows of %d heads of %d values (2 .. 512, even)", who, rows, n_heads, head_dim);
        return -1;
    }
    const int width = n_heads * head_dim;
    if (x_stride == 0) x_stride = width;
    if (out_stride == 0) out_stride = width;
    if (x_stride < width || out_stride < width) { vt_set_error("%s: rows of %d values %d and %d apart", who, width, x_stride, out_stride); return -1; }
    if (!turn_ok(who, how, head_dim)) return -1;
    if (how->rot_dim && (!d_positions || ((uintptr_t)d_positions & 3))) { vt_set_error("%s: no positions", who); return -1; }
    if (!vt_mx4_ready(who)) return -1;
    if (rows == 0) return 0;
    turn_job a = {d_x, NULL, d_out, NULL, d_positions, NULL, how->d_turns, how->d_gain, how->magnitude, how->eps, 1.f / head_dim, 0, n_heads, head_dim, x_stride,
                  out_stride, 2 * how->rot_dim + how->half, 0, {0, 1}};
    const int aligned = ((((uintptr_t)d_out | (uintptr_t)d_x) & (4 * size - 1)) | (x_stride & 3) | (out_stride & 3) | ((uintptr_t)how->d_gain & 15)) == 0;
    turn_launch<false>(a, rows, x_bf16, aligned);
    return vt_check(hipGetLastError(), who) ? -1 : 0;
}

extern "C" int tts_hip_paged_append(const tts_hip_paged_t *b, void *d_k_pages, void *d_v_pages, const void *d_K, const void *d_V, int x_bf16, int stride,
                                    const tts_hip_rotary_t *how) {
    static const char who[] = "tts_hip_paged_append";
    const int size = x_bf16 ? 2 : 4;
    if (!b) { vt_set_error("%s: no batch", who); return -1; }
    if (!d_k_pages || !d_v_pages || !d_K || !d_V || (((uintptr_t)d_k_pages | (uintptr_t)d_v_pages) & 15) || (((uintptr_t)d_K | (uintptr_t)d_V) & (size - 1))) {
        vt_set_error("%s: a NULL pointer, pages that do not lie on 16 bytes, or rows that do not lie on %d", who, size);
        return -1;
    }
    const int width = b->shape.n_kv_heads * b->shape.head_dim;
    if (stride == 0) stride = width;
    if (stride < width) { vt_set_error("%s: rows of %d values %d apart", who, width, stride); return -1; }
    if (how && !turn_ok(who, how, b->shape.head_dim)) return -1;
    if (!vt_paged_ready(who, b)) return -1;
    if (b->n_rows == 0) return 0;
    turn_job a = {d_K, d_V, d_k_pages, d_v_pages, (const int *)b->dev, (const int *)(b->dev + b->at_place), how ? how->d_turns : NULL, how ? how->d_gain : NULL,
                  how ? how->magnitude : 1.f, how ? how->eps : 0.f, 1.f / b->shape.head_dim, 0, b->shape.n_kv_heads, b->shape.head_dim, stride, b->shape.page_rows,
                  how ? 2 * how->rot_dim + how->half : 0, 0, {0, 1}};
    const int aligned = ((((uintptr_t)d_K | (uintptr_t)d_V) & (4 * size - 1)) | (stride & 3) | (how ? (uintptr_t)how->d_gain & 15 : 0)) == 0;
    turn_launch<true>(a, b->n_rows, x_bf16, aligned);
    return vt_check(hipGetLastError(), who) ? -1 : 0;
}
