/*
 * vt_mx4.hip - matrices of microscaled 4-bit floats (vt_mx4.h): quantisation of fp32 and bf16 rows, the way back, and the
 * linear layer whose weights are held that way.  A matrix [rows, cols] is codes [rows, 64 P] and scales [rows, 4 P] with P =
 * cols / 128 rounded up: panels of 128 columns, 64 bytes of codes and a dword of four scales each, zeros behind the last column.
 */
#include "vt_state.h"
#include "vt_gemm.h"
#include "vt_mx4.h"
#include "vt_mx4_plans.h"
#include "vt_requests.h"

#include <math.h>

int vt_mx4_ready(const char *who) {
    if (!g_vt.initialized) { vt_set_error("%s: backend not initialised", who); return 0; }
    int dev = -1;
    if (vt_check(hipGetDevice(&dev), "hipGetDevice")) return 0;
    if (dev == g_vt.device) return 1;
    vt_set_error("%s: current device %d is not the device of the context (%d)", who, dev, g_vt.device);
    return 0;
}

/* ---- quantisation and the way back -------------------------------------------------------------------------------
 * A lane takes a unit of a row, eight consecutive values (a quad of lanes a block) on the way in, four on the way back.  Bound by
 * memory: 9216 x 3072 from bf16 12.3 us, 5.8 TB/s in and out, from fp32 23.3, 5.5 (two, four or eight rows a lane: 12.6 to 26). */
struct mx4_shape { int rows, cols, stride, units, wide_log; vt_divisor chunks; int whole; };

static __device__ __forceinline__ bool mx4_place(const mx4_shape &s, int &row, int &unit) {
    const int wg = (int)blockIdx.x, rb = vt_div(wg, s.chunks), cc = wg - rb * s.chunks.d;
    row = (rb << (8 - s.wide_log)) + ((int)threadIdx.x >> s.wide_log);
    unit = (cc << s.wide_log) + ((int)threadIdx.x & ((1 << s.wide_log) - 1));
    return row < s.rows && unit < s.units;
}

template <class T>
__global__ void __launch_bounds__(256) vt_mx4_quantize_kernel(unsigned *codes, uint8_t *scales, const T *x, mx4_shape s) {
    int row, unit;
    if (!mx4_place(s, row, unit)) return;                /* whole quads: a row has a multiple of 16 units */
    const int left = s.cols - 8 * unit;
    f32x4 a, b;
    vt_mx4_load8(x + (size_t)row * s.stride + 8 * (size_t)unit, left, s.whole && left >= 8, a, b);
    unsigned scale;
    const unsigned c = vt_mx4_encode8(a, b, scale);
    codes[(size_t)row * s.units + unit] = c;
    if ((unit & 3) == 0) scales[((size_t)row * s.units + unit) >> 2] = (uint8_t)scale;
}

/* The way back: four values a lane, so that a wave's store is one piece of memory, past the caches, which do not hold what is bigger
 * than they are anyway: 9216 x 3072 19.0 us (6.8 TB/s), through them 28, and 29.5 with eight values and two stores a lane. */
__global__ void __launch_bounds__(256) vt_mx4_dequantize_kernel(float *x, const uint16_t *codes, const uint8_t *scales, mx4_shape s) {
    int row, unit;
    if (!mx4_place(s, row, unit)) return;
    const int left = s.cols - 4 * unit;
    if (left <= 0) return;
    const size_t at = (size_t)row * s.units + unit;
    const f32x4 v = vt_mx4_decode4(codes[at], scales[at >> 3]);
    vt_mx4_store4(x + (size_t)row * s.stride + 4 * (size_t)unit, left, s.whole && left >= 4, v);
}

/* The launch for as many of `rows` as it has threads for; -> its workgroups */
static int mx4_grid(mx4_shape *s, const void *x, int item, int rows, int cols, int stride, int values) {
    const vt_mx4_lanes l = vt_mx4_lanes_of(rows, cols, values);
    *s = mx4_shape{l.rows, cols, stride, l.units, l.wide_log, vt_divisor_of(l.chunks, l.grid), ((uintptr_t)x & 15) == 0 && (size_t)stride * item % 16 == 0};
    return l.grid;
}

static int mx4_shape_ok(const char *who, const void *x, const uint8_t *codes, const uint8_t *scales, int rows, int cols, int stride, int item) {
    if (!x || !codes || !scales) { vt_set_error("%s: NULL pointer", who); return 0; }
    if (rows < 1 || rows > 1 << 30 || cols < 1 || cols > 1 << 27 || stride < cols) {
        vt_set_error("%s: %d rows (1 .. 2^30) of %d columns (1 .. 2^27) %d apart", who, rows, cols, stride);
        return 0;
    }
    if (((uintptr_t)codes & 15) || ((uintptr_t)scales & 3) || (uintptr_t)x % item) {
        vt_set_error("%s: codes lie on 16 bytes, scales on 4, values on their own size", who);
        return 0;
    }
    return 1;
}

extern "C" int tts_hip_mx4_quantize(uint8_t *d_codes, uint8_t *d_scales, const void *d_x, int x_bf16, int rows, int cols, int x_stride) {
    static const char who[] = "tts_hip_mx4_quantize";
    if (x_stride == 0) x_stride = cols;
    if (!mx4_shape_ok(who, d_x, d_codes, d_scales, rows, cols, x_stride, x_bf16 ? 2 : 4) || !vt_mx4_ready(who)) return -1;
    const size_t row = (size_t)vt_mx4_panels(cols) * 64, item = x_bf16 ? 2 : 4;
    mx4_shape s;
    for (int r = 0; r < rows; r += s.rows) {
        const char *x = (const char *)d_x + (size_t)r * x_stride * item;
        unsigned *codes = (unsigned *)(d_codes + r * row);
        uint8_t *scales = d_scales + r * (row / 16);
        const int grid = mx4_grid(&s, x, (int)item, rows - r, cols, x_stride, 8);
        if (x_bf16) hipLaunchKernelGGL(vt_mx4_quantize_kernel<uint16_t>, dim3(grid), dim3(256), 0, g_vt.stream, codes, scales, (const uint16_t *)x, s);
        else hipLaunchKernelGGL(vt_mx4_quantize_kernel<float>, dim3(grid), dim3(256), 0, g_vt.stream, codes, scales, (const float *)x, s);
        if (vt_check(hipGetLastError(), who)) return -1;
    }
    return 0;
}

extern "C" int tts_hip_mx4_dequantize(float *d_x, const uint8_t *d_codes, const uint8_t *d_scales, int rows, int cols, int x_stride) {
    static const char who[] = "tts_hip_mx4_dequantize";
    if (x_stride == 0) x_stride = cols;
    if (!mx4_shape_ok(who, d_x, d_codes, d_scales, rows, cols, x_stride, 4) || !vt_mx4_ready(who)) return -1;
    const size_t row = (size_t)vt_mx4_panels(cols) * 64;
    mx4_shape s;
    for (int r = 0; r < rows; r += s.rows) {
        float *x = d_x + (size_t)r * x_stride;
        const int grid = mx4_grid(&s, x, 4, rows - r, cols, x_stride, 4);
        hipLaunchKernelGGL(vt_mx4_dequantize_kernel, dim3(grid), dim3(256), 0, g_vt.stream, x, (const uint16_t *)(d_codes + r * row), d_scales + r * (row / 16), s);
        if (vt_check(hipGetLastError(), who)) return -1;
    }
    return 0;
}

/* ---- linear layer: up to eight rows --------------------------------------------------------------------------------
 * y^T[weight row][column] on v_mfma_scale_f32_16x16x128_f8f6f4: 16 weight rows go in as they lie in memory, nothing is decoded, and the five
 * e2m3 planes of x (vt_mx4.h) are columns or instructions: the smallest plane in the first of G instructions, the other four in the
 * columns of the second (up to four rows of x, four columns each) or in those of two more (up to eight rows, two columns each).  Every
 * workgroup splits x (a cut of K of it) itself, while its first weights are on their way.  Its waves share K, or groups of four of
 * them share K and take blocks of 16 weight rows in turn where there are several blocks; a wave's weights come in parts of 16 rows x
 * 2 panels (lines of 128 bytes) straight into LDS of its own, three parts (five rows and more: two) ahead of the one that is
 * multiplied, and it waits for nothing but its own loads; the waves' sums of 16 rows meet in LDS behind a bare barrier.  A panel's
 * products start from zero and are added to the sum by the vector unit, which rounds; the matrix unit cuts at 2^-23.  x's planes have
 * to fit LDS: where they do not, K is cut, the cuts' sums go to memory and the last workgroup of a block of rows to arrive adds them.
 * Bound: one row by 131072 x 3072 39.0 us, the stream of the weights at 5.5 TB/s; by 9216 x 3072 8.0 us, launch and first touch; eight
 * rows 45 and 12.7 (78 and 14.3 with a ring of four parts, which leaves no room for the planes of 3072 columns). */
#define MXR_ROWS 8
#define MXR_WAVES 8
#define MXR_PLANES 5                       /* the last one's scale follows from the fourth's */
#define MXR_PART (16 * 128 + 256)          /* codes, then 16 x 2 words of scales and as much room */

struct mxr_job {
    float *y;
    const float *x;
    const uint8_t *codes, *scales;
    int seq_len, in_dim, out_dim, panels, cut_panels, cuts, rows_per_wg, share_log, whole;       /* 1 << share_log waves share K */
    float *part;
    unsigned *cnt;
};

/* columns of a block: the planes of all rows, and one of zeros; an odd number, so that consecutive blocks lie in different banks */
static __host__ __device__ constexpr int mxr_columns(int seq_len) { return (MXR_PLANES * seq_len + 1) | 1; }
/* parts of a wave's ring: the planes of five and more rows need the room of the fourth */
static constexpr int mxr_ring(int g) { return g > 2 ? 3 : 4; }

template <int G>
__global__ void __launch_bounds__(64 * MXR_WAVES) vt_mx4_rows_kernel(mxr_job a) {
    constexpr int THREADS = 64 * MXR_WAVES, PP = 4 / (G - 1);         /* planes of an instruction but the first */
    constexpr int RING = mxr_ring(G);
    constexpr int BUF = MXR_WAVES * MXR_PART;
    __shared__ __attribute__((aligned(16))) unsigned char buf0[BUF], buf1[BUF], buf2[BUF], buf3[RING > 3 ? BUF : 16];
    __shared__ float red[2][MXR_WAVES][64 * (G - 1)];          /* [row of x][weight row] */
    __shared__ int last;
    extern __shared__ __attribute__((aligned(16))) unsigned char planes[];
    const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
    const int row0 = (int)blockIdx.x * a.rows_per_wg, rows = min(a.rows_per_wg, a.out_dim - row0);
    /* waves that share K, and the blocks that are under way at once */
    const int share = 1 << a.share_log, groups = MXR_WAVES >> a.share_log, group = wave >> a.share_log;
    const int k0 = (int)blockIdx.y * a.cut_panels, k1 = min(k0 + a.cut_panels, a.panels), per_wave = (a.cut_panels + share - 1) >> a.share_log;
    const int p0 = min(k0 + (wave & (share - 1)) * per_wave, k1), p1 = min(p0 + per_wave, k1), parts = (per_wave + 1) / 2, blocks = (rows + 15) / 16;
    const int total = (blocks + groups - 1) / groups * parts;
    /* x: block u % nb of row u / nb of the cut.  [panel][group of lanes][instruction][column] of 16 and of 8 bytes, and the scales; column PP row +
     * plane.  The first blocks are asked for in front of the weights, the next ones while these are split: loads return in order. */
    const int nb = 4 * (k1 - k0), nc = mxr_columns(a.seq_len), units = a.seq_len * nb;
    unsigned char *lo8 = planes + nb * nc * 16, *sc = lo8 + nb * nc * 8;
    const __amdgpu_buffer_rsrc_t xd = vt_buffer(a.x, a.seq_len * a.in_dim * 4);
    int xr = (int)threadIdx.x / nb, xb = (int)threadIdx.x - xr * nb;
    const int xr_step = THREADS / nb, xb_step = THREADS - xr_step * nb;
    vt_f32x16 even, odd, next_even, next_odd;
    auto ask_x = [&](vt_f32x16 &e, vt_f32x16 &o) __attribute__((always_inline)) {
        vt_mx4_load32(xd, xr * a.in_dim * 4, xr < a.seq_len ? 128 * k0 + 32 * xb : a.in_dim, a.in_dim, a.whole, e, o);
    };
    ask_x(even, odd);
    /* codes: lane i brings piece i % 8 of a line, exchanged so that eight rows' same piece lie in different banks; scales: word i % 2 of row i / 2 */
    const int w_at = (lane >> 3) * 64 * a.panels + ((lane & 7) ^ (lane >> 3)) * 16;                /* and 8 rows on: the same exchange */
    const int s_at = lane < 32 ? (lane >> 1) * 4 * a.panels + (lane & 1) * 4 : 0x7ffffff0;
    int ask_block = group, ask_part = 0;                      /* where the next request is: no division */
    auto ask = [&](unsigned char *buf) __attribute__((always_inline)) {
        const bool live = ask_block < blocks && p0 + 2 * ask_part < p1;         /* else zeros, which nobody reads */
        const int left = live ? min(16, rows - 16 * ask_block) : 0, panel = live ? p0 + 2 * ask_part : 0;
        const size_t r = (size_t)row0 + (live ? 16 * ask_block : 0);
        /* from the panel on, with no scalar offset: the range check need not know of one.  (Past the last of an odd number of panels the
         * last row's lanes read zeros, others the next row.) */
        const size_t first = r * a.panels + panel;
        const int size = max(left * a.panels - panel, 0);
        const __amdgpu_buffer_rsrc_t wd = vt_buffer(a.codes + first * 64, size * 64), sd = vt_buffer(a.scales + first * 4, size * 4);
        unsigned char *b = buf + wave * MXR_PART;
#pragma unroll
        for (int d = 0; d < 2; d++)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(wd, (__attribute__((address_space(3))) void *)(b + d * 1024), 16, w_at + d * 8 * 64 * a.panels, 0, 0, 2);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(sd, (__attribute__((address_space(3))) void *)(b + 2048), 4, s_at, 0, 0, 2);
        if (++ask_part >= parts) { ask_part = 0; ask_block += groups; }
    };
    ask(buf0);
    ask(buf1);
    if (RING > 3) ask(buf2);
    for (int u = THREADS;; u += THREADS) {
        const int row = xr, xb_at = xb * nc, at0 = xb_at + a.seq_len + row * PP;
        xr += xr_step;
        xb += xb_step;
        if (xb >= nb) { xb -= nb; xr++; }
        if (u < units) ask_x(next_even, next_odd);
        vt_u32x6 q[MXR_PLANES];
        unsigned s[MXR_PLANES];
        vt_mx4_planes<MXR_PLANES, true>(even, odd, q, s);
        if (row < a.seq_len) {
#pragma unroll
            for (int p = 0; p < MXR_PLANES; p++) {
                const int at = p == MXR_PLANES - 1 ? xb_at + row : at0 + (G - 2 - p / PP) * PP * a.seq_len + p % PP;
                *reinterpret_cast<u32x4 *>(planes + at * 16) = u32x4{q[p][0], q[p][1], q[p][2], q[p][3]};
                *reinterpret_cast<u32x2 *>(lo8 + at * 8) = u32x2{q[p][4], q[p][5]};
                sc[at] = (unsigned char)s[p];
            }
        }
        if (row == 0) {                                  /* the column of zeros */
            const int at = xb_at + nc - 1;
            *reinterpret_cast<u32x4 *>(planes + at * 16) = u32x4{0u, 0u, 0u, 0u};
            *reinterpret_cast<u32x2 *>(lo8 + at * 8) = u32x2{0u, 0u};
            sc[at] = 0;
        }
        if (u >= units) break;
        even = next_even;
        odd = next_odd;
    }
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xc07f);                  /* lgkmcnt(0); weights stay on their way */
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    const int col = min(n, PP * a.seq_len - 1), mine = g * nc + a.seq_len + col;        /* columns past the last repeat it: nobody looks at their sums */
    const int smallest = g * nc + (n % PP == 0 ? col / PP : nc - 1);       /* the smallest plane is in one of a row's columns */
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    float *y = a.cuts > 1 ? a.part + (size_t)blockIdx.y * a.seq_len * a.out_dim : a.y;
    /* the waves' sums: element v of lane l is weight row 4 (l / 16) + v, column l % 16; a row's planes of an instruction are PP lanes */
    auto finish = [&](int turn) __attribute__((always_inline)) {
        f32x4 sum = acc;
#pragma unroll
        for (int v = 0; v < 4; v++) {
            if (PP > 1) sum[v] += vt_dpp<0xB1>(sum[v]);
            if (PP > 2) sum[v] += vt_dpp<0x4E>(sum[v]);
        }
        if (n % PP == 0) *reinterpret_cast<f32x4 *>(&red[turn & 1][wave][n / PP * 16 + 4 * g]) = sum;
        acc = f32x4{0.f, 0.f, 0.f, 0.f};
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0xc07f);
        __builtin_amdgcn_s_barrier();                    /* the other half of red is read before a wave is through the next one */
        asm volatile("" ::: "memory");
        /* the first 64 (G - 1) threads of a group of waves: row of x, weight row */
        const int t = (int)threadIdx.x & (64 * share - 1), s = t >> 4, r = 16 * (turn * groups + group) + (t & 15);
        if (s < a.seq_len && r < rows) {
            const float *from = &red[turn & 1][group << a.share_log][t];
            float p[4];
#pragma unroll
            for (int w = 0; w < 4; w++) p[w] = from[w * 64 * (G - 1)];
            float v = (p[0] + p[2]) + (p[1] + p[3]);
            if (share > 4) {
#pragma unroll
                for (int w = 0; w < 4; w++) p[w] = from[(4 + w) * 64 * (G - 1)];
                v += (p[0] + p[2]) + (p[1] + p[3]);
            }
            float *at = y + (size_t)s * a.out_dim + row0 + r;
            if (a.cuts > 1) vt_stc(at, v);
            else *at = v;
        }
    };
    int turn = 0, part = 0;
    auto item = [&](const unsigned char *here, unsigned char *later) __attribute__((always_inline)) {
        asm volatile("" ::: "memory");
        /* vmcnt: two later parts, or one, may be on their way; lgkmcnt(0): what is asked for below overwrites what the last part read */
        __builtin_amdgcn_s_waitcnt(0x0070 | 3 * (RING - 2));
        asm volatile("" ::: "memory");
        ask(later);
        asm volatile("" ::: "memory");
        const unsigned char *b = here + wave * MXR_PART;
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const int panel = p0 + 2 * part + k;
            if (panel >= p1) break;
            const u32x4 w = *reinterpret_cast<const u32x4 *>(b + n * 128 + ((4 * k + g) ^ (n & 7)) * 16);
            const int ws = b[2048 + n * 8 + 4 * k + g];
            f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < G; i++) {
                const int at = (panel - k0) * 4 * nc + (i ? (i - 1) * PP * a.seq_len + mine : smallest);
                const u32x4 x4 = *reinterpret_cast<const u32x4 *>(planes + at * 16);
                const u32x2 x2 = *reinterpret_cast<const u32x2 *>(lo8 + at * 8);
                const vt_u32x6 xq = {x4.x, x4.y, x4.z, x4.w, x2.x, x2.y};
                sum = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(vt_mfma_e2m1(w), vt_mfma_e2m3(xq), sum, VT_MFMA_E2M1, VT_MFMA_E2M3, 0, ws, 0, (int)sc[at]);
            }
            acc = acc + sum;
        }
        if (++part == parts) { part = 0; finish(turn++); }
    };
    for (int t = 0; t < total; t += RING) {                 /* every wave goes through the same parts and barriers, whatever it has of them */
        item(buf0, RING > 3 ? buf3 : buf2);
        if (t + 1 >= total) break;
        item(buf1, buf0);
        if (t + 2 >= total) break;
        item(buf2, buf1);
        if (RING == 3) continue;
        if (t + 3 >= total) break;
        item(buf3, buf2);
    }
    __builtin_amdgcn_s_waitcnt(0x0f70);                  /* nothing arrives in the buffers any more, and what was stored is acknowledged */
    if (a.cuts == 1) return;
    __syncthreads();
    if (threadIdx.x == 0) last = __hip_atomic_fetch_add(a.cnt + blockIdx.x, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)(a.cuts - 1);
    __syncthreads();
    if (!last) return;
    if (threadIdx.x == 0) vt_stc_u32(a.cnt + blockIdx.x, 0u);    /* ready for the next launch */
    for (int s = 0; s < a.seq_len; s++)
        for (int r = (int)threadIdx.x; r < rows; r += THREADS) {
            const size_t at = (size_t)s * a.out_dim + row0 + r;
            float v = 0.f;
            for (int c = 0; c < a.cuts; c += 4) {
                float p[4];
#pragma unroll
                for (int k = 0; k < 4; k++) p[k] = vt_ldc(a.part + (size_t)min(c + k, a.cuts - 1) * a.seq_len * a.out_dim + at);
#pragma unroll
                for (int k = 0; k < 4; k++) v = c + k < a.cuts ? __fadd_rn(v, p[k]) : v;
            }
            a.y[at] = v;
        }
}

/* LDS: the rings and the sums of eight waves, 25 bytes a block of 32 values of x and plane */
#define MXR_LDS_MOST (160 * 1024)
static size_t mxr_lds(int g) { return (size_t)MXR_WAVES * (MXR_PART * mxr_ring(g) + 2 * 64 * (g - 1) * 4) + 256; }
static size_t mxr_planes_bytes(int seq_len, int panels) { return (size_t)4 * panels * mxr_columns(seq_len) * 25; }

/* ---- linear layer: more rows -----------------------------------------------------------------------------------------
 * x is split into its planes first, [column tile of 32 rows][64 columns of W's K][plane] in the order of the matrix instruction's operand, 16
 * and 8 bytes a lane, and the scales of a lane's first four planes in a word (the fifth's follows).  y[row of x][weight row] then runs on
 * v_mfma_scale_f32_32x32x64_f8f6f4, x as operand A, weights as they lie as B.  A workgroup's tile of BM weight rows and BN rows of x goes
 * through K by panels of 128: both operands come straight into LDS, one panel ahead.  A wave has 32 rows of x and FM x 32 weight rows, so
 * that an operand of x, the larger one (3.75 bytes a value), is read once for FM products.  Ten products of a panel, the smallest planes
 * first, start from zero and are added by the vector unit (the matrix unit's sums are cut at 2^-23).  Few tiles: K is cut and the parts
 * are added by a kernel of their own.  Bound: 1531 x 9216 x 3072 119 to 127 us, 10 of them the planes; the product's 108 to 117 are five
 * products of 43 GMAC, which keep the matrix units busy 47 % of the time (in two rounds of which the second is 69 % full), and 190 KB that its
 * eight waves read from LDS per panel, 1500 cycles of the 2600 that the matrix instructions take, with the next panel's 80 KB on their
 * way there.  226 x 3072 x 9216 38 to 40 us: 6 the planes, 6 the sums of 8 cuts, 27 the product, 192 workgroups. */
#define MXT_STEP (MXR_PLANES * 1536 + 256)               /* bytes of 32 rows x 64 columns of x */

/* A wave has 32 rows by 64 columns; they go through LDS so that its loads are lines (a lane's own 128 bytes come in eight pieces, and
 * with twenty waves on a CU the rest of a line is gone from the first cache by the time of the next piece). */
__global__ void __launch_bounds__(256) vt_mx4_planes_kernel(unsigned char *out, const float *x, int seq_len, int in_dim, int panels, int tiles, int whole) {
    constexpr int ROW = 64 + 4;                          /* floats: eight rows' same piece lie in different banks */
    __shared__ __attribute__((aligned(16))) float turn[4][32 * ROW];
    const int wave = (int)(threadIdx.x >> 6), unit = (int)blockIdx.x * 4 + wave, lane = (int)threadIdx.x & 63;
    if (unit >= tiles * 2 * panels) return;
    /* [panel][tile][half] */
    const int panel = unit / (2 * tiles), rest = unit - panel * 2 * tiles, at = 128 * panel + 64 * (rest & 1), row0 = (rest >> 1) * 32;
    const __amdgpu_buffer_rsrc_t xd = vt_buffer(x + (size_t)row0 * in_dim, min(32, seq_len - row0) * in_dim * 4);      /* zeros past the last row */
    if (whole) {
        f32x4 v[8];
        const int c = at + 4 * (lane & 15);
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = vt_buffer_ld4(xd, c < in_dim ? ((4 * i + (lane >> 4)) * in_dim + c) * 4 : 0x7ffffff0);
#pragma unroll
        for (int i = 0; i < 8; i++) *reinterpret_cast<f32x4 *>(&turn[wave][(4 * i + (lane >> 4)) * ROW + 4 * (lane & 15)]) = v[i];
    } else {
#pragma unroll 8
        for (int i = 0; i < 32; i++)
            turn[wave][i * ROW + lane] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(xd, at + lane < in_dim ? (i * in_dim + at + lane) * 4 : 0x7ffffff0, 0, 0));
    }
    __builtin_amdgcn_wave_barrier();                     /* the wave's own LDS, in order */
    vt_f32x16 even, odd;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const f32x4 v = *reinterpret_cast<const f32x4 *>(&turn[wave][(lane & 31) * ROW + 32 * (lane >> 5) + 4 * i]);
        even[2 * i] = v.x; odd[2 * i] = v.y; even[2 * i + 1] = v.z; odd[2 * i + 1] = v.w;
    }
    vt_u32x6 q[MXR_PLANES];
    unsigned s[MXR_PLANES], all = 0;
    vt_mx4_planes<MXR_PLANES, true>(even, odd, q, s);
    unsigned char *to = out + (size_t)unit * MXT_STEP;
#pragma unroll
    for (int p = 0; p < MXR_PLANES; p++) {
        *reinterpret_cast<u32x4 *>(to + p * 1536 + lane * 16) = u32x4{q[p][0], q[p][1], q[p][2], q[p][3]};
        *reinterpret_cast<u32x2 *>(to + p * 1536 + 1024 + lane * 8) = u32x2{q[p][4], q[p][5]};
        if (p < 4) all |= s[p] << (8 * p);
    }
    *reinterpret_cast<unsigned *>(to + MXR_PLANES * 1536 + lane * 4) = all;
}

struct mxt_job { float *y; const unsigned char *planes; const uint8_t *codes, *scales; int seq_len, out_dim, panels, tiles, cuts, m_tiles; };

/* FM 32 weight rows a wave, NM x NN waves.  AHEAD: a workgroup with the CU to itself.  Its barrier stands in front of the products of a
 * panel's first plane, the last of five, whose x is in registers by then: behind it the next panel's operands come from LDS while these
 * are multiplied (else the matrix units wait for them at every panel), half of the panel after that is asked for there and the other
 * half a plane later.  Workgroups that share a CU fill such waits for each other and need the longer time to memory: they ask for a
 * quarter of the next panel behind each of this one's first four planes, with the barrier between panels.  us, with AHEAD and without, as
 * measured with four planes of x: 512 and 1531 x 9216 x 3072 47.5 and 107 (53 and 114), 1000 x 3072 x 4096 and 16 x 131072 x 3072 51 and
 * 80 (48 and 73). */
template <int FM, int NM, int NN, bool AHEAD>
__global__ void __launch_bounds__(64 * NM * NN) vt_mx4_tile_kernel(mxt_job a) {
    constexpr int THREADS = 64 * NM * NN, BM = 32 * FM * NM, W_BYTES = BM * 64, X_AT = W_BYTES + BM * 4, X_BYTES = NN * 2 * MXT_STEP;
    constexpr int SPARE = X_AT + (X_BYTES + 1023) / 1024 * 1024, BUF = SPARE + (AHEAD ? 1024 : 0);       /* a wave's request brings 1 KB */
    __shared__ __attribute__((aligned(16))) unsigned char buf0[BUF], buf1[BUF];         /* two arrays: reading one need not wait for what arrives in the other */
    const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), n = lane & 31, g = lane >> 5, wm = wave % NM, wn = wave / NM;
    const int cut = (int)blockIdx.x % a.cuts, tile = (int)blockIdx.x / a.cuts, mt = tile % a.m_tiles, nt = tile / a.m_tiles;
    const int p0 = (int)((long long)a.panels * cut / a.cuts), p1 = (int)((long long)a.panels * (cut + 1) / a.cuts);
    const size_t row0 = (size_t)mt * BM;
    const int rows = (int)min((long long)BM, a.out_dim - (long long)row0), t0 = nt * NN, xt = min(NN, a.tiles - t0);
    const __amdgpu_buffer_rsrc_t wd = vt_buffer(a.codes + row0 * 64 * a.panels, rows * 64 * a.panels), sd = vt_buffer(a.scales + row0 * 4 * a.panels, rows * 4 * a.panels);
    /* weights: unit u of 16 bytes is row u / 4, piece u % 4, exchanged so that eight rows' same piece lie in different banks */
    constexpr int WU = W_BYTES / 16 / THREADS, XU = (X_BYTES / 16 + THREADS - 1) / THREADS;
    static_assert(W_BYTES / 16 % THREADS == 0, "whole requests");
    int w_at[8];                                         /* WU of them (with that size the host pass drops the kernel) */
    static_assert(WU <= 8, "w_at");
#pragma unroll
    for (int i = 0; i < WU; i++) { const int u = i * THREADS + (int)threadIdx.x, r = u >> 2; w_at[i] = r * 64 * a.panels + ((u & 3) ^ ((r >> 1) & 3)) * 16; }
    const int s_at = (int)threadIdx.x * 4 * a.panels;
    /* part q of `of` of a panel's requests; past the last panel: zeros, which nobody reads */
    auto ask = [&](unsigned char *b, int panel, int q, int of) __attribute__((always_inline)) {
        const __amdgpu_buffer_rsrc_t xd = vt_buffer(a.planes + ((size_t)min(panel, p1 - 1) * a.tiles + t0) * 2 * MXT_STEP, panel < p1 ? xt * 2 * MXT_STEP : 0);
        const int dead = panel < p1 ? 0 : 0x40000000;
#define LDS(at) (__attribute__((address_space(3))) void *)(b + (at))
#pragma unroll
        for (int i = 0; i < WU; i++)
            if (i % of == q) __builtin_amdgcn_raw_ptr_buffer_load_lds(wd, LDS(i * THREADS * 16 + wave * 1024), 16, (w_at[i] + panel * 64) | dead, 0, 0, 0);
        /* a wave without a share of a request: AHEAD sends it all the same, for nothing to a spare place, because products move across a branch */
        const bool has = wave * 64 < BM;
        if (q == of - 1 && (AHEAD || has))
            __builtin_amdgcn_raw_ptr_buffer_load_lds(sd, LDS(has ? W_BYTES + wave * 256 : SPARE), 4, has ? (s_at + panel * 4) | dead : 0x40000000, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < XU; i++) {
            const int at = i * THREADS * 16 + wave * 1024;
            if ((i + of / 2) % of == q && (AHEAD || at < X_BYTES))
                __builtin_amdgcn_raw_ptr_buffer_load_lds(xd, LDS(at < X_BYTES ? X_AT + at : SPARE), 16, (i * THREADS + (int)threadIdx.x) * 16, 0, 0, 0);
        }
#undef LDS
    };
    vt_f32x16 acc[FM];
#pragma unroll
    for (int f = 0; f < FM; f++) acc[f] = vt_f32x16{};
    u32x4 w[FM][2];
    int ws[FM], xs[2];
    vt_u32x6 first[2];                                   /* x's smallest plane */
    const int x_at = wn * 2 * MXT_STEP, x16 = x_at + lane * 16, x8 = x_at + lane * 8, x4_at = x_at + lane * 4;
    const int w_row = wm * FM * 32 + n, w_piece[2] = {w_row * 64 + (g ^ ((n >> 1) & 3)) * 16, w_row * 64 + ((2 + g) ^ ((n >> 1) & 3)) * 16}, ws_at = w_row * 4;
    auto x_of = [&](const unsigned char *b, int p, int h) __attribute__((always_inline)) {
        const u32x4 x4 = *reinterpret_cast<const u32x4 *>(b + x16 + (X_AT + h * MXT_STEP + p * 1536));
        const u32x2 x2 = *reinterpret_cast<const u32x2 *>(b + x8 + (X_AT + h * MXT_STEP + p * 1536 + 1024));
        return vt_u32x6{x4.x, x4.y, x4.z, x4.w, x2.x, x2.y};
    };
    auto fetch_x = [&](const unsigned char *b) __attribute__((always_inline)) {
        first[0] = x_of(b, MXR_PLANES - 1, 0);
        first[1] = x_of(b, MXR_PLANES - 1, 1);
    };
    auto fetch_w = [&](const unsigned char *b, int h) __attribute__((always_inline)) {
        xs[h] = *reinterpret_cast<const int *>(b + x4_at + (X_AT + h * MXT_STEP + MXR_PLANES * 1536));
#pragma unroll
        for (int f = 0; f < FM; f++) {
            w[f][h] = *reinterpret_cast<const u32x4 *>(b + w_piece[h] + f * 2048);
        }
        if (!h) return;
        int at = ws_at;
        asm("" : "+v"(at));                              /* else a register for each sum with a buffer's place */
        /* bytes 0 and 2: the lane's block of either half */
#pragma unroll
        for (int f = 0; f < FM; f++) ws[f] = (int)(*reinterpret_cast<const unsigned *>(b + at + (W_BYTES + f * 128)) >> (8 * g));
    };
    auto meet = [&]() __attribute__((always_inline)) {   /* what was asked for is there, and everybody is through with what the next requests overwrite */
        __builtin_amdgcn_s_waitcnt(0x0070);
        __syncthreads();
    };
    auto step = [&](int panel, unsigned char *here, unsigned char *other) __attribute__((always_inline)) {
        constexpr int PIN = AHEAD ? 0 : 0x387;           /* what may not cross: nothing may, or products and requests may not */
        if (!AHEAD) { meet(); fetch_x(here); fetch_w(here, 0); fetch_w(here, 1); }
        vt_f32x16 sum[FM];
#pragma unroll
        for (int f = 0; f < FM; f++) sum[f] = vt_f32x16{};
        const int last[2] = {vt_mx4_below((unsigned)xs[0] >> 24), vt_mx4_below((unsigned)xs[1] >> 24)};
#define PRODUCTS(x, h, byte, scales) \
        _Pragma("unroll") for (int f = 0; f < FM; f++) \
            sum[f] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(vt_mfma_e2m3(x[h]), vt_mfma_e2m1(w[f][h]), sum[f], VT_MFMA_E2M3, VT_MFMA_E2M1, \
                                                                    byte, scales[h], 2 * h, ws[f]);
#define PINNED(...) __builtin_amdgcn_sched_barrier(PIN); __VA_ARGS__ __builtin_amdgcn_sched_barrier(PIN);
        const vt_u32x6 x3[2] = {x_of(here, 3, 0), x_of(here, 3, 1)};
        PINNED()
        PRODUCTS(first, 0, 0, last) PRODUCTS(first, 1, 0, last)
        PINNED(if (AHEAD) ask(other, panel + 1, 1, 2); else ask(other, panel + 1, 0, 4);)
        const vt_u32x6 x2[2] = {x_of(here, 2, 0), x_of(here, 2, 1)};
        PINNED()
        PRODUCTS(x3, 0, 3, xs) PRODUCTS(x3, 1, 3, xs)
        PINNED(if (!AHEAD) ask(other, panel + 1, 1, 4);)
        const vt_u32x6 x1[2] = {x_of(here, 1, 0), x_of(here, 1, 1)};
        PINNED()
        PRODUCTS(x2, 0, 2, xs) PRODUCTS(x2, 1, 2, xs)
        PINNED(if (!AHEAD) ask(other, panel + 1, 2, 4);)
        const vt_u32x6 x0[2] = {x_of(here, 0, 0), x_of(here, 0, 1)};
        PINNED()
        PRODUCTS(x1, 0, 1, xs) PRODUCTS(x1, 1, 1, xs)
        PINNED(if (AHEAD) { meet(); fetch_x(other); } else ask(other, panel + 1, 3, 4);)
        PINNED(if (AHEAD) ask(here, panel + 2, 0, 2);)
        PRODUCTS(x0, 0, 0, xs)
        PINNED(if (AHEAD) fetch_w(other, 0);)
        PRODUCTS(x0, 1, 0, xs)
        PINNED(if (AHEAD) fetch_w(other, 1);)
#undef PINNED
#undef PRODUCTS
#pragma unroll
        for (int f = 0; f < FM; f++) acc[f] = acc[f] + sum[f];
        __builtin_amdgcn_sched_barrier(PIN);
    };
    /* every cut has a panel */
    if (AHEAD) {
        ask(buf0, p0, 0, 2);
        ask(buf0, p0, 1, 2);
        ask(buf1, p0 + 1, 0, 2);
        meet();
        fetch_x(buf0);
        fetch_w(buf0, 0);
        fetch_w(buf0, 1);
    } else {
#pragma unroll
        for (int q = 0; q < 4; q++) ask(buf0, p0, q, 4);
    }
    for (int panel = p0; panel < p1; panel += 2) {
        step(panel, buf0, buf1);
        if (panel + 1 >= p1) break;
        step(panel + 1, buf1, buf0);
    }
    __builtin_amdgcn_s_waitcnt(0x0f70);                  /* nothing arrives in the buffers any more */
    /* element v of lane l: row 8 (v / 4) + 4 (l / 32) + v % 4 of x, weight row l % 32 */
    float *y = a.y + (size_t)cut * a.seq_len * a.out_dim;
#pragma unroll
    for (int f = 0; f < FM; f++) {
        const int r = (wm * FM + f) * 32 + n;
        if (r >= rows) continue;
#pragma unroll
        for (int v = 0; v < 16; v++) {
            const int s = (t0 + wn) * 32 + 8 * (v >> 2) + 4 * g + (v & 3);
            if (s < a.seq_len) y[(size_t)s * a.out_dim + row0 + r] = acc[f][v];
        }
    }
}

template <int G> static int mxr_prepare(void) {
    return vt_check(hipFuncSetAttribute((const void *)vt_mx4_rows_kernel<G>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)(MXR_LDS_MOST - mxr_lds(G))),
                    "tts_hip_linear_mx4: LDS");
}
int vt_mx4_prepare(void) { return mxr_prepare<2>() || mxr_prepare<3>() ? -1 : 0; }

static int mx4_linear_rows(float *d_y, const float *d_x, const uint8_t *d_codes, const uint8_t *d_scales, int seq_len, int in_dim, int out_dim, int whole) {
    const int n_cu = g_vt.n_cu > 0 ? g_vt.n_cu : 256, panels = vt_mx4_panels(in_dim), g = seq_len <= 4 ? 2 : 3;
    const int most = (int)((MXR_LDS_MOST - mxr_lds(g)) / mxr_planes_bytes(seq_len, 1)), cuts = (panels + most - 1) / most, wgs = n_cu / cuts > 0 ? n_cu / cuts : 1;
    mxr_job a = {d_y, d_x, d_codes, d_scales, seq_len, in_dim, out_dim, panels, (panels + cuts - 1) / cuts, cuts,
                 (int)(((long long)out_dim + wgs - 1) / wgs), 2, whole, NULL, g_vt.d_mx4_cnt};
    if (a.rows_per_wg <= 16) a.share_log = 3;          /* no second block for the other waves */
    a.cuts = (panels + a.cut_panels - 1) / a.cut_panels;
    if (a.cuts > 1 && !(a.part = (float *)vt_scratch(sizeof(float) * (size_t)a.cuts * seq_len * out_dim))) return -1;
    const dim3 grid((out_dim + a.rows_per_wg - 1) / a.rows_per_wg, a.cuts);
    const size_t lds = mxr_planes_bytes(seq_len, a.cut_panels);
    if (g == 2) hipLaunchKernelGGL(vt_mx4_rows_kernel<2>, grid, dim3(64 * MXR_WAVES), lds, g_vt.stream, a);
    else hipLaunchKernelGGL(vt_mx4_rows_kernel<3>, grid, dim3(64 * MXR_WAVES), lds, g_vt.stream, a);
    return 0;
}

static int mx4_linear_tiles(float *d_y, const float *d_x, const uint8_t *d_codes, const uint8_t *d_scales, int seq_len, int in_dim, int out_dim, int whole) {
    const int n_cu = g_vt.n_cu > 0 ? g_vt.n_cu : 256, panels = vt_mx4_panels(in_dim), tiles = (seq_len + 31) / 32;
    const vt_mxt_plan p = vt_mxt_plan_of(n_cu, seq_len, out_dim, panels);
    const size_t planes = (size_t)tiles * 2 * panels * MXT_STEP, part = p.cuts > 1 ? sizeof(float) * (size_t)seq_len * out_dim * p.cuts : 0;
    unsigned char *area = (unsigned char *)vt_scratch(planes + part);
    if (!area) return -1;
    hipLaunchKernelGGL(vt_mx4_planes_kernel, dim3((tiles * 2 * panels + 3) / 4), dim3(256), 0, g_vt.stream, area, d_x, seq_len, in_dim, panels, tiles, whole);
    const mxt_job a = {p.cuts > 1 ? (float *)(area + planes) : d_y, area, d_codes, d_scales, seq_len, out_dim, panels, tiles, p.cuts, p.m_tiles};
    const dim3 grid((unsigned)p.grid), block(vt_mxt_tiles[p.tile].threads);
    if (p.tile == 0) hipLaunchKernelGGL((vt_mx4_tile_kernel<4, 2, 4, true>), grid, block, 0, g_vt.stream, a);
    else if (p.tile == 1) hipLaunchKernelGGL((vt_mx4_tile_kernel<2, 2, 2, false>), grid, block, 0, g_vt.stream, a);
    else hipLaunchKernelGGL((vt_mx4_tile_kernel<1, 4, 1, false>), grid, block, 0, g_vt.stream, a);
    if (p.cuts > 1) vt_launch_sum_planes(d_y, (float *)(area + planes), p.cuts, (size_t)seq_len * out_dim, (size_t)seq_len * out_dim);
    return 0;
}

extern "C" int tts_hip_linear_mx4(float *d_y, const float *d_x, const uint8_t *d_codes, const uint8_t *d_scales, int seq_len, int in_dim, int out_dim) {
    static const char who[] = "tts_hip_linear_mx4";
    if (!d_y || ((uintptr_t)d_y & 3) || seq_len < 1 || seq_len > 1 << 30) { vt_set_error("%s: %d rows (1 .. 2^30) to %p", who, seq_len, (void *)d_y); return -1; }
    if (!mx4_shape_ok(who, d_x, d_codes, d_scales, out_dim, in_dim, in_dim, 4)) return -1;
    if (in_dim > 1 << 23) { vt_set_error("%s: %d columns (1 .. 2^23)", who, in_dim); return -1; }
    if (!vt_mx4_ready(who)) return -1;
    const int whole = ((uintptr_t)d_x & 15) == 0 && in_dim % 4 == 0;
    if (seq_len <= MXR_ROWS) {
        if (mx4_linear_rows(d_y, d_x, d_codes, d_scales, seq_len, in_dim, out_dim, whole)) return -1;
    } else {
        const int most = vt_mxt_rows(out_dim, vt_mx4_panels(in_dim));
        for (int s = 0; s < seq_len; s += most) {
            const int n = seq_len - s < most ? seq_len - s : most;
            if (mx4_linear_tiles(d_y + (size_t)s * out_dim, d_x + (size_t)s * in_dim, d_codes, d_scales, n, in_dim, out_dim, whole)) return -1;
        }
    }
    return vt_check(hipGetLastError(), who) ? -1 : 0;
}
