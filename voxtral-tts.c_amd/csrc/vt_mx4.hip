/*
 * vt_mx4.hip - matrices of microscaled 4-bit floats (vt_mx4.h): quantisation of fp32 and bf16 rows, the way back, and the
 * linear layer whose weights are held that way.  A matrix [rows, cols] is codes [rows, 64 P] and scales [rows, 4 P] with P =
 * cols / 128 rounded up: panels of 128 columns, 64 bytes of codes and a dword of four scales each, zeros behind the last column.
 */
#include "vt_state.h"
#include "vt_mx4.h"
#include "vt_requests.h"

static int panels_of(int cols) { return cols / 128 + (cols % 128 != 0); }

int vt_mx4_ready(const char *who) {
    if (!g_vt.initialized) { vt_set_error("%s: backend not initialised", who); return 0; }
    int dev = -1;
    if (vt_check(hipGetDevice(&dev), "hipGetDevice")) return 0;
    if (dev == g_vt.device) return 1;
    vt_set_error("%s: current device %d is not the device of the context (%d)", who, dev, g_vt.device);
    return 0;
}

/* ---- quantisation and the way back -------------------------------------------------------------------------------
 * A lane takes eight consecutive values (a quad of lanes a block), 2^wide_log lanes lie along a row and the rest of the workgroup on
 * the rows below, whichever width leaves the fewest lanes behind the row's end.  Bound by memory: 32 bytes in and 4 out per lane. */
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

__global__ void __launch_bounds__(256) vt_mx4_dequantize_kernel(float *x, const unsigned *codes, const uint8_t *scales, mx4_shape s) {
    int row, unit;
    if (!mx4_place(s, row, unit)) return;
    const int left = s.cols - 8 * unit;
    if (left <= 0) return;
    const size_t at = (size_t)row * s.units + unit;
    f32x4 a, b;
    vt_mx4_decode8(codes[at], scales[at >> 2], a, b);
    vt_mx4_store8(x + (size_t)row * s.stride + 8 * (size_t)unit, left, s.whole && left >= 8, a, b);
}

/* Workgroups of a launch over [rows, cols], or 0 where they are too many. */
static int mx4_grid(mx4_shape *s, const void *x, int item, int rows, int cols, int stride) {
    s->rows = rows;
    s->cols = cols;
    s->stride = stride;
    s->units = 16 * panels_of(cols);
    s->whole = ((uintptr_t)x & 15) == 0 && (size_t)stride * item % 16 == 0;
    int best = 8;
    long long lanes = 0;
    for (int w = 8; w >= 4; w--) {
        const long long n = ((long long)(s->units + (1 << w) - 1) >> w) << w;
        if (lanes == 0 || n < lanes) { best = w; lanes = n; }
    }
    s->wide_log = best;
    const long long chunks = (s->units + (1ll << best) - 1) >> best, tall = ((long long)rows + (256 >> best) - 1) / (256 >> best);
    if (chunks * tall > 0x7fffffffll) return 0;
    s->chunks = vt_divisor_of((int)chunks, chunks * tall);
    return (int)(chunks * tall);
}

static int mx4_shape_ok(const char *who, const void *x, const uint8_t *codes, const uint8_t *scales, int rows, int cols, int stride, int item) {
    if (!x || !codes || !scales) { vt_set_error("%s: NULL pointer", who); return 0; }
    if (rows < 1 || cols < 1 || cols > 1 << 27 || stride < cols) {
        vt_set_error("%s: %d rows of %d columns %d apart (columns: 1 .. 2^27)", who, rows, cols, stride);
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
    mx4_shape s;
    const int grid = mx4_grid(&s, d_x, x_bf16 ? 2 : 4, rows, cols, x_stride);
    if (!grid) { vt_set_error("%s: %d x %d is too large for one call", who, rows, cols); return -1; }
    if (x_bf16) hipLaunchKernelGGL(vt_mx4_quantize_kernel<uint16_t>, dim3(grid), dim3(256), 0, g_vt.stream, (unsigned *)d_codes, d_scales, (const uint16_t *)d_x, s);
    else hipLaunchKernelGGL(vt_mx4_quantize_kernel<float>, dim3(grid), dim3(256), 0, g_vt.stream, (unsigned *)d_codes, d_scales, (const float *)d_x, s);
    return vt_check(hipGetLastError(), who) ? -1 : 0;
}

extern "C" int tts_hip_mx4_dequantize(float *d_x, const uint8_t *d_codes, const uint8_t *d_scales, int rows, int cols, int x_stride) {
    static const char who[] = "tts_hip_mx4_dequantize";
    if (x_stride == 0) x_stride = cols;
    if (!mx4_shape_ok(who, d_x, d_codes, d_scales, rows, cols, x_stride, 4) || !vt_mx4_ready(who)) return -1;
    mx4_shape s;
    const int grid = mx4_grid(&s, d_x, 4, rows, cols, x_stride);
    if (!grid) { vt_set_error("%s: %d x %d is too large for one call", who, rows, cols); return -1; }
    hipLaunchKernelGGL(vt_mx4_dequantize_kernel, dim3(grid), dim3(256), 0, g_vt.stream, d_x, (const unsigned *)d_codes, d_scales, s);
    return vt_check(hipGetLastError(), who) ? -1 : 0;
}

/* ---- linear layer ------------------------------------------------------------------------------------------------ */

/* A wave per weight row and four rows of x, which share the decoded weights. */
#define MXL_ROWS 4
__global__ void __launch_bounds__(256)
vt_mx4_linear_kernel(float *y, const float *x, const unsigned *codes, const uint8_t *scales, int seq_len, int in_dim, int out_dim, int units, int whole) {
    const int o = (int)blockIdx.x * 4 + ((int)threadIdx.x >> 6), lane = (int)threadIdx.x & 63;
    if (o >= out_dim) return;
    for (int s0 = 0; s0 < seq_len; s0 += MXL_ROWS) {
        float acc[MXL_ROWS] = {};
        for (int u = lane; u < units && 8 * u < in_dim; u += 64) {
            const size_t at = (size_t)o * units + u;
            f32x4 wa, wb;
            vt_mx4_decode8(codes[at], scales[at >> 2], wa, wb);
#pragma unroll
            for (int s = 0; s < MXL_ROWS; s++) {
                if (s0 + s >= seq_len) break;
                f32x4 a, b;
                vt_mx4_load8(x + (size_t)(s0 + s) * in_dim + 8 * u, in_dim - 8 * u, whole && 8 * u + 8 <= in_dim, a, b);
#pragma unroll
                for (int i = 0; i < 4; i++) acc[s] = fmaf(wb[i], b[i], fmaf(wa[i], a[i], acc[s]));
            }
        }
#pragma unroll
        for (int s = 0; s < MXL_ROWS; s++) {
            const float v = vt_wave_sum(acc[s]);
            if (lane == 0 && s0 + s < seq_len) y[(size_t)(s0 + s) * out_dim + o] = v;
        }
    }
}

extern "C" int tts_hip_linear_mx4(float *d_y, const float *d_x, const uint8_t *d_codes, const uint8_t *d_scales, int seq_len, int in_dim, int out_dim) {
    static const char who[] = "tts_hip_linear_mx4";
    if (!d_y || ((uintptr_t)d_y & 3) || seq_len < 1) { vt_set_error("%s: %d rows to %p", who, seq_len, (void *)d_y); return -1; }
    if (!mx4_shape_ok(who, d_x, d_codes, d_scales, out_dim, in_dim, in_dim, 4) || !vt_mx4_ready(who)) return -1;
    const int whole = ((uintptr_t)d_x & 15) == 0 && in_dim % 4 == 0;
    hipLaunchKernelGGL(vt_mx4_linear_kernel, dim3((out_dim + 3) / 4), dim3(256), 0, g_vt.stream, d_y, d_x, (const unsigned *)d_codes, d_scales, seq_len,
                       in_dim, out_dim, 16 * panels_of(in_dim), whole);
    return vt_check(hipGetLastError(), who) ? -1 : 0;
}
