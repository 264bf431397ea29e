/*
 * vt_kv4.hip - a key/value cache in microscaled 4-bit floats (vt_mx4.h) and the attention that reads it.  Per kv head the
 * rows lie one behind the other, codes [kv heads, max_rows, head_dim / 2] and scales [kv heads, max_rows, head_dim / 32], for K
 * and for V: what one head's attention reads is one piece of memory.
 */
#include "vt_state.h"
#include "vt_mx4.h"
#include "vt_requests.h"

#include <math.h>

int vt_mx4_ready(const char *who);

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

/* ---- rows into the cache and back: a lane per eight values, K in blockIdx.y = 0 and V in 1 ----------------------------- */
struct kv4_rows { int n, pos, max_rows, stride, whole; vt_divisor per_row, per_head; };      /* lanes of a row, of a row of one head */

static __device__ __forceinline__ bool kv4_place(const kv4_rows &r, long long &from, size_t &at) {
    const int i = (int)(blockIdx.x * 256 + threadIdx.x);
    if (i >= r.n * r.per_row.d) return false;
    const int row = vt_div(i, r.per_row), u = i - row * r.per_row.d, h = vt_div(u, r.per_head), d = u - h * r.per_head.d;
    from = (long long)row * r.stride + 8 * u;
    at = ((size_t)h * r.max_rows + r.pos + row) * r.per_head.d + d;
    return true;
}

__global__ void __launch_bounds__(256) vt_kv4_append_kernel(tts_hip_kv4_t c, const float *K, const float *V, kv4_rows r) {
    long long from;
    size_t at;
    if (!kv4_place(r, from, at)) return;
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
    if (!kv4_place(r, to, at)) return;
    f32x4 a, b;
    vt_mx4_decode8(((const unsigned *)(blockIdx.y ? c.v_codes : c.k_codes))[at], (blockIdx.y ? c.v_scales : c.k_scales)[at >> 2], a, b);
    vt_mx4_store8((blockIdx.y ? V : K) + to, 8, r.whole, a, b);
}

static int kv4_rows_ok(const char *who, kv4_rows *r, const tts_hip_kv4_t *c, const float *K, const float *V, int n, int pos, int stride) {
    if (!cache_ok(who, c, pos, n)) return 0;
    const long long width = (long long)c->n_kv_heads * c->head_dim;
    if (stride == 0) stride = (int)(width > 0x7fffffff ? 0x7fffffff : width);
    if (!K || !V || (((uintptr_t)K | (uintptr_t)V) & 3) || stride < width || width / 8 * n > 0x7fffff00ll) {
        vt_set_error("%s: %d rows of %lld values %d apart", who, n, width, stride);
        return 0;
    }
    *r = kv4_rows{n, pos, c->max_rows, stride, (((uintptr_t)K | (uintptr_t)V) & 15) == 0 && stride % 4 == 0,
                  vt_divisor_of((int)(width / 8), width / 8 * n), vt_divisor_of(c->head_dim / 8, width / 8)};
    return vt_mx4_ready(who);
}

extern "C" int tts_hip_kv4_append(const tts_hip_kv4_t *cache, const float *d_K, const float *d_V, int n_rows, int pos, int stride) {
    static const char who[] = "tts_hip_kv4_append";
    kv4_rows r;
    if (!kv4_rows_ok(who, &r, cache, d_K, d_V, n_rows, pos, stride)) return -1;
    hipLaunchKernelGGL(vt_kv4_append_kernel, dim3((r.n * r.per_row.d + 255) / 256, 2), dim3(256), 0, g_vt.stream, *cache, d_K, d_V, r);
    return vt_check(hipGetLastError(), who) ? -1 : 0;
}

extern "C" int tts_hip_kv4_read(float *d_K, float *d_V, const tts_hip_kv4_t *cache, int n_rows, int pos, int stride) {
    static const char who[] = "tts_hip_kv4_read";
    kv4_rows r;
    if (!kv4_rows_ok(who, &r, cache, d_K, d_V, n_rows, pos, stride)) return -1;
    hipLaunchKernelGGL(vt_kv4_read_kernel, dim3((r.n * r.per_row.d + 255) / 256, 2), dim3(256), 0, g_vt.stream, d_K, d_V, *cache, r);
    return vt_check(hipGetLastError(), who) ? -1 : 0;
}

/* ---- attention ------------------------------------------------------------------------------------------------------- */

/* A workgroup per head and query; its waves stride over the rows, a lane owns the values lane, lane + 64, ... of a row. */
__global__ void __launch_bounds__(256) vt_kv4_attention_kernel(float *out, const float *Q, tts_hip_kv4_t c, int start_pos, int n_heads, float scale) {
    __shared__ float part[4][2 + 256];
    const int h = (int)blockIdx.x, i = (int)blockIdx.y, hd = c.head_dim, per = hd / 64, lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
    const int kvh = h / (n_heads / c.n_kv_heads);
    const float *q = Q + ((size_t)i * n_heads + h) * hd;
    float qv[4], o[4], m = -INFINITY, l = 0.f;
    for (int e = 0; e < 4; e++) { qv[e] = e < per ? q[lane + 64 * e] : 0.f; o[e] = 0.f; }
    auto value = [&](const uint8_t *codes, const uint8_t *scales, size_t row, int d) {
        const f32x2 p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4((unsigned)codes[(row * hd + d) >> 1], vt_mx4_scale(scales[(row * hd + d) >> 5]), 0);
        return d & 1 ? p.y : p.x;
    };
    for (int j = wave; j <= start_pos + i; j += 4) {
        const size_t row = (size_t)kvh * c.max_rows + j;
        float s = 0.f;
        for (int e = 0; e < per; e++) s = fmaf(qv[e], value(c.k_codes, c.k_scales, row, lane + 64 * e), s);
        s = vt_wave_sum(s) * scale;
        const float mn = fmaxf(m, s), old = m == -INFINITY ? 0.f : expf(m - mn), p = expf(s - mn);
        l = fmaf(l, old, p);
        for (int e = 0; e < per; e++) o[e] = fmaf(o[e], old, p * value(c.v_codes, c.v_scales, row, lane + 64 * e));
        m = mn;
    }
    if (lane == 0) { part[wave][0] = m; part[wave][1] = l; }
    for (int e = 0; e < per; e++) part[wave][2 + lane + 64 * e] = o[e];
    __syncthreads();
    for (int d = (int)threadIdx.x; d < hd; d += 256) {
        float M = -INFINITY, L = 0.f, O = 0.f;
        for (int w = 0; w < 4; w++) M = fmaxf(M, part[w][0]);
        for (int w = 0; w < 4; w++) {
            if (part[w][0] == -INFINITY && part[w][1] == 0.f) continue;
            const float e = expf(part[w][0] - M);
            L = fmaf(part[w][1], e, L);
            O = fmaf(part[w][2 + d], e, O);
        }
        out[((size_t)i * n_heads + h) * hd + d] = O / L;
    }
}

extern "C" int tts_hip_kv4_attention(float *d_out, const float *d_Q, const tts_hip_kv4_t *cache, int seq_len, int start_pos, int n_heads, float scale) {
    static const char who[] = "tts_hip_kv4_attention";
    if (!d_out || !d_Q || (((uintptr_t)d_out | (uintptr_t)d_Q) & 15)) { vt_set_error("%s: queries and results lie on 16 bytes", who); return -1; }
    if (seq_len < 1 || start_pos < 0) { vt_set_error("%s: %d queries behind %d rows", who, seq_len, start_pos); return -1; }
    if (!cache_ok(who, cache, 0, (long long)start_pos + seq_len)) return -1;
    if (n_heads < 1 || n_heads % cache->n_kv_heads) { vt_set_error("%s: %d heads on %d kv heads", who, n_heads, cache->n_kv_heads); return -1; }
    if (!vt_mx4_ready(who)) return -1;
    hipLaunchKernelGGL(vt_kv4_attention_kernel, dim3(n_heads, seq_len), dim3(256), 0, g_vt.stream, d_out, d_Q, *cache, start_pos, n_heads, scale);
    return vt_check(hipGetLastError(), who) ? -1 : 0;
}
