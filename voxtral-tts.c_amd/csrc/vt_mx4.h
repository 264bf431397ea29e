/*
 * vt_mx4.h - microscaled 4-bit floats (e2m1 codes, one e8m0 scale per 32 values): the conversions that the operators on
 * weights (vt_mx4.hip) and on the 4-bit key/value cache (vt_kv4.hip) share.
 *
 * A block of 32 consecutive values with largest magnitude t has the scale 2^(s - 127), s = floor(log2 t) - 2 + 127 held in
 * 0 .. 254 (2 is the exponent of the largest code, 6); a value's code is the nearest of {0, .5, 1, 1.5, 2, 3, 4, 6} times the
 * scale, of two equally near ones the even one, at most 6, and a sign.  s = 255 stands for a block of NaN: one with an
 * infinity or a NaN in it.  gfx950 converts both ways in hardware (v_cvt_scalef32_pk_*_fp4), with these roundings and, on the
 * way back, NaN for s = 255; what it takes of the scale operand are the exponent's bits, 0 for 2^-127 among them.
 */
#ifndef VT_MX4_H
#define VT_MX4_H

#include "vt_device.h"

__device__ __forceinline__ float vt_mx4_scale(unsigned s) { return __uint_as_float(s << 23); }

/* the scale of a block by the bits of its largest magnitude: the exponent field is floor(log2 t) + 127, and 0 below 2^-126 */
__device__ __forceinline__ unsigned vt_mx4_scale_of(unsigned top) {
    const int e = (int)(top >> 23);
    return e == 255 ? 255u : (unsigned)max(e - 2, 0);
}

/* Eight values of a block whose other 24 the three other lanes of the quad hold -> their codes, and the block's scale. */
__device__ __forceinline__ unsigned vt_mx4_encode8(const f32x4 &a, const f32x4 &b, unsigned &scale) {
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) top = max(top, max(__float_as_uint(a[i]) & 0x7fffffffu, __float_as_uint(b[i]) & 0x7fffffffu));
    top = max(top, (unsigned)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xf, 0xf, false));
    top = max(top, (unsigned)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xf, 0xf, false));
    scale = vt_mx4_scale_of(top);
    const float f = vt_mx4_scale(scale);
    unsigned c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, a.x, a.y, f, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, a.z, a.w, f, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, b.x, b.y, f, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, b.z, b.w, f, 3);
    return scale == 255u ? 0u : c;
}

__device__ __forceinline__ void vt_mx4_decode8(unsigned c, unsigned scale, f32x4 &a, f32x4 &b) {
    const float f = vt_mx4_scale(scale);
    const f32x2 p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, f, 0), q = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, f, 1);
    const f32x2 r = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, f, 2), t = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, f, 3);
    a = f32x4{p.x, p.y, q.x, q.y};
    b = f32x4{r.x, r.y, t.x, t.y};
}

/* n (at most 8) of eight values at p, zeros behind them; whole: all eight there and p on 16 bytes */
__device__ __forceinline__ void vt_mx4_load8(const float *p, int n, bool whole, f32x4 &a, f32x4 &b) {
    if (whole) {
        a = *reinterpret_cast<const f32x4 *>(p);
        b = *reinterpret_cast<const f32x4 *>(p + 4);
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        a[i] = i < n ? p[i] : 0.f;
        b[i] = i + 4 < n ? p[i + 4] : 0.f;
    }
}
__device__ __forceinline__ void vt_mx4_load8(const uint16_t *p, int n, bool whole, f32x4 &a, f32x4 &b) {
    if (whole) {
        const u32x4 w = *reinterpret_cast<const u32x4 *>(p);
        a = f32x4{vt_bf16_lo(w.x), vt_bf16_hi(w.x), vt_bf16_lo(w.y), vt_bf16_hi(w.y)};
        b = f32x4{vt_bf16_lo(w.z), vt_bf16_hi(w.z), vt_bf16_lo(w.w), vt_bf16_hi(w.w)};
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        a[i] = i < n ? vt_bf16_lo(p[i]) : 0.f;
        b[i] = i + 4 < n ? vt_bf16_lo(p[i + 4]) : 0.f;
    }
}
__device__ __forceinline__ void vt_mx4_store8(float *p, int n, bool whole, const f32x4 &a, const f32x4 &b) {
    if (whole) {
        *reinterpret_cast<f32x4 *>(p) = a;
        *reinterpret_cast<f32x4 *>(p + 4) = b;
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (i < n) p[i] = a[i];
        if (i + 4 < n) p[i + 4] = b[i];
    }
}

#endif /* VT_MX4_H */
