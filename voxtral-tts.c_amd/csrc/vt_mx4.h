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

__device__ __forceinline__ f32x4 vt_mx4_decode4(unsigned c, unsigned scale) {
    const float f = vt_mx4_scale(scale);
    const f32x2 p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, f, 0), q = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, f, 1);
    return f32x4{p.x, p.y, q.x, q.y};
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
/* four values back, past the caches where they lie on 16 bytes */
__device__ __forceinline__ void vt_mx4_store4(float *p, int n, bool whole, const f32x4 &v) {
    if (whole) {
        __builtin_nontemporal_store(v, reinterpret_cast<f32x4 *>(p));
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (i < n) p[i] = v[i];
}

/* ---- fp32 operands of the scaled matrix instructions --------------------------------------------------------------
 * v_mfma_scale_f32_*_f8f6f4 multiplies blocks of 32 values with a scale each: the 4-bit operand goes in as it lies in memory, and
 * fp32 values as a sum of NP planes of e2m3 (six bits: 0 .. 2 in steps of 1/8, 2 .. 4 of 1/4, 4 .. 7.5 of 1/2): plane 0 is the nearest
 * e2m3 of the block, every next one that of what is left, each with a scale of its own that puts the largest magnitude at 3.875 .. 7.75 of
 * it.  A plane leaves at most 2^-4 of that magnitude; on values ~N(0, 1) five planes leave 9e-9 of their norm, and 2.0e-8 where the fifth's
 * scale is 2^-4 of the fourth's, each value to 2^-24 of its block's largest (2^-21 at the worst).  Fewer are not enough for fp32: four
 * leave 5.2e-7 of the norm, and 1.3e-4 of the values beside one that is 1000 times as large.  Subtracting what a plane holds is exact.
 * With an infinity or a NaN in it a block's scales say NaN. */
typedef float vt_f32x16 __attribute__((ext_vector_type(16)));
typedef float vt_f32x32 __attribute__((ext_vector_type(32)));
typedef unsigned vt_u32x6 __attribute__((ext_vector_type(6)));
typedef int vt_i32x8 __attribute__((ext_vector_type(8)));
#define VT_MFMA_E2M1 4                    /* formats of an operand, as the instruction numbers them */
#define VT_MFMA_E2M3 2

/* the scale of a plane that stands in a fixed ratio to the one before: 2^-4 of its */
__device__ __forceinline__ int vt_mx4_below(unsigned s) { return max((int)s - 4, 0); }

/* The next plane of a block, and what it leaves of it; even[i], odd[i]: values 2 i and 2 i + 1.  tied: its scale follows from the one
 * before, `scale`. */
__device__ __forceinline__ vt_u32x6 vt_mx4_plane(vt_f32x16 &even, vt_f32x16 &odd, bool tied, unsigned &scale) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < 16; i++) t = __builtin_elementwise_maximum(__builtin_elementwise_maximum(t, fabsf(even[i])), fabsf(odd[i]));
    const unsigned top = __float_as_uint(t);
    scale = tied ? (unsigned)vt_mx4_below(scale) : top >= 0x7f800000u ? 255u : (unsigned)max((int)((top + 0x80000u) >> 23) - 2, 0);
    const float f = vt_mx4_scale(scale);
    const vt_u32x6 q = __builtin_amdgcn_cvt_scalef32_2xpk16_fp6_f32(even, odd, f);
    const vt_f32x32 held = __builtin_amdgcn_cvt_scalef32_pk32_f32_fp6(q, f);
#pragma unroll
    for (int i = 0; i < 16; i++) {
        even[i] = __fsub_rn(even[i], held[2 * i]);
        odd[i] = __fsub_rn(odd[i], held[2 * i + 1]);
    }
    return q;
}

template <int NP, bool TIED = false>
__device__ __forceinline__ void vt_mx4_planes(vt_f32x16 even, vt_f32x16 odd, vt_u32x6 (&q)[NP], unsigned (&s)[NP]) {
#pragma unroll
    for (int p = 0; p < NP; p++) {
        s[p] = p ? s[p - 1] : 0u;
        q[p] = vt_mx4_plane(even, odd, TIED && p == NP - 1, s[p]);
    }
}

/* 32 values of a row from column `at` on, through a buffer that holds the row `row_at` bytes in; zeros from column `cols` on.  whole:
 * rows lie on 16 bytes. (No branch around a load: behind one the compiler waits for it, a trip to memory each.) */
__device__ __forceinline__ void vt_mx4_load32(__amdgpu_buffer_rsrc_t x, int row_at, int at, int cols, int whole, vt_f32x16 &even, vt_f32x16 &odd) {
    if (whole) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const f32x4 v = vt_buffer_ld4(x, at + 4 * i < cols ? row_at + (at + 4 * i) * 4 : 0x7ffffff0);
            even[2 * i] = v.x; odd[2 * i] = v.y; even[2 * i + 1] = v.z; odd[2 * i + 1] = v.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; i++) {
            even[i] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(x, at + 2 * i < cols ? row_at + (at + 2 * i) * 4 : 0x7ffffff0, 0, 0));
            odd[i] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(x, at + 2 * i + 1 < cols ? row_at + (at + 2 * i + 1) * 4 : 0x7ffffff0, 0, 0));
        }
    }
}

__device__ __forceinline__ vt_i32x8 vt_mfma_e2m1(const u32x4 &v) { return __builtin_bit_cast(vt_i32x8, __builtin_shufflevector(v, v, 0, 1, 2, 3, -1, -1, -1, -1)); }
__device__ __forceinline__ vt_i32x8 vt_mfma_e2m3(const vt_u32x6 &v) { return __builtin_bit_cast(vt_i32x8, __builtin_shufflevector(v, v, 0, 1, 2, 3, 4, 5, -1, -1)); }

#endif /* VT_MX4_H */
