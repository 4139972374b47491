/*
 * mx4_dev.h - device code shared by the MXFP4 kernels (k_mx4.hip, k_mx4_gemm.hip): element types,
 * the quantisation of one block, the block-scaled MFMA operands.
 *
 * MXFP4: 32 consecutive values along K share a power of two 2^(byte - 127); each value is a 4-bit
 * code (sign, magnitude 0, 0.5, 1, 1.5, 2, 3, 4 or 6). A packed row is ceil(K/32) blocks of 16
 * bytes (the even element in the low nibble, the last block's tail zero) and ceil(K/32) scale bytes.
 */
#ifndef ARIA_MX4_DEV_H
#define ARIA_MX4_DEV_H

#include "aria_dev.h"
#include "aria_hip_kernels.h"

typedef int i32x8_t __attribute__((ext_vector_type(8)));
typedef float mx_f32x4_t __attribute__((ext_vector_type(4)));
typedef float mx_f32x16_t __attribute__((ext_vector_type(16)));
typedef unsigned mx_u32x4_t __attribute__((ext_vector_type(4)));

/* element types of activations and outputs: the values of aria_dtype */
enum { MX_F32 = 0, MX_F16 = 1, MX_BF16 = 2 };

template <int T> struct MxT;
template <> struct MxT<MX_F32> { using type = float; };
template <> struct MxT<MX_F16> { using type = _Float16; };
template <> struct MxT<MX_BF16> { using type = __bf16; };
template <int T> using mx_t = typename MxT<T>::type;

/* elements off .. off + V - 1 of x as fp32; those past n (counted from off) read as zero. vec: x + off is 16-byte
 * aligned (else aligned to an element) */
template <int T, int V>
__device__ __forceinline__ void mx_load(const void *x, size_t off, int n, bool vec, float (&f)[V]) {
    typedef mx_t<T> v_t __attribute__((ext_vector_type(V)));
    const mx_t<T> *p = (const mx_t<T> *)x + off;
    if (n >= V) {
        v_t v;
        if (vec) {
            if constexpr (sizeof v == 32) {    /* eight fp32 */
                typedef mx_t<T> h_t __attribute__((ext_vector_type(V / 2)));
                const h_t a = *reinterpret_cast<const h_t *>(p), b = *reinterpret_cast<const h_t *>(p + V / 2);
                __builtin_memcpy(&v, &a, 16);
                __builtin_memcpy((char *)&v + 16, &b, 16);
            } else {
                v = *reinterpret_cast<const v_t *>(p);
            }
        } else {
            __builtin_memcpy(&v, p, sizeof v);
        }
#pragma unroll
        for (int i = 0; i < V; i++) f[i] = (float)v[i];
    } else {
#pragma unroll
        for (int i = 0; i < V; i++) f[i] = i < n ? (float)p[i] : 0.0f;
    }
}

/* |v| as ordered bits: an Inf or NaN is above every finite value */
__device__ __forceinline__ unsigned mx_abs_bits(float v) { return __builtin_bit_cast(unsigned, v) & 0x7FFFFFFFu; }

/* the block's scale byte from the largest |value| bits: floor(log2 amax) - 2, biased by 127, at
 * least 0 (amax below 2^-124, zero included); 255 (NaN) where a value is not finite */
__device__ __forceinline__ unsigned mx_scale_byte(unsigned amax_bits) {
    const unsigned e = amax_bits >> 23;
    return e == 255u ? 255u : max(e, 2u) - 2u;
}

/* four values over 2^(byte - 127) -> 16 bits of codes; the rule of mx_pack8 */
__device__ __forceinline__ unsigned mx_pack4(const float (&f)[4], unsigned byte) {
    const float r = __builtin_bit_cast(float, (254u - min(byte, 253u)) << 23);
    unsigned w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[0] * r, f[1] * r, 1.0f, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[2] * r, f[3] * r, 1.0f, 1);
    return byte == 255u ? 0u : w;
}

/* eight values over 2^(byte - 127) -> eight codes, ties to even, saturating at 6. The scaling is a
 * multiplication by the exact reciprocal power (2^127 .. 2^-125), the conversion runs at scale 1 */
__device__ __forceinline__ unsigned mx_pack8(const float (&f)[8], unsigned byte) {
    const float r = __builtin_bit_cast(float, (254u - min(byte, 253u)) << 23);
    unsigned w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[0] * r, f[1] * r, 1.0f, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[2] * r, f[3] * r, 1.0f, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[4] * r, f[5] * r, 1.0f, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[6] * r, f[7] * r, 1.0f, 3);
    return byte == 255u ? 0u : w;
}

/* 16 bytes of codes as an MFMA operand (the fp4 forms read the first four registers) */
__device__ __forceinline__ i32x8_t mx_op(const uint4 &u) {
    return i32x8_t{(int)u.x, (int)u.y, (int)u.z, (int)u.w, 0, 0, 0, 0};
}

/* g / (1 + e^-g). EXACT (fp32 outputs): to a few fp32 steps at any g; what the exponent's rounding leaves out of -g log2 e, r,
 * comes back as the factor 2^r = 1 + r ln 2, and beyond 104 e^-g is infinite or nothing. Else silu_f, which leaves r out: 64
 * half steps at g = -85, 2^-18, nothing beside the rounding to 16 bits (2592 x 1024 -> 2 x 4096, bf16: 24.5 us, 25.5 with it) */
template <bool EXACT>
__device__ __forceinline__ float mx_silu(float g) {
    if constexpr (!EXACT) return silu_f(g);
    constexpr float lo = 1.925963033e-8f;      /* log2 e - ARIA_LOG2E */
    const float x = __builtin_amdgcn_fmed3f(-g, -104.0f, 104.0f), t = x * ARIA_LOG2E;
    const float r = __builtin_fmaf(x, lo, __builtin_fmaf(x, ARIA_LOG2E, -t));
    const float e = __builtin_amdgcn_exp2f(t) * __builtin_fmaf(r, 0.69314718f, 1.0f);
    return g * rcp_fast(1.0f + e);
}

/* store one fp32 result as element type t (uniform) */
__device__ __forceinline__ void mx_store(void *y, int t, size_t i, float v) {
    if (t == MX_F32) ((float *)y)[i] = v;
    else if (t == MX_F16) ((_Float16 *)y)[i] = (_Float16)v;
    else ((__bf16 *)y)[i] = (__bf16)v;
}

#endif /* ARIA_MX4_DEV_H */
