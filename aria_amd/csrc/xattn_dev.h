/*
 * xattn_dev.h - device code shared by the attention kernels on v_mfma_f32_32x32x16 (k_xattn.hip,
 * k_pattn.hip): element types, and the constants of the running reference of a softmax.
 */
#ifndef ARIA_XATTN_DEV_H
#define ARIA_XATTN_DEV_H

#include "aria_dev.h"

typedef float xa_f32x16_t __attribute__((ext_vector_type(16)));
typedef short xa_i16x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) xa_i16x4_t xa_lds_i16x4_t;

#define XA_TOP 7.0f        /* log2 of the largest weight where the reference has just moved */
#define XA_SLACK 8.0f      /* log2 units that the maximum may rise above that before the reference moves again */
#define XA_MIN (-3.40282347e38f)   /* the reference before any key */
#define XA_FAR 16777216.0f /* from here on fp32's steps are over 1 */

template <typename T> struct Xa;
template <> struct Xa<_Float16> {
    typedef _Float16 v8 __attribute__((ext_vector_type(8)));
    typedef _Float16 v2 __attribute__((ext_vector_type(2)));
    static constexpr unsigned ONE = 0x3C00u, NINF = 0xFC00u;
    static __device__ __forceinline__ xa_f32x16_t mfma8(uint2 a, uint2 b, xa_f32x16_t c) {
        typedef _Float16 v4 __attribute__((ext_vector_type(4)));
        return __builtin_amdgcn_mfma_f32_32x32x8f16(__builtin_bit_cast(v4, a), __builtin_bit_cast(v4, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ xa_f32x16_t mfma(v8 a, v8 b, xa_f32x16_t c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ float dot2(v2 a, v2 b, float c) { return __builtin_amdgcn_fdot2(a, b, c, false); }
};
template <> struct Xa<__bf16> {
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    typedef __bf16 v2 __attribute__((ext_vector_type(2)));
    static constexpr unsigned ONE = 0x3F80u, NINF = 0xFF80u;
    static __device__ __forceinline__ xa_f32x16_t mfma8(uint2 a, uint2 b, xa_f32x16_t c) {
        return __builtin_amdgcn_mfma_f32_32x32x8bf16_1k(__builtin_bit_cast(xa_i16x4_t, a), __builtin_bit_cast(xa_i16x4_t, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ xa_f32x16_t mfma(v8 a, v8 b, xa_f32x16_t c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ float dot2(v2 a, v2 b, float c) { return __builtin_amdgcn_fdot2_f32_bf16(a, b, c, false); }
};

#endif /* ARIA_XATTN_DEV_H */
