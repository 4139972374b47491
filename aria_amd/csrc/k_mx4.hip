/*
 * k_mx4.hip - MXFP4 quantisation and dequantisation of rows (gfx950).
 *
 * Block b of a row: byte = floor(log2 max|x|) - 2 + 127, codes = x 2^(127 - byte) rounded to the
 * nearest e2m1 value (ties to the even code, saturated at 6). A block that holds an Inf or NaN gets
 * scale byte 255 and reads back as NaN. All steps are exact but the one rounding to four bits.
 *
 * Both passes are bound by HBM: sizeof(x) + 17/32 bytes per element. Eight values per lane (one
 * 32-byte fp32 or 16-byte fp16 / bf16 read, one 4-byte code word), so a block is a quad of lanes
 * and its maximum two DPP steps.
 */
#include "mx4_dev.h"

template <int T>
__global__ __launch_bounds__(256) void k_mx4_quant(uint8_t *q, uint8_t *scale, const void *x, unsigned total, int K,
                                                   unsigned nb, long ld, int vec) {
    const unsigned i = blockIdx.x * 256u + threadIdx.x;
    if (i >= total) return;                    /* total counts whole quads */
    const unsigned row = i / (4 * nb), o = i - row * 4 * nb;
    float f[8];
    mx_load8<T>(x, (size_t)row * ld + 8 * o, K - 8 * (int)o, vec, f);
    unsigned m = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) m = max(m, mx_abs_bits(f[e]));
    m = max(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, DPP_QUAD_XOR1, 0xF, 0xF, false));
    m = max(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, DPP_QUAD_XOR2, 0xF, 0xF, false));
    const unsigned byte = mx_scale_byte(m);
    ((unsigned *)q)[(size_t)row * 4 * nb + o] = mx_pack8(f, byte);
    if ((o & 3) == 0) scale[(size_t)row * nb + (o >> 2)] = (uint8_t)byte;
}

/* value of a 4-bit code under scale byte b (255: NaN): magnitude bits e2 m1 as fp32, times a power
 * of two; 2^-127 is the fp32 subnormal 0x00400000 */
__device__ __forceinline__ float mx_value(unsigned code, float s) {
    const unsigned e = (code >> 1) & 3, m = code & 1;
    const float mag = e ? __builtin_bit_cast(float, ((126u + e) << 23) | (m << 22)) : (m ? 0.5f : 0.0f);
    const float v = mag * s;
    return (code & 8) ? -v : v;
}
__device__ __forceinline__ float mx_scale_value(unsigned byte) {
    return __builtin_bit_cast(float, byte == 255u ? 0x7FC00000u : byte ? byte << 23 : 0x00400000u);
}

template <int T>
__global__ __launch_bounds__(256) void k_mx4_dequant(void *y, const uint8_t *q, const uint8_t *scale, unsigned total, int K,
                                                     unsigned nb, int vec) {
    const unsigned i = blockIdx.x * 256u + threadIdx.x;
    if (i >= total) return;
    const unsigned row = i / (4 * nb), o = i - row * 4 * nb;
    const int n = K - 8 * (int)o;
    if (n <= 0) return;
    const unsigned w = ((const unsigned *)q)[(size_t)row * 4 * nb + o];
    const float s = mx_scale_value(scale[(size_t)row * nb + (o >> 2)]);
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; e++) f[e] = mx_value((w >> (4 * e)) & 15u, s);
    mx_t<T> *p = (mx_t<T> *)y + (size_t)row * K + 8 * o;
    if (vec) {
        typedef mx_t<T> v8_t __attribute__((ext_vector_type(8)));
        v8_t v;
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = (mx_t<T>)f[e];
        *reinterpret_cast<v8_t *>(p) = v;
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (e < n) p[e] = (mx_t<T>)f[e];
    }
}

/* rows per launch: the kernels count lanes (4 per block) in 32 bits */
static int rows_per_launch(int nb) { return (int)(((1u << 30) - 1) / (4u * (unsigned)nb)); }
static size_t el_size(int t) { return t == MX_F32 ? 4 : 2; }

extern "C" hipError_t aria_k_mx4_quant(uint8_t *q, uint8_t *scale, const void *x, int xtype, int rows, int K, long ld,
                                       hipStream_t s) {
    if (rows <= 0 || K <= 0) return hipSuccess;
    const int nb = (K + 31) / 32, per = rows_per_launch(nb);
    const size_t es = el_size(xtype);
    const int vec = ld % 8 == 0 && ((uintptr_t)x & 15u) == 0;
    for (int r0 = 0; r0 < rows; r0 += per) {
        const int n = rows - r0 < per ? rows - r0 : per;
        const unsigned total = (unsigned)n * 4u * (unsigned)nb;
        uint8_t *qr = q + (size_t)r0 * nb * 16, *sr = scale + (size_t)r0 * nb;
        const char *xr = (const char *)x + (size_t)r0 * ld * es;
        const dim3 grid((total + 255) / 256), block(256);
        if (xtype == MX_F32) hipLaunchKernelGGL(k_mx4_quant<MX_F32>, grid, block, 0, s, qr, sr, xr, total, K, nb, ld, vec);
        else if (xtype == MX_F16) hipLaunchKernelGGL(k_mx4_quant<MX_F16>, grid, block, 0, s, qr, sr, xr, total, K, nb, ld, vec);
        else hipLaunchKernelGGL(k_mx4_quant<MX_BF16>, grid, block, 0, s, qr, sr, xr, total, K, nb, ld, vec);
    }
    return hipGetLastError();
}

extern "C" hipError_t aria_k_mx4_dequant(void *y, int ytype, const uint8_t *q, const uint8_t *scale, int rows, int K,
                                         hipStream_t s) {
    if (rows <= 0 || K <= 0) return hipSuccess;
    const int nb = (K + 31) / 32, per = rows_per_launch(nb);
    const size_t es = el_size(ytype);
    const int vec = K % 8 == 0 && ((uintptr_t)y & 15u) == 0;
    for (int r0 = 0; r0 < rows; r0 += per) {
        const int n = rows - r0 < per ? rows - r0 : per;
        const unsigned total = (unsigned)n * 4u * (unsigned)nb;
        const uint8_t *qr = q + (size_t)r0 * nb * 16, *sr = scale + (size_t)r0 * nb;
        char *yr = (char *)y + (size_t)r0 * K * es;
        const dim3 grid((total + 255) / 256), block(256);
        if (ytype == MX_F32) hipLaunchKernelGGL(k_mx4_dequant<MX_F32>, grid, block, 0, s, yr, qr, sr, total, K, nb, vec);
        else if (ytype == MX_F16) hipLaunchKernelGGL(k_mx4_dequant<MX_F16>, grid, block, 0, s, yr, qr, sr, total, K, nb, vec);
        else hipLaunchKernelGGL(k_mx4_dequant<MX_BF16>, grid, block, 0, s, yr, qr, sr, total, K, nb, vec);
    }
    return hipGetLastError();
}
