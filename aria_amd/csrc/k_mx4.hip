/*
 * k_mx4.hip - MXFP4 quantisation and dequantisation of rows (gfx950).
 *
 * Block b of a row: byte = floor(log2 max|x|) - 2 + 127, codes = x 2^(127 - byte) rounded to the
 * nearest e2m1 value (ties to the even code, saturated at 6). A block that holds an Inf or NaN gets
 * scale byte 255 and reads back as NaN. All steps are exact but the one rounding to four bits.
 *
 * Both passes are bound by HBM: sizeof(x) + 17/32 bytes per element. A lane's unit of work is 16 bytes of x, so that a wave's
 * accesses are contiguous: 8 (fp32) or 4 lanes are a block, whose maximum is three or two DPP steps. Each lane
 * takes two units 64 lanes apart, both loaded before either is used.
 */
#include "mx4_dev.h"

/* unit i of V values (16 bytes: four fp32, eight fp16 or bf16) of the rows taken one after another, 32 nb / V to a row */
template <int T>
__global__ __launch_bounds__(256) void k_mx4_quant(uint8_t *q, uint8_t *scale, const void *x, unsigned total, int K,
                                                   unsigned nb, long ld, int vec) {
    constexpr int V = T == MX_F32 ? 4 : 8, L = 32 / V;         /* values per lane, lanes per block */
    const unsigned i0 = blockIdx.x * 512u + (threadIdx.x & ~63u) * 2 + (threadIdx.x & 63u);
    float f[2][V];
#pragma unroll
    for (int u = 0; u < 2; u++) {
        const unsigned i = i0 + 64 * u, row = i / (L * nb), o = i - row * L * nb;
        const int n = i < total ? K - V * (int)o : 0;
        mx_load<T, V>(x, (size_t)row * ld + V * o, n, vec, f[u]);
    }
#pragma unroll
    for (int u = 0; u < 2; u++) {
        const unsigned i = i0 + 64 * u;
        unsigned m = 0;
#pragma unroll
        for (int e = 0; e < V; e++) m = max(m, mx_abs_bits(f[u][e]));
        m = max(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, DPP_QUAD_XOR1, 0xF, 0xF, false));
        m = max(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, DPP_QUAD_XOR2, 0xF, 0xF, false));
        if constexpr (L == 8) m = max(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, DPP_ROW_HALF_MIRROR, 0xF, 0xF, false));
        if (i >= total) return;                /* total counts whole blocks: their lanes leave together */
        const unsigned byte = mx_scale_byte(m);
        if constexpr (V == 4) ((uint16_t *)q)[i] = (uint16_t)mx_pack4(f[u], byte);
        else ((unsigned *)q)[i] = mx_pack8(f[u], byte);
        if ((i & (L - 1)) == 0) scale[i / L] = (uint8_t)byte;
    }
}

/* value of a 4-bit code times the block's power of two s: magnitude bits e2 m1 as fp32 */
__device__ __forceinline__ float mx_value(unsigned code, float s) {
    const unsigned e = (code >> 1) & 3, m = code & 1;
    const float mag = e ? __builtin_bit_cast(float, ((126u + e) << 23) | (m << 22)) : (m ? 0.5f : 0.0f);
    const float v = mag * s;
    return (code & 8) ? -v : v;
}
/* 2^(byte - 127); 2^-127 is the fp32 subnormal 0x00400000 */
__device__ __forceinline__ float mx_scale_value(unsigned byte) {
    return __builtin_bit_cast(float, byte == 255u ? 0x7FC00000u : byte ? byte << 23 : 0x00400000u);
}

template <int T>
__global__ __launch_bounds__(256) void k_mx4_dequant(void *y, const uint8_t *q, const uint8_t *scale, unsigned total, int K,
                                                     unsigned nb, int vec) {
    const unsigned i0 = blockIdx.x * 512u + (threadIdx.x & ~63u) * 2 + (threadIdx.x & 63u);
    unsigned w[2], b[2];
#pragma unroll
    for (int u = 0; u < 2; u++) {
        const unsigned i = min(i0 + 64 * u, total - 1);
        w[u] = ((const uint16_t *)q)[i];
        b[u] = scale[i >> 3];
    }
    typedef mx_t<T> v4_t __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int u = 0; u < 2; u++) {
        const unsigned i = i0 + 64 * u, row = i / (8 * nb), o = i - row * 8 * nb;
        const int n = K - 4 * (int)o;
        if (i >= total || n <= 0) continue;
        const float s = mx_scale_value(b[u]);
        v4_t v;
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = (mx_t<T>)mx_value((w[u] >> (4 * e)) & 15u, s);
        mx_t<T> *p = (mx_t<T> *)y + (size_t)row * K + 4 * o;
        if (vec && n >= 4) {
            __builtin_nontemporal_store(v, reinterpret_cast<v4_t *>(p));
        } else if (n >= 4) {
            __builtin_memcpy(p, &v, sizeof v); /* rows start at any element */
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (e < n) p[e] = v[e];
        }
    }
}

/* rows per launch: the kernels count quads of values (8 per block) in 32 bits */
static int rows_per_launch(int nb) { return (int)(((1u << 31) - 512) / (8u * (unsigned)nb)); }
static size_t el_size(int t) { return t == MX_F32 ? 4 : 2; }

extern "C" hipError_t aria_k_mx4_quant(uint8_t *q, uint8_t *scale, const void *x, int xtype, int rows, int K, long ld,
                                       hipStream_t s) {
    if (rows <= 0 || K <= 0) return hipSuccess;
    const int nb = (K + 31) / 32, per = rows_per_launch(nb);
    const size_t es = el_size(xtype);
    const int vec = ld % (16 / es) == 0 && ((uintptr_t)x & 15u) == 0;
    for (int r0 = 0; r0 < rows; r0 += per) {
        const int n = rows - r0 < per ? rows - r0 : per;
        const unsigned total = (unsigned)n * (xtype == MX_F32 ? 8u : 4u) * (unsigned)nb;
        uint8_t *qr = q + (size_t)r0 * nb * 16, *sr = scale + (size_t)r0 * nb;
        const char *xr = (const char *)x + (size_t)r0 * ld * es;
        const dim3 grid((total + 511) / 512), block(256);
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
    const int vec = K % 4 == 0 && ((uintptr_t)y & (4 * es - 1)) == 0;
    for (int r0 = 0; r0 < rows; r0 += per) {
        const int n = rows - r0 < per ? rows - r0 : per;
        const unsigned total = (unsigned)n * 8u * (unsigned)nb;
        const uint8_t *qr = q + (size_t)r0 * nb * 16, *sr = scale + (size_t)r0 * nb;
        char *yr = (char *)y + (size_t)r0 * K * es;
        const dim3 grid((total + 511) / 512), block(256);
        if (ytype == MX_F32) hipLaunchKernelGGL(k_mx4_dequant<MX_F32>, grid, block, 0, s, yr, qr, sr, total, K, nb, vec);
        else if (ytype == MX_F16) hipLaunchKernelGGL(k_mx4_dequant<MX_F16>, grid, block, 0, s, yr, qr, sr, total, K, nb, vec);
        else hipLaunchKernelGGL(k_mx4_dequant<MX_BF16>, grid, block, 0, s, yr, qr, sr, total, K, nb, vec);
    }
    return hipGetLastError();
}
