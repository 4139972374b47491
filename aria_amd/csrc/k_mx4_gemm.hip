/*
 * k_mx4_gemm.hip - products of MXFP4 rows on gfx950's block-scaled MFMA:
 * y[m, n] = sum over blocks b of 2^(ex[m,b] + ew[n,b] - 254) sum_i cx[m,b,i] cw[n,b,i] (+ bias[n]),
 * and the gated form y[m, i] = v * g / (1 + e^-g) with v, g the products of weight rows i and
 * inner + i. fp4 x fp4 products and their block sums are exact; sums over blocks are fp32.
 *
 * v_mfma_scale_f32_32x32x64_f8f6f4 takes one block of 32 codes (16 bytes) and one scale byte per
 * lane and operand, so a packed row is the operand as it lies in memory: no unpacking at all. Weights
 * are the A operand and activations the B operand: a lane's accumulators are then 4 consecutive
 * columns n of one row m.
 */
#include "mx4_dev.h"

struct MxArgs {
    void *y;
    const uint8_t *xq, *xs, *wq, *ws;
    const float *bias;
    int M, N;          /* N: output columns (GLU: inner) */
    int nb;            /* blocks of 32 along K */
    int ytype;
    int tn, T;         /* tiles along N, tiles in all */
};

__device__ __forceinline__ float mx_glu(float v, float g) { return v * silu_f(g); }

/* One wave per 32 x 32 outputs (GLU: two accumulators). */
template <bool GLU>
__global__ __launch_bounds__(64) void k_mx4_tile(MxArgs a) {
    const int t = blockIdx.x, lane = threadIdx.x, l32 = lane & 31, h = lane >> 5;
    const int m0 = (t / a.tn) * 32, n0 = (t % a.tn) * 32;
    const int m = min(m0 + l32, a.M - 1), n = min(n0 + l32, a.N - 1);
    const uint4 *xr = (const uint4 *)a.xq + (size_t)m * a.nb;
    const uint8_t *xsr = a.xs + (size_t)m * a.nb;
    mx_f32x16_t acc[GLU ? 2 : 1];
#pragma unroll
    for (int g = 0; g < (GLU ? 2 : 1); g++)
#pragma unroll
        for (int r = 0; r < 16; r++) acc[g][r] = 0.0f;
    for (int b = 0; b < a.nb; b += 2) {
        const bool in = b + h < a.nb;          /* an absent block: codes zero, scale one */
        const uint4 z = make_uint4(0, 0, 0, 0);
        const uint4 xv = in ? xr[b + h] : z;
        const int xsc = in ? xsr[b + h] : 127;
#pragma unroll
        for (int g = 0; g < (GLU ? 2 : 1); g++) {
            const size_t wr = (size_t)(n + g * a.N) * a.nb + b + h;
            const uint4 wv = in ? ((const uint4 *)a.wq)[wr] : z;
            const int wsc = in ? a.ws[wr] : 127;
            acc[g] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(mx_op(wv), mx_op(xv), acc[g], 4, 4, 0, wsc, 0, xsc);
        }
    }
    if (m0 + l32 >= a.M) return;
#pragma unroll
    for (int r = 0; r < 16; r++) {
        const int c = n0 + 8 * (r >> 2) + 4 * h + (r & 3);
        if (c >= a.N) continue;
        float v = acc[0][r];
        if (a.bias) v += a.bias[c];
        if constexpr (GLU) {
            float g = acc[1][r];
            if (a.bias) g += a.bias[a.N + c];
            v = mx_glu(v, g);
        }
        mx_store(a.y, a.ytype, (size_t)(m0 + l32) * a.N + c, v);
    }
}

extern "C" hipError_t aria_k_mx4_gemm(void *y, int ytype, const uint8_t *xq, const uint8_t *xs, const uint8_t *wq,
                                      const uint8_t *ws, const float *bias, int M, int K, int N, int glu, hipStream_t s) {
    if (M <= 0 || N <= 0) return hipSuccess;
    MxArgs a = {y, xq, xs, wq, ws, bias, M, N, (K + 31) / 32, ytype, 0, 0};
    a.tn = (N + 31) / 32;
    a.T = a.tn * ((M + 31) / 32);
    if (glu) hipLaunchKernelGGL(k_mx4_tile<true>, dim3(a.T), dim3(64), 0, s, a);
    else hipLaunchKernelGGL(k_mx4_tile<false>, dim3(a.T), dim3(64), 0, s, a);
    return hipGetLastError();
}
