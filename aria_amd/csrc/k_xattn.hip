/*
 * k_xattn.hip - cross attention to an encoder's states whose number differs from sequence to
 * sequence (gfx950): o = sum_j p_j v_j, p = softmax over the valid keys of scale * q . k_j, where key
 * j of sequence b is valid when j < kv_len[b] and mask[b, j] != 0. A row without a valid key is zero.
 * H query heads share Hkv key/value heads (H / Hkv consecutive query heads to each).
 */
#include "aria_dev.h"
#include "aria_hip_kernels.h"

/* One wave per query row: scores of 64 keys by lane, running maximum and sum, output dims by lane. */
template <typename T>
__global__ __launch_bounds__(64) void k_xattn_row(aria_k_xattn a) {
    __shared__ float P[64];
    const int lane = threadIdx.x;
    const long long w = blockIdx.x;            /* (b * H + h) * Nq + t */
    const int t = (int)(w % a.Nq), h = (int)(w / a.Nq % a.H), b = (int)(w / a.Nq / a.H), hk = h / (a.H / a.Hkv);
    const T *q = (const T *)a.q + b * a.q_batch + h * a.q_head + t * a.q_token;
    const T *k = (const T *)a.k + b * a.k_batch + hk * a.k_head;
    const T *v = (const T *)a.v + b * a.v_batch + hk * a.v_head;
    const int n = a.kv_len ? min(max(a.kv_len[b], 0), a.Nk) : a.Nk;
    float m = -INFINITY, l = 0.0f, o0 = 0.0f, o1 = 0.0f;
    for (int j0 = 0; j0 < n; j0 += 64) {
        const int j = j0 + lane;
        const bool ok = j < n && (!a.mask || a.mask[b * a.mask_stride + j] != 0);
        float s = 0.0f;
        if (ok)
            for (int d = 0; d < a.D; d++) s = __builtin_fmaf((float)q[d], (float)k[j * a.k_token + d], s);
        s = ok ? s * a.scale : -INFINITY;
        const float mn = fmaxf(m, grp_max<64>(s));
        const float ref = mn == -INFINITY ? 0.0f : mn;
        const float p = ok ? expf(s - ref) : 0.0f, al = expf(m - ref);
        l = l * al + grp_sum<64>(p);
        o0 *= al; o1 *= al; m = mn;
        P[lane] = p;
        __syncthreads();
        for (int i = 0; i < 64 && j0 + i < n; i++) {
            if (P[i] == 0.0f) continue;
            const T *vj = v + (j0 + i) * a.v_token;
            if (lane < a.D) o0 = __builtin_fmaf(P[i], (float)vj[lane], o0);
            if (64 + lane < a.D) o1 = __builtin_fmaf(P[i], (float)vj[64 + lane], o1);
        }
        __syncthreads();
    }
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
    const long long ob = b * a.o_batch + h * a.o_head + t * a.o_token;
    if (a.out_f32) {
        if (lane < a.D) ((float *)a.out)[ob + lane] = o0 * inv;
        if (64 + lane < a.D) ((float *)a.out)[ob + 64 + lane] = o1 * inv;
    } else {
        if (lane < a.D) ((T *)a.out)[ob + lane] = (T)(o0 * inv);
        if (64 + lane < a.D) ((T *)a.out)[ob + 64 + lane] = (T)(o1 * inv);
    }
}

extern "C" size_t aria_k_xattn_ws_bytes(const aria_k_xattn *a) { return 0; }

extern "C" hipError_t aria_k_xattn_run(const aria_k_xattn *a, void *ws, hipStream_t s) {
    if (a->B <= 0 || a->Nq <= 0) return hipSuccess;
    const dim3 grid((unsigned)((long long)a->B * a->H * a->Nq));
    if (a->type == 1) hipLaunchKernelGGL(k_xattn_row<_Float16>, grid, dim3(64), 0, s, *a);
    else hipLaunchKernelGGL(k_xattn_row<__bf16>, grid, dim3(64), 0, s, *a);
    return hipGetLastError();
}
