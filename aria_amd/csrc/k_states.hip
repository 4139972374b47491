/*
 * k_states.hip - rotary positions and the 8-bit cache of keys and values (gfx950): tables of
 * cos and sin, rotation of queries and keys, keys and values written as e4m3 rows and read back.
 *
 * Rotation: (a, b) -> (a c - b s, b c + a s) on the pairs (i, i + rot/2) or (2i, 2i + 1); c and s are row p
 * of fp32 tables. A row of the cache is D codes x / 2^e to nearest even under the smallest power of two 2^e that
 * brings the row's largest magnitude to 448 or less: a power of two scales exactly, so a code is the value rounded
 * once, and e4m3's own exponent makes a finer scale unnecessary.
 *
 * All of it is bound by bytes (or, for single tokens, by the launch): a group of lanes holds one row in registers
 * from load to store, the row's maximum goes through lane exchanges, and a group takes several heads of one token, so that
 * table rows are read once for them and more loads are in flight.
 */
#include "aria_dev.h"
#include "aria_hip_kernels.h"

#include <algorithm>

template <int T> struct StT;
template <> struct StT<0> { using type = float; };
template <> struct StT<1> { using type = _Float16; };
template <> struct StT<2> { using type = __bf16; };

/* ---- tables ---- */

struct TabArgs {
    float *c, *s;
    int64_t first;
    int n, rh;
    float gain;
    double turns[128];
};

/* The angle in turns, t = p f / 2 pi, loses its whole turns in 64 bits; what is left, at most half a turn, is an fp32 number
 * of half turns to a relative 2^-24. */
__global__ __launch_bounds__(256) void k_rotary_table(TabArgs a) {
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (at >= (int64_t)a.n * a.rh) return;
    const int p = (int)(at / a.rh), i = (int)(at % a.rh);
    const double t = (double)(a.first + p) * a.turns[i];
    float c, s;
    s = sinpif(2.0f * (float)(t - __builtin_rint(t)));
    c = cospif(2.0f * (float)(t - __builtin_rint(t)));
    a.c[at] = c * a.gain;
    a.s[at] = s * a.gain;
}

extern "C" hipError_t aria_k_rotary_table(float *cos_t, float *sin_t, const double *turns, int rot, double gain,
                                          int64_t first, int n, hipStream_t s) {
    TabArgs a;
    a.c = cos_t;
    a.s = sin_t;
    a.first = first;
    a.n = n;
    a.rh = rot / 2;
    a.gain = (float)gain;
    for (int i = 0; i < 128; i++) a.turns[i] = i < rot / 2 ? turns[i] : 0.0;
    const int64_t blocks = ((int64_t)n * a.rh + 255) / 256;
    hipLaunchKernelGGL(k_rotary_table, dim3((unsigned)blocks), dim3(256), 0, s, a);
    return hipGetLastError();
}

/* ---- rotation and the cache ---- */

/* elements off .. off + n - 1 of p (n at most 8, the others read as zero) as eight elements; p + off has its element's
 * alignment only */
template <typename T>
__device__ __forceinline__ void ld8(const T *p, int n, T (&f)[8]) {
    if (n >= 8) {
        __builtin_memcpy(f, p, sizeof f);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) f[i] = i < n ? p[i] : (T)0.0f;
    }
}
template <typename T>
__device__ __forceinline__ void st8(T *p, int n, const T (&f)[8]) {
    if (n >= 8) {
        __builtin_memcpy(p, f, sizeof f);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i < n) p[i] = f[i];
    }
}

/* the larger of two magnitudes as bits: an Inf or a NaN is above every finite value */
struct OpMaxBits {
    __device__ __forceinline__ float operator()(float a, float b) const {
        return __builtin_bit_cast(float, max(__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b)));
    }
};

#define ST_GRID (1 << 20)    /* workgroups of a launch at most */

/* one section of heads: states to states (rotated), or to rows of the cache */
struct StSec {
    const void *src;
    void *dst;               /* states, or codes */
    uint8_t *scale;          /* the cache's bytes; NULL: states to states */
    int64_t sb, st, sh;      /* source strides, elements */
    int64_t db, dt, dh;      /* destination strides, elements or bytes; of the cache dt is per slot */
    int64_t cb, ch;          /* strides of scale */
    int heads, rotate, chunks;
};
struct StArgs {
    StSec sec[3];
    const float *cos_t, *sin_t;
    const int32_t *pos, *first, *count;
    int64_t pos_stride;
    int B, N, D, rot, npos, cap, inverse;
    int nsec, chunks;        /* sections, and groups of HG heads in all of them */
    int64_t blocks;          /* workgroups' shares: one, or every ST_GRID-th, to each */
    int lr;                  /* lanes that hold rotated pairs */
};

/* A group of LPR lanes takes HG heads of one token. Lane l < lr holds the pairs 8 l .. 8 l + 7, the others 16 plain
 * dims each, as two runs of eight: a at ia, b at ib. The products and the sum of a rotation are fp32 where the result is rounded
 * to 16 bits; where it is an fp32 number (fp32 states, keys before they are quantised) they are 64 bits wide, so that it is
 * the rounded exact value and a code does not depend on the order of two roundings. */
template <int TY, bool INTER, int LPR, int HG>
__global__ __launch_bounds__(256) void k_states(StArgs x) {
    using T = typename StT<TY>::type;
    const int l = threadIdx.x % LPR;
    auto work = [&](int64_t blk) __attribute__((always_inline)) {
        int chunk = (int)(blk % x.chunks);
        const unsigned tok = (unsigned)(blk / x.chunks) * (256 / LPR) + threadIdx.x / LPR;   /* B N is at most 2^30 */
        int si = 0;
        while (si + 1 < x.nsec && chunk >= x.sec[si].chunks) chunk -= x.sec[si++].chunks;
        const StSec &s = x.sec[si];
        if (tok >= (unsigned)x.B * x.N) return;
        const int b = (int)(tok / (unsigned)x.N), t = (int)(tok % (unsigned)x.N);
        if (x.count && t >= x.count[b]) return;
        const int64_t slot = (x.first ? (int64_t)x.first[b] : 0) + t;
        const int64_t p = x.pos ? (int64_t)x.pos[b * x.pos_stride + t] : slot;
        if (x.rot && (p < 0 || p >= x.npos)) return;
        if (s.scale && (slot < 0 || slot >= x.cap)) return;

        const int rh = x.rot / 2;
        const bool turn = l < x.lr && s.rotate;      /* this lane's pairs are rotated */
        int ia, ib, na, nb, np;                      /* runs, their lengths, pairs */
        if (l < x.lr) {
            if (INTER) {
                ia = 16 * l;
                ib = ia + 8;
                na = min(8, x.rot - ia);
                nb = max(0, min(8, x.rot - ib));
                np = (na + nb) / 2;
            } else {
                ia = 8 * l;
                ib = rh + ia;
                na = nb = np = min(8, rh - ia);
            }
        } else {
            ia = x.rot + 16 * (l - x.lr);
            ib = ia + 8;
            na = max(0, min(8, x.D - ia));
            nb = max(0, min(8, x.D - ib));
            np = 0;
        }
        const int h0 = chunk * HG, hn = min(HG, s.heads - h0);
        T fa[HG][8], fb[HG][8];
        const T *src = (const T *)s.src + b * s.sb + t * s.st + h0 * s.sh;
#pragma unroll
        for (int h = 0; h < HG; h++) {
            if (h < hn) {
                ld8(src + h * s.sh + ia, na, fa[h]);
                ld8(src + h * s.sh + ib, nb, fb[h]);
            }
        }
        float c[8], sn[8];
        if (turn) {
            ld8(x.cos_t + p * rh + 8 * l, np, c);
            ld8(x.sin_t + p * rh + 8 * l, np, sn);
#pragma unroll
            for (int i = 0; i < 8; i++) sn[i] = x.inverse ? -sn[i] : sn[i];
        }
#pragma unroll
        for (int h = 0; h < HG; h++) {
            if (h >= hn) break;
            float v[16];                             /* run a, then run b */
#pragma unroll
            for (int i = 0; i < 8; i++) {
                v[i] = (float)fa[h][i];
                v[8 + i] = (float)fb[h][i];
            }
            if (turn) {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int ja = INTER ? 2 * i : i, jb = INTER ? 2 * i + 1 : 8 + i;
                    const float u = v[ja], w = v[jb];
                    if (TY == 0 || s.scale) {        /* uniform */
                        v[ja] = (float)__builtin_fma((double)u, (double)c[i], -((double)w * (double)sn[i]));
                        v[jb] = (float)__builtin_fma((double)w, (double)c[i], (double)u * (double)sn[i]);
                    } else {
                        v[ja] = __builtin_fmaf(u, c[i], -(w * sn[i]));
                        v[jb] = __builtin_fmaf(w, c[i], u * sn[i]);
                    }
                }
            }
            if (!s.scale) {
                T *d = (T *)s.dst + b * s.db + t * s.dt + (h0 + h) * s.dh;
                T ya[8], yb[8];
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    ya[i] = (T)v[i];
                    yb[i] = (T)v[8 + i];
                }
                st8(d + ia, na, ya);
                st8(d + ib, nb, yb);
            } else {
                float m = 0.0f;
#pragma unroll
                for (int i = 0; i < 16; i++) m = OpMaxBits()(m, fabsf(v[i]));
                m = grp_reduce<LPR>(m, OpMaxBits());
                const unsigned bits = __builtin_bit_cast(unsigned, m), e = bits >> 23;
                /* 448 = 1.75 * 2^8 */
                const unsigned byte = e == 255u ? 255u : (unsigned)max(1, (int)e - 8 + ((bits & 0x7FFFFFu) > 0x600000u ? 1 : 0));
                const float r = __builtin_bit_cast(float, (254u - min(byte, 253u)) << 23);
                unsigned w[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    int u = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i] * r, v[4 * i + 1] * r, 0, false);
                    u = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i + 2] * r, v[4 * i + 3] * r, u, true);
                    w[i] = byte == 255u ? 0x7F7F7F7Fu : (unsigned)u;
                }
                uint8_t *d = (uint8_t *)s.dst + b * s.db + slot * s.dt + (h0 + h) * s.dh;
                uint8_t wa[8], wb[8];
                __builtin_memcpy(wa, w, 8);
                __builtin_memcpy(wb, w + 2, 8);
                st8(d + ia, na, wa);
                st8(d + ib, nb, wb);
                if (l == 0) s.scale[b * s.cb + (h0 + h) * s.ch + slot] = (uint8_t)byte;
            }
        }
    };
    for (int64_t blk = blockIdx.x; blk < x.blocks; blk += gridDim.x) work(blk);
}

template <int TY, bool INTER, int LPR>
static void st_launch(StArgs &x, hipStream_t s) {
    const int64_t blocks = ((int64_t)x.B * x.N + 256 / LPR - 1) / (256 / LPR);
    /* four heads to a group where that still fills the CUs */
    int64_t four = 0, one = 0;
    for (int i = 0; i < x.nsec; i++) {
        four += (x.sec[i].heads + 3) / 4;
        one += x.sec[i].heads;
    }
    const bool hg4 = blocks * four >= 1024;
    for (int i = 0; i < x.nsec; i++) x.sec[i].chunks = hg4 ? (x.sec[i].heads + 3) / 4 : x.sec[i].heads;
    x.chunks = (int)(hg4 ? four : one);
    x.blocks = blocks * x.chunks;
    const dim3 grid((unsigned)std::min<int64_t>(x.blocks, ST_GRID));
    if (hg4) hipLaunchKernelGGL((k_states<TY, INTER, LPR, 4>), grid, dim3(256), 0, s, x);
    else hipLaunchKernelGGL((k_states<TY, INTER, LPR, 1>), grid, dim3(256), 0, s, x);
}
template <int TY, bool INTER>
static void st_lanes(StArgs &x, int lanes, hipStream_t s) {
    if (lanes <= 4) st_launch<TY, INTER, 4>(x, s);
    else if (lanes <= 8) st_launch<TY, INTER, 8>(x, s);
    else if (lanes <= 16) st_launch<TY, INTER, 16>(x, s);
    else st_launch<TY, INTER, 32>(x, s);
}
template <int TY>
static void st_pairs(StArgs &x, int interleaved, hipStream_t s) {
    const int rh = x.rot / 2;
    x.lr = interleaved ? (x.rot + 15) / 16 : (rh + 7) / 8;
    const int lanes = x.lr + (x.D - x.rot + 15) / 16;     /* at most 17: D 256 with few dims rotated */
    if (interleaved) st_lanes<TY, true>(x, lanes, s);
    else st_lanes<TY, false>(x, lanes, s);
}
static hipError_t st_run(StArgs &x, int type, int interleaved, hipStream_t s) {
    if (x.B <= 0 || x.N <= 0 || x.nsec == 0) return hipSuccess;
    if (type == 0) st_pairs<0>(x, interleaved, s);
    else if (type == 1) st_pairs<1>(x, interleaved, s);
    else st_pairs<2>(x, interleaved, s);
    return hipGetLastError();
}

static void st_add(StArgs &x, const void *src, void *dst, int heads, int64_t sb, int64_t st, int64_t sh, int64_t db, int64_t dt,
                   int64_t dh) {
    if (heads <= 0) return;
    StSec &s = x.sec[x.nsec++];
    s = StSec{src, dst, nullptr, sb, st, sh, db, dt, dh, 0, 0, heads, x.rot > 0, 0};
}

extern "C" hipError_t aria_k_rotary(const aria_hip_rotary *a, hipStream_t s) {
    StArgs x{};
    x.cos_t = a->cos;
    x.sin_t = a->sin;
    x.pos = a->pos;
    x.first = a->first;
    x.pos_stride = a->pos_stride;
    x.B = a->B;
    x.N = a->N;
    x.D = a->D;
    x.rot = a->rot;
    x.npos = a->npos;
    x.inverse = a->inverse != 0;
    if (a->q) st_add(x, a->q, a->q_out, a->Hq, a->q_batch, a->q_token, a->q_head, a->qo_batch, a->qo_token, a->qo_head);
    if (a->k) st_add(x, a->k, a->k_out, a->Hk, a->k_batch, a->k_token, a->k_head, a->ko_batch, a->ko_token, a->ko_head);
    return st_run(x, a->type, a->interleaved, s);
}

extern "C" hipError_t aria_k_kv_write(const aria_hip_kv_write *a, hipStream_t s) {
    const aria_hip_kv &c = a->cache;
    StArgs x{};
    x.cos_t = a->cos;
    x.sin_t = a->sin;
    x.pos = a->pos;
    x.first = a->first;
    x.count = a->count;
    x.pos_stride = a->pos_stride;
    x.B = c.B;
    x.N = a->N;
    x.D = c.D;
    x.rot = a->cos ? a->rot : 0;
    x.npos = a->npos;
    x.cap = c.cap;
    if (c.cap > 0) {
        st_add(x, a->k, c.k, c.Hkv, a->k_batch, a->k_token, a->k_head, c.batch, c.token, c.head);
        st_add(x, a->v, c.v, c.Hkv, a->v_batch, a->v_token, a->v_head, c.batch, c.token, c.head);
        for (int i = 0; i < 2; i++) {
            x.sec[i].scale = i ? c.v_scale : c.k_scale;
            x.sec[i].cb = c.s_batch;
            x.sec[i].ch = c.s_head;
        }
        x.sec[1].rotate = 0;
    }
    if (a->q) st_add(x, a->q, a->q_out, a->Hq, a->q_batch, a->q_token, a->q_head, a->qo_batch, a->qo_token, a->qo_head);
    return st_run(x, a->type, a->interleaved, s);
}

/* ---- the cache read back ---- */

struct RdArgs {
    aria_hip_kv_read a;
    int chunks, two;         /* groups of HG heads of one operand; both operands are read */
    int64_t blocks;
};

/* LPR lanes to a row, 16 codes to a lane; keys and values in one launch. A row's largest code may lie past the type's
 * largest number (65504 in fp16 is 65536 as a code): it is held to it; a NaN stays one */
template <int TY, int LPR, int HG>
__global__ __launch_bounds__(256) void k_kv_read(RdArgs x) {
    using T = typename StT<TY>::type;
    const aria_hip_kv_read &a = x.a;
    const aria_hip_kv &c = a.cache;
    constexpr float most = TY == 0 ? 3.40282347e38f : TY == 1 ? 65504.0f : 3.38953139e38f;
    auto held = [](float v) __attribute__((always_inline)) {
        return (T)__builtin_elementwise_minimum(__builtin_elementwise_maximum(v, -most), most);
    };
    const int per = x.chunks * (x.two ? 2 : 1);
    const int l = threadIdx.x % LPR;
    auto work = [&](int64_t blk) __attribute__((always_inline)) {
        int chunk = (int)(blk % per);
        const unsigned tok = (unsigned)(blk / per) * (256 / LPR) + threadIdx.x / LPR;
        const bool is_v = x.two ? chunk >= x.chunks : a.k == nullptr;
        if (x.two && is_v) chunk -= x.chunks;
        if (tok >= (unsigned)c.B * a.N || 16 * l >= c.D) return;
        const int b = (int)(tok / (unsigned)a.N), t = (int)(tok % (unsigned)a.N);
        if (a.count && t >= a.count[b]) return;
        const int64_t slot = (a.first ? (int64_t)a.first[b] : 0) + t;
        if (slot < 0 || slot >= c.cap) return;
        const int h0 = chunk * HG, hn = min(HG, c.Hkv - h0);
        const uint8_t *src = (is_v ? c.v : c.k) + b * c.batch + slot * c.token + h0 * c.head + 16 * l;
        const uint8_t *sp = (is_v ? c.v_scale : c.k_scale) + b * c.s_batch + h0 * c.s_head + slot;
        T *dst = is_v ? (T *)a.v + b * a.v_batch + t * a.v_token + h0 * a.v_head + 16 * l
                      : (T *)a.k + b * a.k_batch + t * a.k_token + h0 * a.k_head + 16 * l;
        const int64_t dh = is_v ? a.v_head : a.k_head;
        uint4 u[HG];
        unsigned e[HG];
#pragma unroll
        for (int h = 0; h < HG; h++)
            if (h < hn) {
                u[h] = *reinterpret_cast<const uint4 *>(src + h * c.head);
                e[h] = sp[h * c.s_head];
            }
#pragma unroll
        for (int h = 0; h < HG; h++) {
            if (h >= hn) break;
            const float f = __builtin_bit_cast(float, e[h] << 23);
            const unsigned w[4] = {u[h].x, u[h].y, u[h].z, u[h].w};
            T y[16];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const auto p = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], false), q = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], true);
                y[4 * i] = held(p[0] * f);
                y[4 * i + 1] = held(p[1] * f);
                y[4 * i + 2] = held(q[0] * f);
                y[4 * i + 3] = held(q[1] * f);
            }
            __builtin_memcpy(dst + h * dh, y, sizeof y);
        }
    };
    for (int64_t blk = blockIdx.x; blk < x.blocks; blk += gridDim.x) work(blk);
}

template <int TY, int LPR>
static void rd_launch(RdArgs &x, hipStream_t s) {
    const int64_t blocks = ((int64_t)x.a.cache.B * x.a.N + 256 / LPR - 1) / (256 / LPR);
    const int ops = x.two ? 2 : 1, four = (x.a.cache.Hkv + 3) / 4;
    const bool hg4 = blocks * four * ops >= 1024;
    x.chunks = hg4 ? four : x.a.cache.Hkv;
    x.blocks = blocks * x.chunks * ops;
    const dim3 grid((unsigned)std::min<int64_t>(x.blocks, ST_GRID));
    if (hg4) hipLaunchKernelGGL((k_kv_read<TY, LPR, 4>), grid, dim3(256), 0, s, x);
    else hipLaunchKernelGGL((k_kv_read<TY, LPR, 1>), grid, dim3(256), 0, s, x);
}
template <int TY>
static void rd_lanes(RdArgs &x, hipStream_t s) {
    const int lanes = x.a.cache.D / 16;
    if (lanes <= 4) rd_launch<TY, 4>(x, s);
    else if (lanes <= 8) rd_launch<TY, 8>(x, s);
    else rd_launch<TY, 16>(x, s);
}

extern "C" hipError_t aria_k_kv_read(const aria_hip_kv_read *a, hipStream_t s) {
    RdArgs x;
    x.a = *a;
    x.two = a->k && a->v;
    if (a->cache.B <= 0 || a->N <= 0 || a->cache.cap <= 0 || a->cache.Hkv <= 0 || (!a->k && !a->v)) return hipSuccess;
    if (a->type == 0) rd_lanes<0>(x, s);
    else if (a->type == 1) rd_lanes<1>(x, s);
    else rd_lanes<2>(x, s);
    return hipGetLastError();
}
