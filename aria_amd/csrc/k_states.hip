/*
 * k_states.hip - rotary positions and the 8-bit cache of keys and values (gfx950): tables of
 * cos and sin, rotation of queries and keys, keys and values written as e4m3 rows and read back.
 *
 * Rotation: (a, b) -> (a c - b s, b c + a s) on the pairs (i, i + rot/2) or (2i, 2i + 1); c and s are row p
 * of fp32 tables. A row of the cache is D codes x / 2^e to nearest even under the smallest power of two 2^e that
 * brings the row's largest magnitude to 448 or less: a power of two scales exactly, so a code is the value rounded
 * once, and e4m3's own exponent makes a finer scale unnecessary.
 *
 * All of it is bound by bytes, or, for single tokens, by the launch: a group of lanes holds one row in registers
 * from load to store, the row's maximum goes through lane exchanges, and a group takes four heads of one token where that still
 * fills the CUs, so that table rows are read once for them and more loads are in flight. 4 x 8192 tokens of 20 heads of 128 rotated
 * in bf16 (353 MB): 72 us, 4.9 TB/s, what a copy of 1 GiB reaches (83 with two heads, 76 with eight, 128 where odd widths branch in
 * the same kernel). Lanes load and store 16 bytes beside their neighbours': 32 bytes to a lane in two pieces took 106 us for 8 x 4096 tokens of 10 interleaved
 * heads of 128 in fp32 (407 MB), now 76, and 177 for 4 x 8192 tokens of 8 heads of 128 from fp32 to the cache and back (671 MB with the codes), now
 * 147, the most of it in reading. 4 x 16384 tokens of 8 heads written and read back in bf16 (804 MB with the codes): 172 us, of which the keys'
 * rotation in 64 bits costs 9. One token of 64 sequences: two launches of 3 us.
 */
#include "aria_dev.h"
#include "aria_hip_kernels.h"

#include <algorithm>

template <int T> struct StT;
template <> struct StT<0> { using type = float; };
template <> struct StT<1> { using type = _Float16; };
template <> struct StT<2> { using type = __bf16; };

/* ---- tables ---- */

#define TAB_EACH 4           /* positions of a thread */
struct TabArgs {
    float *c, *s;
    int64_t first, threads;
    int n, rh, groups;       /* positions, pairs, groups of V pairs */
    HostDiv dgroups;
    float gain;
    double turns[128];
};

/* cos and sin of a turns' fraction. The nearest quarter leaves t in 64 bits, exactly; of what is left, at most an eighth, the
 * Taylor series to x^10 and x^9 (the next terms are below 1.2e-10 and 1.8e-9), 2 pi in two parts */
__device__ __forceinline__ void tab_cos_sin(double t, float &c, float &s) {
    const double r = t - __builtin_rint(t), q = __builtin_rint(4.0 * r);
    const float x = (float)__builtin_fma(q, -0.25, r), z = x * x;
    const int k = (int)q;
    const float ps = __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, 42.0586939f, -76.7058598f), 81.6052493f), -41.3417022f), -1.7484556e-07f);
    const float a = __builtin_fmaf(x, 6.28318531f, x * ps);
    const float pc = __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, -26.4262568f, 60.2446414f), -85.4568172f), 64.939394f), -19.7392088f);
    const float b = __builtin_fmaf(z, pc, 1.0f);
    const float u = k & 1 ? b : a, v = k & 1 ? a : b;
    s = k & 2 ? -u : u;
    c = (k + 1) & 2 ? -v : v;
}

/* A thread makes V neighbouring pairs of TAB_EACH positions, whose frequencies it loads once: 131072 x 64 pairs (67 MB) in 13.4 us,
 * where a fill of as many bytes takes 11.4 (20 us with the device library's functions of half turns, a pair to a thread) */
template <int V>
__global__ __launch_bounds__(256) void k_rotary_table(TabArgs a) {
    typedef float fv __attribute__((ext_vector_type(V), aligned(4)));
    fetch_args(a);
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (at >= a.threads) return;
    const unsigned row = a.dgroups.of((unsigned)at), g = (unsigned)at - row * a.groups, rows = (unsigned)(a.n + TAB_EACH - 1) / TAB_EACH;
    double f[V];
#pragma unroll
    for (int i = 0; i < V; i++) f[i] = a.turns[V * g + i];
#pragma unroll
    for (int j = 0; j < TAB_EACH; j++) {
        const unsigned n = row + j * rows;                   /* neighbouring threads write neighbouring positions */
        if (n >= (unsigned)a.n) break;
        const double p = (double)(a.first + n);
        fv c, s;
#pragma unroll
        for (int i = 0; i < V; i++) {
            float u, w;
            tab_cos_sin(p * f[i], u, w);
            c[i] = u * a.gain;
            s[i] = w * a.gain;
        }
        const int64_t o = (int64_t)n * a.rh + V * g;
        *reinterpret_cast<fv *>(a.c + o) = c;
        *reinterpret_cast<fv *>(a.s + o) = s;
    }
}

extern "C" hipError_t aria_k_rotary_table(float *cos_t, float *sin_t, const double *turns, int rot, double gain,
                                          int64_t first, int n, hipStream_t s) {
    TabArgs a{};
    a.c = cos_t;
    a.s = sin_t;
    a.first = first;
    a.n = n;
    a.rh = rot / 2;
    a.gain = (float)gain;
    for (int i = 0; i < rot / 2; i++) a.turns[i] = turns[i];
    const int V = a.rh % 4 == 0 ? 4 : 1;
    a.groups = a.rh / V;
    a.dgroups = HostDiv(a.groups);
    a.threads = (int64_t)((n + TAB_EACH - 1) / TAB_EACH) * a.groups;      /* below 2^30: n is at most 2^24 + 1 */
    const dim3 grid((unsigned)((a.threads + 255) / 256));
    if (V == 4) hipLaunchKernelGGL((k_rotary_table<4>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((k_rotary_table<1>), grid, dim3(256), 0, s, a);
    return hipGetLastError();
}

/* ---- rotation and the cache ---- */

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
    HostDiv dn, dchunks;
};

/* a and b of a pair, rotated. The products and the sum are fp32 where the result is rounded to 16 bits; where it is an fp32
 * number (fp32 states, keys before they are quantised) they are 64 bits wide, so that it is the rounded exact value and a code
 * does not hang on the order of two roundings */
__device__ __forceinline__ void st_turn(float &a, float &b, float c, float s) {
    const float u = a, w = b;
    a = __builtin_fmaf(u, c, -(w * s));
    b = __builtin_fmaf(w, c, u * s);
}
__device__ __forceinline__ void st_turn(float &a, float &b, double c, double s) {
    const double u = a, w = b;
    a = (float)__builtin_fma(u, c, -(w * s));
    b = (float)__builtin_fma(w, c, u * s);
}
/* the byte of a row from the bits of its largest magnitude; 448 = 1.75 * 2^8 */
__device__ __forceinline__ unsigned st_byte(unsigned bits) {
    const unsigned e = bits >> 23;
    return e == 255u ? 255u : (unsigned)max(1, (int)e - 8 + ((bits & 0x7FFFFFu) > 0x600000u ? 1 : 0));
}
/* 2^(127 - byte) */
__device__ __forceinline__ float st_inverse(unsigned byte) { return __builtin_bit_cast(float, (254u - min(byte, 253u)) << 23); }

/* where a share's token lies; false: it is none, or not to be written */
struct StTok {
    int b, t;
    int64_t slot, p;
};
__device__ __forceinline__ bool st_token(const StArgs &x, const StSec &s, unsigned tok, StTok &k) {
    if (tok >= (unsigned)x.B * x.N) return false;
    k.b = x.dn.of(tok);
    k.t = tok - k.b * x.N;
    if (x.count && k.t >= x.count[k.b]) return false;
    k.slot = (x.first ? (int64_t)x.first[k.b] : 0) + k.t;
    k.p = x.pos ? (int64_t)x.pos[k.b * x.pos_stride + k.t] : k.slot;
    if (x.rot && (k.p < 0 || k.p >= x.npos)) return false;
    return !(s.scale && (k.slot < 0 || k.slot >= x.cap));
}

/* Whole chunks of 16 bytes, CW elements: D and rot multiples of CW (interleaved), rot of 2 CW (halves). A group of LPR lanes takes
 * HG heads of one token, two chunks of each to a lane, so that neighbouring lanes' chunks are neighbours: interleaved the chunks l and
 * l + (half of them), else those of the pairs CW l .. CW l + CW - 1, and behind the rotated dims two plain ones. Every load of the
 * HG rows is on its way before the first is used; chunks and heads past the last repeat it, are not stored and do not count in a row's
 * maximum. */
template <int TY, bool INTER, int LPR, int HG>
__global__ __launch_bounds__(256) void k_states(StArgs x) {
    using T = typename StT<TY>::type;
    constexpr int CW = 16 / sizeof(T), CH = CW / 2;
    typedef T vc __attribute__((ext_vector_type(CW), aligned(alignof(T))));
    typedef float fh __attribute__((ext_vector_type(CH), aligned(4)));
    fetch_args(x);
    const int l = threadIdx.x % LPR, rh = x.rot / 2, nc = x.D / CW;
    /* the lane's chunks, and whether their pairs are rotated */
    int ca, cb;
    bool ra, rb, ha;
    if (INTER) {
        const int half = (nc + 1) / 2;
        ca = l;
        cb = l + half;
        ha = l < half;
        ra = CW * ca < x.rot;
        rb = CW * cb < x.rot;
    } else {
        const int lr = rh / CW, half = (nc - 2 * lr + 1) / 2;
        ra = rb = l < lr;
        ca = ra ? l : l + lr;
        cb = ra ? l + lr : ca + half;
        ha = l < lr + half;
    }
    const bool hb = ha && cb < nc;
    const int ia = CW * min(ca, nc - 1), ib = CW * min(cb, nc - 1);
    /* their tables' columns */
    const int ta = min(INTER ? CH * ca : CW * l, max(rh - CH, 0)), tb = min(INTER ? CH * cb : CW * l + CH, max(rh - CH, 0));

    for (int64_t blk = blockIdx.x; blk < x.blocks; blk += gridDim.x) {
        const unsigned tb_ = x.blocks <= 0x7FFFFFFF ? x.dchunks.of((unsigned)blk) : (unsigned)(blk / x.chunks);
        int chunk = (int)(blk - (int64_t)tb_ * x.chunks), si = 0;
        while (si + 1 < x.nsec && chunk >= x.sec[si].chunks) chunk -= x.sec[si++].chunks;
        const StSec &s = x.sec[si];
        StTok k;
        if (!st_token(x, s, tb_ * (256 / LPR) + threadIdx.x / LPR, k)) continue;
        const int h0 = chunk * HG, hn = min(HG, s.heads - h0);
        vc fa[HG], fb[HG];
        const T *src = (const T *)s.src + k.b * s.sb + k.t * s.st + h0 * s.sh;
#pragma unroll
        for (int h = 0; h < HG; h++) {
            const T *r = src + min(h, hn - 1) * s.sh;
            fa[h] = *reinterpret_cast<const vc *>(r + ia);
            fb[h] = *reinterpret_cast<const vc *>(r + ib);
        }
        fh c[2], sn[2];
        const bool turn = s.rotate;                  /* uniform */
        if (turn) {
            const float *ct = x.cos_t + k.p * rh, *st = x.sin_t + k.p * rh;
            c[0] = *reinterpret_cast<const fh *>(ct + ta);
            c[1] = *reinterpret_cast<const fh *>(ct + tb);
            sn[0] = *reinterpret_cast<const fh *>(st + ta);
            sn[1] = *reinterpret_cast<const fh *>(st + tb);
#pragma unroll
            for (int i = 0; i < CH; i++) {
                c[0][i] = ra ? c[0][i] : 1.0f;       /* plain dims: by one and zero */
                c[1][i] = rb ? c[1][i] : 1.0f;
                sn[0][i] = ra ? (x.inverse ? -sn[0][i] : sn[0][i]) : 0.0f;
                sn[1][i] = rb ? (x.inverse ? -sn[1][i] : sn[1][i]) : 0.0f;
            }
        }
        auto rows = [&](auto TURN, auto CACHE) __attribute__((always_inline)) {
            constexpr bool turned = decltype(TURN)::value != 0, cache = decltype(CACHE)::value != 0;
            using W = std::conditional_t<TY == 0 || cache, double, float>;
            W cw[CW], sw[CW];
            if constexpr (turned)
#pragma unroll
                for (int i = 0; i < CW; i++) {
                    cw[i] = c[i / CH][i % CH];
                    sw[i] = sn[i / CH][i % CH];
                }
#pragma unroll
            for (int h = 0; h < HG; h++) {
                float v[2 * CW];                         /* chunk a, then chunk b */
#pragma unroll
                for (int i = 0; i < CW; i++) {
                    v[i] = (float)fa[h][i];
                    v[CW + i] = (float)fb[h][i];
                }
                if constexpr (turned) {
#pragma unroll
                    for (int i = 0; i < CW; i++) {
                        const int ja = INTER ? 2 * i : i, jb = INTER ? 2 * i + 1 : CW + i;
                        st_turn(v[ja], v[jb], cw[i], sw[i]);
                    }
                    if (!(ra && rb)) {               /* plain dims as they came: 0 times an Inf is none of theirs */
#pragma unroll
                        for (int i = 0; i < CW; i++) {
                            v[i] = ra ? v[i] : (float)fa[h][i];
                            v[CW + i] = rb ? v[CW + i] : (float)fb[h][i];
                        }
                    }
                }
                if constexpr (!cache) {
                    if (h >= hn) break;
                    T *d = (T *)s.dst + k.b * s.db + k.t * s.dt + (h0 + h) * s.dh;
                    vc y;
                    if (ha) {
#pragma unroll
                        for (int i = 0; i < CW; i++) y[i] = (T)v[i];
                        *reinterpret_cast<vc *>(d + ia) = y;
                    }
                    if (hb) {
#pragma unroll
                        for (int i = 0; i < CW; i++) y[i] = (T)v[CW + i];
                        *reinterpret_cast<vc *>(d + ib) = y;
                    }
                } else {
                    float ma = 0.0f, mb = 0.0f;
#pragma unroll
                    for (int i = 0; i < CW; i++) {
                        ma = OpMaxBits()(ma, fabsf(v[i]));
                        mb = OpMaxBits()(mb, fabsf(v[CW + i]));
                    }
                    /* a repeated chunk does not count: it is not rotated as its owner's is */
                    const float m = grp_reduce<LPR>(OpMaxBits()(ha ? ma : 0.0f, hb ? mb : 0.0f), OpMaxBits());
                    const unsigned byte = st_byte(__builtin_bit_cast(unsigned, m));
                    const float r = st_inverse(byte);
                    unsigned w[CH];
#pragma unroll
                    for (int i = 0; i < CH; i++) {
                        int u = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i] * r, v[4 * i + 1] * r, 0, false);
                        u = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i + 2] * r, v[4 * i + 3] * r, u, true);
                        w[i] = byte == 255u ? 0x7F7F7F7Fu : (unsigned)u;
                    }
                    if (h >= hn) break;
                    uint8_t *d = (uint8_t *)s.dst + k.b * s.db + k.slot * s.dt + (h0 + h) * s.dh;
                    if (ha) __builtin_memcpy(__builtin_assume_aligned(d + ia, CW), w, CW);
                    if (hb) __builtin_memcpy(__builtin_assume_aligned(d + ib, CW), w + CW / 4, CW);
                    if (l == 0) s.scale[k.b * s.cb + (h0 + h) * s.ch + k.slot] = (uint8_t)byte;
                }
            }
        };
        if (s.scale) {
            if (turn) rows(IC<1>{}, IC<1>{});
            else rows(IC<0>{}, IC<1>{});
        } else {
            if (turn) rows(IC<1>{}, IC<0>{});
            else rows(IC<0>{}, IC<0>{});
        }
    }
}

/* Any even D and rot: a wave takes HG heads of one token, a pair of dims to a lane (two, where D is over 128); pair p is
 * (p, p + rot/2) or (2p, 2p + 1) and, behind the rotated ones, (2p, 2p + 1). */
template <int TY, bool INTER, int HG>
__global__ __launch_bounds__(256) void k_states_any(StArgs x) {
    using T = typename StT<TY>::type;
    constexpr int PL = 2;
    fetch_args(x);
    const int lane = threadIdx.x & 63, rh = x.rot / 2, np = x.D / 2;
    int ia[PL], ib[PL], col[PL];
    bool turns[PL], have[PL];
#pragma unroll
    for (int i = 0; i < PL; i++) {
        const int p = min(lane + 64 * i, np - 1);
        have[i] = lane + 64 * i < np;
        turns[i] = p < rh;
        ia[i] = !INTER && turns[i] ? p : 2 * p;
        ib[i] = !INTER && turns[i] ? p + rh : 2 * p + 1;
        col[i] = min(p, max(rh - 1, 0));
    }
    const bool two = np > 64;
    for (int64_t blk = blockIdx.x; blk < x.blocks; blk += gridDim.x) {
        const unsigned tb = x.blocks <= 0x7FFFFFFF ? x.dchunks.of((unsigned)blk) : (unsigned)(blk / x.chunks);
        int chunk = (int)(blk - (int64_t)tb * x.chunks), si = 0;
        while (si + 1 < x.nsec && chunk >= x.sec[si].chunks) chunk -= x.sec[si++].chunks;
        const StSec &s = x.sec[si];
        StTok k;
        if (!st_token(x, s, tb * 4 + threadIdx.x / 64, k)) continue;
        const int h0 = chunk * HG, hn = min(HG, s.heads - h0);
        T fa[HG][PL], fb[HG][PL];
        const T *src = (const T *)s.src + k.b * s.sb + k.t * s.st + h0 * s.sh;
#pragma unroll
        for (int h = 0; h < HG; h++) {
            const T *r = src + min(h, hn - 1) * s.sh;
#pragma unroll
            for (int i = 0; i < PL; i++) {
                if (i && !two) break;
                fa[h][i] = r[ia[i]];
                fb[h][i] = r[ib[i]];
            }
        }
        float c[PL] = {1.0f, 1.0f}, sn[PL] = {0.0f, 0.0f};
        if (s.rotate) {
#pragma unroll
            for (int i = 0; i < PL; i++) {
                if (i && !two) break;
                c[i] = x.cos_t[k.p * rh + col[i]];
                sn[i] = x.sin_t[k.p * rh + col[i]];
                sn[i] = x.inverse ? -sn[i] : sn[i];
            }
        }
#pragma unroll
        for (int h = 0; h < HG; h++) {
            if (h >= hn) break;
            float a[PL], b[PL], m = 0.0f;
#pragma unroll
            for (int i = 0; i < PL; i++) {
                if (i && !two) break;
                a[i] = (float)fa[h][i];
                b[i] = (float)fb[h][i];
                if (s.rotate && turns[i]) {
                    if (TY == 0 || s.scale) st_turn(a[i], b[i], (double)c[i], (double)sn[i]);
                    else st_turn(a[i], b[i], c[i], sn[i]);
                }
                m = OpMaxBits()(m, OpMaxBits()(fabsf(a[i]), fabsf(b[i])));
            }
            if (!s.scale) {
                T *d = (T *)s.dst + k.b * s.db + k.t * s.dt + (h0 + h) * s.dh;
#pragma unroll
                for (int i = 0; i < PL; i++)
                    if (have[i]) {
                        d[ia[i]] = (T)a[i];
                        d[ib[i]] = (T)b[i];
                    }
                continue;
            }
            m = grp_reduce<64>(m, OpMaxBits());
            const unsigned byte = st_byte(__builtin_bit_cast(unsigned, m));
            const float r = st_inverse(byte);
            uint8_t *d = (uint8_t *)s.dst + k.b * s.db + k.slot * s.dt + (h0 + h) * s.dh;
#pragma unroll
            for (int i = 0; i < PL; i++)
                if (have[i]) {
                    const unsigned w = byte == 255u ? 0x7F7Fu : (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(a[i] * r, b[i] * r, 0, false);
                    d[ia[i]] = (uint8_t)w;
                    d[ib[i]] = (uint8_t)(w >> 8);
                }
            if (lane == 0) s.scale[k.b * s.cb + (h0 + h) * s.ch + k.slot] = (uint8_t)byte;
        }
    }
}

/* shares of `per` tokens, and how many heads a group takes: four, or two where no section has more (two heads of 32 in groups of
 * four: 80 us, 59 x 9154 tokens in fp16; of two: 50), where that makes `enough` workgroups to fill the CUs; else two, where that makes
 * half as many (2 x 1296 tokens of 16 heads of 64, written and read back: 12.1 us with one head, 11.2 with two; 26 x 373 tokens of 20 heads
 * of 32 rotated 8.1 and 6.5; of 366 shapes the worst lost 7 %); else one. Whole chunks: 1024 (thresholds of 256 and 512 for four heads cost
 * some shapes of 500 to 1000 workgroups up to 12 %, 2048 gained one 15 % and lost others 4 %). A wave to a row: 320, since starting four
 * times the workgroups costs more (rotated heads of 128: 192 groups of four 3.41 us with one head and 3.54 with four, 384 4.28 and
 * 3.78, 1536 10.2 and 6.0) */
static int st_shares(StArgs &x, int per, int enough) {
    const int64_t blocks = ((int64_t)x.B * x.N + per - 1) / per;
    int most = 0;
    for (int i = 0; i < x.nsec; i++) most = std::max(most, x.sec[i].heads);
    auto chunks = [&](int hg) {
        int64_t n = 0;
        for (int i = 0; i < x.nsec; i++) n += (x.sec[i].heads + hg - 1) / hg;
        return n;
    };
    int hg = most > 2 ? 4 : most;
    if (hg == 4 && blocks * chunks(4) < enough) hg = 2;
    if (hg == 2 && blocks * chunks(2) < enough / 2) hg = 1;
    for (int i = 0; i < x.nsec; i++) x.sec[i].chunks = (x.sec[i].heads + hg - 1) / hg;
    x.chunks = (int)chunks(hg);
    x.blocks = blocks * x.chunks;
    x.dn = HostDiv(x.N);
    x.dchunks = HostDiv(x.chunks);
    return hg;
}
template <int TY, bool INTER, int LPR>
static void st_launch(StArgs &x, hipStream_t s) {
    const int hg = st_shares(x, 256 / LPR, 1024);
    const dim3 grid((unsigned)std::min<int64_t>(x.blocks, ST_GRID));
    if (hg == 4) hipLaunchKernelGGL((k_states<TY, INTER, LPR, 4>), grid, dim3(256), 0, s, x);
    else if (hg == 2) hipLaunchKernelGGL((k_states<TY, INTER, LPR, 2>), grid, dim3(256), 0, s, x);
    else hipLaunchKernelGGL((k_states<TY, INTER, LPR, 1>), grid, dim3(256), 0, s, x);
}
template <int TY, bool INTER>
static void st_pairs(StArgs &x, hipStream_t s) {
    constexpr int CW = TY == 0 ? 4 : 8;
    if (x.D % CW == 0 && x.rot % (INTER ? CW : 2 * CW) == 0) {
        const int lanes = (x.D + 2 * CW - 1) / (2 * CW);
        if (lanes <= 2) st_launch<TY, INTER, 2>(x, s);
        else if (lanes <= 4) st_launch<TY, INTER, 4>(x, s);
        else if (lanes <= 8) st_launch<TY, INTER, 8>(x, s);
        else if (TY || lanes <= 16) st_launch<TY, INTER, 16>(x, s);
        else if constexpr (TY == 0) st_launch<TY, INTER, 32>(x, s);
        return;
    }
    const int hg = st_shares(x, 4, 320);
    const dim3 grid((unsigned)std::min<int64_t>(x.blocks, ST_GRID));
    if (hg == 4) hipLaunchKernelGGL((k_states_any<TY, INTER, 4>), grid, dim3(256), 0, s, x);
    else if (hg == 2) hipLaunchKernelGGL((k_states_any<TY, INTER, 2>), grid, dim3(256), 0, s, x);
    else hipLaunchKernelGGL((k_states_any<TY, INTER, 1>), grid, dim3(256), 0, s, x);
}
static hipError_t st_run(StArgs &x, int type, int interleaved, hipStream_t s) {
    if (x.B <= 0 || x.N <= 0 || x.nsec == 0) return hipSuccess;
    if (type == 0) interleaved ? st_pairs<0, true>(x, s) : st_pairs<0, false>(x, s);
    else if (type == 1) interleaved ? st_pairs<1, true>(x, s) : st_pairs<1, false>(x, s);
    else interleaved ? st_pairs<2, true>(x, s) : st_pairs<2, false>(x, s);
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
    x.rot = a->rot;
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
    constexpr int CW = 16 / sizeof(T);
    typedef T vc __attribute__((ext_vector_type(CW), aligned(alignof(T))));
    typedef unsigned uc __attribute__((ext_vector_type(CW / 4), aligned(CW)));
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
        if (tok >= (unsigned)c.B * a.N || CW * l >= c.D / 2) return;
        const int b = (int)(tok / (unsigned)a.N), t = (int)(tok % (unsigned)a.N);
        if (a.count && t >= a.count[b]) return;
        const int64_t slot = (a.first ? (int64_t)a.first[b] : 0) + t;
        if (slot < 0 || slot >= c.cap) return;
        const int h0 = chunk * HG, hn = min(HG, c.Hkv - h0);
        const uint8_t *src = (is_v ? c.v : c.k) + b * c.batch + slot * c.token + h0 * c.head + CW * l;
        const uint8_t *sp = (is_v ? c.v_scale : c.k_scale) + b * c.s_batch + h0 * c.s_head + slot;
        T *dst = is_v ? (T *)a.v + b * a.v_batch + t * a.v_token + h0 * a.v_head + CW * l
                      : (T *)a.k + b * a.k_batch + t * a.k_token + h0 * a.k_head + CW * l;
        const int64_t dh = is_v ? a.v_head : a.k_head;
        const int other = c.D / 2;
        uc u[HG][2];
        unsigned e[HG];
#pragma unroll
        for (int h = 0; h < HG; h++)
            if (h < hn) {
                u[h][0] = *reinterpret_cast<const uc *>(src + h * c.head);
                u[h][1] = *reinterpret_cast<const uc *>(src + h * c.head + other);
                e[h] = sp[h * c.s_head];
            }
#pragma unroll
        for (int h = 0; h < HG; h++) {
            if (h >= hn) break;
            const float f = __builtin_bit_cast(float, e[h] << 23);
#pragma unroll
            for (int j = 0; j < 2; j++) {
                vc y;
#pragma unroll
                for (int i = 0; i < CW / 4; i++) {
                    const unsigned w = u[h][j][i];
                    const auto p = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), q = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
                    y[4 * i] = held(p[0] * f);
                    y[4 * i + 1] = held(p[1] * f);
                    y[4 * i + 2] = held(q[0] * f);
                    y[4 * i + 3] = held(q[1] * f);
                }
                *reinterpret_cast<vc *>(dst + h * dh + j * other) = y;
            }
        }
    };
    for (int64_t blk = blockIdx.x; blk < x.blocks; blk += gridDim.x) work(blk);
}

template <int TY, int LPR>
static void rd_launch(RdArgs &x, hipStream_t s) {
    const int64_t blocks = ((int64_t)x.a.cache.B * x.a.N + 256 / LPR - 1) / (256 / LPR);
    const int ops = x.two ? 2 : 1, heads = x.a.cache.Hkv;
    /* as in st_shares() */
    const int hg = blocks * ((heads + 3) / 4) * ops >= 1024 ? 4 : blocks * ((heads + 1) / 2) * ops >= 512 ? 2 : 1;
    x.chunks = (heads + hg - 1) / hg;
    x.blocks = blocks * x.chunks * ops;
    const dim3 grid((unsigned)std::min<int64_t>(x.blocks, ST_GRID));
    if (hg == 4) hipLaunchKernelGGL((k_kv_read<TY, LPR, 4>), grid, dim3(256), 0, s, x);
    else if (hg == 2) hipLaunchKernelGGL((k_kv_read<TY, LPR, 2>), grid, dim3(256), 0, s, x);
    else hipLaunchKernelGGL((k_kv_read<TY, LPR, 1>), grid, dim3(256), 0, s, x);
}
template <int TY>
static void rd_lanes(RdArgs &x, hipStream_t s) {
    const int lanes = x.a.cache.D / (TY == 0 ? 8 : 16);
    if (lanes <= 2) rd_launch<TY, 2>(x, s);
    else if (lanes <= 4) rd_launch<TY, 4>(x, s);
    else if (lanes <= 8) rd_launch<TY, 8>(x, s);
    else if (TY || lanes <= 16) rd_launch<TY, 16>(x, s);
    else if constexpr (TY == 0) rd_launch<TY, 32>(x, s);
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
