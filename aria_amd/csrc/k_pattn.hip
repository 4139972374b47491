/*
 * k_pattn.hip - attention of a batch over shared prefixes and each sequence's own keys, both cached as e4m3
 * rows (gfx950): o = sum_j p_j v_j, p = softmax over the keys j that a row sees of scale * q . k_j. A row that
 * sees no key is zero.
 *
 * A row is a (sequence, token, query head of the group) triple. Two forms: where a sequence's own rows fill a
 * workgroup (or nothing is shared), a workgroup walks through the prefix's key tiles and then through the own ones. Else the rows
 * of all sequences of a prefix go over its keys together, the rows of each sequence over its own keys, and a second kernel joins
 * what they found: the prefix is read, converted and multiplied once for all of them.
 *
 * The arithmetic is that of k_xattn.hip: S^T = K Q^T and O^T = V^T P^T with v_mfma_f32_32x32x16, scores in registers, weights
 * 2^(scale_log2 s - ref) with a lazy reference, P rounded to the 16-bit type. Codes become 16-bit values on their way to LDS: a
 * lane loads 16 codes and their row's byte, converts them with the row's power of two (one instruction per two
 * values) and stores two 16-byte chunks where the swizzle wants them; the next tile's codes are on their way meanwhile.
 * Slots that no row sees become zeros there, and their scores -inf. A key or value row of byte 255 (NaN) is staged
 * as a key of NaNs and a value of zeros: a row that sees it gets a NaN weight, one that does not (a later token's slot) is not
 * touched by it.
 */
#include "xattn_dev.h"
#include "aria_hip_kernels.h"

#include <algorithm>

/* 16-byte source of chunks that hold no slot or no dim */
__device__ const uint4 pa_zero = {0, 0, 0, 0};

template <typename T> struct Pc;
template <> struct Pc<_Float16> {
    template <bool HI> static __device__ __forceinline__ Xa<_Float16>::v2 cvt(unsigned u, float s) { return __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(u, s, HI); }
};
template <> struct Pc<__bf16> {
    template <bool HI> static __device__ __forceinline__ Xa<__bf16>::v2 cvt(unsigned u, float s) { return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(u, s, HI); }
};

/* one kind of workgroup: `sets` sets of R rows (a prefix's, or a sequence's), nrb row blocks to each and key head, ns splits of
 * `per` key tiles */
struct PaJobs {
    int sets, R, nrb, ns, per, jobs;
    int use_prefix, use_own;
    size_t part;             /* floats in front of its partial results */
};
struct PaArgs {
    aria_hip_prefix_attn a;
    int G, Bp;               /* query heads per key head; sequences per prefix */
    int kinds, group;        /* one kind of workgroup or two; the first takes the rows of a prefix's sequences together */
    PaJobs j[2];
    int jobs;
    float scale_log2;
    float *part;
};

/* keys of a tile */
__host__ __device__ constexpr int pa_tile(int DP, int QW) { return DP == 64 || QW > 1 ? 64 : 32; }
/* floats of a row's partial result: sums, reference, weights' sum, remainder of the reference */
__host__ __device__ constexpr int pa_row(int DP) { return DP + 4; }

template <typename T, int DP, int QW, int KS>
__global__ __launch_bounds__(64 * QW * KS) void k_pattn(PaArgs x) {
    constexpr int KT = pa_tile(DP, QW);
    constexpr int NW = QW * KS;
    constexpr int NST = QW > 1 ? 2 : 1;             /* LDS stages */
    constexpr int CPR = DP / 8;                     /* 16-byte chunks of values per key row */
    constexpr int C16 = DP / 16;                    /* 16-byte chunks of codes per key row */
    constexpr int NC = KT * C16 / (64 * QW);        /* code chunks per lane, tile and operand */
    constexpr int TB = KT * DP * 2;                 /* bytes of a tile of values */
    constexpr int ES = DP + 4;                      /* floats per staged output row */
    constexpr int KB = KT / 32, DT = DP / 32, DS = DP / 16;
    constexpr int STAGE = 2 * TB * KS;              /* K and V of every slice */
    constexpr int EPI = NW * 32 * ES * 4 + NW * 96 * 4;
    __shared__ __attribute__((aligned(16))) uint8_t smem[NST * STAGE > EPI ? NST * STAGE : EPI];
    typedef typename Xa<T>::v8 v8;
    typedef typename Xa<T>::v2 v2;
    const aria_hip_prefix_attn &a = x.a;
    const int D = a.own.D, Hkv = a.own.Hkv;

    const int lane = threadIdx.x & 63, g = lane >> 5, l32 = lane & 31;
    const int wid = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int qw = wid % QW, ks = wid / QW;

    int job = xcd_tile(blockIdx.x, x.jobs);
    if (job >= x.jobs) return;
    const int kind = job >= x.j[0].jobs;
    if (kind) job -= x.j[0].jobs;
    const PaJobs &J = x.j[kind];
    const int rb = job % J.nrb, split = job / J.nrb % J.ns, sh = job / J.nrb / J.ns, hk = sh % Hkv, set = sh / Hkv;
    /* a set is a prefix's rows (kind 0 of 2: several sequences), or a sequence's */
    const bool group = x.group && kind == 0;
    const int per_seq = a.Nq * x.G;                 /* rows of one sequence and key head */
    const int pf = group ? set : set / x.Bp;
    auto where = [&](int row, int &b, int &tok, int &hd) __attribute__((always_inline)) {
        const int r = group ? row % per_seq : row;
        b = group ? set * x.Bp + row / per_seq : set;
        tok = r / x.G;
        hd = hk * x.G + r % x.G;
    };
    const int row0 = rb * 32 * QW + qw * 32;        /* the wave's first row; rows past R repeat the last */
    int qb, tok, hd;
    where(min(row0 + l32, J.R - 1), qb, tok, hd);

    v8 qf[DS];
    {
        const T *q = (const T *)a.q + qb * a.q_batch + hd * a.q_head + tok * a.q_token;
#pragma unroll
        for (int i = 0; i < DS; i++) {
            const int d = 16 * i + 8 * g;
            uint4 u = make_uint4(0, 0, 0, 0);
            if (d < D) u = *reinterpret_cast<const uint4 *>(q + d);
            qf[i] = __builtin_bit_cast(v8, u);
        }
    }

    /* the slots that rows see: n0 of the prefix, and of the own part n1 (causal: lim of this lane's row, lim_lo of the
     * wave's first, lim_hi of the block's last) */
    int n0 = 0, n1 = 0, lim = 0, lim_lo = 0, lim_hi = 0;
    if (J.use_prefix) n0 = a.prefix_len ? min(max(a.prefix_len[pf], 0), a.prefix.cap) : a.prefix.cap;
    if (J.use_own) {
        n1 = a.own_len ? min(max(a.own_len[set], 0), a.own.cap) : a.own.cap;
        lim = lim_lo = lim_hi = n1;
        if (a.first) {
            const long long f = (long long)a.first[set] + 1;
            auto at = [&](int t) __attribute__((always_inline)) { return (int)min(max(f + t, 0ll), (long long)n1); };
            lim = at(tok);
            lim_lo = at(min(row0, J.R - 1) / x.G);
            lim_hi = at((min((rb + 1) * 32 * QW, J.R) - 1) / x.G);
        }
    }
    /* key tiles: nt0 of the prefix, then the own ones. A split has J.per of them, and a set with few of them fewer splits */
    const int nt0 = (n0 + KT - 1) / KT, nt = nt0 + (lim_hi + KT - 1) / KT;
    const int w0 = split * J.per;
    if (split > 0 && w0 >= nt0 + (n1 + KT - 1) / KT) return;      /* uniform per workgroup, before any barrier */
    const int w1 = max(w0, min(w0 + J.per, nt));
    const int sp = (w1 - w0 + KS - 1) / KS;
    const int t0 = min(w0 + ks * sp, w1), t1 = min(t0 + sp, w1);

    /* codes of a tile on their way */
    uint4 kc[NC], vc[NC];
    unsigned kb[NC], vb[NC];
    auto load = [&](int i) __attribute__((always_inline)) {
        const bool own = i >= nt0;
        const aria_hip_kv &c = own ? a.own : a.prefix;
        const long long b = own ? set : pf;
        const int base = (own ? i - nt0 : i) * KT, left = (own ? n1 : n0) - base;
        const uint8_t *k = c.k + b * c.batch + hk * c.head + base * c.token, *v = c.v + b * c.batch + hk * c.head + base * c.token;
        const uint8_t *se = c.k_scale + b * c.s_batch + hk * c.s_head + base, *sv = c.v_scale + b * c.s_batch + hk * c.s_head + base;
#pragma unroll
        for (int j = 0; j < NC; j++) {
            const int p = 64 * (QW * j + qw) + lane, r = p / C16, cc = p % C16;
            const bool ok = r < left && 16 * cc < D;
            const long long off = r * c.token + 16 * cc;
            kc[j] = *reinterpret_cast<const uint4 *>(ok ? k + off : (const uint8_t *)&pa_zero);
            vc[j] = *reinterpret_cast<const uint4 *>(ok ? v + off : (const uint8_t *)&pa_zero);
            kb[j] = *(ok ? se + r : (const uint8_t *)&pa_zero);
            vb[j] = *(ok ? sv + r : (const uint8_t *)&pa_zero);
        }
    };
    auto put = [&](uint8_t *to, const uint4 &u, unsigned byte, int at0, int at1) __attribute__((always_inline)) {
        const float s = __builtin_bit_cast(float, byte << 23);
        const v2 c0 = Pc<T>::template cvt<false>(u.x, s), c1 = Pc<T>::template cvt<true>(u.x, s);
        const v2 c2 = Pc<T>::template cvt<false>(u.y, s), c3 = Pc<T>::template cvt<true>(u.y, s);
        const v2 c4 = Pc<T>::template cvt<false>(u.z, s), c5 = Pc<T>::template cvt<true>(u.z, s);
        const v2 c6 = Pc<T>::template cvt<false>(u.w, s), c7 = Pc<T>::template cvt<true>(u.w, s);
        *reinterpret_cast<v8 *>(to + at0) = v8{c0[0], c0[1], c1[0], c1[1], c2[0], c2[1], c3[0], c3[1]};
        *reinterpret_cast<v8 *>(to + at1) = v8{c4[0], c4[1], c5[0], c5[1], c6[0], c6[1], c7[0], c7[1]};
    };
    auto store = [&](int buf) __attribute__((always_inline)) {
        uint8_t *K = smem + buf * STAGE + ks * 2 * TB, *V = K + TB;
#pragma unroll
        for (int j = 0; j < NC; j++) {
            const bool bad = kb[j] == 255u || vb[j] == 255u;
            if (__builtin_expect(__ballot(bad) != 0, 0)) {
                kc[j] = bad ? make_uint4(0x7F7F7F7Fu, 0x7F7F7F7Fu, 0x7F7F7F7Fu, 0x7F7F7F7Fu) : kc[j];
                vc[j] = bad ? make_uint4(0, 0, 0, 0) : vc[j];
                kb[j] = bad ? 127u : kb[j];
                vb[j] = bad ? 127u : vb[j];
            }
            const int p = 64 * (QW * j + qw) + lane, r = p / C16, cp = 2 * (p % C16);
            const int zk = DP == 64 ? (r >> 1) & 7 : r & 15, zv = DP == 64 ? ((r >> 1) & 1) << 2 : (r & 3) << 2;
            put(K, kc[j], kb[j], (r * CPR + (cp ^ zk)) * 16, (r * CPR + ((cp + 1) ^ zk)) * 16);
            put(V, vc[j], vb[j], (r * CPR + (cp ^ zv)) * 16, (r * CPR + ((cp + 1) ^ zv)) * 16);
        }
    };

    xa_f32x16_t o[DT];
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
        for (int r = 0; r < 16; r++) o[d][r] = 0.0f;
    float l = 0.0f, ref = XA_MIN, lo = 0.0f;
    bool far = false;                               /* a row of the wave has a lo */
    const v2 one2 = {(T)1.0f, (T)1.0f};

    /* byte offsets of the fragment reads */
    int koff[DS], voff[DT];
#pragma unroll
    for (int i = 0; i < DS; i++) {
        const int c = 2 * i + g;
        koff[i] = (l32 * CPR + (DP == 64 ? c ^ ((l32 >> 1) & 7) : c ^ (l32 & 15))) * 16;
    }
    {
        const int v = (lane & 15) >> 2, w = lane & 3, Gq = lane >> 4, key = 4 * (Gq >> 1) + v;
#pragma unroll
        for (int d = 0; d < DT; d++) {
            const int dd = 32 * d + 16 * (Gq & 1) + 4 * w, c = dd >> 3;
            voff[d] = (key * CPR + (DP == 64 ? c ^ (((key >> 1) & 1) << 2) : c ^ ((key & 3) << 2))) * 16 + (dd & 7) * 2;
        }
    }

    auto scores = [&](int buf, int i, xa_f32x16_t (&s)[KB]) __attribute__((always_inline)) {
        const uint8_t *K = smem + buf * STAGE + ks * 2 * TB;
#pragma unroll
        for (int kb = 0; kb < KB; kb++)
#pragma unroll
            for (int r = 0; r < 16; r++) s[kb][r] = 0.0f;
#pragma unroll
        for (int i = 0; i < DS; i++)
#pragma unroll
            for (int kb = 0; kb < KB; kb++)
                s[kb] = Xa<T>::mfma(*reinterpret_cast<const v8 *>(K + koff[i] + kb * 32 * CPR * 16), qf[i], s[kb]);
        /* slots that a row of the wave does not see: the last tile of a part, the tiles that a causal limit crosses */
        const bool own = i >= nt0;
        const int base = (own ? i - nt0 : i) * KT;
        if (base + KT > (own ? lim_lo : n0)) {
            const int left = (own ? lim : n0) - base - 4 * g;
#pragma unroll
            for (int kb = 0; kb < KB; kb++)
#pragma unroll
                for (int r = 0; r < 16; r++) s[kb][r] = 32 * kb + 8 * (r >> 2) + (r & 3) < left ? s[kb][r] : -INFINITY;
        }
    };
    /* behind it the exponent of a weight is s * scale_log2 - ref, or, where far, s - lo */
    auto move_ref = [&](xa_f32x16_t (&s)[KB]) __attribute__((always_inline)) {
        float mt = s[0][0];
#pragma unroll
        for (int i = 1; i + 1 < 16 * KB; i += 2) mt = max3_f32(mt, s[i >> 4][i & 15], s[(i + 1) >> 4][(i + 1) & 15]);
        mt = max3_f32(mt, s[KB - 1][15], s[KB - 1][15]);
        const float mo = xor32_f32(mt, lane);
        mt = max3_f32(mt, mo, mo);
        const float d = __builtin_fmaf(mt, x.scale_log2, -ref) - lo;
        if (__ballot(d > XA_TOP + XA_SLACK)) {
            asm volatile("" ::: "memory");   /* a branch, not 16 DT predicated multiplies */
            const bool up = d > XA_TOP;
            const float r2 = up ? __builtin_fmaf(mt, x.scale_log2, -XA_TOP) : ref;
            const float left = fabsf(r2) >= XA_FAR ? __builtin_fmaf(mt, x.scale_log2, -r2) - XA_TOP : 0.0f;
            const float lo2 = up ? left : lo, al = __builtin_amdgcn_exp2f((ref - r2) + (lo - lo2));
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int r = 0; r < 16; r++) o[d][r] *= al;
            l *= al;
            ref = r2;
            lo = lo2;
            far = __ballot(lo != 0.0f) != 0;
        }
        if (__builtin_expect(far, 0)) {
#pragma unroll
            for (int i = 0; i < 16 * KB; i++) s[i >> 4][i & 15] = __builtin_fmaf(s[i >> 4][i & 15], x.scale_log2, -ref);
        }
    };
    auto add = [&](int buf, const xa_f32x16_t (&s)[KB]) __attribute__((always_inline)) {
        const uint8_t *V = smem + buf * STAGE + ks * 2 * TB + TB;
        const float sc = far ? 1.0f : x.scale_log2, rr = far ? lo : ref;
#pragma unroll
        for (int kb = 0; kb < KB; kb++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int s16 = 2 * kb + h;      /* keys 16 s16 .. 16 s16 + 15 */
                v8 vf[DT];
#pragma unroll
                for (int d = 0; d < DT; d++) {
                    const uint8_t *p = V + voff[d] + 16 * s16 * CPR * 16;
                    const xa_i16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((xa_lds_i16x4_t *)p);
                    const xa_i16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((xa_lds_i16x4_t *)(p + 8 * CPR * 16));
                    vf[d] = __builtin_bit_cast(v8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
                }
                v8 p;
#pragma unroll
                for (int i = 0; i < 8; i++)
                    p[i] = (T)__builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][8 * h + i], sc, -rr));
#pragma unroll
                for (int d = 0; d < DT; d++) o[d] = Xa<T>::mfma(vf[d], p, o[d]);
#pragma unroll
                for (int i = 0; i < 4; i++) l = Xa<T>::dot2(v2{p[2 * i], p[2 * i + 1]}, one2, l);
            }
    };
    auto tile = [&](int buf, int i) __attribute__((always_inline)) {
        xa_f32x16_t s[KB];
        scores(buf, i, s);
        move_ref(s);
        add(buf, s);
    };

    if constexpr (NST == 2) {
        if (t0 < t1) {
            load(t0);
            store(0);
            if (t0 + 1 < t1) load(t0 + 1);
        }
        __syncthreads();
        for (int i = t0; i < t0 + sp; i++) {        /* every slice meets as often; its tiles end at t1 */
            const int buf = (i - t0) & 1;
            if (i + 1 < t1) {
                store(buf ^ 1);
                if (i + 2 < t1) load(i + 2);
            }
            if (i < t1) tile(buf, i);
            __syncthreads();
        }
    } else {
        /* one wave's tiles: its LDS accesses are in order */
        if (t0 < t1) load(t0);
        for (int i = t0; i < t1; i++) {
            store(0);
            if (i + 1 < t1) load(i + 1);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            tile(0, i);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
        __syncthreads();                            /* slices still reading their stages */
    }

    /* join: lanes l and l ^ 32 hold half of a row's sum each */
    l += xor32_f32(l, lane);
    float *E = (float *)smem + wid * 32 * ES;
    float *ML = (float *)smem + NW * 32 * ES;       /* per wave 32 references, 32 sums, 32 remainders of the references */
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
        for (int r = 0; r < 4; r++)
            *reinterpret_cast<float4 *>(E + l32 * ES + 32 * d + 8 * r + 4 * g) =
                make_float4(o[d][4 * r], o[d][4 * r + 1], o[d][4 * r + 2], o[d][4 * r + 3]);
    if (g == 0) { ML[wid * 96 + l32] = ref; ML[wid * 96 + 32 + l32] = l; ML[wid * 96 + 64 + l32] = lo; }
    __syncthreads();

    /* a group of CPR lanes finishes one row, 8 dims per lane; the KS waves of a block of rows take them in turn */
    constexpr int RPW = 64 / CPR;                    /* rows per wave at once */
    const int c8 = 8 * (lane % CPR);
#pragma unroll 1
    for (int i = ks; i < 32 / RPW; i += KS) {
        const int q = i * RPW + lane / CPR;          /* row within the block */
        float v[8], m[KS], c[KS];
#pragma unroll
        for (int w = 0; w < KS; w++) {
            m[w] = ML[(w * QW + qw) * 96 + q];
            c[w] = ML[(w * QW + qw) * 96 + 64 + q];
        }
        float rm = m[0], rl = c[0];                  /* the largest reference, and of those that have it the largest remainder */
#pragma unroll
        for (int w = 1; w < KS; w++) {
            rl = m[w] > rm ? c[w] : m[w] == rm ? fmaxf(rl, c[w]) : rl;
            rm = fmaxf(rm, m[w]);
        }
        float rs = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = 0.0f;
#pragma unroll
        for (int w = 0; w < KS; w++) {
            const float f = __builtin_amdgcn_exp2f((m[w] - rm) + (c[w] - rl));
            rs = __builtin_fmaf(f, ML[(w * QW + qw) * 96 + 32 + q], rs);
            const float *e = (const float *)smem + ((w * QW + qw) * 32 + q) * ES + c8;
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = __builtin_fmaf(f, e[j], v[j]);
        }
        const int orow = rb * 32 * QW + qw * 32 + q;
        if (orow >= J.R || c8 >= D) continue;
        if (x.part) {
            float *P = x.part + J.part + ((size_t)(sh * J.ns + split) * J.R + orow) * pa_row(DP);
            *reinterpret_cast<float4 *>(P + c8) = make_float4(v[0], v[1], v[2], v[3]);
            *reinterpret_cast<float4 *>(P + c8 + 4) = make_float4(v[4], v[5], v[6], v[7]);
            if (c8 == 0) *reinterpret_cast<float4 *>(P + DP) = make_float4(rm, rs, rl, 0.0f);
            continue;
        }
        const float inv = rs == 0.0f ? 0.0f : 1.0f / rs;
        int b, t, h;
        where(orow, b, t, h);
        const long long at = b * a.o_batch + h * a.o_head + t * a.o_token + c8;
        if (a.out_f32) {
            float *y = (float *)a.out + at;
            *reinterpret_cast<float4 *>(y) = make_float4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
            *reinterpret_cast<float4 *>(y + 4) = make_float4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv);
        } else {
            v8 y;
#pragma unroll
            for (int j = 0; j < 8; j++) y[j] = (T)(v[j] * inv);
            *reinterpret_cast<v8 *>((T *)a.out + at) = y;
        }
    }
}

/* Joins the partial results of one row: those of the prefix's splits, then those of the own part's. A group of DP / 8 lanes per
 * 8 dims, the wave's 64 / (DP / 8) groups take the splits in turn and add up through lane exchanges */
template <typename T, int DP>
__global__ __launch_bounds__(64) void k_pattn_join(PaArgs x, int KT) {
    constexpr int CPR = DP / 8, NG = 64 / CPR;
    const aria_hip_prefix_attn &a = x.a;
    const int per_seq = a.Nq * x.G;
    for (int i = blockIdx.x; i < a.B * a.H * a.Nq; i += gridDim.x) {
        const int hk = i / per_seq % a.own.Hkv, b = i / per_seq / a.own.Hkv, row = i % per_seq;
        const int lane = threadIdx.x, grp = lane / CPR, c8 = 8 * (lane % CPR), D = a.own.D;
        const int pf = b / x.Bp;
        const int n0 = a.prefix_len ? min(max(a.prefix_len[pf], 0), a.prefix.cap) : a.prefix.cap;
        const int n1 = a.own_len ? min(max(a.own_len[b], 0), a.own.cap) : a.own.cap;
        const int nt0 = (n0 + KT - 1) / KT, nt1 = (n1 + KT - 1) / KT;
        auto splits = [&](const PaJobs &J, int nt) { return max(1, (nt + J.per - 1) / J.per); };   /* those that hold keys */
        const int s0 = splits(x.j[0], x.group ? nt0 : nt0 + nt1), s1 = x.kinds == 2 ? splits(x.j[1], nt1) : 0;
        const int set0 = x.group ? pf : b, row_0 = x.group ? (b - pf * x.Bp) * per_seq + row : row;
        auto at = [&](int s) __attribute__((always_inline)) -> const float * {
            if (s < s0) return x.part + x.j[0].part + ((size_t)((set0 * a.own.Hkv + hk) * x.j[0].ns + s) * x.j[0].R + row_0) * pa_row(DP);
            return x.part + x.j[1].part + ((size_t)((b * a.own.Hkv + hk) * x.j[1].ns + s - s0) * x.j[1].R + row) * pa_row(DP);
        };
        const int ns = s0 + s1;
        float m = XA_MIN, ml = -INFINITY;                          /* the largest reference and its largest remainder */
        for (int s = lane; s < ns; s += 64) {
            const float *p = at(s) + DP;
            ml = p[0] > m ? p[2] : p[0] == m ? fmaxf(ml, p[2]) : ml;
            m = fmaxf(m, p[0]);
        }
        const float ma = grp_max<64>(m);
        ml = grp_max<64>(m == ma ? ml : -INFINITY);
        m = ma;
        float rs = 0.0f, v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (c8 < D)
#pragma unroll 4
            for (int s = grp; s < ns; s += NG) {
                const float *p = at(s);
                const float f = __builtin_amdgcn_exp2f((p[DP] - m) + (p[DP + 2] - ml));
                rs = __builtin_fmaf(f, p[DP + 1], rs);
                const float4 u = *reinterpret_cast<const float4 *>(p + c8), w = *reinterpret_cast<const float4 *>(p + c8 + 4);
                const float e[8] = {u.x, u.y, u.z, u.w, w.x, w.y, w.z, w.w};
#pragma unroll
                for (int j = 0; j < 8; j++) v[j] = __builtin_fmaf(f, e[j], v[j]);
            }
#pragma unroll
        for (int k = CPR; k < 64; k *= 2) {
            rs += __shfl_xor(rs, k, 64);
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] += __shfl_xor(v[j], k, 64);
        }
        if (grp != 0 || c8 >= D) continue;
        const float inv = rs == 0.0f ? 0.0f : 1.0f / rs;
        const long long out = b * a.o_batch + (hk * x.G + row % x.G) * a.o_head + (row / x.G) * a.o_token + c8;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            if (a.out_f32) ((float *)a.out)[out + j] = v[j] * inv;
            else ((T *)a.out)[out + j] = (T)(v[j] * inv);
        }
    }
}

/* How a call runs */
struct PaPlan { int qw, ks, DP, join; };
static PaPlan pa_plan(const aria_hip_prefix_attn *a, PaArgs &x) {
    PaPlan p;
    const int Hkv = a->own.Hkv, P = a->prefix.B;
    x.G = a->H / Hkv;
    x.Bp = a->B / P;
    p.DP = a->own.D <= 64 ? 64 : 128;
    const int R = a->Nq * x.G;
    const bool has_p = a->prefix.cap > 0, has_o = a->own.cap > 0;
    const bool share = has_p && x.Bp > 1 && R < 128;
    const long long rows = share ? (long long)R * x.Bp : R, sets = share ? P : a->B;
    p.qw = rows <= 32 || sets * Hkv * ((rows + 127) / 128) < 64 ? 1 : 4;
    p.ks = p.qw == 1 ? 4 : 1;
    const int KT = pa_tile(p.DP, p.qw), br = 32 * p.qw;
    auto tiles = [&](int cap) { return (cap + KT - 1) / KT; };
    auto set_up = [&](PaJobs &J, int sets, long long R, int nt, int up, int uo, size_t part) {
        J.sets = sets;
        J.R = (int)R;
        J.nrb = (int)((R + br - 1) / br);
        J.use_prefix = up;
        J.use_own = uo;
        J.part = part;
        /* at least 256 keys to a workgroup, and two workgroups to a CU */
        const long long wg = (long long)sets * Hkv * J.nrb;
        J.ns = p.qw == 1 ? (int)std::max<long long>(1, std::min<long long>((long long)nt * KT / 256, 512 / wg)) : 1;
        J.per = std::max(1, (nt + J.ns - 1) / J.ns);
        J.jobs = (int)(wg * J.ns);
        return part + (size_t)sets * Hkv * J.ns * R * pa_row(p.DP);
    };
    x.group = share;
    if (share) {
        const size_t n = set_up(x.j[0], P, rows, tiles(a->prefix.cap), 1, 0, 0);
        x.kinds = 1;
        x.j[1] = PaJobs{};
        if (has_o) {
            x.kinds = 2;
            set_up(x.j[1], a->B, R, tiles(a->own.cap), 0, 1, n);
        }
        p.join = x.kinds == 2 || x.j[0].ns > 1;
    } else {
        x.kinds = 1;
        set_up(x.j[0], a->B, R, (has_p ? tiles(a->prefix.cap) : 0) + (has_o ? tiles(a->own.cap) : 0), has_p, has_o, 0);
        x.j[1] = PaJobs{};
        p.join = x.j[0].ns > 1;
    }
    x.jobs = x.j[0].jobs + x.j[1].jobs;
    return p;
}

extern "C" size_t aria_k_pattn_ws_bytes(const aria_hip_prefix_attn *a) {
    PaArgs x{};
    const PaPlan p = pa_plan(a, x);
    size_t n = 0;
    for (int i = 0; i < 2; i++) n += (size_t)x.j[i].sets * a->own.Hkv * x.j[i].ns * x.j[i].R * pa_row(p.DP);
    return p.join ? n * sizeof(float) : 0;
}

template <typename T>
static hipError_t pa_launch(const PaPlan &p, const PaArgs &x, hipStream_t s) {
    const dim3 grid((unsigned)((x.jobs + 7) / 8 * 8));
    if (p.qw == 1) {
        if (p.DP == 64) hipLaunchKernelGGL((k_pattn<T, 64, 1, 4>), grid, dim3(256), 0, s, x);
        else hipLaunchKernelGGL((k_pattn<T, 128, 1, 4>), grid, dim3(256), 0, s, x);
    } else {
        if (p.DP == 64) hipLaunchKernelGGL((k_pattn<T, 64, 4, 1>), grid, dim3(256), 0, s, x);
        else hipLaunchKernelGGL((k_pattn<T, 128, 4, 1>), grid, dim3(256), 0, s, x);
    }
    if (p.join) {
        const dim3 rows((unsigned)std::min(x.a.B * x.a.H * x.a.Nq, 1 << 20));
        const int KT = pa_tile(p.DP, p.qw);
        if (p.DP == 64) hipLaunchKernelGGL((k_pattn_join<T, 64>), rows, dim3(64), 0, s, x, KT);
        else hipLaunchKernelGGL((k_pattn_join<T, 128>), rows, dim3(64), 0, s, x, KT);
    }
    return hipGetLastError();
}

extern "C" hipError_t aria_k_pattn_run(const aria_hip_prefix_attn *a, void *ws, hipStream_t s) {
    if (a->B <= 0 || a->Nq <= 0) return hipSuccess;
    PaArgs x{};
    x.a = *a;
    const PaPlan p = pa_plan(a, x);
    x.scale_log2 = a->scale * ARIA_LOG2E;
    x.part = p.join ? (float *)ws : nullptr;
    return a->type == 1 ? pa_launch<_Float16>(p, x, s) : pa_launch<__bf16>(p, x, s);
}
