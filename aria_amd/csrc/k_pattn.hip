/*
 * k_pattn.hip - attention of a batch over shared prefixes and each sequence's own keys, both cached as e4m3
 * rows (gfx950): o = sum_j p_j v_j, p = softmax over the keys j that a row sees of scale * q . k_j. A row that
 * sees no key is zero.
 *
 * A row is a (sequence, token, query head of the group) triple. Where it pays, the rows of all sequences of a prefix go over its
 * keys together, the rows of each sequence over its own keys in the same launch, and a second kernel joins what they found: the prefix
 * is read, converted and multiplied once for all of them. Else a workgroup walks through the prefix's key tiles and then through the
 * own ones. Either way the keys may be split over workgroups, to be joined too.
 *
 * The arithmetic is that of k_xattn.hip: S^T = K Q^T and O^T = V^T P^T with v_mfma_f32_32x32x16, scores in registers, weights
 * 2^(scale_log2 s - ref) with a lazy reference, P rounded to the 16-bit type (half a step of it per weight; the row sum adds the rounded
 * values). Codes become 16-bit values on their way to LDS: a lane loads 16 codes and their row's byte, converts them with
 * the row's power of two (one instruction per two values, exact in bf16) and stores two 16-byte chunks where the swizzle wants
 * them; the next tile's codes are on their way meanwhile. Converted once, a tile serves up to 128 rows.
 * The scores of slots that a row does not see become -inf. A key or value row of byte 255 (NaN) is staged
 * as a key of NaNs and a value of zeros: a row that sees it gets a NaN weight, one that does not (a later token's slot) is not
 * touched by it. So are slots behind a length, whose scores are -inf for every row. A row whose byte lets codes pass the type's largest number
 * (65504 in fp16 is 65536 as a code) is held to it: an infinity would reach the rows that do not see it as 0 times itself.
 *
 * What bounds it (us of a call among others):
 *  - many rows: the chain of one tile, which two waves a SIMD do not hide. 8 sequences of 512 tokens, 4 heads to each of 4 key heads of
 *    128, over 8192 + up to 1024 keys: 309, 0.95 PFLOP/s; matrix pipe, VALU and LDS are busy 38 % each, 29 % of the waves' cycles are waits
 *    and barriers. No gain there (306 that day) from the scores of the next 32 keys beside this step's softmax (311), more workgroups of 32-key tiles
 *    (331), other orders (317); the next tile's scores need 329 registers (470).
 *    4 sequences of 1296 tokens, 16 heads of 64, over 2048 + 1296 keys: 104, 0.68 PFLOP/s; 704 workgroups are 2.75 a CU, where three
 *    run at once, and end together only on some of them (CUs busy 83 %).
 *  - few rows over many keys: their bytes (8 tokens over 131072 shared keys, 135 MB: 27 in the kernel and 6 in the join).
 *  - little of both: the launch and the latency of a tile. 172 tokens over 257 keys of 64: 10.6; in the kernel the arguments are there after
 *    0.3 us, the lengths after 1.7, the first tile in LDS after 2.4 and done after 3.3.
 */
#include "xattn_dev.h"
#include "aria_hip_kernels.h"

#include <algorithm>

typedef float pa_f32x2_t __attribute__((ext_vector_type(2)));
#define PA_AHEAD 6           /* key fragments on their way to a score product */

/* cvt: two codes of a dword times their row's power of two. LARGE: the first byte under which a code may lie past the type's largest
 * number MOST (448 * 2^7 and 448 * 2^119 do not) */
template <typename T> struct Pc;
template <> struct Pc<_Float16> {
    static constexpr unsigned LARGE = 135;
    static constexpr float MOST = 65504.0f;
    template <bool HI> static __device__ __forceinline__ Xa<_Float16>::v2 cvt(unsigned u, float s) { return __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(u, s, HI); }
};
template <> struct Pc<__bf16> {
    static constexpr unsigned LARGE = 247;
    static constexpr float MOST = 3.38953139e38f;
    template <bool HI> static __device__ __forceinline__ Xa<__bf16>::v2 cvt(unsigned u, float s) { return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(u, s, HI); }
};

/* One kind of workgroup: `sets` sets of R rows (a prefix's, or a sequence's), nrb row blocks to each and key head, ns splits of
 * `per` key tiles. Form 0, 1, 2: a row block of 32, 64 or 128 rows, whose keys 4, 2 or 1 slices of waves share out. Form 0 has one LDS
 * stage to a wave and no barriers in its loop, the others two stages */
struct PaJobs {
    int sets, R, nrb, ns, per, jobs, form;
    int use_prefix, use_own, tp;                    /* tp: tiles of a prefix's capacity */
    HostDiv dnrb, dns, dper;
    size_t part;             /* floats in front of its partial results */
};
struct PaArgs {
    aria_hip_prefix_attn a;
    int G, Bp;               /* query heads per key head; sequences per prefix */
    int kinds, group;        /* one kind of workgroup or two; the first takes the rows of a prefix's sequences together */
    PaJobs j[2];
    HostDiv dhkv, dseq, dg, dbp;                      /* Hkv, rows of a sequence and key head, G, Bp */
    float scale_log2;
    float *part;
};

/* keys of a tile */
__host__ __device__ constexpr int pa_tile(int DV, int form) { return DV <= 64 || form == 2 ? 64 : 32; }
/* floats of a row's partial result: sums, reference, weights' sum, remainder of the reference */
__host__ __device__ constexpr int pa_row(int DV) { return DV + 4; }
/* LDS bytes of a form: the stages of every slice, later the output rows and each wave's 32 references, sums and remainders */
__host__ __device__ constexpr int pa_lds(int DV, int form) {
    const int ks = 4 >> form, st = (form ? 2 : 1) * ks * 2 * pa_tile(DV, form) * (DV <= 64 ? 64 : 128) * 2;
    const int epi = form == 2 ? 0 : 4 * 32 * (DV + 4) * 4 + 4 * 96 * 4;
    return st > epi ? st : epi;
}

/* DV: the width as products see it, 32, 64, 96 or 128; a row in LDS has 64 or 128 dims (DP) */
template <typename T, int DV, int FORM>
__device__ __forceinline__ void pa_work(const PaArgs &x, int kind, int job, uint8_t *smem) {
    constexpr int QW = 1 << FORM, KS = 4 >> FORM, NW = 4;
    constexpr int DP = DV <= 64 ? 64 : 128, KT = pa_tile(DV, FORM);
    constexpr int NST = QW > 1 ? 2 : 1;             /* LDS stages */
    constexpr int CPR = DP / 8;                     /* 16-byte chunks of values per key row */
    constexpr int C16 = DP / 16;                    /* 16-byte chunks of codes per key row */
    constexpr int NC = KT * C16 / (64 * QW);        /* code chunks per lane, tile and operand */
    constexpr int TB = KT * DP * 2;                 /* bytes of a tile of values */
    constexpr int ES = DV + 4;                      /* floats per staged output row */
    constexpr int KB = KT / 32, DT = DV / 32, DS = DV / 16;
    constexpr int STAGE = 2 * TB * KS;              /* K and V of every slice */
    typedef typename Xa<T>::v8 v8;
    typedef typename Xa<T>::v2 v2;
    const aria_hip_prefix_attn &a = x.a;
    const int D = a.own.D, Hkv = a.own.Hkv;

    const int lane = threadIdx.x & 63, g = lane >> 5, l32 = lane & 31;
    const int wid = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int qw = wid % QW, ks = wid / QW;

    const PaJobs &J = x.j[kind];
    unsigned rest = x.j[kind].dnrb.of(job), next;
    const int rb = job - rest * J.nrb;
    const int split = rest - (next = J.dns.of(rest)) * J.ns, set = x.dhkv.of(next), hk = next - set * Hkv, sh = next;
    /* a set is a prefix's rows (several sequences), or a sequence's */
    const bool group = x.group && kind == 0;
    const int pf = group ? set : x.dbp.of(set);

    /* codes of a tile on their way. Slots behind the capacity repeat its last one and chunks past D the last chunk: the
     * former are not seen, the latter's dims meet zeros of q or are not stored */
    typedef __attribute__((address_space(1))) const uint8_t gu8;
    typedef __attribute__((address_space(4))) const int ci32;
    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
    u32x4 kc[NC], vc[NC];
    unsigned kb[NC], vb[NC];
    const uint8_t *kp, *vp, *se, *sv;
    unsigned tb;                                    /* bytes from slot to slot (below 2^24) */
    int left;                                       /* slots from the tile's first to the capacity */
    bool at_own;
    auto seek = [&](bool own, int i) __attribute__((always_inline)) {
        const aria_hip_kv &c = own ? a.own : a.prefix;
        const long long b = own ? set : pf, at = b * c.batch + hk * c.head + (long long)i * KT * c.token;
        const long long sat = b * c.s_batch + hk * c.s_head + (long long)i * KT;
        kp = c.k + at;
        vp = c.v + at;
        se = c.k_scale + sat;
        sv = c.v_scale + sat;
        tb = (unsigned)c.token;
        left = c.cap - i * KT;
        at_own = own;
    };
    auto load = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < NC; j++) {
            const int p = 64 * (QW * j + qw) + lane;
            const unsigned r = min(p / C16, left - 1), off = r * tb + 16 * min(p % C16, D / 16 - 1);
            kc[j] = *(__attribute__((address_space(1))) const u32x4 *)((gu8 *)kp + off);
            vc[j] = *(__attribute__((address_space(1))) const u32x4 *)((gu8 *)vp + off);
            kb[j] = ((gu8 *)se)[r];
            vb[j] = ((gu8 *)sv)[r];
        }
    };
    /* A split has J.per of the tiles, of which its slices take every KS-th. The first tile goes out before the lengths are here:
     * it is the one that full caches would have */
    const int w0 = split * J.per, i0 = w0 + ks, g_own = i0 >= J.tp, g_tile = g_own ? i0 - J.tp : i0;
    const bool guess = !g_own || (J.use_own && g_tile * KT < a.own.cap);
    if (guess) {
        seek(g_own, g_tile);
        load();
    }

    auto where = [&](int row, int &b, int &tok, int &hd) __attribute__((always_inline)) {
        const int s = group ? x.dseq.of(row) : 0, r = row - s * (int)x.dseq.d;
        b = group ? set * x.Bp + s : set;
        tok = x.dg.of(r);
        hd = hk * x.G + r - tok * x.G;
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
    if (J.use_prefix) n0 = a.prefix_len ? min(max(((ci32 *)a.prefix_len)[pf], 0), a.prefix.cap) : a.prefix.cap;
    if (J.use_own) {
        n1 = a.own_len ? min(max(((ci32 *)a.own_len)[set], 0), a.own.cap) : a.own.cap;
        lim = lim_lo = lim_hi = n1;
        if (a.first) {
            const long long f = (long long)((ci32 *)a.first)[set] + 1;
            auto at = [&](int t) __attribute__((always_inline)) { return (int)min(max(f + t, 0ll), (long long)n1); };
            lim = at(tok);
            lim_lo = at(x.dg.of(min(row0, J.R - 1)));
            lim_hi = at(x.dg.of(min((rb + 1) * 32 * QW, J.R) - 1));
        }
    }
    /* key tiles: nt0 of the prefix, then the own ones; a set with few of them has fewer splits */
    const int nt0 = (n0 + KT - 1) / KT, nt = nt0 + (lim_hi + KT - 1) / KT;
    if (split > 0 && w0 >= nt0 + (n1 + KT - 1) / KT) return;      /* uniform per workgroup, before any barrier */
    const int w1 = min(w0 + J.per, nt);
    if (i0 < w1 && !(guess && (g_own ? i0 >= nt0 && i0 - nt0 == g_tile : i0 < nt0))) {
        seek(i0 >= nt0, i0 >= nt0 ? i0 - nt0 : i0);
        load();
    }
    /* behind load(): on to the slice's next tile, i */
    auto move = [&](int i) __attribute__((always_inline)) {
        if (!at_own && i >= nt0) {
            seek(true, i - nt0);
        } else {
            kp += (unsigned long long)tb * (KT * KS);
            vp += (unsigned long long)tb * (KT * KS);
            se += KT * KS;
            sv += KT * KS;
            left -= KT * KS;
        }
    };
    auto put = [&](auto HELD, uint8_t *to, const u32x4 &u, unsigned byte, int at0, int at1) __attribute__((always_inline)) {
        const float s = __builtin_bit_cast(float, byte << 23);
        if constexpr (decltype(HELD)::value != 0) {
            T y[16];
            auto held = [&](float v) __attribute__((always_inline)) {
                return (T)__builtin_elementwise_minimum(__builtin_elementwise_maximum(v * s, -Pc<T>::MOST), Pc<T>::MOST);
            };
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const auto p = __builtin_amdgcn_cvt_pk_f32_fp8((int)u[i], false), q = __builtin_amdgcn_cvt_pk_f32_fp8((int)u[i], true);
                y[4 * i] = held(p[0]);
                y[4 * i + 1] = held(p[1]);
                y[4 * i + 2] = held(q[0]);
                y[4 * i + 3] = held(q[1]);
            }
            __builtin_memcpy(__builtin_assume_aligned(to + at0, 16), y, 16);
            __builtin_memcpy(__builtin_assume_aligned(to + at1, 16), y + 8, 16);
            return;
        }
        const v2 c0 = Pc<T>::template cvt<false>(u.x, s), c1 = Pc<T>::template cvt<true>(u.x, s);
        const v2 c2 = Pc<T>::template cvt<false>(u.y, s), c3 = Pc<T>::template cvt<true>(u.y, s);
        const v2 c4 = Pc<T>::template cvt<false>(u.z, s), c5 = Pc<T>::template cvt<true>(u.z, s);
        const v2 c6 = Pc<T>::template cvt<false>(u.w, s), c7 = Pc<T>::template cvt<true>(u.w, s);
        *reinterpret_cast<v8 *>(to + at0) = v8{c0[0], c0[1], c1[0], c1[1], c2[0], c2[1], c3[0], c3[1]};
        *reinterpret_cast<v8 *>(to + at1) = v8{c4[0], c4[1], c5[0], c5[1], c6[0], c6[1], c7[0], c7[1]};
    };
    /* rows of tile i that stand for NaN or lie behind its last slot; whether others may hold more than the type does */
    auto fix = [&](int i) __attribute__((always_inline)) {
        const int valid = i < nt0 ? n0 - i * KT : n1 - (i - nt0) * KT;
        bool any = false;
#pragma unroll
        for (int j = 0; j < NC; j++) any |= max(kb[j], vb[j]) >= Pc<T>::LARGE || (64 * (QW * j + qw) + lane) / C16 >= valid;
        bool large = false;
        if (__builtin_expect(__ballot(any) != 0, 0)) {
#pragma unroll
            for (int j = 0; j < NC; j++) {
                const bool bad = kb[j] == 255u || vb[j] == 255u || (64 * (QW * j + qw) + lane) / C16 >= valid;
                kc[j] = bad ? u32x4{0x7F7F7F7Fu, 0x7F7F7F7Fu, 0x7F7F7F7Fu, 0x7F7F7F7Fu} : kc[j];
                vc[j] = bad ? u32x4{0, 0, 0, 0} : vc[j];
                kb[j] = bad ? 127u : kb[j];
                vb[j] = bad ? 127u : vb[j];
                large |= max(kb[j], vb[j]) >= Pc<T>::LARGE;
            }
            large = __ballot(large) != 0;
        }
        return large;
    };
    auto put_k = [&](auto HELD, int buf) __attribute__((always_inline)) {
        uint8_t *K = smem + buf * STAGE + ks * 2 * TB;
#pragma unroll
        for (int j = 0; j < NC; j++) {
            const int p = 64 * (QW * j + qw) + lane, r = p / C16, cp = 2 * (p % C16);
            const int z = DP == 64 ? (r >> 1) & 7 : r & 15;
            put(HELD, K, kc[j], kb[j], (r * CPR + (cp ^ z)) * 16, (r * CPR + ((cp + 1) ^ z)) * 16);
        }
    };
    auto put_v = [&](auto HELD, int buf) __attribute__((always_inline)) {
        uint8_t *V = smem + buf * STAGE + ks * 2 * TB + TB;
#pragma unroll
        for (int j = 0; j < NC; j++) {
            const int p = 64 * (QW * j + qw) + lane, r = p / C16, cp = 2 * (p % C16);
            const int z = DP == 64 ? ((r >> 1) & 1) << 2 : (r & 3) << 2;
            put(HELD, V, vc[j], vb[j], (r * CPR + (cp ^ z)) * 16, (r * CPR + ((cp + 1) ^ z)) * 16);
        }
    };
    auto store = [&](int buf, int i) __attribute__((always_inline)) {
        const bool large = fix(i);
        put_k(IC<0>{}, buf);
        put_v(IC<0>{}, buf);
        if (__builtin_expect(large, 0)) {           /* once more: the fast path keeps its straight line */
            put_k(IC<1>{}, buf);
            put_v(IC<1>{}, buf);
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

    auto scores = [&](int buf, xa_f32x16_t (&s)[KB]) __attribute__((always_inline)) {
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
        /* fragments PA_AHEAD products ahead */
        constexpr int N = DS * KB, AH = PA_AHEAD < N ? PA_AHEAD : N;
        __builtin_amdgcn_sched_group_barrier(0x100, AH, 0);
#pragma unroll
        for (int i = 0; i < N - AH; i++) {
            __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x8, AH, 0);
    };
    auto hide = [&](int i, xa_f32x16_t (&s)[KB]) __attribute__((always_inline)) {
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
                v2 p2[4];
#pragma unroll
                for (int i = 0; i < 4; i++)
                    p2[i] = __builtin_convertvector((pa_f32x2_t{__builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][8 * h + 2 * i], sc, -rr)),
                                                          __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][8 * h + 2 * i + 1], sc, -rr))}), v2);
                const v8 p = __builtin_shufflevector(__builtin_shufflevector(p2[0], p2[1], 0, 1, 2, 3), __builtin_shufflevector(p2[2], p2[3], 0, 1, 2, 3), 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
                for (int d = 0; d < DT; d++) o[d] = Xa<T>::mfma(vf[d], p, o[d]);
#pragma unroll
                for (int i = 0; i < 4; i++) l = Xa<T>::dot2(p2[i], one2, l);
            }
    };
    auto tile = [&](int buf, int i) __attribute__((always_inline)) {
        if (row0 >= J.R) return;                    /* the last row block's waves without rows: they only fetch */
        xa_f32x16_t s[KB];
        scores(buf, s);
        hide(i, s);
        move_ref(s);
        add(buf, s);
    };

    /* the rows of q are here: this use tells the compiler, which else would wait for them, and with them for the next
     * tile's codes, at every tile's first product */
    auto have_q = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < DS; i++) asm volatile("" : "+v"(qf[i]));
    };
    have_q();
    if constexpr (NST == 2) {
        if (i0 < w1) {
            store(0, i0);
            move(i0 + KS);
            if (i0 + KS < w1) load();
        }
        __syncthreads();
        for (int n = 0, i = i0; n < w1 - w0; n += KS, i += KS) {    /* every slice meets as often; its tiles end at w1 */
            const int buf = n / KS & 1;
            if (i < w1) tile(buf, i);
            if (i + KS < w1) {
                store(buf ^ 1, i + KS);
                move(i + 2 * KS);
                if (i + 2 * KS < w1) load();
            }
            __syncthreads();
        }
    } else {
        /* one wave's tiles: its LDS accesses are in order */
        for (int i = i0; i < w1; i += KS) {
            store(0, i);
            move(i + KS);
            if (i + KS < w1) load();
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            tile(0, i);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
        __syncthreads();                            /* slices still reading their stages */
    }

    /* lanes l and l ^ 32 hold half of a row's sum each */
    l += xor32_f32(l, lane);
    if constexpr (KS == 1) {
        /* from the accumulators: through LDS, in whole rows, this took 2 us more */
        if (row0 + l32 < J.R) {
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            float *P = x.part + J.part + ((size_t)(sh * J.ns + split) * J.R + row0 + l32) * pa_row(DV);
            const long long at = qb * a.o_batch + hd * a.o_head + tok * a.o_token;
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int c = 32 * d + 8 * r + 4 * g;
                    const float y[4] = {o[d][4 * r], o[d][4 * r + 1], o[d][4 * r + 2], o[d][4 * r + 3]};
                    if (x.part) {
                        *reinterpret_cast<float4 *>(P + c) = make_float4(y[0], y[1], y[2], y[3]);
                    } else if (c < D) {
                        if (a.out_f32) {
                            *reinterpret_cast<float4 *>((float *)a.out + at + c) = make_float4(y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv);
                        } else {
                            typedef T v4 __attribute__((ext_vector_type(4)));
                            *reinterpret_cast<v4 *>((T *)a.out + at + c) = v4{(T)(y[0] * inv), (T)(y[1] * inv), (T)(y[2] * inv), (T)(y[3] * inv)};
                        }
                    }
                }
            if (x.part && g == 0) *reinterpret_cast<float4 *>(P + DV) = make_float4(ref, l, lo, 0.0f);
        }
        return;
    }
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
    const int c8 = 8 * (lane % CPR), rows = min(32, J.R - row0);
#pragma unroll 1
    for (int i = ks; i * RPW < rows; i += KS) {
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
            const float *e = (const float *)smem + ((w * QW + qw) * 32 + q) * ES + min(c8, DV - 8);
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = __builtin_fmaf(f, e[j], v[j]);
        }
        if (q >= rows || c8 >= D) continue;
        if (x.part) {
            float *P = x.part + J.part + ((size_t)(sh * J.ns + split) * J.R + row0 + q) * pa_row(DV);
            *reinterpret_cast<float4 *>(P + c8) = make_float4(v[0], v[1], v[2], v[3]);
            *reinterpret_cast<float4 *>(P + c8 + 4) = make_float4(v[4], v[5], v[6], v[7]);
            if (c8 == 0) *reinterpret_cast<float4 *>(P + DV) = make_float4(rm, rs, rl, 0.0f);
            continue;
        }
        const float inv = rs == 0.0f ? 0.0f : 1.0f / rs;
        int b, t, h;
        where(row0 + q, b, t, h);
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

/* FORMS: the forms that the launch's kinds have, a bit to each */
template <typename T, int DV, int FORMS>
__global__ __launch_bounds__(256) void k_pattn(PaArgs x) {
    constexpr int l0 = FORMS & 1 ? pa_lds(DV, 0) : 0, l1 = FORMS & 2 ? pa_lds(DV, 1) : 0, l2 = FORMS & 4 ? pa_lds(DV, 2) : 0;
    __shared__ __attribute__((aligned(16))) uint8_t smem[l0 > l1 ? (l0 > l2 ? l0 : l2) : l1 > l2 ? l1 : l2];
    fetch_args(x);
    /* each kind spreads over all XCDs by itself, neighbouring jobs (which read the same keys) to one */
    const int first = (x.j[0].jobs + 7) & ~7, kind = (int)blockIdx.x >= first;
    const int job = xcd_tile(blockIdx.x - (kind ? first : 0), x.j[kind].jobs);
    if (job >= x.j[kind].jobs) return;
    const int form = x.j[kind].form;
    if constexpr ((FORMS & 1) != 0) if (form == 0) pa_work<T, DV, 0>(x, kind, job, smem);
    if constexpr ((FORMS & 2) != 0) if (form == 1) pa_work<T, DV, 1>(x, kind, job, smem);
    if constexpr ((FORMS & 4) != 0) if (form == 2) pa_work<T, DV, 2>(x, kind, job, smem);
}

/* Joins the partial results of a row: those of the prefix's splits, then those of the own part's. WR waves to a row: first
 * each thread takes a split's reference and sum, then groups of 8 or 16 lanes, 8 dims to a lane, take the splits' sums in turn */
template <typename T, int DV, int WR>
__global__ __launch_bounds__(256) void k_pattn_join(PaArgs x) {
    constexpr int CPR = DV <= 64 ? 8 : 16, TR = 64 * WR, NG = TR / CPR, RB = 4 / WR, MOST = 512;
    constexpr int FIRST = 2;                                   /* a group's splits that are on their way before the factors are known */
    __shared__ float fac[RB][MOST], red[RB][WR][4];
    __shared__ __attribute__((aligned(16))) float acc[RB][WR][8 * CPR];
    fetch_args(x);
    const aria_hip_prefix_attn &a = x.a;
    const int per_seq = a.Nq * x.G, rows = a.B * a.H * a.Nq;
    const int sub = threadIdx.x / TR, tr = threadIdx.x % TR, wv = tr / 64, lane = threadIdx.x & 63;
    const int grp = tr / CPR, c8 = 8 * (tr % CPR), D = a.own.D;
    for (int i0 = blockIdx.x * RB; i0 < rows; i0 += gridDim.x * RB) {
        const int i = min(i0 + sub, rows - 1);
        const int bh = x.dseq.of(i), row = i - bh * per_seq, b = x.dhkv.of(bh), hk = bh - b * a.own.Hkv, pf = x.dbp.of(b);
        const int n0 = a.prefix_len ? min(max(a.prefix_len[pf], 0), a.prefix.cap) : a.prefix.cap;
        const int n1 = a.own_len ? min(max(a.own_len[b], 0), a.own.cap) : a.own.cap;
        auto splits = [&](int kind, bool p, bool o) __attribute__((always_inline)) {   /* those that hold keys */
            const PaJobs &J = x.j[kind];
            const int KT = pa_tile(DV, J.form), nt = (p ? (n0 + KT - 1) / KT : 0) + (o ? (n1 + KT - 1) / KT : 0);
            return max(1u, J.dper.of(nt + J.per - 1));
        };
        const int s0 = splits(0, true, !x.group), s1 = x.kinds == 2 ? (int)splits(1, false, true) : 0, ns = s0 + s1;
        const int set0 = x.group ? pf : b, row_0 = x.group ? (b - pf * x.Bp) * per_seq + row : row;
        const float *p0 = x.part + x.j[0].part + ((size_t)(set0 * a.own.Hkv + hk) * x.j[0].ns * x.j[0].R + row_0) * pa_row(DV);
        const float *p1 = x.part + x.j[1].part + ((size_t)(b * a.own.Hkv + hk) * x.j[1].ns * x.j[1].R + row) * pa_row(DV);
        const size_t st0 = (size_t)x.j[0].R * pa_row(DV), st1 = (size_t)x.j[1].R * pa_row(DV);
        auto at = [&](int s) __attribute__((always_inline)) { return s < s0 ? p0 + s * st0 : p1 + (s - s0) * st1; };
        float4 u[FIRST], w[FIRST];
#pragma unroll
        for (int j = 0; j < FIRST; j++) {
            const float *p = at(min(grp + j * NG, ns - 1)) + min(c8, DV - 8);
            u[j] = *reinterpret_cast<const float4 *>(p);
            w[j] = *reinterpret_cast<const float4 *>(p + 4);
        }
        float4 h = make_float4(XA_MIN, 0.0f, -INFINITY, 0.0f);  /* reference, sum, remainder of this thread's split */
        if (tr < ns) h = *reinterpret_cast<const float4 *>(at(tr) + DV);
        float m = h.x, ml = h.z;                               /* the largest reference and its largest remainder */
        for (int s = tr + TR; s < ns; s += TR) {
            const float4 g = *reinterpret_cast<const float4 *>(at(s) + DV);
            ml = g.x > m ? g.z : g.x == m ? fmaxf(ml, g.z) : ml;
            m = fmaxf(m, g.x);
        }
        const float mw = grp_max<64>(m), lw = grp_max<64>(m == mw ? ml : -INFINITY);
        m = mw;
        ml = lw;
        if constexpr (WR > 1) {
            if (lane == 0) { red[sub][wv][0] = m; red[sub][wv][1] = ml; }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < WR; k++) {
                const float mk = red[sub][k][0], lk = red[sub][k][1];
                ml = mk > m ? lk : mk == m ? fmaxf(ml, lk) : ml;
                m = fmaxf(m, mk);
            }
        }
        float rs = 0.0f;
        for (int s = tr; s < ns; s += TR) {
            const float4 g = s == tr ? h : *reinterpret_cast<const float4 *>(at(s) + DV);
            const float f = __builtin_amdgcn_exp2f((g.x - m) + (g.z - ml));
            fac[sub][s] = f;
            rs = __builtin_fmaf(f, g.y, rs);
        }
        rs = grp_sum<64>(rs);
        if constexpr (WR > 1) {
            if (lane == 0) red[sub][wv][2] = rs;
        }
        __syncthreads();
        if constexpr (WR > 1) {
            rs = 0.0f;
#pragma unroll
            for (int k = 0; k < WR; k++) rs += red[sub][k][2];
        }
        float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        auto more = [&](float f, const float4 &u, const float4 &w) __attribute__((always_inline)) {
            const float e[8] = {u.x, u.y, u.z, u.w, w.x, w.y, w.z, w.w};
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = __builtin_fmaf(f, e[j], v[j]);
        };
#pragma unroll
        for (int j = 0; j < FIRST; j++)
            if (grp + j * NG < ns) more(fac[sub][grp + j * NG], u[j], w[j]);
#pragma unroll 4
        for (int s = grp + FIRST * NG; s < ns; s += NG) {
            const float *p = at(s) + min(c8, DV - 8);
            more(fac[sub][s], *reinterpret_cast<const float4 *>(p), *reinterpret_cast<const float4 *>(p + 4));
        }
#pragma unroll
        for (int k = CPR; k < 64; k *= 2)
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] += __shfl_xor(v[j], k, 64);
        if constexpr (WR > 1) {
            if (lane < CPR) {
                *reinterpret_cast<float4 *>(&acc[sub][wv][c8]) = make_float4(v[0], v[1], v[2], v[3]);
                *reinterpret_cast<float4 *>(&acc[sub][wv][c8 + 4]) = make_float4(v[4], v[5], v[6], v[7]);
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < WR; k++)
                if (k != wv)
#pragma unroll
                    for (int j = 0; j < 8; j++) v[j] += acc[sub][k][c8 + j];
        }
        if (grp == 0 && c8 < D && i0 + sub < rows) {
            const float inv = rs == 0.0f ? 0.0f : 1.0f / rs;
            const int t = x.dg.of(row);
            const long long out = b * a.o_batch + (hk * x.G + row - t * x.G) * a.o_head + t * a.o_token + c8;
            if (a.out_f32) {
                float *y = (float *)a.out + out;
                *reinterpret_cast<float4 *>(y) = make_float4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
                *reinterpret_cast<float4 *>(y + 4) = make_float4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv);
            } else {
                typename Xa<T>::v8 y;
#pragma unroll
                for (int j = 0; j < 8; j++) y[j] = (T)(v[j] * inv);
                *reinterpret_cast<typename Xa<T>::v8 *>((T *)a.out + out) = y;
            }
        }
        __syncthreads();                                       /* fac and acc serve the next rows */
    }
}

/* How a call runs: whether the rows of a prefix's sequences share its tiles, each kind's form and number of splits, by an
 * estimate of the launches' time, whose constants were measured (a workgroup's time for 1024 keys, alone on its CU, one of two and
 * one of as many as fit; 2.5 us for the rest of it; 4 us and 1.6 TB/s for what is joined). One token of 32 sequences over 8192
 * shared and 512 own keys takes 18 us with the prefix's rows together and 38 with each sequence's alone; 1296 tokens of 4 sequences
 * over 2048 + 1296 keys 104 us alone and 144 together; 14 x 58 tokens over 2 x 75761 keys 317 together and 541 alone (128 rows), 428 (64), 495
 * (32). Over 40 drawn shapes the form taken was within 8 % of
 * the best of the forced ones, and 1 % behind in the mean. Splits may make up to 2304 workgroups, several to a place one after the
 * other: their rounds even out, where 257 to 400 unsplit ones leave most CUs with one while others have two (24 x 348 tokens of 4
 * heads of 32 over 21135 keys 392 -> 205 us). Such rounds are estimated less well, so they have to win by 8 %: of 750 drawn shapes 27
 * took 5 to 48 % less for it and three 3 to 9 % more (without the 8 %, one took 21 % more). */
#define PA_SPLITS 256        /* of one kind at most: the join holds a factor of each in LDS */
struct PaPlan {
    int DV, join;
};
static PaPlan pa_plan(const aria_hip_prefix_attn *a, PaArgs &x) {
    const int Hkv = a->own.Hkv, P = a->prefix.B, np = a->prefix.cap, no = a->own.cap;
    PaPlan p;
    p.DV = (a->own.D + 31) / 32 * 32;
    x.G = a->H / Hkv;
    x.Bp = a->B / P;
    const long long R = (long long)a->Nq * x.G;
    /* us for 1024 keys of a workgroup that has its CU alone, of one of two, and of one of as many as a CU holds, and that number:
     * of forms 0, 1 and 2 at widths 32, 64, 96 and 128 */
    static const double alone[4][3] = {{5.2, 9.5, 15.5}, {5.2, 9.5, 17.0}, {9.9, 17.8, 22.5}, {10.0, 17.0, 25.0}};
    static const double paired[4][3] = {{7.4, 12.7, 21.0}, {8.6, 14.7, 25.3}, {14.5, 24.3, 33.2}, {15.0, 25.4, 38.4}};
    static const double full[4][3] = {{7.4, 12.7, 28.0}, {8.6, 14.7, 33.0}, {14.5, 24.3, 33.2}, {15.0, 25.4, 38.4}};
    static const int hold[4][3] = {{2, 2, 3}, {2, 2, 3}, {2, 2, 2}, {2, 2, 2}};
    const int wide = p.DV / 32 - 1;
    const double begin = 2.5;                                 /* us of a workgroup beside its tiles */
    struct Kind {
        long long sets, R, wg;
        int n0, n1, form, nt, ns, per;
    };
    auto kind = [&](long long sets, long long R, int n0, int n1, int form) {
        const int br = 32 << form, KT = pa_tile(p.DV, form);
        Kind k{sets, R, sets * Hkv * ((R + br - 1) / br), n0, n1, form, (n0 + KT - 1) / KT + (n1 + KT - 1) / KT, 1, 1};
        return k;
    };
    auto split = [&](Kind &k, long long ns) {
        k.ns = (int)std::max<long long>(1, std::min<long long>(ns, std::min(PA_SPLITS, k.nt)));
        k.per = std::max(1, (k.nt + k.ns - 1) / k.ns);
        k.ns = std::max(1, (k.nt + k.per - 1) / k.per);
    };
    auto estimate = [&](const Kind *k, int kinds) {
        long long jobs = 0;
        int slots = 768;
        double all = 0, longest = 0, shortest = 1e30, bytes = 0;
        for (int i = 0; i < kinds; i++) {
            jobs += k[i].wg * k[i].ns;
            slots = std::min(slots, 256 * hold[wide][k[i].form]);
        }
        for (int i = 0; i < kinds; i++) {
            const double keys = (double)k[i].per * pa_tile(p.DV, k[i].form) / 1024;
            all += (double)k[i].wg * k[i].ns * (begin + keys * full[wide][k[i].form]) / (256 * hold[wide][k[i].form]);
            longest = std::max(longest, begin + keys * (jobs <= 256 ? alone : jobs <= 512 ? paired : full)[wide][k[i].form]);
            shortest = std::min(shortest, begin + keys * alone[wide][k[i].form]);
            bytes += (double)k[i].sets * Hkv * k[i].ns * k[i].R * pa_row(p.DV) * sizeof(float);
        }
        /* what does not fit the CUs at once begins when something ends, and the last round is not full */
        const double t = jobs > slots ? std::max(all + 0.25 * longest, longest + shortest) : std::max(all, longest);
        return kinds == 2 || k[0].ns > 1 ? t + 4.0 + bytes / 1.6e6 : t;
    };
    double best = 1e30;
    Kind got[2];
    int got_kinds = 1, got_group = 0;
    auto attempt = [&](Kind *k, int kinds, int group, double more = 1.0) {
        const double t = more * estimate(k, kinds);
        if (t < best) {
            best = t;
            got[0] = k[0];
            if (kinds == 2) got[1] = k[1];
            got_kinds = kinds;
            got_group = group;
        }
    };
    for (int group = 0; group < (np > 0 && x.Bp > 1 ? 2 : 1); group++) {
        const int kinds = group && no > 0 ? 2 : 1;
        for (int form = 0; form < 3; form++) {
            Kind k[2];
            k[0] = group ? kind(P, R * x.Bp, np, 0, form) : kind(a->B, R, np, no, form);
            if (form && k[0].R <= 16 << form) continue;       /* half of the block idle */
            for (int j = 0; j < (kinds == 2 ? 3 : 1); j++) {
                if (kinds == 2) {
                    k[1] = kind(a->B, R, 0, no, R <= 32 ? 0 : R <= 64 ? 1 : 2);
                    split(k[1], j == 0 ? 1 : j == 1 ? (k[1].nt + 7) / 8 : (k[1].nt + 3) / 4);
                    if (j && k[1].ns == 1) break;
                }
                const long long others = kinds == 2 ? k[1].wg * k[1].ns : 0;
                const long long room[8] = {0, 256 - others, 512 - others, 512, 768 - others, 1024 - others, 1536 - others, 2304 - others};
                int last = 0;
                for (int i = 0; i < 8; i++) {
                    split(k[0], room[i] / k[0].wg);
                    if (k[0].ns != last) attempt(k, kinds, group, i < 4 ? 1.0 : 1.08);
                    last = k[0].ns;
                }
                split(k[0], (k[0].nt + 3) / 4);
                if (k[0].wg * k[0].ns < 256) attempt(k, kinds, group);
            }
        }
    }
    x.dhkv = HostDiv(Hkv);
    x.dseq = HostDiv((int)R);
    x.dg = HostDiv(x.G);
    x.dbp = HostDiv(x.Bp);
    x.group = got_group;
    x.kinds = got_kinds;
    x.j[0] = x.j[1] = PaJobs{};
    size_t part = 0;
    for (int i = 0; i < got_kinds; i++) {
        const Kind &k = got[i];
        PaJobs &J = x.j[i];
        J.sets = (int)k.sets;
        J.R = (int)k.R;
        J.nrb = (int)(k.wg / (k.sets * Hkv));
        J.form = k.form;
        J.ns = k.ns;
        J.per = k.per;
        J.jobs = (int)(k.wg * k.ns);
        J.use_prefix = k.n0 > 0;
        J.use_own = k.n1 > 0;
        J.tp = (k.n0 + pa_tile(p.DV, k.form) - 1) / pa_tile(p.DV, k.form);
        J.dnrb = HostDiv(J.nrb);
        J.dns = HostDiv(J.ns);
        J.dper = HostDiv(J.per);
        J.part = part;
        part += (size_t)k.sets * Hkv * k.ns * k.R * pa_row(p.DV);
    }
    p.join = got_kinds == 2 || got[0].ns > 1;
    return p;
}

extern "C" size_t aria_k_pattn_ws_bytes(const aria_hip_prefix_attn *a) {
    PaArgs x{};
    const PaPlan p = pa_plan(a, x);
    size_t n = 0;
    for (int i = 0; i < x.kinds; i++) n += (size_t)x.j[i].sets * a->own.Hkv * x.j[i].ns * x.j[i].R * pa_row(p.DV);
    return p.join ? n * sizeof(float) : 0;
}

template <typename T, int DV>
static void pa_launch(const PaPlan &p, const PaArgs &x, hipStream_t s) {
    const dim3 grid((unsigned)(((x.j[0].jobs + 7) & ~7) + ((x.j[1].jobs + 7) & ~7)));
    switch (1 << x.j[0].form | (x.kinds == 2 ? 1 << x.j[1].form : 0)) {
    case 1: hipLaunchKernelGGL((k_pattn<T, DV, 1>), grid, dim3(256), 0, s, x); break;
    case 2: hipLaunchKernelGGL((k_pattn<T, DV, 2>), grid, dim3(256), 0, s, x); break;
    case 3: hipLaunchKernelGGL((k_pattn<T, DV, 3>), grid, dim3(256), 0, s, x); break;
    case 4: hipLaunchKernelGGL((k_pattn<T, DV, 4>), grid, dim3(256), 0, s, x); break;
    case 5: hipLaunchKernelGGL((k_pattn<T, DV, 5>), grid, dim3(256), 0, s, x); break;
    case 6: hipLaunchKernelGGL((k_pattn<T, DV, 6>), grid, dim3(256), 0, s, x); break;
    }
    if (!p.join) return;
    const int rows = x.a.B * x.a.H * x.a.Nq;
    if (x.j[0].ns + x.j[1].ns > 16)
        hipLaunchKernelGGL((k_pattn_join<T, DV, 4>), dim3(std::min(rows, 1 << 20)), dim3(256), 0, s, x);
    else
        hipLaunchKernelGGL((k_pattn_join<T, DV, 1>), dim3(std::min((rows + 3) / 4, 1 << 20)), dim3(256), 0, s, x);
}

template <typename T>
static void pa_width(const PaPlan &p, const PaArgs &x, hipStream_t s) {
    if (p.DV == 32) pa_launch<T, 32>(p, x, s);
    else if (p.DV == 64) pa_launch<T, 64>(p, x, s);
    else if (p.DV == 96) pa_launch<T, 96>(p, x, s);
    else pa_launch<T, 128>(p, x, s);
}

extern "C" hipError_t aria_k_pattn_run(const aria_hip_prefix_attn *a, void *ws, hipStream_t s) {
    if (a->B <= 0 || a->Nq <= 0) return hipSuccess;
    PaArgs x{};
    x.a = *a;
    const PaPlan p = pa_plan(a, x);
    x.scale_log2 = a->scale * ARIA_LOG2E;
    x.part = p.join ? (float *)ws : nullptr;
    if (a->type == 1) pa_width<_Float16>(p, x, s);
    else pa_width<__bf16>(p, x, s);
    return hipGetLastError();
}
