/*
 * k_xattn.hip - cross attention to an encoder's states whose number differs from sequence to
 * sequence (gfx950): o = sum_j p_j v_j, p = softmax over the valid keys of scale * q . k_j, where key
 * j of sequence b is valid when j < kv_len[b] and mask[b, j] != 0. A row without a valid key is zero.
 * H query heads share Hkv key/value heads (H / Hkv consecutive query heads to each).
 *
 * One pass over the keys: each wave keeps 32 rows' running maximum, sum and fp32 output while key
 * tiles go by; scores never leave registers. The rows of one key/value head are (token, query head of
 * its group) pairs, so grouped heads and single tokens fill the 32 columns of an MFMA together.
 *
 * S^T = K Q^T and O^T = V^T P^T with v_mfma_f32_32x32x16: the accumulator of lane l (row l % 32, keys
 * 8 (r / 4) + 4 (l / 32) + r % 4) is the second product's B operand once rounded to 16 bits; V's
 * operand comes from key-major LDS by the transpose read in the same key order. Lanes l and l ^ 32
 * share a row, so a maximum needs one exchange.
 *
 * K and V tiles arrive by LDS DMA. Slots of keys that are not valid, and of dims past D, are
 * filled from 16 bytes of zeros: whatever lies in masked places (NaN, Inf, memory behind the last
 * state) never enters LDS. In a tile that has such keys one more product per 32 keys, of -inf at theirs and a column of ones,
 * adds -inf to their scores (0 before): 2 MFMAs in place of 32 selects on the busier VALU (4 x 16 x 4096 rows x up to
 * 2048 masked keys of 64: 109 us, 118 with selects).
 *
 * The weights are 2^(scale_log2 s - ref) with a lazy reference: it lies 7 below a tile's largest exponent where it moves,
 * and moves when a tile exceeds that by 8, which leaves O / l unchanged. The largest weight of a row is thus between 2^7 and
 * 2^15 (fp16 reaches 2^16), and in fp16 a weight vanishes only below 2^-32 of it. The reference starts at the lowest
 * finite value, so a slice whose keys all score -inf has weight zero instead of NaN.
 * Where fp32's steps at the reference are over 1 (2^24), what its rounding leaves out is kept beside it (lo, else 0), and the
 * exponents of a tile are taken in two steps: without that the largest weight could be anything up to 2^(half a step).
 * P is rounded to the type of V: the second product takes 16-bit operands, and its weights in two parts would double the
 * matrix work. That is half a step, 2^-11 or 2^-8, per weight at most (errors of an output against 64 bits 2.8e-4 in fp16
 * and 2.3e-3 in bf16, 2.1e-4 and 1.7e-3 with fp32 weights; the output's own rounding is in both); the row sum adds the
 * rounded values, so the weights still sum to one.
 */
#include "xattn_dev.h"
#include "aria_hip_kernels.h"

#include <algorithm>

/* 16-byte source of slots that hold no valid key or no dim */
__device__ const uint4 xa_zero = {0, 0, 0, 0};

struct XaArgs {
    aria_k_xattn a;
    int G, R;            /* query heads per key head; rows per (batch, key head) */
    int nrb, T;          /* row blocks per (batch, key head); workgroups per split */
    int ns, per;         /* splits of the keys across workgroups, key tiles to each */
    int plain;           /* every chunk holds dims, and lane offsets within a tile fit 32 bits */
    float scale_log2;
    float *part;         /* ns > 1: per (tile, split) 32 x DP sums, 32 references, 32 row sums, 32 remainders of the references */
};

/* keys of a tile where KS waves take tiles in turn */
__host__ __device__ constexpr int xa_tile(int DP) { return DP == 64 ? 64 : 32; }
/* floats of one partial result */
__host__ __device__ constexpr int xa_part(int DP) { return 32 * DP + 96; }

/* KS slices of the keys, each of QW waves of 32 rows that share its tiles; the slices' results are joined at the end. With
 * QW > 1 there are two stages, the next tile moving under the current one's products. With QW = 1 a wave works by itself,
 * without barriers, is bound by the keys' bytes, and has one stage, so that two workgroups fit a CU (16 x 4 key heads x up to
 * 8192 keys of 128: 56 us with two stages and one workgroup, 45 with one and two, the join included); the next tile's keys
 * then move while this one's values are added, its values while the scores are made (45 to 42). That overlap needs a call without a
 * mask: the compiler waits for a mask byte with everything that is on its way, the next tile's transfers included (the
 * same sequences, their keys in the last-level cache: 35.5 us with a mask that keeps 7 of 8 keys, 31.8 without).
 * Widths other than 64 and 128 are padded to the next of the two, and their chunks past D are looked at in every transfer: 4 x 16 x
 * 4096 rows x 2048 keys of 72 or 96 take 313 and 316 us, of 128 273, of 32 144 and of 64 148; one row over 16 x 4 x 8192
 * keys of 72 46 us, of 96 50, of 128 46.
 * What bounds it: with many rows the VALU, 69 % busy beside the MFMAs' 46 % at 4 x 16 x 4096 rows x 2048 keys of 64 (0.88
 * PFLOP/s; an exponential, a fused multiply-add, half a maximum, half a conversion and half a dot product per score);
 * with a single row the keys' bytes (4.9 TB/s without the join); at a few tiles a wave the latency of one tile, about 1 us. */
template <typename T, int DP, int KT, int QW, int KS>
__global__ __launch_bounds__(64 * QW * KS) void k_xattn(XaArgs x) {
    static_assert( (DP == 64 || DP == 128) && (KT == 64 || KT == 32), "");
    constexpr int NW = QW * KS;
    constexpr int NST = QW > 1 ? 2 : 1;             /* LDS stages */
    constexpr int CPR = DP / 8;                     /* 16-byte chunks per key row */
    constexpr uint64_t ALL = KT == 64 ? ~0ull : 0xFFFFFFFFull;   /* every key of a tile */
    constexpr int SLOTS = KT * CPR;                 /* per tile and operand */
    constexpr int ND = SLOTS / 64 / QW;             /* DMA instructions per wave, tile and operand */
    constexpr int TB = SLOTS * 16;                  /* bytes of a tile */
    constexpr int ES = DP + 4;                      /* floats per staged output row */
    constexpr int KB = KT / 32, DT = DP / 32, DS = DP / 16;
    constexpr int STAGE = 2 * TB * KS;              /* K and V of every slice */
    constexpr int EPI = NW * 32 * ES * 4 + NW * 96 * 4;
    __shared__ __attribute__((aligned(16))) uint8_t smem[NST * STAGE > EPI ? NST * STAGE : EPI];
    typedef typename Xa<T>::v8 v8;
    typedef typename Xa<T>::v2 v2;
    const aria_k_xattn &a = x.a;

    const int lane = threadIdx.x & 63, g = lane >> 5, l32 = lane & 31;
    const int wid = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int qw = wid % QW, ks = wid / QW;

    /* row blocks of one key head run on one XCD, whose L2 then holds its K and V; batches alternate
     * fastest so that unequal lengths spread over the XCDs */
    const int wg = xcd_tile(blockIdx.x, x.T * x.ns);
    if (wg >= x.T * x.ns) return;
    const int split = wg % x.ns, t = wg / x.ns;
    const int rb = t % x.nrb, bh = t / x.nrb, b = bh % a.B, hk = bh / a.B;
    const int n = a.kv_len ? min(max(a.kv_len[b], 0), a.Nk) : a.Nk;
    const uint8_t *mask = a.mask ? a.mask + b * a.mask_stride : nullptr;
    const int row = rb * 32 * QW + qw * 32 + l32;   /* this lane's row; rows past R repeat the last */
    const int rr = min(row, x.R - 1), tok = rr / x.G, hd = hk * x.G + rr % x.G;

    v8 qf[DS];
    {
        const T *q = (const T *)a.q + b * a.q_batch + hd * a.q_head + tok * a.q_token;
#pragma unroll
        for (int i = 0; i < DS; i++) {
            const int d = 16 * i + 8 * g;
            uint4 u = make_uint4(0, 0, 0, 0);
            if (d < a.D) u = *reinterpret_cast<const uint4 *>(q + d);
            qf[i] = __builtin_bit_cast(v8, u);
        }
    }

    /* this workgroup's tiles, and this slice's share of them: [t0, t1). Every split has as many tiles, and a short
     * sequence fewer splits, so that workgroups are equally long */
    const int nt = (n + KT - 1) / KT;
    const int w0 = x.ns > 1 ? split * x.per : 0, w1 = x.ns > 1 ? min(w0 + x.per, nt) : nt;
    if (split > 0 && w0 >= nt) return;      /* uniform per workgroup, before any barrier */
    const int sp = (w1 - w0 + KS - 1) / KS;
    const int t0 = min(w0 + ks * sp, w1), t1 = min(t0 + sp, w1);

    /* DMA sources: slot p of the tile holds chunk cp of key row r, and receives the chunk that the swizzle puts there.
     * Scalar bases move from tile to tile; a lane's offset within a tile stays */
    const char *kb = (const char *)((const T *)a.k + b * a.k_batch + hk * a.k_head + (long long)t0 * KT * a.k_token);
    const char *vb = (const char *)((const T *)a.v + b * a.v_batch + hk * a.v_head + (long long)t0 * KT * a.v_token);
    const long long kstep = KT * a.k_token * 2, vstep = KT * a.v_token * 2;
    auto slot = [&](int i, int &r, int &ck, int &cv) __attribute__((always_inline)) {
        const int p = 64 * (QW * i + qw) + lane, cp = p % CPR;
        r = p / CPR;
        ck = DP == 64 ? cp ^ ((r >> 1) & 7) : cp ^ (r & 15);
        cv = DP == 64 ? cp ^ (((r >> 1) & 1) << 2) : cp ^ ((r & 3) << 2);
    };
    unsigned koff_g[ND], voff_g[ND];
#pragma unroll
    for (int i = 0; i < ND; i++) {
        int r, ck, cv;
        slot(i, r, ck, cv);
        koff_g[i] = (unsigned)(r * a.k_token + 8 * ck) * 2;
        voff_g[i] = (unsigned)(r * a.v_token + 8 * cv) * 2;
    }
    auto dma_one = [&](auto IS_V, int buf, uint64_t bits) __attribute__((always_inline)) {
        constexpr bool is_v = decltype(IS_V)::value != 0;
        const uint32_t S = (uint32_t)(uintptr_t)smem + buf * STAGE + ks * 2 * TB + (is_v ? TB : 0) + 1024 * qw;
        const char *&base = is_v ? vb : kb;
        if (x.plain && bits == ALL) {
#pragma unroll
            for (int i = 0; i < ND; i++) dma16_s(base, is_v ? voff_g[i] : koff_g[i], S + 1024 * QW * i);
        } else {
#pragma unroll 1   /* unrolled, half as much code again, which every launch fetches first: 0.2 us */
            for (int i = 0; i < ND; i++) {
                int r, ck, cv;
                slot(i, r, ck, cv);
                const int c = is_v ? cv : ck;
                const bool ok = ((bits >> r) & 1) && 8 * c < a.D;
                dma16(ok ? base + (r * (is_v ? a.v_token : a.k_token) + 8 * c) * 2 : (const char *)&xa_zero, S + 1024 * QW * i);
            }
        }
        base += is_v ? vstep : kstep;
    };
    auto dma = [&](int buf, uint64_t bits) __attribute__((always_inline)) {
        dma_one(IC<0>{}, buf, bits);
        dma_one(IC<1>{}, buf, bits);
    };
    /* the valid keys of tile i (bit j: key KT i + j) where no mask says otherwise */
    auto in_len = [&](int i) __attribute__((always_inline)) -> uint64_t {
        const int left = n - i * KT;
        return left >= KT ? ALL : left <= 0 ? 0ull : (1ull << left) - 1;
    };
    auto mask_byte = [&](int i) __attribute__((always_inline)) -> int {
        const int j = i * KT + (lane & (KT - 1));
        return mask && i < t1 && j < n ? mask[j] : 1;
    };
    auto to_bits = [&](int i, int byte) __attribute__((always_inline)) -> uint64_t {
        return i < t1 ? in_len(i) & __ballot(byte != 0) : 0ull;
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

    const unsigned ninf = g ? 0u : Xa<T>::NINF;     /* element 0 of lanes 0 .. 31, whose keys are their numbers */
    auto scores = [&](int buf, uint64_t bits, xa_f32x16_t (&s)[KB]) __attribute__((always_inline)) {
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
        if (bits != ALL) {   /* one more product adds -inf (a 16-bit value) times 1 to the scores of the other keys */
#pragma unroll
            for (int kb = 0; kb < KB; kb++) {
                const unsigned w = ~(unsigned)(bits >> (32 * kb)) >> l32;
                s[kb] = Xa<T>::mfma8(make_uint2(0u - (w & 1u) & ninf, 0), make_uint2(Xa<T>::ONE, 0), s[kb]);
            }
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
    /* this wave's transfers have landed and its fragment reads have returned: without the latter a read
     * still in flight would race with the next transfer into its stage. The compiler does not know of
     * the transfers, so this is also its fence */
    auto drain = []() __attribute__((always_inline)) { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory"); };
    auto meet = [&]() __attribute__((always_inline)) {
        if constexpr (QW > 1) __syncthreads();
    };

    uint64_t cur = to_bits(t0, mask_byte(t0));
    if constexpr (NST == 2) {
        uint64_t nxt = to_bits(t0 + 1, mask_byte(t0 + 1));
        if (t0 < t1) dma(0, cur);
        drain();
        /* the rows are here: this use tells the compiler, which else would wait for them, and with them for the next
         * tile's transfer, at every tile's first product */
#pragma unroll
        for (int i = 0; i < DS; i++) asm volatile("" : "+v"(qf[i]));
        meet();
        /* one tile from stage BUF; a compile-time stage keeps every LDS offset an immediate */
        auto turn = [&](auto BUF, int i) __attribute__((always_inline)) {
            constexpr int buf = decltype(BUF)::value;
            const int byte = mask_byte(i + 2);
            if (i + 1 < t1) dma(buf ^ 1, nxt);
            if (cur) {
                xa_f32x16_t s[KB];
                scores(buf, cur, s);
                move_ref(s);
                add(buf, s);
            }
            drain();
            meet();
            cur = nxt;
            nxt = to_bits(i + 2, byte);
        };
        for (int i = t0; i < t0 + sp; i += 2) {     /* every slice meets as often; its tiles end at t1 */
            turn(IC<0>{}, i);
            if (i + 1 >= t0 + sp) break;
            turn(IC<1>{}, i + 1);
        }
    } else {
        /* keys of tile i + 1 leave when the scores of tile i stand, its values when tile i is added: one of the two is
         * always on its way. Newer transfers may be in flight behind the ones waited for */
        auto behind = [](bool more) __attribute__((always_inline)) {
            if (more) asm volatile("s_waitcnt vmcnt(%0)" : : "i"(ND) : "memory");
            else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        };
        auto have_read = []() __attribute__((always_inline)) { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); };
        int byte = mask_byte(t0 + 1);
        if (t0 < t1) dma(0, cur);
        behind(t0 < t1);
#pragma unroll
        for (int i = 0; i < DS; i++) asm volatile("" : "+v"(qf[i]));
        for (int i = t0; i < t1; i++) {
            const bool more = i + 1 < t1;
            uint64_t nxt = in_len(i + 1);
            if (mask) nxt &= __ballot(byte != 0);
            behind(true);
            xa_f32x16_t s[KB];
            if (cur) scores(0, cur, s);
            have_read();
            if (more) dma_one(IC<0>{}, 0, nxt);
            if (mask) byte = mask_byte(i + 2);
            if (cur) move_ref(s);
            behind(more);
            if (cur) add(0, s);
            have_read();
            if (more) dma_one(IC<1>{}, 0, nxt);
            cur = nxt;
        }
    }

    /* join: lanes l and l ^ 32 hold half of a row's sum each */
    l += xor32_f32(l, lane);
    float *E = (float *)smem + wid * 32 * ES;
    float *ML = (float *)smem + NW * 32 * ES;       /* per wave 32 references, 32 sums, 32 remainders of the references */
    if (QW == 1) __syncthreads();                    /* slices still reading their stages */
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
        for (int r = 0; r < 4; r++)
            *reinterpret_cast<float4 *>(E + l32 * ES + 32 * d + 8 * r + 4 * g) =
                make_float4(o[d][4 * r], o[d][4 * r + 1], o[d][4 * r + 2], o[d][4 * r + 3]);
    if (KS > 1 && g == 0) { ML[wid * 96 + l32] = ref; ML[wid * 96 + 32 + l32] = l; ML[wid * 96 + 64 + l32] = lo; }
    __syncthreads();

    /* a group of CPR lanes finishes one row, 8 dims per lane; the KS waves of a block of rows take them in turn */
    constexpr int RPW = 64 / CPR;                    /* rows per wave at once */
    const int c8 = 8 * (lane % CPR);
#pragma unroll 1
    for (int i = ks; i < 32 / RPW; i += KS) {
        const int q = i * RPW + lane / CPR;          /* row within the block */
        float v[8], rs, rm, rl;
        if constexpr (KS == 1) {
            const float *e = E + q * ES + c8;
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = e[j];
            rs = __shfl(l, q, 64);
            rm = __shfl(ref, q, 64);
            rl = __shfl(lo, q, 64);
        } else {
            float m[KS], c[KS];
#pragma unroll
            for (int w = 0; w < KS; w++) {
                m[w] = ML[(w * QW + qw) * 96 + q];
                c[w] = ML[(w * QW + qw) * 96 + 64 + q];
            }
            rm = m[0];                               /* the largest reference, and of those that have it the largest remainder */
            rl = c[0];
#pragma unroll
            for (int w = 1; w < KS; w++) {
                rl = m[w] > rm ? c[w] : m[w] == rm ? fmaxf(rl, c[w]) : rl;
                rm = fmaxf(rm, m[w]);
            }
            rs = 0.0f;
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
        }
        const int orow = rb * 32 * QW + qw * 32 + q;
        if (orow >= x.R || c8 >= a.D) continue;
        if (x.ns > 1) {
            float *P = x.part + (size_t)(t * x.ns + split) * xa_part(DP);
            *reinterpret_cast<float4 *>(P + q * DP + c8) = make_float4(v[0], v[1], v[2], v[3]);
            *reinterpret_cast<float4 *>(P + q * DP + c8 + 4) = make_float4(v[4], v[5], v[6], v[7]);
            if (c8 == 0) { P[32 * DP + q] = rm; P[32 * DP + 32 + q] = rs; P[32 * DP + 64 + q] = rl; }
            continue;
        }
        const float inv = rs > 0.0f ? 1.0f / rs : 0.0f;
        const long long at = b * a.o_batch + (hk * x.G + orow % x.G) * a.o_head + (orow / x.G) * a.o_token + c8;
        /* non-temporal: the L2s keep keys and values (2 x 16 x 1296 rows x up to 257 keys 12.2 us, 11.9 so) */
        if (a.out_f32) {
            typedef float f4_t __attribute__((ext_vector_type(4)));
            f4_t *y = reinterpret_cast<f4_t *>((float *)a.out + at);
            __builtin_nontemporal_store(f4_t{v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv}, y);
            __builtin_nontemporal_store(f4_t{v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv}, y + 1);
        } else {
            v8 y;
#pragma unroll
            for (int j = 0; j < 8; j++) y[j] = (T)(v[j] * inv);
            __builtin_nontemporal_store(y, reinterpret_cast<v8 *>((T *)a.out + at));
        }
    }
}

/* Joins the partial results of one row: a group of DP / 8 lanes per 8 dims, the wave's 64 / (DP / 8) groups take the
 * splits in turn and add up through lane exchanges */
template <typename T, int DP>
__global__ __launch_bounds__(64) void k_xattn_join(XaArgs x) {
    constexpr int CPR = DP / 8, NG = 64 / CPR;
    const aria_k_xattn &a = x.a;
    const int rows = min(32, x.R);                             /* one row block where R is smaller */
    const int t = blockIdx.x / rows, q = blockIdx.x % rows;
    const int rb = t % x.nrb, bh = t / x.nrb, b = bh % a.B, hk = bh / a.B, row = rb * 32 + q;
    if (row >= x.R) return;
    const int lane = threadIdx.x, grp = lane / CPR, c8 = 8 * (lane % CPR);
    const float *P = x.part + (size_t)t * x.ns * xa_part(DP);
    const int n = a.kv_len ? min(max(a.kv_len[b], 0), a.Nk) : a.Nk;
    const int ns = max(1, (n + x.per * xa_tile(DP) - 1) / (x.per * xa_tile(DP)));   /* the splits that hold keys */
    float m = XA_MIN, ml = -INFINITY;                          /* the largest reference and its largest remainder */
    for (int s = lane; s < ns; s += 64) {
        const float *p = P + (size_t)s * xa_part(DP) + 32 * DP + q;
        ml = p[0] > m ? p[64] : p[0] == m ? fmaxf(ml, p[64]) : ml;
        m = fmaxf(m, p[0]);
    }
    const float ma = grp_max<64>(m);
    ml = grp_max<64>(m == ma ? ml : -INFINITY);
    m = ma;
    float rs = 0.0f, v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (c8 < a.D)
#pragma unroll 4
        for (int s = grp; s < ns; s += NG) {
            const float *p = P + (size_t)s * xa_part(DP);
            const float f = __builtin_amdgcn_exp2f((p[32 * DP + q] - m) + (p[32 * DP + 64 + q] - ml));
            rs = __builtin_fmaf(f, p[32 * DP + 32 + q], rs);
            const float4 u = *reinterpret_cast<const float4 *>(p + q * DP + c8), w = *reinterpret_cast<const float4 *>(p + q * DP + c8 + 4);
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
    if (grp != 0 || c8 >= a.D) return;
    const float inv = rs > 0.0f ? 1.0f / rs : 0.0f;
    const long long at = b * a.o_batch + (hk * x.G + row % x.G) * a.o_head + (row / x.G) * a.o_token + c8;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        if (a.out_f32) ((float *)a.out)[at + j] = v[j] * inv;
        else ((T *)a.out)[at + j] = (T)(v[j] * inv);
    }
}

/* How a call runs: qw blocks of 32 rows and ks slices of the keys to a workgroup, ns splits of the keys across workgroups.
 *  qw 1, ks 4: up to 32 rows a key head, and where blocks of 128 rows would leave CUs idle, which blocks of 32 rows then
 *    fill, each reading the keys for itself (16 heads x 172 rows x 257 keys of 64: 6.2 us, 8.5 with qw 4; x 710 rows x 1024 keys: 25.2 and 14.5);
 *  qw 4, ks 2: up to a workgroup per CU, and up to 700 of them over long keys of 64 (2 x 16 x 710 rows x 257 keys: 8.9 us, 9.5 with
 *    one slice; 2 x 16 x 1296 x 1296: 29.1 and 31.4, of 128 54.2 and 49.4);
 *  qw 4, ks 1; and qw 8, width 64, from four rounds of 256 rows on: it gains 3 - 7 % from two rounds on (2 x 16 x 4096 x 2048
 *    82.5 and 77.8 us, 4 x 16 x 4096 x 2048 158 and 152, 8 x 16 x 3000 x 257 47.5 and 46.0) and loses below (1296 rows of 64 heads,
 *    1.5 rounds, x 2048: 62.6 and 69.9); of 128, where 8 waves' registers fill the CU: 164 and 168.
 * Over 444 shapes (8 to 128 heads in all, 40 to 4096 rows, 64 to 2048 keys, widths 64 and 128) the form taken is within 5 % of
 * the best in 348 and 4 % behind in the mean. It is furthest behind at 64 to 128 blocks of 128 rows over 1300 keys and more, where
 * single waves' slices would be faster (8 heads x 1296 x 2048: 23.1 us, 15.1 with qw 1). */
struct XaPlan { int qw, ks, DP, nrb, T, ns, per; };
static XaPlan xa_plan(const aria_k_xattn *a) {
    XaPlan p;
    const long long R = (long long)a->Nq * (a->H / a->Hkv), bh = (long long)a->B * a->Hkv;
    auto tiles = [&](int qw) { return bh * ((R + 32 * qw - 1) / (32 * qw)); };
    p.DP = a->D <= 64 ? 64 : 128;
    const long long w4 = tiles(4);
    p.qw = R <= 32 || w4 < 64 || (w4 < 128 && a->Nk <= 512) ? 1 : p.DP == 64 && tiles(8) >= 1024 ? 8 : 4;
    p.ks = p.qw == 1 ? 4 : p.qw == 4 && (w4 < 300 || (w4 < 700 && p.DP == 64 && a->Nk >= 1024)) ? 2 : 1;
    p.T = (int)tiles(p.qw);
    p.nrb = (int)(p.T / bh);
    p.ns = 1;
    if (p.qw == 1) {
        /* at least 256 keys to a workgroup, and as many workgroups as the CUs hold at once, two each (16 x 4 key heads x up
         * to 8192 keys of 128: 39.4 us, 42 with twice as many, 47 with three quarters) */
        p.ns = std::max(1, std::min(a->Nk / 256, 512 / p.T));
    }
    p.per = ((a->Nk + xa_tile(p.DP) - 1) / xa_tile(p.DP) + p.ns - 1) / p.ns;
    return p;
}

extern "C" size_t aria_k_xattn_ws_bytes(const aria_k_xattn *a) {
    const XaPlan p = xa_plan(a);
    return p.ns > 1 ? (size_t)p.T * p.ns * xa_part(p.DP) * sizeof(float) : 0;
}

template <typename T>
static hipError_t xa_launch(const XaPlan &p, const XaArgs &x, hipStream_t s) {
    const int n = p.T * p.ns;
    const dim3 grid((unsigned)((n + 7) / 8 * 8));
    if (p.qw == 1) {
        if (p.DP == 64) hipLaunchKernelGGL((k_xattn<T, 64, 64, 1, 4>), grid, dim3(256), 0, s, x);
        else hipLaunchKernelGGL((k_xattn<T, 128, 32, 1, 4>), grid, dim3(256), 0, s, x);
        if (p.ns > 1) {
            const dim3 rows((unsigned)p.T * (unsigned)(x.R < 32 ? x.R : 32));
            if (p.DP == 64) hipLaunchKernelGGL((k_xattn_join<T, 64>), rows, dim3(64), 0, s, x);
            else hipLaunchKernelGGL((k_xattn_join<T, 128>), rows, dim3(64), 0, s, x);
        }
    } else if (p.qw == 8) {
        hipLaunchKernelGGL((k_xattn<T, 64, 64, 8, 1>), grid, dim3(512), 0, s, x);
    } else if (p.ks == 2) {
        if (p.DP == 64) hipLaunchKernelGGL((k_xattn<T, 64, 64, 4, 2>), grid, dim3(512), 0, s, x);
        else hipLaunchKernelGGL((k_xattn<T, 128, 64, 4, 2>), grid, dim3(512), 0, s, x);
    } else {
        if (p.DP == 64) hipLaunchKernelGGL((k_xattn<T, 64, 64, 4, 1>), grid, dim3(256), 0, s, x);
        else hipLaunchKernelGGL((k_xattn<T, 128, 64, 4, 1>), grid, dim3(256), 0, s, x);
    }
    return hipGetLastError();
}

extern "C" hipError_t aria_k_xattn_run(const aria_k_xattn *a, void *ws, hipStream_t s) {
    if (a->B <= 0 || a->Nq <= 0) return hipSuccess;
    const XaPlan p = xa_plan(a);
    XaArgs x;
    x.a = *a;
    x.G = a->H / a->Hkv;
    x.R = a->Nq * x.G;
    x.nrb = p.nrb;
    x.T = p.T;
    x.ns = p.ns;
    x.per = p.per;
    x.plain = a->D == p.DP && a->k_token < (1 << 24) && a->v_token < (1 << 24);   /* 64 keys x 2 bytes x 2^24 = 2^31 */
    x.scale_log2 = a->scale * ARIA_LOG2E;
    x.part = (float *)ws;
    return a->type == 1 ? xa_launch<_Float16>(p, x, s) : xa_launch<__bf16>(p, x, s);
}
