/*
 * k_mx4_gemm.hip - products of MXFP4 rows on gfx950's block-scaled MFMA:
 * y[m, n] = sum over blocks b of 2^(ex[m,b] + ew[n,b] - 254) sum_i cx[m,b,i] cw[n,b,i] (+ bias[n]),
 * and the gated form y[m, i] = v * g / (1 + e^-g) with v, g the products of weight rows i and
 * inner + i. fp4 x fp4 products and their block sums are exact; sums over blocks are fp32.
 *
 * v_mfma_scale_f32_32x32x64_f8f6f4 takes one block of 32 codes (16 bytes) and one scale byte per
 * lane and operand, so a packed row is the operand as it lies in memory: no unpacking at all. Weights
 * are the A operand and activations the B operand: a lane's accumulators are then 4 consecutive
 * columns n of one row m. Sums over K do not depend on which block a lane half takes, so half h takes
 * blocks 4h .. 4h + 3 of each 8-block chunk: its four scale bytes are one dword, picked by op_sel.
 */
#include "mx4_dev.h"

struct MxArgs {
    void *y;
    const uint8_t *xq, *xs, *wq, *ws;
    const float *bias;
    int M, N;          /* N: output columns (GLU: inner) */
    int nb;            /* blocks of 32 along K */
    int ytype;
    int tm, tn, T;     /* tiles along M and N, tiles in all */
    int vec;           /* rows of y are 16-byte aligned */
};

/* the scale bytes of a row's last blocks, b to b + 15; absent ones read as 0 */
__device__ __forceinline__ uint4 mx_scale_end(const uint8_t *row, int b, int nb) {
    unsigned w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16; i++)
        if (b + i < nb) w[i >> 2] |= (unsigned)row[b + i] << (8 * (i & 3));
    return make_uint4(w[0], w[1], w[2], w[3]);
}

/* V results of one row from column n on: four fp32 or eight 16-bit values. Non-temporal: they are not read here, and in
 * the L2s they would take the operands' place (2592 x 1024 -> 4096 to bf16 13.4 us, 14.6 else; to fp32 15.0 and 15.8; 8192 x
 * 1024 -> 8192, 57 to bf16 and 69 to fp32, within 3 % either way) */
template <int V>
__device__ __forceinline__ void mx_store_row(const MxArgs &a, int m, int n, const float (&v)[V]) {
    const size_t at = (size_t)m * a.N + n;
    if (a.vec && n + V <= a.N) {
        if constexpr (V == 4) {
            typedef float v4_t __attribute__((ext_vector_type(4)));
            __builtin_nontemporal_store(v4_t{v[0], v[1], v[2], v[3]}, reinterpret_cast<v4_t *>((float *)a.y + at));
        } else if (a.ytype == MX_F16) {
            typedef _Float16 v8_t __attribute__((ext_vector_type(8)));
            v8_t o;
#pragma unroll
            for (int i = 0; i < 8; i++) o[i] = (_Float16)v[i];
            __builtin_nontemporal_store(o, reinterpret_cast<v8_t *>((_Float16 *)a.y + at));
        } else {
            typedef __bf16 v8_t __attribute__((ext_vector_type(8)));
            v8_t o;
#pragma unroll
            for (int i = 0; i < 8; i++) o[i] = (__bf16)v[i];
            __builtin_nontemporal_store(o, reinterpret_cast<v8_t *>((__bf16 *)a.y + at));
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; i++)
            if (n + i < a.N) mx_store(a.y, a.ytype, at + i, v[i]);
    }
}

/* v, as a value that the compiler knows nothing of: what is computed from it is not kept in registers from further up */
__device__ __forceinline__ int fresh(int v) {
    asm volatile("" : "+v"(v));
    return v;
}

/* the same for a value that is one for the wave, which stays in a scalar register */
__device__ __forceinline__ uint32_t fresh_s(uint32_t v) {
    v = __builtin_amdgcn_readfirstlane(v);
    asm volatile("" : "+s"(v));
    return v;
}

/* LDS written by some lanes of a wave stands for its other lanes behind this, and what was read before it has been: LDS is in
 * order within a wave, so only the compiler has to keep the order, and no instruction comes of it */
__device__ __forceinline__ void wave_order() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

/*
 * WK groups of WM x WN waves; a group's waves share LDS stages and take one of WK parts of K; a wave owns
 * FM x FN blocks of 32 x 32 outputs (GLU: the first half of its FN are value rows, the second half
 * the gate rows of the same columns). Chunks of 256 K (128 bytes of every row) move to LDS by DMA, NST stages;
 * chunk c of a row sits at c ^ ((row >> 1) & 7), so that each eight lanes of a fragment read (32 rows x 16 bytes per lane half)
 * meet every bank once. (The conflicts that are counted, a third of the LDS' active cycles at 8192 x 4096 x 8192, are 8 % in the
 * form that reads the same fragments but no scales from LDS: they come from the scale dwords, 16 bytes apart, and
 * the output's staging.) With two stages the next chunk moves under the current one's products; with one, the CU's other
 * workgroups fill the wait.
 * Barriers (none where a group is one wave) follow the wait for this wave's transfers and fragment reads, so behind one the
 * chunk is whole and, with two stages, the other stage free.
 * What bounds it: at 8192 x 4096 x 8192 waiting: the matrix pipes are busy in 41 - 43 % of the launch's cycles, with one workgroup a
 * CU whose waves all wait for their transfers and meet at every chunk (the fp4 MFMA from registers reaches 6.6 - 6.9
 * PFLOP/s on random codes, 8.9 on zeros; the chunk loop 4.4, the launch with its prologue and output 3.6). Power shows
 * in the clock, 1.9 - 2.0 GHz of 2.4 in that launch;
 * at a few rounds of tiles the latency of a tile's first chunk and of its output.
 */
template <int FM, int FN, int WM, int WN, int WK, int NST, bool GLU>
__global__ __launch_bounds__(64 * WM * WN * WK) void k_mx4_gemm(MxArgs a) {
    constexpr int NW = WM * WN * WK, GW = WM * WN;
    constexpr int BM = 32 * FM * WM, BN = 32 * FN * WN;          /* rows of x and of w per tile */
    constexpr int OW = GLU ? 16 * FN : 32 * FN;                  /* columns of y per wave */
    constexpr int NR = BM + BN, STAGE = NR * 128;
    constexpr int ND = NR / 8 / GW;                              /* DMA instructions per wave and chunk */
    constexpr int NDX = BM / 8 / GW;                             /* the first of them move x */
    static_assert(BM % (8 * GW) == 0 && BN % (8 * GW) == 0 && (!GLU || FN % 2 == 0), "");
    constexpr int ES = 32 * FN + 4;                              /* floats per staged row */
    constexpr int EPI = NW * 32 * ES * 4;
    constexpr bool SHARED = GW > 1;                              /* scales go through LDS */
    constexpr int SCALES = SHARED ? NR * 16 : 0;                 /* scale bytes of two chunks */
    constexpr int NS = SHARED ? NR / (64 * GW) : 1;              /* scale rows per lane */
    static_assert(SHARED ? NR % (64 * GW) == 0 && WK == 1 : NST == 1, "");
    constexpr int GROUP = NST * STAGE + 2 * SCALES;              /* LDS of one K group */
    constexpr int BIAS = WK * GROUP > EPI ? WK * GROUP : EPI;    /* biases of the tile's w rows behind the rest */
    __shared__ __attribute__((aligned(16))) uint8_t smem[BIAS + (SHARED ? 4 * BN : 0)];
    const int lane = threadIdx.x & 63, l32 = lane & 31, h = lane >> 5;
    const int wid = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int wk = wid / GW, gw = wid % GW, wm = gw / WN, wn = gw % WN;

    /* tiles in bands of 4 tile rows, columns fastest after them: the tiles that run side by side on an XCD then
     * share few panels of both operands */
    const int t = xcd_tile(blockIdx.x, a.T);
    if (t >= a.T) return;
    const int band = t / (4 * a.tn), gm = min(4, a.tm - 4 * band), r = t - band * 4 * a.tn;
    const int m0 = (4 * band + r % gm) * BM, n0 = (r / gm) * (OW * WN);

    /* w rows of the LDS tile lie behind its x rows; GLU: wave by wave, value rows before gate rows. The column of
     * w row i, counted from n0, and whether it is a gate row */
    auto is_gate = [&](int i) __attribute__((always_inline)) { return GLU && i % (32 * FN) >= OW; };
    auto w_col = [&](int i) __attribute__((always_inline)) {
        const int c = GLU ? i / (32 * FN) * OW + i % OW : i;
        return min(c, a.N - 1 - n0);
    };
    /* lane offsets of the DMA slots: slot lane of instruction i fills 16 bytes of LDS row 8 (GW i + gw) + lane / 8 */
    unsigned off[ND];
    const size_t rb = (size_t)a.nb * 16;
    auto source = [&](int i, int c) __attribute__((always_inline)) -> unsigned {
        const int row = 8 * (GW * i + gw) + (lane >> 3);
        if (i < NDX) return (unsigned)((min(m0 + row, a.M - 1) - m0) * rb) + 16 * c;
        return (unsigned)(w_col(row - BM) * rb) + 16 * c;
    };
#pragma unroll
    for (int i = 0; i < ND; i++) {
        const int row = 8 * (GW * i + gw) + (lane >> 3);
        off[i] = source(i, (lane & 7) ^ ((row >> 1) & 7));
    }
    const uint8_t *xb = a.xq + (size_t)m0 * rb, *wb = a.wq + (size_t)n0 * rb;
    const size_t gate = (size_t)a.N * rb;                        /* from a value row to its gate row */
    const uint32_t sb = (uint32_t)(uintptr_t)smem + wk * GROUP;

    /* SHARED: scales of two chunks at a time, 16 bytes of a row per lane, through registers to LDS. (A dword per fragment row
     * and lane half, straight to registers, kept the address unit busy for longer than the products took: 200 us
     * against 155 at 8192 x 4096 x 8192) */
    const uint8_t *srow[NS];
#pragma unroll
    for (int i = 0; i < NS; i++) {
        const int row = 64 * (GW * i + gw) + lane;
        srow[i] = row < BM ? a.xs + (size_t)min(m0 + row, a.M - 1) * a.nb
                           : a.ws + ((size_t)(n0 + w_col(row - BM)) + (is_gate(row - BM) ? a.N : 0)) * a.nb;
    }
    uint4 sreg[NS];
    auto load_scales = [&](int c) __attribute__((always_inline)) {   /* a row's scales start at any byte */
#pragma unroll
        for (int i = 0; i < NS; i++) __builtin_memcpy(&sreg[i], srow[i] + 8 * c, 16);
    };
    auto put_scales = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < NS; i++)
            *reinterpret_cast<uint4 *>(smem + wk * GROUP + NST * STAGE + buf * SCALES + (64 * (GW * i + gw) + lane) * 16) = sreg[i];
    };

    /* a one-wave group takes its few scales straight to registers, a dword per fragment row and lane half */
    const uint8_t *xsr[FM], *wsr[FN];
#pragma unroll
    for (int i = 0; i < FM; i++) xsr[i] = a.xs + (size_t)min(m0 + (wm * FM + i) * 32 + l32, a.M - 1) * a.nb + 4 * h;
#pragma unroll
    for (int j = 0; j < FN; j++) {
        const int i = (wn * FN + j) * 32 + l32;
        wsr[j] = a.ws + ((size_t)(n0 + w_col(i)) + (is_gate(i) ? a.N : 0)) * a.nb + 4 * h;
    }
    auto scales = [&](unsigned (&x)[FM], unsigned (&w)[FN], int c) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < FM; i++) __builtin_memcpy(&x[i], xsr[i] + 8 * c, 4);
#pragma unroll
        for (int j = 0; j < FN; j++) __builtin_memcpy(&w[j], wsr[j] + 8 * c, 4);
    };

    /* chunk c to stage buf. In a row's last, short chunk (END) the slots of absent blocks take the chunk's first
     * block instead: their scales are 0, and 2^-127 times 2^-127 leaves nothing of any code */
    const uint32_t mb = fresh_s(sb + gw * 1024);
    auto issue = [&](auto END, int buf, int c) __attribute__((always_inline)) {
        static_for<ND>([&](auto I) __attribute__((always_inline)) {
            constexpr int i = decltype(I)::value;
            const int row0 = 8 * (GW * i + gw);
            unsigned o = off[i];
            if constexpr (decltype(END)::value != 0) {
                const int ln = fresh(lane), row = row0 + (ln >> 3), k = (ln & 7) ^ ((row >> 1) & 7);
                if (k >= a.nb - 8 * c) o -= 16 * k;
            }
            const size_t at = (size_t)c * 128;
            const uint8_t *p;
            if constexpr (i < NDX) p = xb + at;
            else p = wb + at + (is_gate(row0 - BM) ? gate : (size_t)0);
            dma16_s(p, o, mb + buf * STAGE + i * (1024 * GW));
        });
    };

    /* The biases end under the first chunk's transfer. SHARED: those of the tile's w rows go to LDS as well, since loads to
     * registers behind a branch are waited for where it ends, before any transfer has left */
    float bias[8], gbias[8];
#pragma unroll
    for (int e = 0; e < 8; e++) { bias[e] = 0.0f; gbias[e] = 0.0f; }
    const int bv = a.ytype == MX_F32 ? 4 : 8, bc = bv * (lane % (OW / bv));   /* this lane's columns of the wave's */
    if constexpr (SHARED) {
        static_assert(BN % 64 == 0 && BN / 64 <= NW, "");
        const int i = 64 * wid + lane;
        if (a.bias && wid < BN / 64) dma4(a.bias + n0 + w_col(i) + (is_gate(i) ? a.N : 0), (uint32_t)(uintptr_t)smem + BIAS + 256 * wid);
    } else if (a.bias) {
        const int n = n0 + wn * OW + bc;
        if (n + bv <= a.N) {
            __builtin_memcpy(bias, a.bias + n, 16);
            if (bv == 8) __builtin_memcpy(bias + 4, a.bias + n + 4, 16);
            if constexpr (GLU) {
                __builtin_memcpy(gbias, a.bias + a.N + n, 16);
                if (bv == 8) __builtin_memcpy(gbias + 4, a.bias + a.N + n + 4, 16);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (e < bv && n + e < a.N) {
                    bias[e] = a.bias[n + e];
                    if constexpr (GLU) gbias[e] = a.bias[a.N + n + e];
                }
        }
    }

    mx_f32x16_t acc[FM][FN];
    static_for<FM * FN>([&](auto I) __attribute__((always_inline)) {
        acc[I / FN][I % FN] = mx_f32x16_t{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
    });

    /* four MFMA steps; the fragments of step J + 1 are read while step J multiplies. Each step is a scheduling
     * region in which the reads are spread over the MFMAs */
    uint32_t fx[4], fw[4];                                       /* where step j's first fragments lie in a stage */
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const uint32_t at = l32 * 128 + (((4 * h + j) ^ ((l32 >> 1) & 7)) << 4);
        fx[j] = at + wm * FM * 4096;
        fw[j] = at + (BM / 32 + wn * FN) * 4096;
    }
    const uint32_t cx = (wm * FM * 32 + l32) * 16 + 4 * h, cw = cx + (BM + (wn * FN - wm * FM) * 32) * 16;
    auto shared_scales = [&](unsigned (&x)[FM], unsigned (&w)[FN], int buf, int sbuf) __attribute__((always_inline)) {
        const uint8_t *C = smem + wk * GROUP + NST * STAGE + sbuf * SCALES + buf * 8;
#pragma unroll
        for (int i = 0; i < FM; i++) x[i] = *reinterpret_cast<const unsigned *>(C + cx + i * 512);
#pragma unroll
        for (int j = 0; j < FN; j++) w[j] = *reinterpret_cast<const unsigned *>(C + cw + j * 512);
    };
    auto compute = [&](int buf, const unsigned (&x)[FM], const unsigned (&w)[FN]) __attribute__((always_inline)) {
        const uint8_t *S = smem + wk * GROUP + buf * STAGE;
        uint4 xf[2][FM], wf[2][FN];
        auto read = [&](auto J) __attribute__((always_inline)) {
            constexpr int j = decltype(J)::value, p = j & 1;
            static_for<FM>([&](auto I) __attribute__((always_inline)) { xf[p][I] = *reinterpret_cast<const uint4 *>(S + fx[j] + I * 4096); });
            static_for<FN>([&](auto I) __attribute__((always_inline)) { wf[p][I] = *reinterpret_cast<const uint4 *>(S + fw[j] + I * 4096); });
        };
        read(IC<0>{});
        __builtin_amdgcn_sched_barrier(0);
        static_for<4>([&](auto J) __attribute__((always_inline)) {
            constexpr int j = decltype(J)::value, p = j & 1;
            if constexpr (j < 3) read(IC<j + 1>{});
            static_for<FM * FN>([&](auto I) __attribute__((always_inline)) {
                constexpr int m = decltype(I)::value / FN, n = decltype(I)::value % FN;
                acc[m][n] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(mx_op(wf[p][n]), mx_op(xf[p][m]), acc[m][n], 4, 4,
                                                                           j, (int)w[n], j, (int)x[m]);
            });
            static_for<FM * FN>([&](auto I) __attribute__((always_inline)) {
                constexpr int i = decltype(I)::value, nr = FM + FN, nm = FM * FN;
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                constexpr int d = nr < nm ? (i < nr) : (nr * (i + 1) / nm - nr * i / nm);   /* early in the step */
                if constexpr (j < 3 && d > 0) __builtin_amdgcn_sched_group_barrier(0x100, d, 0);
            });
            /* holds the step's MFMAs here: nothing else keeps them from sinking below the reads of all later steps */
#pragma unroll
            for (int i = 0; i < FM * FN; i++) asm volatile("" : "+v"(acc[i / FN][i % FN]));
            __builtin_amdgcn_sched_barrier(0);
        });
    };
    /* this wave's transfers have landed and its fragment reads have returned; then the group's */
    auto turn = [&]() __attribute__((always_inline)) {
        if constexpr (GW == 1) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    };

    /* Scale loads are behind the wait of turn(): arrived() is a use that tells the compiler so, which else would wait for
     * them, and with them for every later transfer, where they are used */
    unsigned xa[FM], wa[FN];
    if constexpr (SHARED) {
        /* Whole pairs of chunks. Behind the turn() before a pair's first product its scales are in LDS and those of the next
         * pair are requested; they are stored behind a later turn(), into the half that no wave reads any more */
        auto arrived = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < NS; i++)
                asm volatile("" : "+v"(sreg[i].x), "+v"(sreg[i].y), "+v"(sreg[i].z), "+v"(sreg[i].w));
        };
        const int np = a.nb / 16;
        int sbuf = 0;
        if constexpr (NST == 1) {
            if (np) {
                load_scales(0);
                issue(IC<0>{}, 0, 0);
                put_scales(0);
                for (int p = 0;; p++) {
                    turn();
                    shared_scales(xa, wa, 0, p & 1);
                    compute(0, xa, wa);
                    turn();                                      /* the stage is still being read */
                    issue(IC<0>{}, 0, 2 * p + 1);
                    load_scales(2 * min(p + 1, np - 1));
                    turn();
                    arrived();
                    shared_scales(xa, wa, 1, p & 1);
                    compute(0, xa, wa);
                    if (p + 1 == np) break;
                    turn();
                    issue(IC<0>{}, 0, 2 * p + 2);
                    put_scales((p + 1) & 1);
                }
            }
        } else {
            if (np) {
                load_scales(0);
                issue(IC<0>{}, 0, 0);
                put_scales(0);
            }
            for (int p = 0; p < np; p++) {
                turn();
                issue(IC<0>{}, 1, 2 * p + 1);
                const bool more = p + 1 < np;
                load_scales(2 * min(p + 1, np - 1));
                shared_scales(xa, wa, 0, sbuf);
                compute(0, xa, wa);
                turn();
                arrived();
                if (more) {
                    issue(IC<0>{}, 0, 2 * p + 2);
                    put_scales(sbuf ^ 1);
                }
                shared_scales(xa, wa, 1, sbuf);
                compute(1, xa, wa);
                sbuf ^= 1;
            }
        }
        const int left = a.nb - 16 * np;                         /* blocks of up to two chunks */
        if (left) {
#pragma unroll
            for (int i = 0; i < NS; i++) sreg[i] = mx_scale_end(srow[i], 16 * np, a.nb);
            turn();                                              /* the last pair is still being read */
            put_scales(0);
            issue(IC<1>{}, 0, 2 * np);
            if (NST == 2 && left > 8) issue(IC<1>{}, 1, 2 * np + 1);
            turn();
            shared_scales(xa, wa, 0, 0);
            compute(0, xa, wa);
            if (left > 8) {
                if constexpr (NST == 1) {
                    turn();
                    issue(IC<1>{}, 0, 2 * np + 1);
                    turn();
                }
                shared_scales(xa, wa, 1, 0);
                compute(NST - 1, xa, wa);
            }
        }
    } else {
        /* the whole chunks [c0, c1) of this wave, then, by the last wave, a short one */
        auto arrived = [](unsigned (&x)[FM], unsigned (&w)[FN]) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < FM; i++) asm volatile("" : "+v"(x[i]));
#pragma unroll
            for (int j = 0; j < FN; j++) asm volatile("" : "+v"(w[j]));
        };
        const int nc = a.nb / 8, per = (nc + WK - 1) / WK;
        const int c0 = min(wk * per, nc), c1 = min(c0 + per, nc);
        for (int c = c0; c < c1; c++) {
            if (c > c0) turn();                                  /* the stage is still being read */
            issue(IC<0>{}, 0, c);
            scales(xa, wa, c);
            turn();
            arrived(xa, wa);
            compute(0, xa, wa);
        }
        if ((a.nb & 7) && wk == WK - 1) {
            turn();
            issue(IC<1>{}, 0, nc);
#pragma unroll
            for (int i = 0; i < FM; i++) xa[i] = mx_scale_end(xsr[i] - 4 * h, 8 * nc + 4 * h, a.nb).x;
#pragma unroll
            for (int j = 0; j < FN; j++) wa[j] = mx_scale_end(wsr[j] - 4 * h, 8 * nc + 4 * h, a.nb).x;
            turn();
            compute(0, xa, wa);
        }
    }

    /* epilogue, 32 rows of every wave at a time: staged in LDS, the groups' parts added in order, whole row
     * segments stored */
    const int el = fresh(lane), el32 = el & 31, eh = el >> 5;
    float *E = (float *)smem + wid * 32 * ES;
    if constexpr (SHARED)
        if (a.bias) {
            const float *p = (const float *)(smem + BIAS) + wn * 32 * FN + bc;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                bias[e] = e < bv ? p[e] : 0.0f;
                if constexpr (GLU) gbias[e] = e < bv ? p[OW + e] : 0.0f;
            }
        }
    __syncthreads();                                             /* stages still being read */
    static_for<FM>([&](auto I) __attribute__((always_inline)) {
        constexpr int i = decltype(I)::value;
        if constexpr (WK == 1) wave_order();                     /* a wave reads what it has written itself */
        else if constexpr (i > 0) __syncthreads();               /* parts still being read */
        static_for<4 * FN>([&](auto JE) __attribute__((always_inline)) {
            constexpr int j = decltype(JE)::value / 4, e = decltype(JE)::value % 4;
            *reinterpret_cast<float4 *>(E + el32 * ES + 32 * j + 8 * e + 4 * eh) =
                make_float4(acc[i][j][4 * e], acc[i][j][4 * e + 1], acc[i][j][4 * e + 2], acc[i][j][4 * e + 3]);
        });
        if constexpr (WK == 1) wave_order();
        else __syncthreads();
        /* 16 bytes of a row per lane: V columns */
        auto rows = [&](auto VV) __attribute__((always_inline)) {
            constexpr int V = decltype(VV)::value, LPR = OW / V, RPI = 64 / LPR;   /* lanes per row, rows per wave at once */
            const int cv = V * (el % LPR), n = n0 + wn * OW + cv;
#pragma unroll
            for (int q0 = 0; q0 < 32; q0 += WK * RPI) {
                const int q = q0 + wk * RPI + el / LPR, m = m0 + (wm * FM + i) * 32 + q;
                if (WK * RPI > 32 && q >= 32) break;
                float v[V], g[V];
#pragma unroll
                for (int k = 0; k < WK; k++) {
                    const float *p = (const float *)smem + (k * GW + gw) * 32 * ES + q * ES + cv;
#pragma unroll
                    for (int e4 = 0; e4 < V; e4 += 4) {
                        const float4 u = *reinterpret_cast<const float4 *>(p + e4);
                        const float w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                        for (int e = 0; e < 4; e++) v[e4 + e] = k ? v[e4 + e] + w[e] : w[e];
                        if constexpr (GLU) {
                            const float4 t4 = *reinterpret_cast<const float4 *>(p + OW + e4);
                            const float z[4] = {t4.x, t4.y, t4.z, t4.w};
#pragma unroll
                            for (int e = 0; e < 4; e++) g[e4 + e] = k ? g[e4 + e] + z[e] : z[e];
                        }
                    }
                }
#pragma unroll
                for (int e = 0; e < V; e++) {
                    v[e] += bias[e];
                    if constexpr (GLU) v[e] *= mx_silu<V == 4>(g[e] + gbias[e]);   /* V = 4: fp32 out */
                }
                if (m < a.M && n < a.N) mx_store_row<V>(a, m, n, v);
            }
        };
        if (a.ytype == MX_F32) rows(IC<4>{});
        else rows(IC<8>{});
    });
}

/* 32 values of a row, kept as loaded until they are quantised */
template <int T>
struct MxRaw {
    typedef mx_t<T> v_t __attribute__((ext_vector_type(16 / sizeof(mx_t<T>))));
    static constexpr int V = 16 / (int)sizeof(mx_t<T>), NV = 32 / V;
    v_t v[NV];
    /* whole blocks on 16-byte addresses */
    __device__ __forceinline__ void load(const mx_t<T> *p) {
#pragma unroll
        for (int i = 0; i < NV; i++) v[i] = reinterpret_cast<const v_t *>(p)[i];
    }
    /* any address; values past the first n are zero */
    __device__ __forceinline__ void load_some(const mx_t<T> *p, int n) {
#pragma unroll
        for (int i = 0; i < NV; i++) {
            if (V * (i + 1) <= n) {
                __builtin_memcpy(&v[i], p + V * i, 16);
            } else {
#pragma unroll
                for (int e = 0; e < V; e++) v[i][e] = V * i + e < n ? p[V * i + e] : (mx_t<T>)0.0f;
            }
        }
    }
    __device__ __forceinline__ uint4 pack(unsigned &byte) const {
        unsigned m = 0, w[4];
#pragma unroll
        for (int i = 0; i < 32; i++) m = max(m, mx_abs_bits((float)v[i / V][i % V]));
        byte = mx_scale_byte(m);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; e++) f[e] = (float)v[(8 * i + e) / V][(8 * i + e) % V];
            w[i] = mx_pack8(f, byte);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};

/*
 * Few rows: quantised by the wave that multiplies them, in the same launch. A workgroup owns 16 rows and 16 weight rows (GLU: 16
 * value and 16 gate rows), its NW waves take K in turn, and the 16 x 16 sums meet in LDS. v_mfma_scale_f32_16x16x128:
 * lane l holds block l / 16 of four, of row l % 16, so a lane reads 32 activations, finds their maximum and packs
 * its own operand: no lane exchange. Every workgroup quantises its rows again, which is little beside the latency
 * of a second launch. What bounds it is latency: WHOLE (whole blocks, 16-byte rows) loads two steps ahead of their use.
 */
template <int XT, bool GLU, int NW, bool WHOLE>
__global__ __launch_bounds__(64 * NW) void k_mx4_rows(MxArgs a, const void *x, long ldx, int K) {
    constexpr int F = GLU ? 2 : 1, U = 2;
    __shared__ __attribute__((aligned(16))) float E[NW][F][16][20];
    const int lane = threadIdx.x & 63, l16 = lane & 15, kg = lane >> 4;
    const int wid = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int n0 = blockIdx.x * 16, n = min(n0 + l16, a.N - 1), steps = (a.nb + 3) / 4, m0 = blockIdx.y * 16;
    mx_f32x4_t acc[F];
#pragma unroll
    for (int f = 0; f < F; f++) acc[f] = mx_f32x4_t{0, 0, 0, 0};
    const mx_t<XT> *xr = (const mx_t<XT> *)x + (size_t)min(m0 + l16, a.M - 1) * ldx;   /* rows past M: not stored */
    for (int s0 = wid; s0 < steps; s0 += U * NW) {
        MxRaw<XT> raw[U];
        uint4 w[U][F];
        int sc[U][F];
        /* an absent block loads the row's last; its codes are taken as zero, its scales as one */
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int b = 4 * (s0 + u * NW) + kg, bc = min(b, a.nb - 1);
#pragma unroll
            for (int f = 0; f < F; f++) {
                const size_t at = (size_t)(n + f * a.N) * a.nb + bc;
                w[u][f] = ((const uint4 *)a.wq)[at];
                sc[u][f] = b < a.nb ? a.ws[at] : 127;
            }
            if constexpr (WHOLE) raw[u].load(xr + 32 * bc);
            else raw[u].load_some(xr + 32 * bc, K - 32 * bc);
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const bool in = 4 * (s0 + u * NW) + kg < a.nb;
            unsigned byte;
            uint4 q = raw[u].pack(byte);
            if (!in) { q = make_uint4(0, 0, 0, 0); byte = 127; }
#pragma unroll
            for (int f = 0; f < F; f++)
                acc[f] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx_op(w[u][f]), mx_op(q), acc[f], 4, 4, 0, sc[u][f], 0, (int)byte);
        }
    }
#pragma unroll
    for (int f = 0; f < F; f++)
        *reinterpret_cast<mx_f32x4_t *>(&E[wid][f][l16][4 * kg]) = acc[f];
    __syncthreads();
    for (int i = threadIdx.x; i < 256; i += 64 * NW) {
        const int m = i >> 4, c = i & 15;
        if (m0 + m >= a.M || n0 + c >= a.N) continue;
        float v = 0.0f, g = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; w++) {
            v += E[w][0][m][c];
            if constexpr (GLU) g += E[w][F - 1][m][c];
        }
        if (a.bias) v += a.bias[n0 + c];
        if constexpr (GLU) {
            if (a.bias) g += a.bias[a.N + n0 + c];
            v *= a.ytype == MX_F32 ? mx_silu<true>(g) : mx_silu<false>(g);
        }
        mx_store(a.y, a.ytype, (size_t)(m0 + m) * a.N + n0 + c, v);
    }
}

template <int FM, int FN, int WM, int WN, int WK, int NST, bool GLU>
static hipError_t launch(MxArgs a, hipStream_t s) {
    constexpr int OW = (GLU ? 16 : 32) * FN * WN;
    a.tm = (a.M + 32 * FM * WM - 1) / (32 * FM * WM);
    a.tn = (a.N + OW - 1) / OW;
    a.T = a.tm * a.tn;
    hipLaunchKernelGGL((k_mx4_gemm<FM, FN, WM, WN, WK, NST, GLU>), dim3((unsigned)((a.T + 7) / 8 * 8)), dim3(64 * WM * WN * WK), 0, s, a);
    return hipGetLastError();
}

/* Which tile: the least estimated time, in us, over one launch. A configuration takes at least the latency of one tile, and where
 * there are many tiles the time that all CUs need for them; both grow with the chunks of K, the large tiles' also
 * with the bytes of output. Fitted to M = 17 .. 8192, N = 1024 .. 8192, K = 256 .. 8192. Over 720 shapes there (both outputs' sizes,
 * gated and not) the estimate of the form that is taken is 7 % off in the median, 21 % or less in nine of ten, 36 % at most, and the
 * form within 5 % of the best one in 641, 10 % in 694, 26 % at most (1.5 % in the mean). A form far from being taken can be
 * misjudged by much more (t64 by 50 %, t256 by 160 %).
 *  t32, t64: 32 x 32 (GLU: 32 x 64) and 64 x 64, K split over four one-wave groups, several workgroups to a CU;
 *  t128a, t128b: 128 x 128 in one stage, three workgroups to a CU, and in two stages, two to a CU, for long K and few tiles;
 *  t256: 256 x 256 in rounds of one to a CU.
 * Measured, in that order, us: M 344, K 1024, N 4096 6.5, 6.2, 7.3, 7.1, 13.2; M 172, K 4096, N 1024 4.9, 7.5, 15.7, 14.7, 29.8;
 * M 2592, K 1024, N 4096 26.3, 23.4, 12.1, 14.5, 14.1; M 2592, K 4096, N 1024 23.7, 17.3, 20.0, 16.4, 31.7; M 8192, K 4096, N 8192
 * 503, 288, 170, 182, 153. */
template <bool GLU>
static hipError_t pick(const MxArgs &a, hipStream_t s) {
    constexpr int H = GLU ? 2 : 1;                               /* weight rows per column */
    const double nc = (a.nb + 7) / 8, es = a.ytype == MX_F32 ? 4 : 2;
    auto tiles = [&](int bm, int cols) { return (double)((a.M + bm - 1) / bm) * (double)((a.N + cols - 1) / cols); };
    auto most = [](double x, double y) { return x > y ? x : y; };
    const double kb = 128 * (128 / H) * es / 1024;               /* output of a 128 x 128 tile */
    const double n128 = tiles(128, 128 / H), rounds = (double)((long)(tiles(256, 256 / H) + 255) / 256);
    const double t32 = GLU ? most(4.4 + 0.2 * nc, 3 + tiles(32, 32) * (0.0006 + 0.00083 * nc))
                           : most(4.4 + 0.04 * nc, 3 + tiles(32, 32) * (0.001 + 0.00043 * nc));
    const double t64 = most(4.0 + 0.25 * nc, 2.7 + tiles(64, 64 / H) * (0.004 + 0.00138 * nc));
    auto half = [&](double at_once) {                            /* past one round, the last one counts half of what it is short of */
        return n128 <= at_once ? n128 : (n128 + at_once * (double)(long)((n128 + at_once - 1) / at_once)) / 2;
    };
    const double t128a = most(3.7 + 1.05 * nc, 3 + half(768) * (0.002 + 0.000075 * kb + 0.0023 * nc));
    const double t128b = most(4.4 + 0.66 * nc, 3 + half(512) * (0.0024 + 0.000075 * kb + 0.0025 * nc));
    const double t256 = 3 + rounds * ((nc < 2 ? 2.4 : -0.6) + 0.16 * kb + 2.02 * nc);
    /* A launch holds less than 2^32 threads: tiles of 256 threads are counted; of 256 x 256 there are never too many
     * (M up to 2^28, M N up to 2^36) */
    const double most_tiles = (double)((1l << 24) - 8);
    const double us[5] = {t32, t64, t128a, t128b, t256}, count[5] = {tiles(32, 32), tiles(64, 64 / H), n128, n128, 0};
    int which = 4;
    for (int i = 3; i >= 0; i--)
        if (us[i] <= us[which] && count[i] <= most_tiles) which = i;
    switch (which) {
    case 0: return launch<1, H, 1, 1, 4, 1, GLU>(a, s);
    case 1: return launch<2, 2, 1, 1, 4, 1, GLU>(a, s);
    case 2: return launch<2, 2, 2, 2, 1, 1, GLU>(a, s);
    case 3: return launch<2, 2, 2, 2, 1, 2, GLU>(a, s);
    default: return launch<4, 2, 2, 4, 1, 2, GLU>(a, s);
    }
}

extern "C" hipError_t aria_k_mx4_gemm(void *y, int ytype, const uint8_t *xq, const uint8_t *xs, const uint8_t *wq,
                                      const uint8_t *ws, const float *bias, int M, int K, int N, int glu, hipStream_t s) {
    if (M <= 0 || N <= 0) return hipSuccess;
    MxArgs a = {y, xq, xs, wq, ws, bias, M, N, (K + 31) / 32, ytype, 0, 0, 0, 0};
    a.vec = N % (ytype == MX_F32 ? 4 : 8) == 0 && ((uintptr_t)y & 15u) == 0;
    return glu ? pick<true>(a, s) : pick<false>(a, s);
}

template <int XT, bool GLU>
static void launch_rows(const MxArgs &a, const void *x, long ldx, int K, hipStream_t s) {
    const bool whole = K % 32 == 0 && ldx * sizeof(mx_t<XT>) % 16 == 0 && ((uintptr_t)x & 15u) == 0;
    const dim3 grid((unsigned)((a.N + 15) / 16), (unsigned)((a.M + 15) / 16));
    if (a.nb > 32) {   /* K past 1024 keeps eight waves busy for two steps */
        if (whole) hipLaunchKernelGGL((k_mx4_rows<XT, GLU, 8, true>), grid, dim3(512), 0, s, a, x, ldx, K);
        else hipLaunchKernelGGL((k_mx4_rows<XT, GLU, 8, false>), grid, dim3(512), 0, s, a, x, ldx, K);
    } else {
        if (whole) hipLaunchKernelGGL((k_mx4_rows<XT, GLU, 4, true>), grid, dim3(256), 0, s, a, x, ldx, K);
        else hipLaunchKernelGGL((k_mx4_rows<XT, GLU, 4, false>), grid, dim3(256), 0, s, a, x, ldx, K);
    }
}

/* Whether one launch of k_mx4_rows beats quantisation and product: x's bytes per workgroup bound its latency (16 fp32 rows of 4096:
 * 11.4 us against 7.5 in two launches; fp16 7.7; one row 6.0; 16 fp16 rows of 1024: 4.2), and beyond 16 rows every
 * 16 columns quantise them again (N 4096, K 1024: 32 rows 5.0 against 7.5, 64 rows 7.7). */
extern "C" int aria_k_mx4_rows_fit(int xtype, int M, int K, int N) {
    const long bytes = (long)(M < 16 ? M : 16) * K * (xtype == MX_F32 ? 4 : 2);
    return bytes <= 96 * 1024 && (M <= 16 || (K <= 1024 && ((M + 15L) / 16) * ((N + 15L) / 16) <= 640));
}

extern "C" hipError_t aria_k_mx4_rows(void *y, int ytype, const void *x, int xtype, long ldx, const uint8_t *wq,
                                      const uint8_t *ws, const float *bias, int M, int K, int N, int glu, hipStream_t s) {
    if (M <= 0 || N <= 0) return hipSuccess;
    const MxArgs a = {y, nullptr, nullptr, wq, ws, bias, M, N, (K + 31) / 32, ytype, 0, 0, 0, 0};
    if (glu) {
        if (xtype == MX_F32) launch_rows<MX_F32, true>(a, x, ldx, K, s);
        else if (xtype == MX_F16) launch_rows<MX_F16, true>(a, x, ldx, K, s);
        else launch_rows<MX_BF16, true>(a, x, ldx, K, s);
    } else {
        if (xtype == MX_F32) launch_rows<MX_F32, false>(a, x, ldx, K, s);
        else if (xtype == MX_F16) launch_rows<MX_F16, false>(a, x, ldx, K, s);
        else launch_rows<MX_BF16, false>(a, x, ldx, K, s);
    }
    return hipGetLastError();
}
