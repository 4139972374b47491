/*
 * aria_hip.h - device-pointer, stream-ordered entry points of the MI355X backend
 * (libaria_hip.so), beside the reference-compatible ABI in aria_gpu.h.
 *
 * These are the hot-path operations the reference's device DiT composes inside
 * src/aria_cuda.cu (fused norm+modulate, gate+residual, GLU, softmax, RoPE, Q8/Q4
 * dequant-on-use GEMM, pingpong), exposed one by one so that a caller holding
 * device buffers can chain them on one stream with no host round trip, and the
 * host-pointer forms of the quantizer/GEMM interfaces of src/aria_quant.h.
 *
 * Conventions:
 *   - Pointers named d* or taking "device" in the comment are device memory;
 *     all others are host memory.
 *   - stream: a hipStream_t passed as void*; NULL means the library's own stream
 *     (aria_hip_default_stream()). Device-pointer calls only enqueue work.
 *   - Return value: 0 on success, a negative ARIA_HIP_E* code on a rejected
 *     argument, or the positive hipError_t of a failed HIP call.
 *     aria_hip_last_error() describes the last failure.
 *   - Shapes are row-major fp32 unless stated; weights are PyTorch Linear
 *     [N = out, K = in] (src/aria_ops.h:10).
 *   - rows_per_batch: per-batch broadcast vectors (adaLN scale/shift/gate) are
 *     [rows / rows_per_batch, dim]; row r uses vector r / rows_per_batch.
 */
#ifndef ARIA_HIP_H
#define ARIA_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define ARIA_HIP_EINVAL  (-1)   /* bad shape, NULL where a buffer is required */
#define ARIA_HIP_ENODEV  (-2)   /* no usable HIP device */
#define ARIA_HIP_ENOMEM  (-3)   /* device allocation failed */

/* ---- runtime ---- */
/* Select device 0 and create the library stream; idempotent, thread-safe.
 * Returns 0, or ARIA_HIP_ENODEV. Every other call initialises on demand. */
int aria_hip_init(void);
const char *aria_hip_last_error(void);
void *aria_hip_default_stream(void);
int aria_hip_stream_sync(void *stream);
/* A further stream (non-blocking, default priority) for callers that run work side by side, or
 * NULL; aria_hip_stream_destroy ignores NULL and the library's own stream. */
void *aria_hip_stream_create(void);
void aria_hip_stream_destroy(void *stream);
/* HIP events for stream-ordered timing (bench harness). */
void *aria_hip_event_create(void);
void aria_hip_event_destroy(void *ev);
int aria_hip_event_record(void *ev, void *stream);
/* milliseconds between two recorded events (synchronises on the second), or -1 */
float aria_hip_event_elapsed_ms(void *ev0, void *ev1);
int aria_hip_memcpy_h2d_async(void *ddst, const void *hsrc, size_t bytes, void *stream);
int aria_hip_memcpy_d2h_async(void *hdst, const void *dsrc, size_t bytes, void *stream);
int aria_hip_memcpy_d2d_async(void *ddst, const void *dsrc, size_t bytes, void *stream);
/* device properties: number of CUs, and the gfx target name ("gfx950") */
int aria_hip_cu_count(void);
int aria_hip_arch(char *buf, size_t buflen);

/* ---- row normalisations (device pointers) ----
 * Replace aria_rmsnorm / aria_gemma_rmsnorm (src/aria_ops.h:91-108,
 * src/aria_cpu.c:643-733). LayerNorm has no reference op: biased variance,
 * y = (x - mean)/sqrt(var + eps) * gamma + beta, gamma/beta may be NULL. */
int aria_hip_rmsnorm_dev(float *dy, const float *dx, const float *dw, int rows, int dim,
                         float eps, void *stream);
int aria_hip_gemma_rmsnorm_dev(float *dy, const float *dx, const float *dw, int rows, int dim,
                               float eps, void *stream);
int aria_hip_layernorm_dev(float *dy, const float *dx, const float *dgamma, const float *dbeta,
                           int rows, int dim, float eps, void *stream);
/* Fused RMSNorm(w) -> adaLN modulate, one pass: y = (x*inv*w)*(1+scale)+shift.
 * The reference runs aria_rmsnorm then adaln_modulate (src/aria_sa3_dit.c:175-176,
 * 255-256); its device twin is k_rmsnorm_adaln(_h) (src/aria_cuda.cu:199-249).
 * out_f16 != 0 writes IEEE half (the GEMM operand) into dy. */
int aria_hip_rmsnorm_adaln_dev(void *dy, int out_f16, const float *dx, const float *dw,
                               const float *dscale, const float *dshift, int rows, int dim,
                               int rows_per_batch, float eps, void *stream);
/* Config 1/2 chain fused into one pass:
 * out = gelu_tanh(LayerNorm(x)*gamma+beta)*(1+scale)+shift) + x. */
int aria_hip_ln_mod_gelu_res_dev(float *dout, const float *dx, const float *dgamma,
                                 const float *dbeta, const float *dscale, const float *dshift,
                                 int rows, int dim, int rows_per_batch, float eps, void *stream);

/* ---- elementwise / broadcast (device pointers; n counts floats) ----
 * aria_add/addto/scale/axpy, aria_silu, aria_gelu_tanh, aria_silu_gate
 * (src/aria_ops.h:111-117,166-170); y may alias x. */
int aria_hip_add_dev(float *dy, const float *da, const float *db, size_t n, void *stream);
int aria_hip_axpy_dev(float *dy, const float *dx, float a, size_t n, void *stream);
int aria_hip_scale_dev(float *dy, const float *dx, float a, size_t n, void *stream);
int aria_hip_gelu_tanh_dev(float *dy, const float *dx, size_t n, void *stream);
int aria_hip_silu_dev(float *dy, const float *dx, size_t n, void *stream);
int aria_hip_silu_gate_dev(float *dout, const float *dgate, const float *dup, size_t n,
                           void *stream);
/* adaln_modulate (src/aria_sa3_dit.c:71-82): y = x*(1+scale)+shift. */
int aria_hip_modulate_dev(float *dy, const float *dx, const float *dscale, const float *dshift,
                          int rows, int dim, int rows_per_batch, void *stream);
/* gate_sigmoid + residual (src/aria_sa3_dit.c:85-97, 211-215) as one pass:
 * out = res + (o [+ bias]) * sigmoid(1 - gate); out may alias res. */
int aria_hip_gate_residual_dev(float *dout, const float *dres, const float *do_,
                               const float *dgate, const float *dbias, int rows, int dim,
                               int rows_per_batch, void *stream);
/* GLU combine (src/aria_sa3_dit.c:108-121): proj [rows, 2*inner] = [value | gate],
 * out[r,i] = silu(gate (+b)) * (value (+b)); out_f16 writes half. */
int aria_hip_glu_combine_dev(void *dout, int out_f16, const float *dproj, const float *dbias,
                             int rows, int inner, void *stream);
/* pingpong (src/aria_sampler.c:216-220): x = (1-tn)*(x - tc*v) + tn*noise,
 * each operation rounded on its own: bit-identical to the host loop. */
int aria_hip_pingpong_dev(float *dx, const float *dv, const float *dnoise, float tc, float tn,
                          size_t n, void *stream);

/* ---- softmax / rotary (device pointers) ---- */
/* aria_softmax_inplace (src/aria_ops.h:164), mask [rows, cols] or NULL. */
int aria_hip_softmax_dev(float *dx, int rows, int cols, const float *dmask, void *stream);
/* aria_rope_apply (src/aria_ops.h:126): x [H, N, D] in place, tables [N, rot/2]. */
int aria_hip_rope_apply_dev(float *dx, const float *dcos, const float *dsin, int H, int N, int D,
                            int rot_dim, void *stream);
/* The same rotation on q and k (same shape, distinct buffers) in one launch, as the
 * DiT applies it (src/aria_sa3_dit.c:193-194). */
int aria_hip_rope_apply2_dev(float *dq, float *dk, const float *dcos, const float *dsin, int H, int N,
                             int D, int rot_dim, void *stream);

/* ---- quantisation (src/aria_quant.h layouts) ---- */
/* Device pack: bit-exact with aria_q8_quant / aria_q4_quant (src/aria_quant.c:78, 353). */
int aria_hip_q8_quant_dev(int8_t *dq, float *dscale, const float *dW, int N, int K, void *stream);
int aria_hip_q4_quant_dev(uint8_t *dq, float *dscale, const float *dW, int N, int K, void *stream);
/* Device unpack to fp32 (the per-weight value the dequant GEMM uses). */
int aria_hip_q8_dequant_dev(float *dW, const int8_t *dq, const float *dscale, int N, int K,
                            void *stream);
int aria_hip_q4_dequant_dev(float *dW, const uint8_t *dq, const float *dscale, int N, int K,
                            void *stream);

/* Dequant-on-use GEMM on MFMA, y[M,N] = x[M,K] W[N,K]^T (+ b[N]); b may be NULL.
 * Replaces aria_linear_q8 / aria_linear_q4 (src/aria_quant.h:45, 65;
 * src/aria_quant.c:98-145, 469-538) and the reference's dequantize-to-fp16 +
 * cublasGemmEx device path (src/aria_cuda.cu:1009-1035). Weights stay packed in HBM.
 * wtype 0 = Q8 (dq int8 [N,K], dscale [N]), 1 = Q4 (dq u8 [N,ceil(K/2)], dscale
 * [N, 2*ceil(K/32)] [min,step] pairs), 2 = fp16 weights (dq = half [N,K], dscale unused).
 * x_f16 / y_f16 select IEEE-half activations / outputs instead of fp32. */
int aria_hip_qlinear_dev(void *dy, int y_f16, const void *dx, int x_f16, int wtype, const void *dq,
                         const float *dscale, const float *db, int M, int K, int N, void *stream);
/* As aria_hip_qlinear_dev with an explicit workgroup tile (M x N): 1 = 192x128,
 * 2 = 128x128, 3 = 96x256, 4 = 96x128, 5 = 128x256, 6 = 64x128, 7 = 128x64, 8 = 64x64
 * (both operands staged through LDS); 9..12 = 32x256, 64x256, 96x256, 128x256 with the
 * weights loaded straight into registers (Q8/Q4 with K % 64 == 0, else the 128x128 LDS
 * kernel); 0 = chosen from the shape (tuning knob; fp32 activations without an fp16
 * staging buffer run 128x128, or with tiles 0 and few outputs the K-split kernel). */
int aria_hip_qlinear_ex_dev(void *dy, int y_f16, const void *dx, int x_f16, int wtype, const void *dq,
                            const float *dscale, const float *db, int M, int K, int N, int tiles,
                            void *stream);
int aria_hip_linear_q8_dev(float *dy, const float *dx, const int8_t *dq, const float *dscale,
                           const float *db, int M, int K, int N, void *stream);
/* aria_hip_qlinear_dev that allocates nothing. No counterpart in the reference: it is for
 * callers that cannot allocate device memory (code under HIP graph capture, tight serving
 * loops, harnesses that forbid hipMalloc). Same arguments and results, bit for bit; the
 * fp16 staging of fp32 activations goes to a static device array of
 * ARIA_HIP_NOALLOC_SCRATCH bytes per GPU instead of per-call pool memory, so M * K * 2 must
 * not exceed it (ARIA_HIP_EINVAL otherwise; fp16 activations need no staging). Every call
 * on one GPU shares that array. A staging call on another stream than the GPU's previous one
 * first waits (hipStreamWaitEvent) for that call's GEMM, so calls from several streams or
 * threads run one after another on the device. Under stream capture the call records no
 * event and waits for none: inside a graph the caller orders the calls. */
#define ARIA_HIP_NOALLOC_SCRATCH ((size_t)32 << 20)
int aria_hip_qlinear_noalloc_dev(void *dy, int y_f16, const void *dx, int x_f16, int wtype, const void *dq,
                                 const float *dscale, const float *db, int M, int K, int N, void *stream);
int aria_hip_linear_q4_dev(float *dy, const float *dx, const uint8_t *dq, const float *dscale,
                           const float *db, int M, int K, int N, void *stream);

/* ---- W8A8: int8 activations x int8 weights on the int8 MFMA ----
 * Replaces the reference's gemm_w8a8 / gemm_w8a8_h (src/aria_cuda.cu:934-1004: per-token
 * activation quantisation k_quant_act_q8(_h), int8 IMMA GEMM into int32, dequant k_deq_i32)
 * with the numbers of aria_linear_q8a8 (src/aria_quant.h:47-51, src/aria_quant.c:253-345),
 * bit for bit. */
/* RMSNorm(w) (-> adaLN modulate with per-batch dscale / dshift [rows / rows_per_batch, dim],
 * or both NULL) with W8A8 output, one pass: the fp32 result row (the aria_hip_rmsnorm_adaln_dev
 * value) is quantised in registers as aria_hip_quant_act_q8_dev does, dyq int8 [rows, dim] and
 * dsx [rows]. The reference's W8A8 block runs k_rmsnorm(_adaln) into fp32 then
 * k_quant_act_q8 (src/aria_cuda.cu:1075, 1094, 1133 with 934-949). dim 256, 512, 768, 1024 or
 * 2048. */
int aria_hip_rmsnorm_adaln_q8_dev(int8_t *dyq, float *dsx, const float *dx, const float *dw, const float *dscale,
                                  const float *dshift, int rows, int dim, int rows_per_batch, float eps,
                                  void *stream);
/* Per-row symmetric int8 activations: sx[m] = amax / 127 (amax = max |x[m,:]|),
 * dxq[m,k] = clamp(rint(x * 127 / amax), -127, 127), all zero when amax == 0. dx is
 * fp32 or fp16 (x_f16) [M, K]; dxq [M, K] int8, dsx [M]. */
int aria_hip_quant_act_q8_dev(int8_t *dxq, float *dsx, const void *dx, int x_f16, int M, int K,
                              void *stream);
/* dy[m,n] = (float)(sum_k dxq[m,k] dq[n,k]) * dsx[m] * dscale[n] (+ db[n], else + 0.0f),
 * exact int32 sums, fp32 (or fp16 with y_f16) output. dq / dscale are the Q8 weight
 * (aria_q8_quant layout). */
int aria_hip_gemm_i8_dev(void *dy, int y_f16, const int8_t *dxq, const float *dsx, const int8_t *dq,
                         const float *dscale, const float *db, int M, int K, int N, void *stream);
/* Both steps, as aria_linear_q8a8 on device data: dws is caller workspace of at least
 * aria_hip_q8a8_ws_bytes(M, K) bytes (the int8 rows and their scales). */
size_t aria_hip_q8a8_ws_bytes(int M, int K);
int aria_hip_linear_q8a8_dev(float *dy, const void *dx, int x_f16, const int8_t *dq, const float *dscale,
                             const float *db, int M, int K, int N, void *dws, void *stream);
/* Host-pointer form with the reference's signature (src/aria_quant.h:50). */
int aria_hip_linear_q8a8(float *y, const float *x, const int8_t *q, const float *scale, const float *b,
                         int M, int K, int N);

/* ---- attention (the DiT's, head dim 64) ----
 * Head preparation, replacing extract_heads + q/k RMSNorm + RoPE of the block
 * (src/aria_sa3_dit.c:183-194, 222-226): dsrc [B*S, ld] fp32 holds nsec sections of
 * H*64 columns (e.g. the qkv projection); section i is written to ddst[i] (a host
 * array of device pointers) as fp16 [B, H, S, 64]. kind[i]: 0 = q, 1 = k (RMSNorm
 * with dw[i] (may be NULL), eps, then RoPE over rot dims with tables [S, rot/2];
 * rot 0 = none), 2 = v (copy). kind and ddst/dw are host arrays of nsec entries. */
int aria_hip_qkv_prep_dev(const float *dsrc, int ld, int B, int S, int H, int nsec, const int *kind,
                          uint16_t *const *ddst, const float *const *dw, const float *dcos,
                          const float *dsin, int rot, float eps, void *stream);
/* Fused attention, replacing aria_attention (src/aria_ops.h:135, src/aria_cpu.c:811-849)
 * for the DiT: q [B*H, Nq, D], k/v [B*H, Nk, D] fp16 -> dout [B, Nq, H*D] with heads
 * merged (the layout the output projection reads), fp16 when out_f16 else fp32.
 * softmax(q k^T / sqrt(D)) v with scores kept on chip. D must be 64. */
int aria_hip_flash_attention_dev(const uint16_t *dq, const uint16_t *dk, const uint16_t *dv, void *dout,
                                 int out_f16, int B, int H, int Nq, int Nk, int D, void *stream);
/* Host form of the fused attention (parity entry): q/k/v fp32 [B*H, N, D] are rounded
 * to fp16 on the device; out fp32 [B, Nq, H*D]. */
int aria_hip_attention_f16(float *out, const float *q, const float *k, const float *v, int B, int H,
                           int Nq, int Nk, int D);

/* ---- cross attention to an encoder's states of another length ----
 * o[b,t,h,:] = sum_j p_j v[b,j,h / (H/Hkv),:], p = softmax over the valid keys j of
 * scale * q[b,t,h,:] . k[b,j,h / (H/Hkv),:]. Key j of sequence b is valid when j < kv_len[b] (kv_len
 * NULL: Nk; values are taken as clamped to 0..Nk) and mask[b * mask_stride + j] != 0 (mask NULL:
 * all). A row with no valid key (Nk = 0 included), or of a finite query whose valid keys all score
 * -Inf, is written as zeros. Keys and values that are not valid may hold anything (Inf and NaN
 * included): they do not reach the result, but all Nk rows must be readable memory. type: 1 = fp16,
 * 2 = bf16 (aria_dtype's values) for q, k, v and out; out_f32 != 0 writes fp32. D: a multiple of 8
 * up to 128. H a multiple of Hkv. B * H at most 2^20, B * H * Nq and Nk at most 2^30. scale:
 * positive, at most 2^127.
 * Strides count elements and are multiples of 8, not negative, pointers are 16-byte aligned (for
 * an fp32 out too); batch / head / token strides of q, k and v may be 0 (broadcast); rows of out lie
 * apart from each other and from every input.
 * Probabilities are rounded to the type before they multiply v, whatever out's type; in fp16 one
 * below 2^-32 of its row's largest may count as zero (an infinite value under one gives NaN). Sums
 * and softmax statistics are fp32.
 * dws: aria_hip_cross_attention_ws_bytes(a) bytes (0: may be NULL), 256-byte aligned, not shared
 * by calls that may run at the same time; the number goes by B, H, Hkv, Nq, Nk and D alone, so a
 * program can ask for it before the rest of the description stands (0 for sizes that are refused).
 * No counterpart in the reference, whose attention takes one length (src/aria_ops.h:135). */
typedef struct {
    const void *q, *k, *v;
    void *out;
    const int32_t *kv_len;   /* [B] or NULL */
    const uint8_t *mask;     /* rows of Nk bytes, mask_stride apart, or NULL */
    int type, out_f32;
    int B, H, Hkv, Nq, Nk, D;
    float scale;
    int64_t q_batch, q_head, q_token, k_batch, k_head, k_token, v_batch, v_head, v_token;
    int64_t o_batch, o_head, o_token, mask_stride;
} aria_hip_cross_attn;
size_t aria_hip_cross_attention_ws_bytes(const aria_hip_cross_attn *a);
int aria_hip_cross_attention_dev(const aria_hip_cross_attn *a, void *dws, void *stream);
/* Host form: q fp32 [B*H, Nq, D] and k/v [B*Hkv, Nk, D] are rounded to fp16 on the device, scale is
 * 1/sqrt(D); kv_len [B] and mask [B, Nk] may be NULL; out fp32 [B, Nq, H*D]. */
int aria_hip_cross_attention_f16(float *out, const float *q, const float *k, const float *v, const int32_t *kv_len,
                                 const uint8_t *mask, int B, int H, int Hkv, int Nq, int Nk, int D);

/* ---- MXFP4: microscaled 4-bit floating point (no counterpart in the reference) ----
 * Blocks of 32 values along K share a power of two 2^(byte - 127); a value is a 4-bit code: sign
 * and magnitude 0, 0.5, 1, 1.5, 2, 3, 4 or 6 (e2m1). A packed row is ceil(K/32) blocks of 16
 * bytes (the even element in the low nibble, codes past K zero) in dq [rows, 16 * ceil(K/32)]
 * and one byte per block in dscale [rows, ceil(K/32)]; dq is 16-byte aligned.
 * Quantisation: byte = floor(log2 max|x|) - 2 + 127 (at least 0; 0 for a block of zeros), codes
 * x / 2^(byte - 127) to nearest, ties to the even code, saturating at 6, the sign of zero kept. A
 * block that holds an Inf or a NaN gets byte 255 and codes 0: it stands for NaN.
 * Element types of activations and outputs are aria_dtype's values: 0 fp32, 1 fp16, 2 bf16;
 * ldx: elements between rows of x (at least K). K at most 2^24, rows at most 2^30; of the
 * products M at most 2^28, N (inner) at most 2^26 and M * N at most 2^36. Outputs and workspaces
 * overlap no input. */
int aria_hip_mx4_quant_dev(uint8_t *dq, uint8_t *dscale, const void *dx, int xtype, int rows, int K, int64_t ldx,
                           void *stream);
/* y [rows, K] from packed rows, rounded to ytype. fp32 holds every value of a pack made here; in one
 * from elsewhere byte 253 with codes 4 and 6 and byte 254 with 2 and above lie past it: Inf. */
int aria_hip_mx4_dequant_dev(void *dy, int ytype, const uint8_t *dq, const uint8_t *dscale, int rows, int K,
                             void *stream);
/* dy[m,n] = sum_k x[m,k] w[n,k] (+ db[n]; db NULL = none) on packed activations [M, K] and weights
 * [N, K]: block-scaled MFMA, fp32 sums, rounded once to ytype. */
int aria_hip_gemm_mx4_dev(void *dy, int ytype, const uint8_t *dxq, const uint8_t *dxs, const uint8_t *dq,
                          const uint8_t *dscale, const float *db, int M, int K, int N, void *stream);
/* The same with the activations quantised in the call. dws: caller workspace of
 * aria_hip_mx4_ws_bytes(M, K) bytes, 256-byte aligned, not shared by calls that may run at the
 * same time. */
size_t aria_hip_mx4_ws_bytes(int M, int K);
int aria_hip_linear_mx4_dev(void *dy, int ytype, const void *dx, int xtype, int64_t ldx, const uint8_t *dq,
                            const uint8_t *dscale, const float *db, int M, int K, int N, void *dws, void *stream);
/* Gated feed-forward up-projection, one pass: dq / dscale / db hold 2 * inner rows [value | gate]
 * (the order of aria_hip_glu_combine_dev), dy[m,i] = v * silu(g) with v = x . w[i] + db[i] and
 * g = x . w[inner + i] + db[inner + i] in fp32; neither projection is stored. */
int aria_hip_glu_mx4_dev(void *dy, int ytype, const void *dx, int xtype, int64_t ldx, const uint8_t *dq,
                         const uint8_t *dscale, const float *db, int M, int K, int inner, void *dws, void *stream);
/* Host forms (fp32): q [rows, 16 * ceil(K/32)], scale [rows, ceil(K/32)]. */
int aria_hip_mx4_quant(uint8_t *q, uint8_t *scale, const float *x, int rows, int K);
int aria_hip_mx4_dequant(float *y, const uint8_t *q, const uint8_t *scale, int rows, int K);
int aria_hip_linear_mx4(float *y, const float *x, const uint8_t *q, const uint8_t *scale, const float *b, int M,
                        int K, int N);
int aria_hip_glu_mx4(float *y, const float *x, const uint8_t *q, const uint8_t *scale, const float *b, int M, int K,
                     int inner);

/* ---- rotary positions by table, a cache of keys and values in 8 bits, attention over shared prefixes
 *      (no counterpart in the reference, whose rotary embedding takes positions 0 .. N-1 in fp32,
 *      src/aria_ops.h:122-126, and whose attention takes one set of keys, src/aria_ops.h:135) ----
 * Element types are aria_dtype's values: 0 fp32, 1 fp16, 2 bf16. Strides count elements (bytes in a
 * cache), are not negative, and those of inputs may be 0 (broadcast); rows of outputs lie apart from
 * each other and, unless stated, from every input. Pointers and strides of states need only their
 * element's alignment. Heads at most 2^16 each, B * N at most 2^30, D at most 256. */

/* Frequencies of the rotated pairs i = 0 .. rot/2 - 1, f_i = base^(-2i/rot), for contexts longer than
 * the trained one. kind 0: f_i; 1 (linear): f_i / factor; 2 (base): base * factor^(rot/(rot-2)) in
 * base's place, which leaves f_0 and divides the last by factor; 3 (by turns): with t = trained * f_i / 2 pi
 * turns over the trained length and w = (t - low) / (high - low) held to 0 .. 1, f_i (w + (1 - w) / factor).
 * gain multiplies both tables. rot even, 2 .. 256 (kind 2: from 4); base > 1; factor > 0 (kinds 1 - 3);
 * trained > 0, high > low (kind 3); all finite, gain in fp32 too. No pair may make more than 16 turns from one position to the
 * next (kinds 1 and 3: factor from 0.01 on). */
typedef struct {
    int rot, kind;
    double base, factor, trained, low, high, gain;
} aria_hip_rotary_scaling;
/* dcos, dsin [n, rot/2] fp32 for positions first .. first + n - 1 (first and all of them 0 .. 2^24): the angle's
 * fraction of a turn to 2^-28 at any of them, so that far positions keep fp32's precision. 4-byte aligned. */
int aria_hip_rotary_table_dev(float *dcos, float *dsin, const aria_hip_rotary_scaling *a, int64_t first, int n,
                              void *stream);

/* Rotates the first rot dims of every head of q [B, N, Hq, D] and, where k is given, of k [B, N, Hk, D]
 * into q_out and k_out; dims from rot on are copied. Pairs are (i, i + rot/2), or (2i, 2i + 1) where
 * interleaved: (a, b) -> (a c - b s, b c + a s), and by the other sign of s where inverse (the adjoint: a
 * gradient's way back). c, s = row p of cos, sin [npos, rot/2], p the token's position: pos[b *
 * pos_stride + t], or without pos first[b] + t (first NULL: t). Rows of a position outside 0 .. npos - 1
 * (padding) are left as they are. Products and sums in fp32 (fp32 states: in 64 bits), rounded once.
 * An output may be its own input with the same strides. D even, rot even, 0 .. D. */
typedef struct {
    const void *q, *k;
    void *q_out, *k_out;
    const float *cos, *sin;
    const int32_t *pos, *first;
    int64_t pos_stride;
    int type, B, N, Hq, Hk, D, rot, npos, interleaved, inverse;
    int64_t q_batch, q_token, q_head, k_batch, k_token, k_head;
    int64_t qo_batch, qo_token, qo_head, ko_batch, ko_token, ko_head;
} aria_hip_rotary;
int aria_hip_rotary_dev(const aria_hip_rotary *a, void *stream);

/* A cache of keys and values: slot t of head h of sequence b is a row of D codes at k (v) + b * batch +
 * h * head + t * token bytes and a scale byte at k_scale (v_scale) + b * s_batch + h * s_head + t. Codes are
 * e4m3 (sign, 4 bits of exponent with bias 7, 3 of mantissa, largest 448, no infinity); the row stands
 * for code * 2^(byte - 127). byte: the smallest, at least 1, for which the row's largest magnitude is at
 * most 448 * 2^(byte - 127); codes to nearest, ties to even. A row that holds an Inf or a NaN gets byte
 * 255 and codes 0x7F: it stands for NaN. (Of a pack from elsewhere: a byte of 0 and NaN codes under another
 * byte than 255 are not supported.) D: a multiple of 16 up to 256. k and v 16-byte aligned, batch, head and token
 * multiples of 16; B and Hkv at most 2^16, cap at most 2^30. */
typedef struct {
    uint8_t *k, *v, *k_scale, *v_scale;
    int64_t batch, head, token, s_batch, s_head;
    int B, Hkv, D, cap;
} aria_hip_kv;
/* Writes tokens t < count[b] (count NULL: N; held to 0 .. N) of k, v [B, N, Hkv, D] to slots first[b] + t (first
 * NULL: t); slots outside 0 .. cap - 1 are skipped. Where rot > 0 keys are rotated before,
 * as in aria_hip_rotary, by position pos[b * pos_stride + t], or the slot without pos; the rotated key is rounded to fp32,
 * then to its code. A token whose position lies outside the table is not written. Queries q [B, N, Hq, D] of the same
 * tokens (q NULL: none), rotated likewise, go to q_out in their own type, whatever their slot; q_out may be q.
 * Two calls in flight must not write the same slot. */
typedef struct {
    aria_hip_kv cache;
    const void *k, *v, *q;
    void *q_out;
    const float *cos, *sin;
    const int32_t *pos, *first, *count;
    int64_t pos_stride;
    int type, N, Hq, rot, npos, interleaved;
    int64_t k_batch, k_token, k_head, v_batch, v_token, v_head;
    int64_t q_batch, q_token, q_head, qo_batch, qo_token, qo_head;
} aria_hip_kv_write;
int aria_hip_kv_write_dev(const aria_hip_kv_write *a, void *stream);
/* Slots first[b] + t, t < count[b], as values in k, v [B, N, Hkv, D] (either NULL: not read), rounded to type
 * and held to its finite range (NaN stays); rows of other t and of slots outside 0 .. cap - 1 are left as they are. */
typedef struct {
    aria_hip_kv cache;
    void *k, *v;
    const int32_t *first, *count;
    int type, N;
    int64_t k_batch, k_token, k_head, v_batch, v_token, v_head;
} aria_hip_kv_read;
int aria_hip_kv_read_dev(const aria_hip_kv_read *a, void *stream);

/* Attention for a batch whose sequences share prefixes: q [B, H, Nq, D] fp16 or bf16 -> out [B, Nq, H, D]
 * (out_f32: fp32). Sequence b sees prefix b / (B / prefix.B), of prefix.B that divide B, and sequence b of own;
 * H / Hkv consecutive query heads read one head of both.
 *   out[b,t,h] = sum_j p_j v_j, p = softmax over the keys j that it sees of scale * q . k_j:
 * the prefix's slots below prefix_len (per prefix; NULL: cap), and own slots below own_len (per sequence; NULL:
 * cap) that, where first is given, are at most first[b] + t (causal: query t stands at slot first[b] + t).
 * Lengths are taken as held to 0 .. cap; a cache of cap 0 is absent (no pointers). Both descriptions give B, Hkv and D.
 * A row that sees no key is zero. What the slots that a row does not see hold does not reach it (byte 255 included). A key
 * or a value of byte 255 that it sees makes the whole row NaN.
 * Cached values are rounded to q's type (exact in bf16; fp16 above 2^-24 steps) and held to its finite range, as reading them is;
 * probabilities are rounded to it too, and in fp16 one below 2^-32 of its row's largest may count as zero. Sums and softmax
 * statistics are fp32: scores times scale, and sums of values under weights of up to 2^15, have to stay within it. D up to
 * 128; scale positive, at most 2^127; B * H at most 2^20, B * H * Nq at most 2^30; a cache's token stride below 2^24. q and out
 * 16-byte aligned, strides multiples of 8. Many sequences' rows together read a prefix once.
 * dws: aria_hip_prefix_attention_ws_bytes(a) bytes (0: may be NULL), 256-byte aligned, not shared by calls that may run at the
 * same time; the number goes by B, H, Nq and both caches' B, Hkv, D and cap alone. It may fall where one of them grows
 * (8 sequences of 300 tokens may need 60 MB and of 400 none): a workspace for several descriptions has the largest number of
 * them all, not that of the largest description. */
typedef struct {
    const void *q;
    void *out;
    aria_hip_kv prefix, own;
    const int32_t *prefix_len, *own_len, *first;
    int type, out_f32, B, H, Nq;
    float scale;
    int64_t q_batch, q_token, q_head, o_batch, o_token, o_head;
} aria_hip_prefix_attn;
size_t aria_hip_prefix_attention_ws_bytes(const aria_hip_prefix_attn *a);
int aria_hip_prefix_attention_dev(const aria_hip_prefix_attn *a, void *dws, void *stream);

/* Host-pointer forms with the reference's signatures (src/aria_quant.h:43-45, 64-65):
 * allocate, copy in, run, copy out, free; synchronous. Return 0 or an error. */
int aria_hip_q8_quant(int8_t *q, float *scale, const float *W, int N, int K);
int aria_hip_q4_quant(uint8_t *q, float *scale, const float *W, int N, int K);
int aria_hip_q8_dequant(float *W, const int8_t *q, const float *scale, int N, int K);
int aria_hip_q4_dequant(float *W, const uint8_t *q, const float *scale, int N, int K);
int aria_hip_linear_q8(float *y, const float *x, const int8_t *q, const float *scale,
                       const float *b, int M, int K, int N);
int aria_hip_linear_q4(float *y, const float *x, const uint8_t *q, const float *scale,
                       const float *b, int M, int K, int N);

/* ---- host-pointer forms of the fused ops (parity entry points) ---- */
int aria_hip_layernorm(float *y, const float *x, const float *gamma, const float *beta,
                       int rows, int dim, float eps);
int aria_hip_rmsnorm_adaln(float *y, const float *x, const float *w, const float *scale,
                           const float *shift, int rows, int dim, int rows_per_batch, float eps);
int aria_hip_ln_mod_gelu_res(float *out, const float *x, const float *gamma, const float *beta,
                             const float *scale, const float *shift, int rows, int dim,
                             int rows_per_batch, float eps);
int aria_hip_modulate(float *y, const float *x, const float *scale, const float *shift,
                      int rows, int dim, int rows_per_batch);
int aria_hip_gate_residual(float *out, const float *res, const float *o, const float *gate,
                           const float *bias, int rows, int dim, int rows_per_batch);
int aria_hip_glu_combine(float *out, const float *proj, const float *bias, int rows, int inner);
int aria_hip_add(float *y, const float *a, const float *b, size_t n);
int aria_hip_pingpong(float *x, const float *v, const float *noise, float tc, float tn, size_t n);

#ifdef __cplusplus
}
#endif
#endif /* ARIA_HIP_H */
