/*
 * hf_fp8.h -- FP8 (e4m3) operators of the B200 MoE library: quantised rows, the
 * block-scaled product, and the routed SwiGLU experts over FP8 weights.
 *
 * The reference keeps every weight in BF16; an FP8 checkpoint of the same model
 * stores each weight matrix as e4m3 values with one fp32 scale per block of
 * 128 x 128 (the value is q * scale), which halves the bytes a decode step
 * streams and doubles the tensor cores' rate.
 *
 * Status, streams and errors as in hf_moe.h: argument errors return HF_ERR_ARG
 * before anything is enqueued, calls are asynchronous on `stream`, pointers
 * belong to the current device. e4m3 values are passed as uint8_t bits.
 */
#ifndef HF_FP8_H
#define HF_FP8_H

#include "hf_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

#define HF_FP8_BLOCK 128 /* columns of a row, and rows and columns of a weight, per scale */

/* Rows to e4m3 with one scale per 128 columns:
 *   s[t, b] = the smallest power of two with max|x[t, 128b ..]| <= 448 s
 *             (1 for a block of zeros, at least 2^-126)
 *   q[t, j] = x[t, j] / s, rounded to nearest even
 * Dividing by a power of two is exact, so each value is rounded once; e4m3 has
 * the same relative precision at either end of a binade, so nothing is lost
 * against a scale of max / 448. A block that holds Inf or NaN becomes NaN
 * (scale and values): it is never saturated.
 * x: device [T x K] BF16 or fp32, rows ldx elements apart, 16-byte aligned
 * (pointer and pitch); q: device [T x K]; scales: device fp32 [T x ceil(K/128)].
 * K a multiple of 16; T, K (and N below) at most 2^31 - 4096. */
HF_API hf_status hf_fp8_quantize(const void* x, hf_dtype x_dtype, long long ldx, int T, int K,
                                 uint8_t* q, float* scales, hf_stream stream);

/* out = (xq * sx) (wq * sw)^T over T rows:
 *   out[t, n] = sum_b sx[t, b] sw[n / 128, b] sum_{j in block b} xq[t, j] wq[n, j]
 * with products and sums in fp32 (the two scales are multiplied first: their product
 * neither overflows nor is subnormal). xq: device e4m3 [T x K]; sx: fp32
 * [T x ceil(K/128)] (any values, not only powers of two); wq: e4m3 [N x K];
 * sw: fp32 [ceil(N/128) x ceil(K/128)]; out: [T x N] of out_dtype. K a multiple
 * of 16, any T and N; xq, wq and the workspace 16-byte (workspace: 256-byte)
 * aligned. Sums of up to 128 products are taken by the tensor cores in fp32; with
 * few output tiles K is cut into runs whose fp32 partial sums lie in the workspace
 * and are added in order, so equal calls give equal bits. */
HF_API size_t hf_fp8_gemm_workspace_size(int T, int N, int K);
HF_API hf_status hf_fp8_gemm(const uint8_t* xq, const float* sx, const uint8_t* wq, const float* sw,
                             int T, int N, int K, void* out, hf_dtype out_dtype, void* workspace,
                             size_t workspace_bytes, hf_stream stream);

/* The routed SwiGLU experts over FP8 weights (expertFFNRaw and the combine,
 * glm_forward.cpp:434-449, 555-556, 639-640, with quantised operands):
 *   xq, sx  = quantise(x)
 *   g, u    = xq Wg^T, xq Wu^T                    (of the token's experts)
 *   mq, ms  = quantise(silu(g) * u)               (per 128 intermediate columns)
 *   y_i     = mq Wd^T
 *   out     = resid + sum_i w_i y_i               (rank order, fp32)
 * experts: device e4m3, E blocks [gate I*H | up I*H | down H*I] (the layout of
 * Scheduler::getExpertPtr, engine/scheduler.h:80-84); scales: device fp32, E
 * blocks [gate ceil(I/128) x ceil(H/128) | up, the same | down ceil(H/128) x
 * ceil(I/128)]. x: device [T x H] BF16 or fp32, rows ldx elements apart.
 * routing: topk_weights [T x k], counts, offsets and perm as written by
 * hf_route_logits or hf_moe_route for the same T and k (a shared segment behind
 * the routed ones is left out; topk_ids is not read). offsets do not decrease and
 * perm names a slot once at most; entries out of range are clipped (offsets) or
 * skipped (perm), and a slot that perm does not name, or at a position outside
 * [offsets[0], offsets[E]), adds nothing to its token. resid: device [T x H] of
 * out_dtype or NULL, may be out itself. out: device [T x H] of out_dtype; until the
 * combine the expert outputs y_i are kept in fp32 for fp32 outputs, and for bf16
 * ones with 16 significant bits (the rest of the fp32 number cut off) or, from a
 * mean of 97 positions an expert on, in FP16 times a power of two per 32 columns
 * (11 significant bits down to 2^-28 of a block's largest). The shared expert, or a
 * dense MLP, is the call with E = 1, k = 1 and the routed output as resid. H and I
 * multiples of 16, k in 1..32, E in 1..1024, T * k and 3 * E * max(H, I) at most
 * 2^31 - 4096; pointers 16-byte aligned, the workspace 256-byte. A workspace serves
 * any number of layers in stream order. */
HF_API size_t hf_fp8_moe_experts_workspace_size(int T, int top_k, int E, int H, int I,
                                                hf_dtype out_dtype);
HF_API hf_status hf_fp8_moe_experts(const uint8_t* experts, const float* scales, int E, int H,
                                    int I, const void* x, hf_dtype x_dtype, long long ldx, int T,
                                    int top_k, const hf_moe_routing* routing, const void* resid,
                                    void* out, hf_dtype out_dtype, void* workspace,
                                    size_t workspace_bytes, hf_stream stream);

/* Waits for `stream` and reports whether a bounded device wait of the last
 * hf_fp8_gemm or hf_fp8_moe_experts on this workspace gave up (HF_ERR_TIMEOUT).
 * Every output of such a call is right or NaN, so that it does not pass unnoticed
 * where nobody asks. */
HF_API hf_status hf_fp8_status(const void* workspace, hf_stream stream);

/* Limit of every bounded device wait of the products launched or captured from now
 * on, in this process, in nanoseconds (default 2 s, 0 restores it), and a test hook
 * (failure detection without a GPU fault): with block b > 0 the products' copies stop
 * ahead of each CTA's b-th block of 128 columns and wait on a barrier that nothing
 * signals (b < 0: those of every CTA pair's second CTA only, ahead of the |b|-th), so
 * that the waits run out and hf_fp8_status reports HF_ERR_TIMEOUT. 0 turns it off.
 * As hf_moe_set_wait_timeout and hf_moe_debug_stall, for calls without a context. */
HF_API hf_status hf_fp8_set_wait_timeout(uint64_t ns);
HF_API hf_status hf_fp8_debug_stall(int block);

#ifdef __cplusplus
}
#endif
#endif /* HF_FP8_H */
