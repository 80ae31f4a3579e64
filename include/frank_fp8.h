/*
 * frank_fp8.h -- C ABI of the 8-bit (e4m3) MoE FFN path: block-scaled
 * quantisation, the expert-grouped product, the expert FFN, the whole block
 * and its sub-layer with norms on both sides.  Additions of this library: the
 * reference computes the same block in fp32 (components/moe/moe_ffn_block.mlir:34-209).
 *
 * Conventions are frank_moe.h's: device pointers, caller-owned buffers, a
 * cudaStream_t as void*, asynchronous calls, 0 or a negative FRANK_E* status
 * with frank_last_error().  16-byte aligned buffers throughout.
 *
 * 8-bit rows.  A row of K values is held as e4m3 values q [T, K] and one fp32
 * scale for each block of 128 consecutive values, block-major:
 * scale [ceil(K/128), T]; the value is q * scale.  Quantising sets
 *   scale = 2^p, p the least integer >= -110 with amax <= 448 * 2^p,
 *   q     = e4m3(v / 2^p), nearest, ties to even
 * so that v / 2^p is exact and the value is rounded once.  A block that holds
 * a NaN or an infinity gets the scale NaN: every product with it is NaN.
 *
 * 8-bit weights.  e4m3 q [E, N, K] and one fp32 scale for each 128 x 128 block:
 * scale [E, ceil(N/128), ceil(K/128)].  Products form (row's scale) * (weights'
 * scale) in fp32.  A row's scale is in [2^-110, 2^120], so weights' scales of
 * magnitude below 2^8 never overflow there; a larger one gives infinities or NaN
 * with those rows whose scale takes the product to 2^128.  A product of
 * scales below 2^-126 keeps fewer bits: an error of up to 2^-125 for each block of K.
 *
 * K, N, H and F are multiples of 16; the last block may be short.
 */
#ifndef FRANK_FP8_H_
#define FRANK_FP8_H_

#include "frank_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

#define FRANK_FP8_BLOCK 128

/*
 * x [T, K] (FRANK_F32 or FRANK_BF16) -> q [T, K], scale [ceil(K/128), T].
 */
int frank_quantize_fp8(int x_dtype, const void* x, int64_t T, int64_t K,
                       void* q, float* scale, void* stream);

/*
 * The norm before an 8-bit block: xn = bf16(x / sqrt(mean(x^2) + eps) * weight)
 * for x [T, H] (FRANK_F32 or FRANK_BF16), then the 8-bit form of xn.
 * xn [T, H] bf16 may be NULL.  H <= 16384.
 */
int frank_rms_norm_fp8(int x_dtype, const void* x, const float* weight,
                       int64_t T, int64_t H, float eps, void* xn, void* q,
                       float* scale, void* stream);

/*
 * One-time weight prepack: [O, I, E] (expert innermost, in_dtype FRANK_F32 or
 * FRANK_BF16) -> 8-bit weights q [E, O, I] and scale [E, ceil(O/128),
 * ceil(I/128)], scales by the rule for rows over each 128 x 128 block.
 */
int frank_prepack_experts_fp8(int in_dtype, const void* w_oie, int64_t O,
                              int64_t I, int64_t E, void* q_eoi, float* scale,
                              void* stream);

/*
 * Product of 8-bit rows and weights: for the rows r of group e (rows
 * [offsets[e], offsets[e+1]) of q; offsets [E+1] ascending int32 from 0 to `rows`,
 * or NULL with E = 1 for one group of all rows)
 *   out[r, n] = sum_b scale[b, r] * w_scale[e, n/128, b] * sum_{k in block b} q[r, k] * w[e, n, k]
 * accumulated in fp32 and stored in out_dtype (FRANK_F32 or FRANK_BF16),
 * out [rows, N].  Rows outside every group are left as they were.
 * E <= 256.
 */
int frank_fp8_matmul(const void* q, const float* scale, const void* w,
                     const float* w_scale, const int32_t* offsets, int64_t E,
                     int64_t rows, int64_t N, int64_t K, int out_dtype,
                     void* out, void* stream);

/*
 * frank_fp8_matmul of rows x [rows, K] (FRANK_F32 or FRANK_BF16) that are quantised
 * first, in a workspace of frank_fp8_linear_workspace_size(rows, K) bytes.
 */
size_t frank_fp8_linear_workspace_size(int64_t rows, int64_t K);
int frank_fp8_linear(int x_dtype, const void* x, const void* w,
                     const float* w_scale, const int32_t* offsets, int64_t E,
                     int64_t rows, int64_t N, int64_t K, int out_dtype,
                     void* out, void* workspace, size_t ws_bytes,
                     void* stream);

/*
 * The expert FFN with the routing given: x [T, H] bf16 is quantised,
 *   h = gate(x) * silu(up(x))   (fp32, then quantised in blocks of 128 of F)
 *   y[t] = sum_j route_w[j, t] * down(h[j, t])     (fp32, j in order; rounded once)
 * route_w [k, T] fp32, route_ids [k, T] int32 in [0, E) (an id that a token names
 * twice counts twice); y [T, H] in y_dtype.  An id outside [0, E) is clamped and recorded
 * in *err_flag (device int32, zeroed by the caller; may be NULL).
 * Workspace: frank_fp8_moe_workspace_size(T, H, F, E, k) bytes, no header, any
 * contents; calls that share one must not overlap.
 */
size_t frank_fp8_moe_workspace_size(int64_t T, int64_t H, int64_t F, int64_t E,
                                    int64_t k);
int frank_fp8_moe_experts(const void* x, const float* route_w,
                          const int32_t* route_ids, const void* w_up,
                          const float* s_up, const void* w_gate,
                          const float* s_gate, const void* w_down,
                          const float* s_down, int64_t T, int64_t E, int64_t k,
                          int64_t H, int64_t F, int y_dtype, void* y,
                          int32_t* err_flag, void* workspace, size_t ws_bytes,
                          void* stream);

/*
 * The whole block: frank_router_topk's routing of x [T, H] bf16 (wr as there,
 * FRANK_F32, FRANK_BF16 or FRANK_ROUTER_PACKED), then frank_fp8_moe_experts.
 * route_w / route_ids [k, T]: optional outputs (may be NULL).
 */
int frank_fp8_moe_block(const void* x, int wr_dtype, const void* wr,
                        const void* w_up, const float* s_up,
                        const void* w_gate, const float* s_gate,
                        const void* w_down, const float* s_down, int64_t T,
                        int64_t E, int64_t k, int64_t H, int64_t F,
                        int normalize, int y_dtype, void* y, float* route_w,
                        int32_t* route_ids, void* workspace, size_t ws_bytes,
                        void* stream);

/*
 * The sub-layer around the 8-bit block, with norms before and after it:
 *   xn  = bf16(rms_norm(residual, norm_w, eps))
 *   y   = block(xn)
 *   out = residual_scale * residual + gate * rms_norm(y, post_w, eps)
 * residual, out [T, H] in res_dtype (FRANK_F32 or FRANK_BF16; out may be
 * residual).  post_w NULL: y is not normalised.  gate: fp32 [gate_rows, H]
 * where gate_rows divides T and rows of T / gate_rows consecutive tokens share
 * a gate, or NULL for 1.  H <= 16384.
 */
int frank_fp8_moe_sublayer(int res_dtype, const void* residual,
                           const float* norm_w, float eps, int wr_dtype,
                           const void* wr, const void* w_up,
                           const float* s_up, const void* w_gate,
                           const float* s_gate, const void* w_down,
                           const float* s_down, int64_t T, int64_t E,
                           int64_t k, int64_t H, int64_t F, int normalize,
                           const float* post_w, const float* gate,
                           int64_t gate_rows, float residual_scale, void* out,
                           float* route_w, int32_t* route_ids, void* workspace,
                           size_t ws_bytes, void* stream);

/*
 * The end of a sub-layer, and the beginning of the next one:
 *   out  = residual_scale * residual + gate * rms_norm(y, weight, eps)
 *   next = rms_norm(out, next_weight, eps)                (when next is not NULL)
 * y [T, H] in y_dtype; residual and out [T, H] in res_dtype (out may be
 * residual; next is computed from the rounded out); next [T, H] in next_dtype.
 * gate and gate_rows as above.  H % 4 == 0, H <= 16384.
 */
int frank_post_norm_residual(int y_dtype, const void* y, int res_dtype,
                             const void* residual, const float* weight,
                             float eps, const float* gate, int64_t gate_rows,
                             float residual_scale, void* out,
                             const float* next_weight, int next_dtype,
                             void* next, int64_t T, int64_t H, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* FRANK_FP8_H_ */
