/*
 * ggml_hip_moe.h -- C ABI of what a mixture-of-experts layer needs around the
 * block-quantized products, in libggml_hip_qmm.so: the choice of each token's
 * experts, matrix products in 8-bit integers with a scale for each token and
 * each channel (dense and by experts), and the weighted sum of the experts'
 * rows.
 *
 * Conventions are those of ggml_hip_qmm.h: device pointers, activations f32,
 * asynchronous on `stream`, no allocation, scratch from the caller, 0 or a
 * hipError_t back (hipErrorInvalidValue = 1 for what an entry does not take,
 * before anything is launched).  Strides are in elements, and f32 and int32
 * tensors aligned to 4 bytes; nothing that is written overlaps what is read, but
 * where a comment allows it.  All results are deterministic.
 */
#ifndef GGML_HIP_MOE_H
#define GGML_HIP_MOE_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* The probability p of expert e, from the logits l of its token. */
#define HIP_QMM_ROUTE_SOFTMAX 0        /* exp(l_e) / sum over all experts */
#define HIP_QMM_ROUTE_SIGMOID 1        /* 1 / (1 + exp(-l_e)) */
#define HIP_QMM_ROUTE_SOFTMAX_CHOSEN 2 /* l_e itself; softmax over the chosen ones makes the weights */

/*
 * The k experts of each token and their weights.  Expert e's score is
 * p_e + bias[e] (bias NULL: 0).  The experts form n_groups groups of
 * n_experts / n_groups neighbours; a group's score is the sum of its
 * `group_top` (1 or 2) best scores, or of the one it has, and the experts of
 * the n_keep best groups stand for choice.  ids[t] are the k best of them, by
 * descending score, weights[t] their p (SOFTMAX_CHOSEN: softmax of their l),
 * divided by max(their sum, min_sum) with `renormalize`, times `scale`.
 *
 * Of equal scores the lower index (of groups: too) comes first, a NaN before
 * all others.  An expert whose l or bias is -infinity is hidden: never chosen,
 * and no part of its group's score.  Places for which no expert is left hold id
 * -1 and weight 0, as hip_qmm_mul_mat_id and hip_qmm_mul_mat_id_i8 take it.
 * A softmax over a NaN or +infinity is NaN, as in IEEE arithmetic.
 * Scores are computed and compared in f64, where those that f32 would round
 * to one value keep their order (without a bias experts are compared by their
 * l), and weights are rounded to f32 once.
 *
 * n_experts 1..1024, k 1..64 and at most n_experts, n_groups 1..64 and a
 * divisor of n_experts, n_keep 1..n_groups; min_sum at least 0 and finite,
 * scale finite; n_tokens at most 2^24.
 */
int hip_qmm_moe_route(const float *logits, int64_t n_tokens, int64_t n_experts, int64_t logits_stride,
                      const float *bias, int gating, int64_t n_groups, int64_t n_keep, int group_top, int64_t k,
                      int renormalize, float min_sum, float scale, int32_t *ids, int64_t ids_stride, float *weights,
                      int64_t weights_stride, void *stream);

/*
 * Rows to 8-bit integers: scale[r] = max|x[r]| * (1/127) and q[r] = x[r] / scale[r]
 * to the nearest, half to even, cut to +-127: one f32 product with the f32 next
 * to 1/127, and IEEE f32 divisions.  A row
 * whose scale rounds to 0 has zeros, and one with a value that is not finite
 * zeros and a scale of NaN.  Only the K values of a row are written.  K 1 to
 * 131071, n_rows at most 2^24.
 */
int hip_qmm_quantize_i8(const float *x, int64_t K, int64_t n_rows, int64_t x_stride, int8_t *q, int64_t q_stride,
                        float *scale, void *stream);

/*
 * dst[n][m] = (sum_k w[m][k] * x[n][k]) * x_scale[n] * w_scale[m], the sum in
 * 32-bit integers (exact), then three f32 roundings (the sum's and the two
 * products'; only the result's range matters, not a product's).  With x_scale
 * NULL x is f32 and quantized in the call as hip_qmm_quantize_i8 does.
 *
 * w is int8, 16-byte aligned with a row stride that is a multiple of 16, and so
 * is an int8 x; the bytes from K to the next multiple of 16 of each of their
 * rows must be readable but do not matter.  K 1 to 131071, nrows and ncols at
 * most 2^22, their product at most 2^38.  The workspace is scratch, 256-byte aligned: its contents do
 * not matter before the call, and it serves one call at a time.  Its size is at
 * most ncols * (K + 131) + 512, and 0 for an int8 x.
 */
size_t hip_qmm_mul_mat_i8_workspace_size(int64_t K, int64_t nrows, int64_t ncols, int quantized);
int hip_qmm_mul_mat_i8(const int8_t *w, const float *w_scale, int64_t K, int64_t nrows, int64_t w_stride,
                       const void *x, const float *x_scale, int64_t ncols, int64_t x_stride, float *dst,
                       int64_t dst_stride, void *workspace, size_t workspace_size, void *stream);

/*
 * hip_qmm_mul_mat_id with such weights: row (t, s) of dst, at
 * dst + (t*n_ids + s)*dst_stride, is the product of expert ids[t][s] (rows at
 * w + e*expert_stride, scales at w_scale + e*nrows) with row t*ne11 + s % ne11 of x
 * (ne11 1 or n_ids; x_stride between rows, x_scale one a row or NULL as above).
 * An id outside [0, n_as) leaves a zero row.  n_as at most 1024, n_tokens*n_ids
 * at most 2^22, times nrows at most 2^38; expert_stride a multiple of 16; otherwise the limits of
 * hip_qmm_mul_mat_i8.
 */
size_t hip_qmm_mul_mat_id_i8_workspace_size(int64_t K, int64_t nrows, int64_t n_as, int64_t ne11, int64_t n_tokens,
                                            int64_t n_ids, int quantized);
int hip_qmm_mul_mat_id_i8(const int8_t *w, const float *w_scale, int64_t K, int64_t nrows, int64_t w_stride,
                          int64_t expert_stride, int64_t n_as, const void *x, const float *x_scale, int64_t ne11,
                          int64_t n_tokens, int64_t x_stride, const int32_t *ids, int64_t n_ids, int64_t ids_stride,
                          float *dst, int64_t dst_stride, void *workspace, size_t workspace_size, void *stream);

/*
 * dst[t] = add[t] + sum_s weights[t][s] * y[t][s], over rows of nrows values,
 * summed in f64 and rounded to f32 once (add NULL: from 0).  With ids, slots whose id
 * is negative are left out, whatever their rows hold.  Row (t, s) of y is at
 * y + t*y_token_stride + s*y_row_stride.  dst may be add with its stride.
 * n_ids 0..65535, n_tokens and nrows at most 2^31 - 1.
 */
int hip_qmm_moe_combine(const float *y, int64_t n_tokens, int64_t n_ids, int64_t nrows, int64_t y_token_stride,
                        int64_t y_row_stride, const float *weights, int64_t weights_stride, const int32_t *ids,
                        int64_t ids_stride, const float *add, int64_t add_stride, float *dst, int64_t dst_stride,
                        void *stream);

#ifdef __cplusplus
}
#endif

#endif /* GGML_HIP_MOE_H */
