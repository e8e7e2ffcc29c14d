/*
 * C ABI of the operators around the grouped GEMM in a mixture-of-experts layer (MI355X, gfx950):
 * RMS norm, router with balance loss, dispatch and combine of the experts' rows, and grouped
 * products with 4-bit weights. Same library and conventions as gg_grouped_gemm.h: plain pointers
 * and sizes, `stream` a hipStream_t passed as void* (NULL = the default stream) of the current
 * device, every entry point returns a gg_status, none exits the process or throws.
 *
 * Every call enqueues kernels on `stream` and returns: it allocates nothing, waits for nothing and
 * keeps nothing for a later call, so any of them may be captured into a graph. Buffers, workspace
 * among them, must stay valid until the work on `stream` is done. Row strides are in elements.
 * Sums, norms and softmax statistics are float32; an output is rounded once, when it is stored.
 * Results do not depend on the order in which workgroups run.
 */
#ifndef GG_MOE_LAYER_H
#define GG_MOE_LAYER_H

#include "gg_grouped_gemm.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Beside gg_dtype: norm weights and router logits may be float32. */
enum { GG_DTYPE_FP32 = 4 };

/* Message of the last failed call of this header on the calling thread ("" if none). */
const char *gg_layer_last_error(void);

/* ---- RMS norm with the residual's addition ---- */

/* How y is written. */
typedef enum gg_norm_scale {
    GG_NORM_PLAIN        = 0, /* y in the type of x */
    GG_NORM_SCALE_TENSOR = 1, /* y fp8, one scale for the tensor from its largest |y|: what the fp8 grouped GEMMs take */
    GG_NORM_SCALE_ROW    = 2, /* y fp8, one scale for each row from its largest |y| */
    GG_NORM_SCALE_GIVEN  = 3  /* y fp8, divided by scale[0], which is read; values past the format's range saturate */
} gg_norm_scale;

/*
 * h = x + residual, rounded to x's type as the layers after this one read it (h = x without a
 * residual); rstd = 1 / sqrt(mean(h^2) + eps) of each row; y = h * rstd * weight, of the rounded h.
 * (A row whose squares add up past 3.4e38, which values of some 10^17 and more can, has an rstd of 0.)
 * fp8: y = round(h * rstd * weight / scale), scale = max |h * rstd * weight| / (the format's largest
 * value), 1 where that is zero or subnormal. A NaN in a row makes its rstd, y and (for a tensor scale, every) scale NaN.
 *   dtype: GG_DTYPE_BF16 or GG_DTYPE_FP16 (x, residual, h; y unless fp8). weight_dtype: the same or
 *   GG_DTYPE_FP32. out_dtype: dtype, or an fp8 type with scale_mode 1-3.
 *   h: [rows, hidden]; may be x or residual itself. Not written (and may be NULL) without a residual.
 *   y: [rows, hidden] contiguous, overlapping no input. rstd: [rows], or NULL but for GG_NORM_SCALE_TENSOR.
 *   scale: written, [1] or [rows] (of no rows it may be NULL), or for GG_NORM_SCALE_GIVEN read, [1].
 *   workspace: GG_NORM_WORKSPACE bytes for GG_NORM_SCALE_TENSOR, else unused.
 * GG_ERR_UNSUPPORTED unless hidden % 8 == 0, hidden <= 32768, strides % 8 == 0 and 16-byte aligned
 * buffers (y of fp8: 8-byte).
 */
enum { GG_NORM_WORKSPACE = 8192 };
int gg_rms_norm(int dtype, int weight_dtype, int out_dtype, int scale_mode, int64_t rows, int64_t hidden, float eps,
                const void *x, int64_t x_stride, const void *residual, int64_t residual_stride, const void *weight,
                void *h, int64_t h_stride, void *y, float *rstd, float *scale, void *workspace, void *stream);

/*
 * Gradients of gg_rms_norm from its h and rstd (an fp8 y is differentiated as if it were not rounded):
 *   grad_x = grad_h + rstd * (weight * grad_y) - h * rstd^3 * mean(weight * grad_y * h)
 *   grad_weight = sum over rows of grad_y * h * rstd
 * grad_x [rows, hidden] contiguous is the gradient of x and of residual alike; grad_h (the gradient
 * that reaches h past the norm) may be NULL. grad_x may take the place of a contiguous grad_y, h or grad_h.
 * grad_weight [hidden] is of weight_dtype.
 * workspace: gg_rms_norm_backward_workspace(rows, hidden) bytes (0 for few rows: then it may be NULL), 16-byte aligned.
 * Rules as above.
 */
size_t gg_rms_norm_backward_workspace(int64_t rows, int64_t hidden);
int gg_rms_norm_backward(int dtype, int weight_dtype, int64_t rows, int64_t hidden, const void *grad_y,
                         int64_t grad_y_stride, const void *h, int64_t h_stride, const void *weight, const float *rstd,
                         const void *grad_h, int64_t grad_h_stride, void *grad_x, void *grad_weight, void *workspace,
                         size_t workspace_bytes, void *stream);

/* ---- router ---- */

/*
 * Top-k routing of logits [tokens, experts] (float32, bf16 or fp16).
 *   experts_out [tokens, top_k] int32: each token's largest logits in descending order, equal ones by
 *               the lower index (NaN counts as the largest value). -1 in the slots of a token that
 *               takes no part, and in slots for which only logits of -infinity are left.
 *   weights     [tokens, top_k]: softmax probabilities (over all experts) of those; with renormalize
 *               divided by their sum over the token. 0 where experts_out is -1.
 *   counts      [experts] int64: rows of each expert, the group sizes that the grouped GEMMs take.
 *   offs        [experts + 1] int64: first row of each expert, in expert order back to back.
 *   rows        [tokens, top_k] int32: the row of each (token, slot) pair: experts in order, within an
 *               expert tokens in order. -1 where experts_out is -1.
 *   lse         [tokens]: log of the sum of exponentials of the token's logits; -infinity for a token
 *               that takes no part.
 *   mask        [tokens] bytes or NULL: 0 = the token takes no part (padding): its logits are not
 *               looked at. A token whose logits are all -infinity takes no part either.
 *   loss, slope [1], [experts], both or neither (NULL): the balance loss
 *               experts * sum_e f_e P_e, f_e = counts_e / sum of counts, P_e = mean probability of e
 *               over the tokens that take part, and its derivative with respect to one token's
 *               probability of e, experts * f_e / (tokens that take part). 0 if there are none.
 *   workspace:  gg_route_workspace(tokens, experts, top_k) bytes, 16-byte aligned.
 * GG_ERR_UNSUPPORTED: more than 1024 experts, top_k > 32, tokens > 2^28 or tokens * top_k >= 2^31. top_k <= experts.
 */
size_t gg_route_workspace(int64_t tokens, int experts, int top_k);
int gg_route(int dtype, int64_t tokens, int experts, int top_k, int renormalize, const void *logits, int64_t stride,
             const uint8_t *mask, int *experts_out, float *weights, int64_t *counts, int64_t *offs, int *rows, float *lse,
             float *loss, float *slope, void *workspace, size_t workspace_bytes, void *stream);

/*
 * grad_logits [tokens, experts] contiguous, of the logits' type, from the gradient of the weights
 * ([tokens, top_k] float32 or NULL) and of the balance loss ([1] device float32, with the forward's
 * slope; or both NULL). Rows of tokens that take no part are 0. (counts are whole numbers: the loss is
 * differentiated through the probabilities.)
 */
int gg_route_backward(int dtype, int64_t tokens, int experts, int top_k, int renormalize, const void *logits,
                      int64_t stride, const int *experts_out, const float *weights, const float *lse,
                      const float *grad_weights, const float *grad_loss, const float *slope, void *grad_logits,
                      void *stream);

/* ---- rows of the experts ---- */

/*
 * dispatch: xs[rows[t, s]] = x[t] for the rows a router gave (xs [tokens * top_k, hidden]); rows of xs
 * past the last expert's (slots of -1 leave as many) are zeroed. elem_size: bytes of an element (1, 2 or 4).
 * dispatch_backward: grad_x[t] = sum over s of grad_xs[rows[t, s]] (bf16 or fp16).
 * combine: out[t] = sum over s of weights[t, s] * y[rows[t, s]] (bf16 or fp16); 0 for a token without rows.
 * combine_backward: grad_y[rows[t, s]] = weights[t, s] * grad_out[t] (rows past the last expert's
 * zeroed), grad_weights[t, s] = grad_out[t] . y[rows[t, s]] (0 where rows is -1).
 * offs: the router's; only offs[experts], the number of rows in use, is read.
 * Matrices are contiguous but for x and grad_out, whose rows are `stride` elements apart.
 * GG_ERR_UNSUPPORTED unless a row is a multiple of 16 bytes and at most 128 KB, strides too, buffers are
 * 16-byte aligned, top_k <= 32 and tokens * top_k < 2^31.
 */
int gg_dispatch(int elem_size, int64_t tokens, int top_k, int64_t hidden, int experts, const void *x, int64_t stride,
                const int *rows, const int64_t *offs, void *xs, void *stream);
int gg_dispatch_backward(int dtype, int64_t tokens, int top_k, int64_t hidden, const void *grad_xs, const int *rows,
                         void *grad_x, void *stream);
int gg_combine(int dtype, int64_t tokens, int top_k, int64_t hidden, const void *y, const int *rows,
               const float *weights, void *out, void *stream);
int gg_combine_backward(int dtype, int64_t tokens, int top_k, int64_t hidden, int experts, const void *grad_out,
                        int64_t stride, const void *y, const int *rows, const int64_t *offs, const float *weights,
                        void *grad_y, float *grad_weights, void *stream);

/* ---- grouped products with 4-bit weights ---- */

/*
 * out[rows of g] = x[rows of g] @ w[g]^T with w[g, n, k] = scale * (q - zero), q in 0..15, one scale (and
 * zero, in 0..15) for each `group` consecutive k; zero = 8 where zeros is NULL. x [total_m, k], out
 * [total_m, n], scales of dtype (bf16 or fp16), zeros bytes. For groups of few rows: decode, short prompts.
 * group_lens / group_offs: device sizes as in gg_prepare_device_lens_op; a group whose rows are not
 * inside [0, total_m) gets no work (and is not reported); rows of out that belong to no group are not
 * written. The products are of 16 + q, less (16 + zero) times the sum of x, exact but for the float32 sums:
 * an infinity in x makes its row's outputs NaN or infinite, and so may finite values of which 62 times the sum
 * of |x| over the `group` k of a scale reaches 3.4e38 (4.3e34 in each of 128).
 *
 * Storage: n in tiles of 16 and k in tiles of 128, padded with zeros:
 *   packed [group_num][ceil(n / 16)][ceil(k / 128)][64][16] bytes: piece 16 a + r of a tile is row r,
 *     its little-endian 32-bit word j holds the eight k from 32 j + 8 a on, k = 0, 2, 4, 6 in its nibbles
 *     0-3 (from the low end) and k = 1, 3, 5, 7 in its nibbles 4-7;
 *   scales, zeros [group_num][ceil(n / 16)][k / group][16].
 * So a wave's load of a tile is 1 KB in a row, and a lane has the operand of four matrix instructions.
 * GG_ERR_UNSUPPORTED unless n % 8 == 0, group is 32, 64 or 128, k % group == 0, x, out, packed, scales
 * 16-byte and zeros 4-byte aligned, n and k at most 2097152, group_num at most 8192 and total_m at most 134217728.
 */
int gg_gemm_w4(int dtype, int group_num, int64_t total_m, int64_t n, int64_t k, int group, const int64_t *group_lens,
               const int64_t *group_offs, const void *x, const void *packed, const void *scales, const uint8_t *zeros,
               void *out, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* GG_MOE_LAYER_H */
