/*
 * C ABI of the operators around the grouped GEMM in a mixture-of-experts layer (MI355X, gfx950):
 * RMS norm, layer norm, gated activation, rows of int8, router with balance loss, dispatch and combine of the
 * experts' rows, and grouped products with 4-bit weights and in 8-bit integers. Same library and conventions as gg_grouped_gemm.h: plain pointers
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

/* Beside gg_dtype: norm weights and router logits may be float32, rows of 8 bits whole numbers in -127 .. 127. */
enum { GG_DTYPE_FP32 = 4, GG_DTYPE_INT8 = 5 };

/* Message of the last failed call of this header on the calling thread ("" if none). */
const char *gg_layer_last_error(void);

/* ---- RMS norm with the residual's addition ---- */

/* How y is written. */
typedef enum gg_norm_scale {
    GG_NORM_PLAIN        = 0, /* y in the type of x */
    GG_NORM_SCALE_TENSOR = 1, /* y fp8, one scale for the tensor from its largest |y|: what the fp8 grouped GEMMs take */
    GG_NORM_SCALE_ROW    = 2, /* y fp8 or int8, one scale for each row from its largest |y|: int8 is what gg_gemm_i8 takes */
    GG_NORM_SCALE_GIVEN  = 3  /* y fp8, divided by scale[0], which is read; values past the format's range saturate */
} gg_norm_scale;

/*
 * h = x + residual, rounded to x's type as the layers after this one read it (h = x without a
 * residual); rstd = 1 / sqrt(mean(h^2) + eps) of each row; y = h * rstd * weight, of the rounded h.
 * (A row whose squares add up past 3.4e38, which values of some 10^17 and more can, has an rstd of 0.)
 * fp8: y = round(h * rstd * weight / scale), scale = max |h * rstd * weight| / (the format's largest
 * value), 1 where that is zero or subnormal. A NaN in a row makes its rstd, y and (for a tensor scale, every) scale NaN.
 * int8: the same with 127 for the format's largest value, rounded to the nearest whole number, halves to even. A row
 * whose largest |y| is a NaN or an infinity has that (a NaN first) for a scale and holds zeros.
 *   dtype: GG_DTYPE_BF16 or GG_DTYPE_FP16 (x, residual, h; y unless 8-bit). weight_dtype: the same or
 *   GG_DTYPE_FP32. out_dtype: dtype, an fp8 type with scale_mode 1-3, or GG_DTYPE_INT8 with GG_NORM_SCALE_ROW.
 *   h: [rows, hidden]; may be x or residual itself. Not written (and may be NULL) without a residual.
 *   y: [rows, hidden] contiguous, overlapping no input. rstd: [rows], or NULL but for GG_NORM_SCALE_TENSOR.
 *   scale: written, [1] or [rows] (of no rows it may be NULL), or for GG_NORM_SCALE_GIVEN read, [1].
 *   workspace: GG_NORM_WORKSPACE bytes for GG_NORM_SCALE_TENSOR, else unused.
 * GG_ERR_UNSUPPORTED unless hidden % 8 == 0, hidden <= 32768, strides % 8 == 0 and 16-byte aligned
 * buffers (y of 8 bits: 8-byte).
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

/* ---- layer norm with the residual's addition ---- */

/*
 * As gg_rms_norm, of h less its row's mean: mean = mean(h), rstd = 1 / sqrt(mean((h - mean)^2) + eps),
 * y = (h - mean) * rstd * weight + bias. The squares are summed about means, so a large mean costs the variance nothing,
 * and y no more than the mean's own rounding to float32 times rstd * weight; a row of one value has that value for its mean
 * and gives its bias (with eps = 0 NaN). bias: [hidden] of weight_dtype, or NULL for none. mean, rstd: [rows], or NULL but
 * for GG_NORM_SCALE_TENSOR. Types, scales, workspace and rules as there; bias 16-byte aligned.
 */
int gg_layer_norm(int dtype, int weight_dtype, int out_dtype, int scale_mode, int64_t rows, int64_t hidden, float eps,
                  const void *x, int64_t x_stride, const void *residual, int64_t residual_stride, const void *weight,
                  const void *bias, void *h, int64_t h_stride, void *y, float *mean, float *rstd, float *scale,
                  void *workspace, void *stream);

/*
 * Gradients of gg_layer_norm from its h, mean and rstd (an 8-bit y is differentiated as if it were not rounded); with
 * d = h - mean and g = weight * grad_y:
 *   grad_x = grad_h + rstd * (g - mean(g)) - d * rstd^3 * mean(g * d)
 *   grad_weight = sum over rows of grad_y * d * rstd, grad_bias = sum over rows of grad_y
 * grad_weight, grad_bias: [hidden] of weight_dtype, both written. The rest as in gg_rms_norm_backward.
 */
size_t gg_layer_norm_backward_workspace(int64_t rows, int64_t hidden);
int gg_layer_norm_backward(int dtype, int weight_dtype, int64_t rows, int64_t hidden, const void *grad_y,
                           int64_t grad_y_stride, const void *h, int64_t h_stride, const void *weight, const float *mean,
                           const float *rstd, const void *grad_h, int64_t grad_h_stride, void *grad_x, void *grad_weight,
                           void *grad_bias, void *workspace, size_t workspace_bytes, void *stream);

/* ---- gated activation, rows of int8 ---- */

/*
 * y = silu(gate) * up, silu(v) = v / (1 + exp(-v)); gu [rows, 2 * inner] holds each row's gates and then its ups, as a
 * product with the weights of both stacked writes them. out_dtype: dtype, or GG_DTYPE_INT8 with scale [rows] as
 * gg_rms_norm's int8 rows (of the float32 values, which are not rounded to dtype first).
 *   y: [rows, inner] contiguous, overlapping no input.
 * gg_silu_product_backward: grad_gu [rows, 2 * inner] contiguous from grad_y [rows, inner]; with p = 1 / (1 + exp(-gate))
 *   grad_gate = grad_y * up * p * (1 + gate * (1 - p)), grad_up = grad_y * gate * p
 * In both, a sigmoid below 2^-126 (a gate below -87.3) may be taken as 0.
 * grad_gu may take the place of a contiguous gu.
 * GG_ERR_UNSUPPORTED unless inner % 8 == 0, inner <= 32768, strides % 8 == 0 and 16-byte aligned buffers (int8 y: 8-byte).
 */
int gg_silu_product(int dtype, int out_dtype, int64_t rows, int64_t inner, const void *gu, int64_t gu_stride, void *y,
                    float *scale, void *stream);
int gg_silu_product_backward(int dtype, int64_t rows, int64_t inner, const void *grad_y, int64_t grad_y_stride,
                             const void *gu, int64_t gu_stride, void *grad_gu, void *stream);

/* y [rows, n] int8 contiguous, overlapping no input, and scale [rows] of the rows of x (bf16 or fp16), as gg_rms_norm's int8
 * rows. Rules as above for n. */
int gg_quantize_rows(int dtype, int64_t rows, int64_t n, const void *x, int64_t x_stride, int8_t *y, float *scale, void *stream);

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
 * dispatch_scaled: the same, and xs_scale[rows[t, s]] = scale[t] (float32) for rows that have a scale each; 0 for the zeroed rows.
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
int gg_dispatch_scaled(int elem_size, int64_t tokens, int top_k, int64_t hidden, int experts, const void *x, int64_t stride,
                       const float *scale, const int *rows, const int64_t *offs, void *xs, float *xs_scale, void *stream);
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

/* ---- grouped products in 8-bit integers ---- */

/*
 * out[rows of g] = x[rows of g] @ w[g]^T * scales: out[m, n] = sum_k x[m, k] w[g, n, k] * w_scale[g, n] * x_scale[m]
 * for x [total_m, k] and w [group_num, n, k] int8 (-128 .. 127), x_scale [total_m] and w_scale [group_num, n] float32,
 * out [total_m, n] of out_dtype (bf16 or fp16), all contiguous. The sums are int32 and exact; each is made a float32,
 * multiplied by w_scale and then by x_scale, and rounded to out_dtype once. Any number of rows a group, one to very many.
 * group_lens / group_offs: device sizes as in gg_prepare_device_lens_op; a group whose rows are not inside
 * [0, total_m) gets no work (and is not reported); rows of out that belong to no group are not written.
 * workspace: gg_gemm_i8_workspace(group_num) bytes, 16-byte aligned, not shared by calls that may overlap.
 * (The first call on a device looks up that device's properties, and so must run outside stream capture.)
 * GG_ERR_UNSUPPORTED unless n % 8 == 0, k % 16 == 0, x, w, w_scale and out 16-byte aligned, n at most 2097152, k below
 * 131072 (past it a sum may leave int32), group_num at most 8192 and total_m at most 134217728.
 */
size_t gg_gemm_i8_workspace(int group_num);
int gg_gemm_i8(int out_dtype, int group_num, int64_t total_m, int64_t n, int64_t k, const int64_t *group_lens,
               const int64_t *group_offs, const int8_t *x, const int8_t *w, const float *x_scale, const float *w_scale,
               void *out, void *workspace, size_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* GG_MOE_LAYER_H */
