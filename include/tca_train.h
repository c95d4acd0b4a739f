/*
 * tca_train.h -- C ABI of the operators beside the sparse product in a
 * training step (libtcaspmm.so, gfx950): layer norm with its backward pass,
 * softmax cross entropy with its gradient, and an AdamW step over many
 * tensors at once.  No counterpart in the reference, which is forward-only.
 *
 * Conventions of tca_spmm.h: int status (TCA_OK == 0), tca_last_error(),
 * pointers named d_* are DEVICE pointers, calls are stream-ordered on `stream`
 * (a hipStream_t, NULL = default stream), do not synchronise and allocate
 * nothing: what a call needs beside its outputs is a workspace that the
 * caller gives it, of the size the matching *_workspace function names (no
 * contents are expected in it, and it may be reused once the call's work has
 * run).  Types are TCA_F16, TCA_F32 or TCA_BF16; sums and statistics are held
 * in fp32 and each output is rounded once.  Results do not depend on the
 * schedule: no atomics, sums in a fixed order.  Tensors need their element's
 * alignment only; outputs overlap no input but where a call updates in place.
 */
#ifndef TCA_TRAIN_H
#define TCA_TRAIN_H

#include "tca_spmm.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- layer norm over the last axis ----
 * y[i, c] = (x[i, c] - mean_i) * rstd_i * w[c] + b[c],
 * rstd_i = 1 / sqrt(mean_c((x[i, c] - mean_i)^2) + eps).
 * x is rows x width with `x_pitch` elements between rows (0 repeats one row),
 * y is dense.  x_dtype any type; y_dtype equal to it, or any type for fp32 x.
 * d_w and d_b (each may be NULL: ones / zeros) have w_dtype, which is x_dtype,
 * y_dtype or fp32.  d_stats: NULL, or [rows][2] fp32 {mean, rstd} for the
 * backward pass.  0 <= rows, 1 <= width <= TCA_LAYER_NORM_MAX_WIDTH. */
#define TCA_LAYER_NORM_MAX_WIDTH 16384
int tca_layer_norm(const void* d_x, int64_t rows, int32_t width, int64_t x_pitch, int32_t x_dtype, const void* d_w,
                   const void* d_b, int32_t w_dtype, float eps, void* d_y, int32_t y_dtype, float* d_stats,
                   void* stream);

/* Gradients of tca_layer_norm: with xh = (x - mean) rstd and g = dy w,
 *   dx = rstd (g - mean_c(g) - xh mean_c(g xh))   (x_dtype, dense)
 *   dw[c] = sum_i dy xh,  db[c] = sum_i dy        (w_dtype)
 * d_dy is rows x width of y_dtype with `dy_pitch` elements between rows.  Each
 * of d_dx, d_dw and d_db may be NULL; with rows == 0 the written ones of dw
 * and db are zeros. */
int tca_layer_norm_backward_workspace(int64_t rows, int32_t width, size_t* bytes);
int tca_layer_norm_backward(const void* d_dy, int64_t dy_pitch, int32_t y_dtype, const void* d_x, int64_t x_pitch,
                            int32_t x_dtype, int64_t rows, int32_t width, const void* d_w, int32_t w_dtype,
                            const float* d_stats, void* d_dx, void* d_dw, void* d_db, void* d_workspace,
                            size_t workspace_bytes, void* stream);

/* ---- softmax cross entropy ----
 * Row i of logits x (rows x classes, `pitch` elements between rows) with
 * target t_i: loss_i = log(sum_c exp(x[i, c] - m_i)) - (x[i, t_i] - m_i),
 * m_i = max_c x[i, c].  A row whose target is ignore_index counts for nothing:
 * its logits are not read, its loss and its gradient are 0.  A target outside
 * [0, classes) that is not ignore_index gives NaN in the loss and in its
 * row's gradient.  Logits of -inf take no part; a row of nothing else has no
 * distribution and gives NaN.
 * rows and pitch are below 2^31, classes at most 2^30.
 * reduction: TCA_LOSS_NONE (d_loss [rows]), TCA_LOSS_SUM or TCA_LOSS_MEAN
 * (d_loss [1]; the mean is over the rows that count, and 0 over none). */
#define TCA_LOSS_NONE 0
#define TCA_LOSS_SUM 1
#define TCA_LOSS_MEAN 2

/* The loss.  d_targets: int64 (target_bytes 8) or int32 (4).  For the backward
 * pass d_stats [rows][2] fp32 receives {m_i, sum_i} of the rows that count, and
 * d_norm [1] fp32 receives 1 / count for the mean, 1 otherwise; each may be
 * NULL. */
int tca_cross_entropy_workspace(int64_t rows, int32_t classes, size_t* bytes);
int tca_cross_entropy(const void* d_logits, int64_t rows, int32_t classes, int64_t pitch, int32_t dtype,
                      const void* d_targets, int32_t target_bytes, int64_t ignore_index, int32_t reduction,
                      float* d_loss, float* d_stats, float* d_norm, void* d_workspace, size_t workspace_bytes,
                      void* stream);

/* d_dlogits (rows x classes, dense, the logits' type) =
 *   (exp(x - m_i) / sum_i - [c == t_i]) * d_gloss[i * gloss_stride] * d_norm[0]
 * from what tca_cross_entropy left in d_stats and d_norm (NULL: 1); d_gloss is the fp32
 * gradient of the loss (gloss_stride 0: one value for all rows). */
int tca_cross_entropy_backward(const float* d_gloss, int64_t gloss_stride, const void* d_logits, int64_t rows,
                               int32_t classes, int64_t pitch, int32_t dtype, const void* d_targets,
                               int32_t target_bytes, int64_t ignore_index, const float* d_stats, const float* d_norm,
                               void* d_dlogits, void* stream);

/* The loss (not multiplied by `scale`) and its gradient times `scale` in one
 * pass over the logits; reduction TCA_LOSS_SUM or TCA_LOSS_MEAN. */
int tca_cross_entropy_grad(const void* d_logits, int64_t rows, int32_t classes, int64_t pitch, int32_t dtype,
                           const void* d_targets, int32_t target_bytes, int64_t ignore_index, int32_t reduction,
                           float scale, float* d_loss, void* d_dlogits, void* d_workspace, size_t workspace_bytes,
                           void* stream);

/* ---- AdamW over many tensors ----
 * Per element, in fp32 and in this order, each operation rounded:
 *   m = m b1 + g (1 - b1);  v = v b2 + (g g) (1 - b2)
 *   p = p keep - m / (sqrt(v) correct + eps) rate
 * keep = 1 - lr weight_decay, rate = lr / (1 - b1^step),
 * correct = 1 / sqrt(1 - b2^step), 1 - b1 and 1 - b2 computed in fp64.
 *
 * state_bits 32: m and v are fp32 [n].  state_bits 8: m and r = sqrt(v) are
 * e4m3 (OCP) codes in blocks of TCA_ADAMW_BLOCK values, the last one padded
 * (codes [blocks * TCA_ADAMW_BLOCK], scales fp32 [blocks]); a value is code *
 * scale.  A block's scale is its largest finite |value| * (1 / 448), or 0 (with
 * codes 0) if that maximum is below 2^-100; a code is value * (1 / scale)
 * rounded to nearest even, NaN for what is not finite, and for r > 0 at least
 * 2^-9, the least code above zero.  p is updated from m and r before they are
 * rounded.
 *
 * param_dtype TCA_F32: p is the parameter, master is NULL.  TCA_F16 / TCA_BF16:
 * p is read from `master` (fp32), written there, and rounded to the parameter. */
#define TCA_ADAMW_BLOCK 256
typedef struct tca_adamw_tensor {
    void* param;        /* [n] param_dtype */
    const void* grad;   /* [n] param_dtype */
    float* master;      /* [n] */
    void* m;            /* fp32 [n], or codes */
    void* v;            /* fp32 [n], or codes of r */
    float* m_scale;     /* state_bits 8 */
    float* v_scale;     /* state_bits 8 */
    int64_t n;
} tca_adamw_tensor;

/* One step over `count` tensors (a HOST array, copied into the launches).  They are
 * worked on side by side: no two share memory (TCA_ERR_INVALID if parameters do). */
int tca_adamw_step(const tca_adamw_tensor* tensors, int32_t count, int32_t param_dtype, int32_t state_bits,
                   int64_t step, double lr, double beta1, double beta2, double eps, double weight_decay,
                   void* stream);

/* The same with the step counts on the device, so that the call can be captured
 * into a graph: d_steps is a HOST array of `count` DEVICE pointers, an int64 of its
 * own for each tensor, which the call raises by one and then uses (1 for the first
 * step).  d_factors: 2 * count floats of workspace.  pow() is the device's, in
 * fp64: rate and correct can differ from the host's by their rounding to fp32. */
int tca_adamw_step_device(const tca_adamw_tensor* tensors, int64_t* const* d_steps, int32_t count, int32_t param_dtype,
                          int32_t state_bits, double lr, double beta1, double beta2, double eps, double weight_decay,
                          float* d_factors, void* stream);

#ifdef __cplusplus
} /* extern "C" */
#endif

#endif /* TCA_TRAIN_H */
