/*
 * b200train -- C ABI of the steps of a fine-tuning step that lie between the attention and expert kernels
 * (b200attn.h, b200moe.h) and the optimizer: the residual sum with its RMS norm, the global gradient norm with
 * clipping, and the clipped SGD update.  Part of libb200attn.so.
 *
 * The reference project leaves them to Hugging Face (GptOssRMSNorm.forward and the two sums of
 * GptOssDecoderLayer.forward, transformers/models/gpt_oss/modeling_gpt_oss.py:48-63, :357-386) and to its launcher
 * (gradient clipping at 1.0, configs/zero3.yaml:6).
 *
 * Conventions as in b200attn.h: device pointers unless said otherwise, no allocation, no synchronisation, calls only
 * enqueue work on `stream` of `device`; 0 on success or a negative B200ATTN_E* code (b200attn_strerror explains it).
 */
#ifndef B200TRAIN_H_
#define B200TRAIN_H_

#include <stddef.h>
#include <stdint.h>

#include "b200attn.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types. */
enum { B200TRAIN_BF16 = 0, B200TRAIN_FP16 = 1, B200TRAIN_FP32 = 2 };

enum { B200TRAIN_EOVERLAP = -10 }; /* two tensors of one call, one of which is written, share memory */

#define B200TRAIN_NORM_MAX_COLS 16384 /* widest row of the norm */

/*
 * h[t,:] = round(x[t,:] + residual[t,:]);  y[t,c] = round(weight[c] * h[t,c] * rsqrt(mean_c(h[t,c]^2) + eps)).
 * The sum is rounded to the element type first (it is the residual stream), the norm is taken of the rounded row in
 * fp32 and rounded once.  residual == NULL: h is x itself, and `h` must be NULL too.
 *   x, residual   (rows x cols), element type `dtype`, element strides x_stride / residual_stride between rows
 *   weight        (cols), element type `weight_dtype`: `dtype` or B200TRAIN_FP32
 *   y, h          (rows x cols) contiguous, fully overwritten; neither may overlap an input
 * Base pointers 16-byte aligned.  Where cols is a multiple of 16 bytes' worth of elements, the strides must be too;
 * otherwise the inputs must be contiguous (stride == cols).  rows >= 0, eps >= 0, 1 <= cols <= B200TRAIN_NORM_MAX_COLS, and
 * 8 elements less (4 of fp32) where cols is no multiple of 16 bytes' worth.
 */
int b200train_add_rms_norm(const void* x, int64_t x_stride, const void* residual, int64_t residual_stride,
                           const void* weight, void* y, void* h, int64_t rows, int32_t cols, float eps, int32_t dtype,
                           int32_t weight_dtype, int32_t device, void* stream);

/* fp32 values of scratch that b200train_add_rms_norm_bwd needs to make dweight (0 where it needs none). */
int64_t b200train_norm_scratch_floats(int64_t rows, int32_t cols, int32_t dtype, int32_t device);

/*
 * The gradients of the above: with n = h * rstd, g = dy * weight,
 *   dx[t,:] = dh[t,:] + rstd * (g - n * mean_c(g * n))      (the gradient of x and of residual alike)
 *   dweight[c] = sum_t dy[t,c] * n[t,c]                     (fp32, in an order fixed by the sizes)
 * rstd is taken from h again.  dh may be NULL (no gradient arrives through h); dweight may be NULL (not wanted; scratch
 * is then not used).  dx (rows x cols) contiguous, dweight (cols) of `weight_dtype`, both fully overwritten.
 * Alignment and strides as above, for dy, dh and h.
 */
int b200train_add_rms_norm_bwd(const void* dy, int64_t dy_stride, const void* dh, int64_t dh_stride, const void* h,
                               int64_t h_stride, const void* weight, void* dx, void* dweight, float* scratch,
                               int64_t scratch_floats, int64_t rows, int32_t cols, float eps, int32_t dtype,
                               int32_t weight_dtype, int32_t device, void* stream);

/*
 * The global norm of many tensors, clipping by it, and the SGD update with the clip folded in.
 *   grads, params, counts, dtypes   HOST arrays of `tensors` entries, read during the call: device addresses (element
 *                                   aligned), elements (>= 0), element types.  A tensor's elements are contiguous; no two
 *                                   tensors of a call that writes may overlap (B200TRAIN_EOVERLAP).
 *   scratch                         device fp64, b200train_clip_scratch_doubles(...) of them
 *   norm                            out, device fp32: n = sqrt(sum of g^2 over all tensors).  Squares are fp32, their sums
 *                                   fp32 within 16 bytes of a tensor and fp64 beyond (n is right to 2.5 * 2^-24): an element
 *                                   above 1.8e19, or a few of 16 bytes near it, makes n infinite.
 * c = min(1, max_norm / (n + 1e-6)), max_norm >= 0; a NaN norm makes c NaN, an infinite one 0; max_norm = inf is no limit, c = 1.
 * No value is read by the host.
 */
int64_t b200train_clip_scratch_doubles(int64_t tensors, int32_t device);

/* norm only. */
int b200train_grad_norm(const int64_t* grads, const int64_t* counts, const int32_t* dtypes, int64_t tensors, double* scratch,
                        int64_t scratch_doubles, float* norm, int32_t device, void* stream);

/* g <- round(c * g); nothing is written where c = 1.  torch.nn.utils.clip_grad_norm_ as one pass each way. */
int b200train_clip_grads(const int64_t* grads, const int64_t* counts, const int32_t* dtypes, int64_t tensors, float max_norm,
                         double* scratch, int64_t scratch_doubles, float* norm, int32_t device, void* stream);

/* p <- round(p - lr * c * g), rounded once; the gradients are left as they are.  A parameter has its gradient's type. */
int b200train_clipped_sgd(const int64_t* grads, const int64_t* params, const int64_t* counts, const int32_t* dtypes, int64_t tensors,
                          float lr, float max_norm, double* scratch, int64_t scratch_doubles, float* norm, int32_t device, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* B200TRAIN_H_ */
