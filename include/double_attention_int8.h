/*
 * C ABI of the 8-bit operators of the blocks' feed-forward: the linear layer
 * on 8-bit integers, the root-mean-square norm with the residual's addition,
 * and activations kept in 8 bits for the backward pass.  No counterpart in the
 * reference.  The conventions are those of double_attention_hip.h: device
 * pointers, element counts, the caller's stream, buffers and workspace,
 * nothing allocated, freed or synchronized, arguments checked before anything
 * is enqueued, 0 or a DA_ERR_* code returned (da_last_error has the message).
 */
#ifndef DOUBLE_ATTENTION_INT8_H
#define DOUBLE_ATTENTION_INT8_H

#include "double_attention_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Rows in 8 bits.  A row of `cols` numbers is kept as signed integers with an
 * fp32 scale for the whole row (group 0) or for each 128 columns of it (group
 * 128, DA_INT8_GROUP; the last group may be shorter):
 *   scale = max(amax, 127 * 2^-126) / 127,  q = rint(x / scale) in [-127, 127]
 * with fp32's division and ties to even; scale is amax times fp32's 1 / 127
 * (da_add_rms_norm multiplies by rstd / scale instead: where n / scale is within
 * fp32's roundings of a half, its q may be either neighbour).
 * A row (group) that holds an infinity or a NaN gets the scale NaN and zeros:
 * all of it then stands for NaN.  values: [rows] rows at a pitch ldv that is a
 * multiple of 16 (>= cols), 16-byte aligned; the bytes of a row's last chunk
 * of 16 behind cols are storage that these calls may write and never use.
 * scales: [rows] or [rows][ceil(cols / 128)] fp32, contiguous.
 *
 * The 16-bit (and fp32) tensors of these operators are rows of any width at
 * any pitch >= that width, aligned to their elements.  No call reads or writes
 * outside of the rows it is given.  No output may overlap an input or another
 * output, values, scales, parameters and the workspace among them: such calls
 * are refused (DA_ERR_INVALID_ARGUMENT).  Rows of one pitch may lie in each
 * other's gaps, and a contiguous tensor in one gap; rows of two pitches whose
 * ranges meet count as overlapping.  A launch takes fewer than 2^32 threads, 16
 * for each group of a row, or 64, 256 or 1024 for a row held whole (up to 1024,
 * 8192 and more columns); calls with more rows are refused (DA_ERR_UNSUPPORTED).
 */
#define DA_INT8_GROUP 128
#define DA_I8 3 /* dtype code of 8-bit rows with one scale each */

/* values, scales = int8(x); x of any dtype.  group 0: cols <= 65536. */
int da_quantize_int8(const void* x, int64_t rows, int64_t cols, int64_t ldx, int dtype, int64_t group, void* values,
                     int64_t ldv, float* scales, da_stream_t stream);

/* out [rows, cols] (pitch ldo, any dtype) = values * scale, rounded once. */
int da_dequantize_int8(const void* values, int64_t rows, int64_t cols, int64_t ldv, const float* scales, int64_t group,
                       void* out, int64_t ldo, int out_dtype, da_stream_t stream);

/*
 * The linear layer on 8-bit rows, one scale per token and per output channel:
 *   out[t, f] = act(x_scales[t] w_scales[f] sum_k x[t, k] weight[f, k] + bias[f]),
 * the sum in 32-bit integers (exact), the rest in fp32, rounded to dtype
 * (DA_F16 or DA_BF16), then + residual (NULL or [rows, out_features] of dtype
 * at pitch ldr; added to the rounded result and rounded again, as the unfused
 * `x + linear(...)` does).  x: [rows, in_features] at pitch ldx, of x_dtype
 * DA_I8 with x_scales, or 16-bit rows (x_scales is not read) that are quantized
 * as by da_quantize_int8, where they are multiplied or into the workspace
 * (16-byte aligned, as many bytes as da_linear_int8_workspace_bytes returns;
 * with 0 it may be NULL).  weight: [out_features, in_features] at pitch ldw.
 * 8-bit rows may hold any integers, -128 too; the bytes behind in_features are
 * not used.  in_features <= 65536, pitches of 8-bit rows at most 2^23.  out:
 * contiguous [rows, out_features].
 */
int64_t da_linear_int8_workspace_bytes(int64_t rows, int64_t in_features, int64_t out_features, int x_dtype, int dtype);
int da_linear_int8(const void* x, int x_dtype, int64_t ldx, const float* x_scales, int64_t rows, int64_t in_features,
                   const void* weight, int64_t ldw, const float* w_scales, int64_t out_features, const void* bias,
                   int bias_dtype, int activation, const void* residual, int64_t ldr, void* out, int dtype,
                   void* workspace, int64_t workspace_bytes, da_stream_t stream);

/*
 * Root-mean-square norm with the residual's addition in front of it:
 *   s = x + residual (rounded to dtype; residual NULL: s is x),
 *   n = s / sqrt(mean(s^2) + eps) * weight   over the last dimension, in fp32,
 * (rows whose squares exceed fp32, |s| above about 1e19, have none),
 * n as out (rounded to dtype), as 8-bit rows with one scale each (values, ldv,
 * scales), or as both (out or values may be NULL, not both).  sum receives s
 * ([rows, dim] contiguous; required with a residual, not written without).
 * x, residual: [rows, dim] of dtype (DA_F16 or DA_BF16) at pitches ldx, ldr;
 * weight: [dim] of param_dtype, or NULL (1).  dim <= 16384, eps > 0.
 */
int da_add_rms_norm(const void* x, int64_t ldx, const void* residual, int64_t ldr, int64_t rows, int64_t dim,
                    const void* weight, int param_dtype, float eps, int dtype, void* sum, void* out, void* values,
                    int64_t ldv, float* scales, da_stream_t stream);

/*
 * Its backward at grad = dL/dn and grad_sum = dL/ds (NULL: 0), with
 * xh = s rstd and g = grad weight:
 *   grad_x = rstd (g - xh mean(g xh)) + grad_sum   (dL/dx and dL/dresidual; rounded once)
 *   grad_weight = sum over the rows of grad xh     (fp32, in an order that the sizes fix;
 *                                                   rounded once to param_dtype)
 * sum, grad, grad_sum: [rows, dim] of dtype at pitches ldsum, ldg, ldgs;
 * grad_x contiguous.  grad_weight: [dim] or NULL; with it, the workspace
 * (16-byte aligned) holds the bytes that
 * da_add_rms_norm_backward_workspace_bytes returns.
 */
int64_t da_add_rms_norm_backward_workspace_bytes(int64_t rows, int64_t dim);
int da_add_rms_norm_backward(const void* sum, int64_t ldsum, const void* grad, int64_t ldg, const void* grad_sum,
                             int64_t ldgs, int64_t rows, int64_t dim, const void* weight, int param_dtype, float eps,
                             int dtype, void* grad_x, void* grad_weight, void* workspace, int64_t workspace_bytes,
                             da_stream_t stream);

/*
 * GELU (exact, as DA_ACT_GELU) that keeps its input in 8 bits for the backward:
 *   out = gelu(z) of the z given (rounded once to dtype), values, scales = int8(z) in groups of 128.
 * Backward at grad = dL/dout, from the kept zt = q scale:
 *   grad_z = grad gelu'(zt),  out = gelu(zt) (NULL: not formed; the operand of the next layer's
 *   weight gradient).  z, grad: [rows, cols] of dtype (DA_F16 or DA_BF16) at pitches ldz, ldg;
 *   out and grad_z contiguous.
 */
int da_gelu_int8(const void* z, int64_t rows, int64_t cols, int64_t ldz, int dtype, void* out, void* values,
                 int64_t ldv, float* scales, da_stream_t stream);
int da_gelu_int8_backward(const void* values, int64_t rows, int64_t cols, int64_t ldv, const float* scales,
                          const void* grad, int64_t ldg, int dtype, void* grad_z, void* out, da_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* DOUBLE_ATTENTION_INT8_H */
