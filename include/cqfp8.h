/*
 * cqfp8.h - C ABI of the B200 8-bit floating-point linear.
 *
 *   y = act(x^ . w^T + b)
 *
 * w: e4m3 codes [output_dims, input_dims] with one f32 scale for each
 * 128 x 128 block (the last blocks may be short): the weight is scale * code.
 * x^: each row of x in e4m3 with one scale for each 128 values, brought there
 * by the call: the scale is the least power of two that brings the largest
 * finite magnitude of the 128 to 448 or less (1 where all are zero, never
 * below 2^-126), and a code is the e4m3 value nearest to x / scale, halves to
 * even.  Dividing by a power of two is exact, so a row's codes do not depend on
 * how they were computed.  Infinities and NaN of x become NaN codes, which make
 * that row of y NaN and no other.  Sums, scales, bias and activation are f32;
 * y is rounded to T once.
 *
 * Next to the affine INT8 linear of cqlinear.h it takes as many bytes for its
 * weights and runs batched calls at the tensor cores' 8-bit rate.  No
 * counterpart in the reference.
 *
 * Conventions (status codes, cq_last_error, one thread per handle, void*
 * streams) are those of cqlinear.h.  No call here allocates device memory
 * except the creation of a layer: scratch is the caller's workspace, used only
 * by work on the call's own stream, so calls of one layer on several streams
 * are independent when each has its own workspace.
 */
#ifndef CQFP8_H
#define CQFP8_H

#include "cqlinear.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct cq_fp8_linear cq_fp8_linear;

/*
 * A layer from e4m3 codes [output_dims, input_dims] and f32 scales
 * [ceil(output_dims / 128), ceil(input_dims / 128)], both row-major without
 * gaps, in host or device memory; the layer owns copies.  bias_or_null: T
 * [output_dims].  dtype T (CQ_F16 or CQ_BF16) is the type of x, y and bias.
 */
cq_status cq_fp8_linear_create(const uint8_t *codes, const float *scales, const void *bias_or_null,
                               int32_t output_dims, int32_t input_dims, cq_dtype dtype,
                               int32_t device, cq_fp8_linear **out);

/*
 * A layer from an f32 weight [output_dims, input_dims] and an f32 bias
 * [output_dims] or NULL (rounded to T), in host or device memory: the weight
 * is brought to codes as cq_fp8_quantize_weight does.
 */
cq_status cq_fp8_linear_create_from_f32(const float *weight, const float *bias_or_null,
                                        int32_t output_dims, int32_t input_dims, cq_dtype dtype,
                                        int32_t device, cq_fp8_linear **out);

/* Bytes of workspace that a forward call on `rows` rows needs (it grows with
 * rows, and is 0 for none); SIZE_MAX for a NULL layer or rows < 0. */
size_t cq_fp8_linear_workspace(const cq_fp8_linear *layer, int32_t rows);

/*
 * y[rows, output_dims] = act(x^ . w^T + b): x and y device T with row strides
 * ldx >= input_dims and ldy >= output_dims (elements), of any alignment that T
 * has.  workspace: device memory of at least cq_fp8_linear_workspace(layer,
 * rows) bytes, 256-byte aligned.  Asynchronous on `stream`; can be captured.
 */
cq_status cq_fp8_linear_forward(cq_fp8_linear *layer, const void *x, int64_t ldx, int32_t rows,
                                void *y, int64_t ldy, cq_act act, void *workspace,
                                size_t workspace_bytes, void *stream);

/*
 * forward on rows already in e4m3 (cq_fp8_quantize_rows), for several layers
 * that share an input: codes [rows, ld], 16-byte aligned rows (ld a multiple
 * of 16), scales f32 [ceil(input_dims / 128), rows].  Same results as forward
 * on the rows that the codes came from.  No workspace.
 */
cq_status cq_fp8_linear_forward_codes(cq_fp8_linear *layer, const uint8_t *codes, int64_t ld,
                                      const float *scales, int32_t rows, void *y, int64_t ldy,
                                      cq_act act, void *stream);

int32_t cq_fp8_linear_input_dims(const cq_fp8_linear *layer);
int32_t cq_fp8_linear_output_dims(const cq_fp8_linear *layer);

/* Frees the layer.  NULL is a no-op. */
void cq_fp8_linear_destroy(cq_fp8_linear *layer);

/*
 * Device rows x [rows, cols] of T (CQ_F16, CQ_BF16 or CQ_F32), row stride ldx,
 * to e4m3: codes [rows, ld], 16-byte aligned rows (ld >= cols, a multiple of
 * 16; columns from cols on, up to the next multiple of 128 or ld, are set to
 * zero) and scales f32 [ceil(cols / 128), rows].  Asynchronous on `stream`.
 */
cq_status cq_fp8_quantize_rows(const void *x, int64_t ldx, int32_t rows, int32_t cols,
                               cq_dtype dtype, uint8_t *codes, int64_t ld, float *scales,
                               void *stream);

/*
 * Device f32 weight [rows, cols] to e4m3 codes [rows, cols] and f32 scales
 * [ceil(rows / 128), ceil(cols / 128)] by the same rule over 128 x 128 blocks.
 * Asynchronous on `stream`.
 */
cq_status cq_fp8_quantize_weight(const float *w, int32_t rows, int32_t cols, uint8_t *codes,
                                 float *scales, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* CQFP8_H */
