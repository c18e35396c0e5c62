/*
 * cqexperts.h - C ABI of the B200 linears of experts: a router, the experts'
 * products, and the sum of what they made, for a feed-forward module whose
 * weights are several experts' of which each token meets a few.
 *
 *   cq_route            token -> its `top` best experts, their weights, and the
 *                       order of (token, expert) pairs by expert
 *   cq_expert_linear    y[r] = act(W[e] x[r] + b[e]) for rows sorted by expert
 *   cq_expert_combine   y[t] = sum_j weight[t, j] z[position[t, j]]
 *   cq_expert_ffn       the four steps of a feed-forward module in one call
 *
 * No counterpart in the reference, whose feed-forward modules are dense
 * (crates/nemotron-mlx/src/model/encoder.rs:300-336).
 *
 * Conventions are those of cqlinear.h and cqfp8.h: status codes, one thread
 * per handle, device pointers, asynchronous on `stream`, scratch in a
 * caller's workspace (256-byte aligned), no device allocation outside of
 * creation.  What a call reads on the device (offsets, tokens, positions) is
 * checked there against its array's bounds: a bad value gives wrong rows, not
 * a wrong access.
 */
#ifndef CQEXPERTS_H
#define CQEXPERTS_H

#include "cqlinear.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct cq_expert_linear cq_expert_linear;

/* How an expert linear holds its weights. */
typedef int32_t cq_weight_format;
enum {
    CQ_WEIGHT_T = 0,   /* 16-bit values of the layer's type T */
    CQ_WEIGHT_E4M3 = 1 /* e4m3 codes with an f32 scale for each 128 x 128 block (cqfp8.h) */
};

/*
 * Weights [experts, output_dims, input_dims] (T or e4m3 codes), for e4m3 also
 * f32 scales [experts, ceil(output_dims / 128), ceil(input_dims / 128)] (else
 * NULL), bias_or_null T [experts, output_dims]; row-major without gaps, host or
 * device memory; the layer owns copies.  1 <= experts <= 1024.
 */
cq_status cq_expert_linear_create(const void *weight, const float *scales, const void *bias_or_null,
                                  int32_t experts, int32_t output_dims, int32_t input_dims,
                                  cq_weight_format format, cq_dtype dtype, int32_t device,
                                  cq_expert_linear **out);

/* Bytes of workspace that a forward call on `rows` rows needs; SIZE_MAX for a
 * NULL layer or rows < 0. */
size_t cq_expert_linear_workspace(const cq_expert_linear *layer, int32_t rows);

/*
 * Rows [offsets[e], offsets[e + 1]) of x meet expert e: y = act(x W[e]^T +
 * b[e]), x and y T with row strides ldx and ldy of any alignment.  offsets:
 * device int32 [experts + 1], rising from 0 to at most `rows`; a group may be
 * empty.  Rows from offsets[experts] on are set to zero.  With e4m3 weights x
 * is brought to e4m3 by the call, as cq_fp8_linear_forward does.  Sums, bias
 * and activation are f32; y is rounded to T once.
 */
cq_status cq_expert_linear_forward(cq_expert_linear *layer, const void *x, int64_t ldx,
                                   int32_t rows, const int32_t *offsets, void *y, int64_t ldy,
                                   cq_act act, void *workspace, size_t workspace_bytes,
                                   void *stream);

int32_t cq_expert_linear_experts(const cq_expert_linear *layer);
int32_t cq_expert_linear_input_dims(const cq_expert_linear *layer);
int32_t cq_expert_linear_output_dims(const cq_expert_linear *layer);

/* Frees the layer.  NULL is a no-op. */
void cq_expert_linear_destroy(cq_expert_linear *layer);

/* Bytes of workspace of cq_route; SIZE_MAX for sizes that it refuses. */
size_t cq_route_workspace(int32_t tokens, int32_t experts, int32_t top);

/*
 * logits [tokens, experts] of CQ_F32, CQ_F16 or CQ_BF16, row stride ld.
 * For each token the `top` experts with the largest logits, largest first, the
 * lower expert first where equal; one whose logit is -infinity or NaN is never
 * taken.  1 <= top <= min(experts, 32), experts <= 1024.
 *   expert   int32 [tokens, top]; -1 where fewer than `top` could be taken
 *   weight   f32 [tokens, top]: softmax of the logits over the experts taken
 *            (renormalize != 0) or over all that could be (0); 0 where none
 *   offsets  int32 [experts + 1]: the rows of expert e, once pairs are sorted
 *            by expert and within one by token, are [offsets[e], offsets[e+1])
 *   token    int32 [tokens * top]: the token of each sorted row, -1 past
 *            offsets[experts]
 *   position int32 [tokens, top]: the sorted row of each pair, -1 where expert is
 */
cq_status cq_route(const void *logits, int64_t ld, cq_dtype dtype, int32_t tokens, int32_t experts,
                   int32_t top, int32_t renormalize, int32_t *expert, float *weight,
                   int32_t *offsets, int32_t *token, int32_t *position, void *workspace,
                   size_t workspace_bytes, void *stream);

/*
 * y[t] = sum over j of weight[t, j] * z[position[t, j]] in f32, rounded to T
 * once: z T [rows, dims] with row stride ldz, position int32 and weight f32
 * [tokens, top]; a position outside [0, rows) adds nothing.
 */
cq_status cq_expert_combine(const void *z, int64_t ldz, int32_t rows, const int32_t *position,
                            const float *weight, int32_t tokens, int32_t top, int32_t dims,
                            cq_dtype dtype, void *y, int64_t ldy, void *stream);

/* Bytes of workspace of cq_expert_ffn_forward; SIZE_MAX where it refuses. */
size_t cq_expert_ffn_workspace(const cq_expert_linear *up, const cq_expert_linear *down,
                               int32_t tokens, int32_t top);

/*
 * A feed-forward module of experts: route by logits (as cq_route), h =
 * act(up(x)), z = down(h), y = combine(z).  up and down agree in experts,
 * format, dtype and device; down's input is up's output and y has down's width.
 * x T [tokens, ldx], logits of logits_dtype [tokens, ld_logits], y T [tokens,
 * ldy]; y is zero for a token without an expert.  With e4m3 weights h goes
 * from f32 to e4m3 at once; with 16-bit weights it is the sum of two values of
 * T, which keeps twice T's fraction (and T's range).  z stays in f32.
 */
cq_status cq_expert_ffn_forward(cq_expert_linear *up, cq_expert_linear *down, const void *x,
                                int64_t ldx, int32_t tokens, const void *logits, int64_t ld_logits,
                                cq_dtype logits_dtype, int32_t top, int32_t renormalize, cq_act act,
                                void *y, int64_t ldy, void *workspace, size_t workspace_bytes,
                                void *stream);

#ifdef __cplusplus
}
#endif

#endif /* CQEXPERTS_H */
