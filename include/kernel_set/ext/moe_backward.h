/*
 * Gradients of the routed layer's steps of kernel_set/moe.h: the gate, the way
 * of the tokens to the experts and the way back with the routing weights.
 *
 * The reference's C ABI has the forward steps only (include/kernel_set/moe.h),
 * so these entry points have no counterpart there. They neither synchronise
 * nor allocate beyond the stream's scratch named below.
 */
#ifndef KERNEL_SET_EXT_MOE_BACKWARD_H_
#define KERNEL_SET_EXT_MOE_BACKWARD_H_

#include "kernel_set/types.h"

KS_BEGIN_EXTERN_C

/*
 * Gradient of ks_moe_gate_softmax_topk with respect to the logits.
 *   d_logits   [num_tokens, num_experts]  `dtype` (f32 / f16 / bf16), written whole
 *   d_weights, weights  [num_tokens, top_k]  fp32; the weights that the gate gave
 *   indices    [num_tokens, top_k]  int32, the experts that it gave; a slot whose id
 *              is out of range takes no part, one that is named twice counts twice
 *   logits     [num_tokens, num_experts]  `dtype`; read without renormalisation only,
 *              may be NULL otherwise
 * With s = sum_k weights_k d_weights_k:
 *   renormalised      d_logits_e = sum over slots k of e: weights_k (d_weights_k - s)
 *   not renormalised  d_logits_e = -softmax(logits)_e s + sum over slots k of e: weights_k d_weights_k
 * At most 1024 experts and top_k 32, as the gate. fp32 inside, one rounding.
 * d_logits may be logits.
 */
KS_API ks_status_t ks_moe_gate_softmax_topk_backward(
    void* d_logits, const float* d_weights, const float* weights,
    const int32_t* indices, const void* logits, int64_t num_tokens,
    int num_experts, int top_k, int renormalize, ks_dtype_t dtype,
    ks_stream_t stream);

/*
 * Gradient of ks_moe_permute: d_input[t, :] = sum of the rows of d_permuted that
 * are token t's, in slot order, in fp32, rounded once; zeros for a token without rows.
 *   d_input [num_tokens, hidden], d_permuted [num_tokens*top_k, hidden], f32 / f16 / bf16
 *   sorted_token_ids [num_tokens*top_k] int32; a pair may occur once, rows with
 *   an id out of range are not read.
 * In all but small calls the inverse permutation lives in the stream's scratch, which
 * this call shares with ks_moe_unpermute (the same rules under stream capture).
 */
KS_API ks_status_t ks_moe_permute_backward(void* d_input,
                                           const void* d_permuted,
                                           const int32_t* sorted_token_ids,
                                           int64_t num_tokens, int top_k,
                                           int64_t hidden, ks_dtype_t dtype,
                                           ks_stream_t stream);

/*
 * Gradient of ks_moe_unpermute. For row r of pair (t, k):
 *   d_permuted[r, :] = routing_weights[t, k] * d_out[t, :], rounded once
 *   d_weights[t, k]  = <d_out[t, :], permuted[r, :]> in fp32
 * Rows whose id is out of range become zeros, and so do the weights' gradients of
 * pairs without a row.
 *   d_permuted, permuted [num_tokens*top_k, hidden], d_out [num_tokens, hidden],
 *   f32 / f16 / bf16; d_weights, routing_weights [num_tokens, top_k] fp32
 * A pair may occur once in sorted_token_ids. d_permuted may be permuted. One launch,
 * no scratch.
 */
KS_API ks_status_t ks_moe_unpermute_backward(
    void* d_permuted, float* d_weights, const void* d_out,
    const void* permuted, const int32_t* sorted_token_ids,
    const float* routing_weights, int64_t num_tokens, int top_k,
    int64_t hidden, ks_dtype_t dtype, ks_stream_t stream);

KS_END_EXTERN_C

#endif /* KERNEL_SET_EXT_MOE_BACKWARD_H_ */
