/*
 * fgqa_rope.h -- C ABI of what comes before attention in libfgqa.so: queries and
 * keys normalised for each head and rotated to their positions, in one pass, and
 * the gradients of that.  Conventions and status codes are fgqa.h's, but for the
 * head dims.
 *
 * No counterpart in the reference (its rotation is an operator of its own, its
 * norms are those of whole rows).
 */
#ifndef FGQA_ROPE_H
#define FGQA_ROPE_H

#include "fgqa.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * For each row x of head_dim elements (a token's query or key of one head):
 *   y = x * w / sqrt(mean(x^2) + eps)         (y = x where the weights are NULL)
 * and, with theta_j = positions[axes[j]][b][s] * inv_freq[j], j < rotary_dim / 2,
 *   (y_a, y_b) -> (y_a cos theta_j - y_b sin theta_j, y_b cos theta_j + y_a sin theta_j)
 * of elements (a, b) = (j, j + rotary_dim / 2), or (2j, 2j + 1) where interleaved;
 * elements from rotary_dim on are not rotated.
 *
 *   q, k           bf16 [B, S, H, D], strides {b, s, h}
 *   q_out, k_out   the same shapes, strides of their own.  Either may be its input
 *                  (same address and strides); all else lies apart.
 *   positions      int32 or (positions_int64) int64 [num_axes, B, S], any strides
 *                  of 0 or more {axis, b, s}
 *   inv_freq       fp32 [rotary_dim / 2], radians
 *   axes           int32 [rotary_dim / 2], the axis of each pair, clamped to
 *                  [0, num_axes) (nullable: all of axis 0)
 *   q_weight, k_weight   [D], bf16 or (weights_bf16 0) fp32; both or neither
 *   head_dim       a multiple of 16 up to 256; rotary_dim one of 0 .. head_dim
 *
 * Angles are formed in 64 bits and reduced to a turn before they are rounded, all
 * else is fp32, with one rounding to bf16 at the end.  Squares are summed in fp32:
 * elements beyond 2^60 overflow.
 */
typedef struct fgqa_rope_args {
    const void* q;
    const void* k;
    void* q_out;
    void* k_out;
    const void* positions;
    const float* inv_freq;
    const int32_t* axes;
    const void* q_weight;
    const void* k_weight;
    int32_t positions_int64;
    int32_t weights_bf16;
    int32_t num_axes;
    int32_t batch;
    int32_t seqlen;
    int32_t num_q_heads;
    int32_t num_kv_heads;
    int32_t head_dim;
    int32_t rotary_dim;
    int32_t interleaved;
    float eps;
    int64_t q_stride[3];
    int64_t k_stride[3];
    int64_t q_out_stride[3];
    int64_t k_out_stride[3];
    int64_t positions_stride[3];
} fgqa_rope_args;

int fgqa_qk_norm_rope(const fgqa_rope_args* args, void* stream);

/*
 * Its gradients: from those of q_out and k_out, those of q, k and the weights.
 *
 *   fwd             the forward call's arguments (q_out and k_out are not used, nor
 *                   q and k without weights)
 *   grad_q_out, grad_k_out   bf16, as q and k
 *   grad_q, grad_k           bf16, as q and k; either may be its grad_*_out
 *                            (same address and strides); all else lies apart
 *   grad_q_weight, grad_k_weight   fp32 [D], the sums over all rows (NULL without
 *                            weights); zeros where there is no row
 *   workspace       256-byte aligned, at least
 *                   fgqa_qk_norm_rope_backward_workspace_bytes (0 without weights);
 *                   NULL and 0: the library's buffer, as for the backward of the prefill
 * No atomics: the same bits from run to run on one kind of device.
 */
typedef struct fgqa_rope_backward_args {
    fgqa_rope_args fwd;
    const void* grad_q_out;
    const void* grad_k_out;
    void* grad_q;
    void* grad_k;
    float* grad_q_weight;
    float* grad_k_weight;
    int64_t grad_q_out_stride[3];
    int64_t grad_k_out_stride[3];
    int64_t grad_q_stride[3];
    int64_t grad_k_stride[3];
    void* workspace;
    size_t workspace_bytes;
} fgqa_rope_backward_args;

int fgqa_qk_norm_rope_backward_workspace_bytes(const fgqa_rope_backward_args* args, size_t* bytes);

int fgqa_qk_norm_rope_backward(const fgqa_rope_backward_args* args, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* FGQA_ROPE_H */
