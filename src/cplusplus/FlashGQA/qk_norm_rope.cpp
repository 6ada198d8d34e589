// C++ operator entry points of the norm and rotation of queries and keys, implemented over
// the C ABI (include/fgqa_rope.h).  Host-only C++: no HIP types or calls in this file.
#include "FlashGQA/qk_norm_rope_kernel.h"

#include <cstdint>

#include "fgqa_rope.h"

namespace fgqa_cpp {
void set_last_status(int status);   // flash_gqa.cpp
}

namespace {
// Strides {b, s, h} of contiguous rows; too far ones are refused by the C ABI.
void contiguous(const QkNormRope& how, int heads, int64_t (&st)[3]) {
    st[2] = how.headDim;
    st[1] = (int64_t)heads * how.headDim;
    if (__builtin_mul_overflow((int64_t)how.seqLength, st[1], &st[0])) st[0] = INT64_MAX;
}

fgqa_rope_args as_c(const QkNormRope& how) {
    fgqa_rope_args a = {};
    a.positions = how.positions;
    a.inv_freq = how.invFreq;
    a.axes = how.axes;
    a.q_weight = how.qWeight;
    a.k_weight = how.kWeight;
    a.weights_bf16 = 1;
    a.num_axes = how.numAxes;
    a.batch = how.batchSize;
    a.seqlen = how.seqLength;
    a.num_q_heads = how.numQueryHeads;
    a.num_kv_heads = how.numKvHeads;
    a.head_dim = how.headDim;
    a.rotary_dim = how.rotaryDim;
    a.interleaved = how.interleaved ? 1 : 0;
    a.eps = how.eps;
    contiguous(how, how.numQueryHeads, a.q_stride);
    contiguous(how, how.numQueryHeads, a.q_out_stride);
    contiguous(how, how.numKvHeads, a.k_stride);
    contiguous(how, how.numKvHeads, a.k_out_stride);
    a.positions_stride[0] = (int64_t)how.batchSize * how.seqLength;
    a.positions_stride[1] = how.seqLength;
    a.positions_stride[2] = 1;
    return a;
}
}  // namespace

void LaunchQkNormRopeBf16Kernel(const QkNormRope& how, const bf16_t* q, const bf16_t* k, bf16_t* qOut, bf16_t* kOut) {
    fgqa_rope_args a = as_c(how);
    a.q = q;
    a.k = k;
    a.q_out = qOut;
    a.k_out = kOut;
    fgqa_cpp::set_last_status(fgqa_qk_norm_rope(&a, nullptr));
}

void LaunchQkNormRopeBackwardBf16Kernel(const QkNormRope& how, const bf16_t* q, const bf16_t* k, const bf16_t* gradQOut,
                                        const bf16_t* gradKOut, bf16_t* gradQ, bf16_t* gradK, float* gradQWeight,
                                        float* gradKWeight) {
    fgqa_rope_backward_args a = {};
    a.fwd = as_c(how);
    a.fwd.q = q;
    a.fwd.k = k;
    a.grad_q_out = gradQOut;
    a.grad_k_out = gradKOut;
    a.grad_q = gradQ;
    a.grad_k = gradK;
    a.grad_q_weight = gradQWeight;
    a.grad_k_weight = gradKWeight;
    contiguous(how, how.numQueryHeads, a.grad_q_out_stride);
    contiguous(how, how.numQueryHeads, a.grad_q_stride);
    contiguous(how, how.numKvHeads, a.grad_k_out_stride);
    contiguous(how, how.numKvHeads, a.grad_k_stride);
    fgqa_cpp::set_last_status(fgqa_qk_norm_rope_backward(&a, nullptr));
}
