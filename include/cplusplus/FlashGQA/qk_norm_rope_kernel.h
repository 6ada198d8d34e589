// Queries and keys normalised for each head and rotated to their positions: C++ operator
// entry points (MI355X / gfx950).
//
// No reference counterpart.  include/fgqa_rope.h states what they compute.
#pragma once

#include <cstdint>

#include "Utils/utils.h"

/** What the forward and the backward pass share. */
struct QkNormRope {
    const int32_t* positions = nullptr;   // device [numAxes, batchSize, seqLength]
    const float* invFreq = nullptr;       // device [rotaryDim / 2]
    const int32_t* axes = nullptr;        // device [rotaryDim / 2], or null: all of axis 0
    const bf16_t* qWeight = nullptr;      // device [headDim], both or neither
    const bf16_t* kWeight = nullptr;
    float eps = 1e-6f;
    int numAxes = 1;
    int batchSize = 0;
    int seqLength = 0;
    int numQueryHeads = 0;
    int numKvHeads = 0;
    int headDim = 128;
    int rotaryDim = 128;
    bool interleaved = false;
};

// Both launch on the default stream, return nothing, and report through
// FlashGqaGetLastStatus(); nothing is launched when it is not 0.

/**
 * @brief Norm and rotation (fgqa_qk_norm_rope).
 * @param q, qOut Device bf16 [batchSize, seqLength, numQueryHeads, headDim]; may be the same.
 * @param k, kOut Device bf16 [batchSize, seqLength, numKvHeads, headDim]; may be the same.
 */
void LaunchQkNormRopeBf16Kernel(const QkNormRope& how, const bf16_t* q, const bf16_t* k, bf16_t* qOut, bf16_t* kOut);

/**
 * @brief Its gradients (fgqa_qk_norm_rope_backward), in the library's device buffer: calls that may run at the
 *        same time take the C ABI with a workspace each.
 * @param q, k The forward pass's inputs (not used without weights).
 * @param gradQOut, gradKOut The outputs' gradients; gradQ, gradK the inputs'.
 * @param gradQWeight, gradKWeight Device fp32 [headDim], or null without weights.
 */
void LaunchQkNormRopeBackwardBf16Kernel(const QkNormRope& how, const bf16_t* q, const bf16_t* k, const bf16_t* gradQOut,
                                        const bf16_t* gradKOut, bf16_t* gradQ, bf16_t* gradK, float* gradQWeight,
                                        float* gradKWeight);
