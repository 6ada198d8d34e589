// Paged KV cache: C++ operator entry points (MI355X / gfx950).
//
// No reference counterpart: the cache that LaunchFlashGqaBf16KernelPaged reads,
// written, read with a scale for each block of 8-bit codes, and cut to a budget.
// include/fgqa_kv.h states what each operator computes.
#pragma once

#include <cstdint>

#include "Utils/utils.h"

/** Element type of a paged cache. */
enum class KvCacheType { Bf16 = 0, Fp8E4m3 = 1, Int8 = 2 };

/**
 * @brief A contiguous paged cache on the device.
 *
 * k, v: [numPages, pageSize, numKvHeads, 128] of `type`, 16-byte aligned.
 * kScales, vScales: fp32 [numPages, numKvHeads], the scale of each block (page
 * and KV head) of 8-bit codes; required for Int8, null for Bf16.  An Fp8E4m3
 * cache without them has kScale and vScale for all of it.  K's and V's data and
 * scales lie apart where a call writes them.
 */
struct KvCache {
    void* k = nullptr;
    void* v = nullptr;
    float* kScales = nullptr;
    float* vScales = nullptr;
    KvCacheType type = KvCacheType::Bf16;
    int numPages = 0;
    int pageSize = 0;
    int numKvHeads = 0;
    float kScale = 1.f;
    float vScale = 1.f;
};

// All of these launch on the default stream, return nothing, and report
// through FlashGqaGetLastStatus(); nothing is launched when it is not 0.

/**
 * @brief Writes new tokens to the cache (fgqa_kv_append).
 * @param k, v Device bf16 [batchSize, maxNew, numKvHeads, 128].
 * @param blockTable Device int32 [batchSize, maxPagesPerSeq].
 * @param seqLengths Device int32 [batchSize]: tokens each sequence holds already.
 * @param newLengths Device int32 [batchSize]: new tokens of each, or null: maxNew.
 */
void LaunchKvCacheAppendKernel(const KvCache& cache, const bf16_t* k, const bf16_t* v, const int32_t* blockTable,
                               const int32_t* seqLengths, const int32_t* newLengths, int batchSize, int maxNew,
                               int maxPagesPerSeq);

/**
 * @brief LaunchFlashGqaBf16KernelPaged over a cache with block scales
 *        (fgqa_decode_blocks), with the LSE.
 * @param q, o Device bf16 [batchSize, numQueryHeads, 128].
 * @param lse Device fp32 [batchSize, numQueryHeads] (natural log), or null.
 */
void LaunchFlashGqaBf16KernelPagedBlocks(const KvCache& cache, const bf16_t* q, float scale, bf16_t* o, float* lse,
                                         const int32_t* blockTable, const int32_t* seqLengths, int batchSize,
                                         int maxPagesPerSeq, int numQueryHeads);

/**
 * @brief Adds to each cached token's weight what a decode step gave it (fgqa_kv_weights).
 * @param lse The step's, as the decode wrote it.
 * @param weights Device fp32 [batchSize, numKvHeads, maxPagesPerSeq * pageSize].
 */
void LaunchKvCacheWeightsKernel(const KvCache& cache, const bf16_t* q, float scale, const float* lse, float* weights,
                                const int32_t* blockTable, const int32_t* seqLengths, int batchSize,
                                int maxPagesPerSeq, int numQueryHeads);

/**
 * @brief Cuts each sequence to `budget` tokens and moves them to new pages (fgqa_kv_evict).
 * @param weights, newWeights Device fp32 [batchSize, numKvHeads, maxPagesPerSeq * pageSize], apart.
 * @param newBlockTable Device int32 [batchSize, maxNewPagesPerSeq].
 * @param newSeqLengths Device int32 [batchSize].
 * @param kept Device int32 [batchSize, numKvHeads, budget].
 */
void LaunchKvCacheEvictKernel(const KvCache& cache, const float* weights, float* newWeights, const int32_t* blockTable,
                              const int32_t* newBlockTable, const int32_t* seqLengths, int32_t* newSeqLengths,
                              int32_t* kept, int budget, int recent, int batchSize, int maxPagesPerSeq,
                              int maxNewPagesPerSeq);
