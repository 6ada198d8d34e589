// Sequences that share pages of a paged KV cache: C++ operator entry points (MI355X / gfx950).
//
// No reference counterpart.  include/fgqa_pages.h states what each operator computes.
#pragma once

#include <cstdint>

#include "FlashGQA/kv_cache_kernel.h"

// All of these launch on the default stream, return nothing, and report
// through FlashGqaGetLastStatus(); nothing is launched when it is not 0.  They use
// the library's device buffer: calls that may run at the same time take the C ABI with a workspace each.

/**
 * @brief Sequences that go on from others and share their pages, with pages for new tokens (fgqa_kv_fork).
 * @param blockTable Device int32 [batchSize, maxPagesPerSeq].
 * @param seqLengths Device int32 [batchSize].
 * @param parents Device int32 [newBatchSize]: the row each new one goes on from, -1: none; or null: row i from row i.
 * @param newLengths Device int32 [newBatchSize]: tokens to have pages for, or null: 0.
 * @param held Device uint8 [numPages]: pages in use elsewhere, or null.
 * @param newBlockTable Device int32 [newBatchSize, maxNewPagesPerSeq].
 * @param newSeqLengths Device int32 [newBatchSize].
 * @param numFree Device int32 [1]: free pages that are left; below 0: missing.
 */
void LaunchKvCacheForkKernel(const KvCache& cache, const int32_t* blockTable, const int32_t* seqLengths,
                             const int32_t* parents, const int32_t* newLengths, const uint8_t* held,
                             int32_t* newBlockTable, int32_t* newSeqLengths, int32_t* numFree, int batchSize,
                             int maxPagesPerSeq, int newBatchSize, int maxNewPagesPerSeq);

/**
 * @brief Moves the pages in use to the lowest page numbers (fgqa_kv_compact).
 * @param newBlockTable Device int32 [batchSize, maxPagesPerSeq].
 * @param numUsed Device int32 [1]: all pages from there on are free.
 */
void LaunchKvCacheCompactKernel(const KvCache& cache, const int32_t* blockTable, const int32_t* seqLengths,
                                const uint8_t* held, int32_t* newBlockTable, int32_t* numUsed, int batchSize,
                                int maxPagesPerSeq);

/**
 * @brief Single-token attention for sequences that begin alike (fgqa_decode_shared), over any cache.
 * @param q, o Device bf16 [batchSize, numQueryHeads, 128].
 * @param lse Device fp32 [batchSize, numQueryHeads] (natural log), or null.
 * @param groupStarts Device int32 [numGroups + 1], ascending.
 * @param sharedLengths Device int32 [numGroups]: tokens that a group's sequences have in common.
 */
void LaunchFlashGqaBf16KernelPagedShared(const KvCache& cache, const bf16_t* q, float scale, bf16_t* o, float* lse,
                                         const int32_t* blockTable, const int32_t* seqLengths,
                                         const int32_t* groupStarts, const int32_t* sharedLengths, int batchSize,
                                         int maxPagesPerSeq, int numQueryHeads, int numGroups);
