// C++ operator entry points of sequences that share pages, implemented over the C ABI
// (include/fgqa_pages.h).  Host-only C++: no HIP types or calls in this file.
#include "FlashGQA/kv_pages_kernel.h"
#include "fgqa_pages.h"
#include "kv_cache_args.h"

using namespace fgqa_cpp;

void LaunchKvCacheForkKernel(const KvCache& cache, const int32_t* blockTable, const int32_t* seqLengths,
                             const int32_t* parents, const int32_t* newLengths, const uint8_t* held,
                             int32_t* newBlockTable, int32_t* newSeqLengths, int32_t* numFree, int batchSize,
                             int maxPagesPerSeq, int newBatchSize, int maxNewPagesPerSeq) {
    fgqa_kv_fork_args a = {};
    a.cache = as_c(cache);
    a.block_table = blockTable;
    a.seqlens = seqLengths;
    a.parents = parents;
    a.new_lens = newLengths;
    a.held = held;
    a.new_block_table = newBlockTable;
    a.new_seqlens = newSeqLengths;
    a.num_free = numFree;
    a.block_table_stride = maxPagesPerSeq;
    a.new_block_table_stride = maxNewPagesPerSeq;
    a.batch = batchSize;
    a.max_pages = maxPagesPerSeq;
    a.new_batch = newBatchSize;
    a.new_max_pages = maxNewPagesPerSeq;
    set_last_status(fgqa_kv_fork(&a, nullptr));
}

void LaunchKvCacheCompactKernel(const KvCache& cache, const int32_t* blockTable, const int32_t* seqLengths,
                                const uint8_t* held, int32_t* newBlockTable, int32_t* numUsed, int batchSize,
                                int maxPagesPerSeq) {
    fgqa_kv_compact_args a = {};
    a.cache = as_c(cache);
    a.block_table = blockTable;
    a.seqlens = seqLengths;
    a.held = held;
    a.new_block_table = newBlockTable;
    a.num_used = numUsed;
    a.block_table_stride = a.new_block_table_stride = maxPagesPerSeq;
    a.batch = batchSize;
    a.max_pages = maxPagesPerSeq;
    set_last_status(fgqa_kv_compact(&a, nullptr));
}

void LaunchFlashGqaBf16KernelPagedShared(const KvCache& cache, const bf16_t* q, float scale, bf16_t* o, float* lse,
                                         const int32_t* blockTable, const int32_t* seqLengths,
                                         const int32_t* groupStarts, const int32_t* sharedLengths, int batchSize,
                                         int maxPagesPerSeq, int numQueryHeads, int numGroups) {
    fgqa_decode_shared_args a = {};
    a.cache = as_c(cache);
    a.q = q;
    a.o = o;
    a.lse = lse;
    a.block_table = blockTable;
    a.seqlens = seqLengths;
    a.group_starts = groupStarts;
    a.shared_lens = sharedLengths;
    a.batch = batchSize;
    if (!max_tokens(cache, maxPagesPerSeq, &a.max_seqlen)) return;
    a.num_q_heads = numQueryHeads;
    a.num_groups = numGroups;
    a.scale = scale;
    a.q_stride[0] = a.o_stride[0] = (int64_t)numQueryHeads * kHeadDim;
    a.q_stride[1] = a.o_stride[1] = kHeadDim;
    a.block_table_stride = maxPagesPerSeq;
    set_last_status(fgqa_decode_shared(&a, nullptr));
}
