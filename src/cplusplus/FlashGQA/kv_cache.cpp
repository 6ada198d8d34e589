// C++ operator entry points of the paged KV cache, implemented over the C ABI
// (include/fgqa_kv.h).  Host-only C++: no HIP types or calls in this file.
#include <climits>
#include <cstdint>

#include "FlashGQA/kv_cache_kernel.h"
#include "fgqa_kv.h"

namespace fgqa_cpp {
void set_last_status(int status);   // flash_gqa.cpp
}

namespace {
constexpr int kHeadDim = 128;

// pageSize * numKvHeads * 128 stays inside 64 bits for any ints.
fgqa_kv_cache as_c(const KvCache& c) {
    fgqa_kv_cache r = {};
    r.k = c.k;
    r.v = c.v;
    r.k_scales = c.kScales;
    r.v_scales = c.vScales;
    r.kv_dtype = static_cast<int32_t>(c.type);
    r.num_kv_heads = c.numKvHeads;
    r.head_dim = kHeadDim;
    r.page_size = c.pageSize;
    r.num_pages = c.numPages;
    r.k_scale = c.kScale;
    r.v_scale = c.vScale;
    int64_t page = 0;
    const int64_t slot = (int64_t)c.numKvHeads * kHeadDim;
    if (__builtin_mul_overflow((int64_t)c.pageSize, slot, &page)) page = INT64_MAX;   // refused as too far
    const int64_t st[3] = {page, slot, kHeadDim};
    for (int i = 0; i < 3; ++i) r.k_stride[i] = r.v_stride[i] = st[i];
    r.k_scales_stride[0] = r.v_scales_stride[0] = c.numKvHeads;
    r.k_scales_stride[1] = r.v_scales_stride[1] = 1;
    return r;
}

// Tokens of a block table row; false (and the status) when the C ABI's int cannot hold them.
bool max_tokens(const KvCache& c, int pages, int32_t* tokens) {
    const int64_t n = pages > 0 && c.pageSize > 0 ? (int64_t)pages * c.pageSize : 0;
    if (n > INT_MAX) {
        fgqa_cpp::set_last_status(FGQA_ERR_UNSUPPORTED);
        return false;
    }
    *tokens = static_cast<int32_t>(n);
    return true;
}
}  // namespace

void LaunchKvCacheAppendKernel(const KvCache& cache, const bf16_t* k, const bf16_t* v, const int32_t* blockTable,
                               const int32_t* seqLengths, const int32_t* newLengths, int batchSize, int maxNew,
                               int maxPagesPerSeq) {
    fgqa_kv_append_args a = {};
    a.cache = as_c(cache);
    a.k_new = k;
    a.v_new = v;
    int64_t row = 0;
    const int64_t token = (int64_t)cache.numKvHeads * kHeadDim;
    if (__builtin_mul_overflow((int64_t)maxNew, token, &row)) row = INT64_MAX;
    const int64_t st[3] = {row, token, kHeadDim};
    for (int i = 0; i < 3; ++i) a.k_new_stride[i] = a.v_new_stride[i] = st[i];
    a.block_table = blockTable;
    a.block_table_stride = maxPagesPerSeq;
    a.seqlens = seqLengths;
    a.new_lens = newLengths;
    a.batch = batchSize;
    a.max_new = maxNew;
    a.max_pages = maxPagesPerSeq;
    fgqa_cpp::set_last_status(fgqa_kv_append(&a, nullptr));
}

void LaunchFlashGqaBf16KernelPagedBlocks(const KvCache& cache, const bf16_t* q, float scale, bf16_t* o, float* lse,
                                         const int32_t* blockTable, const int32_t* seqLengths, int batchSize,
                                         int maxPagesPerSeq, int numQueryHeads) {
    fgqa_decode_blocks_args a = {};
    a.cache = as_c(cache);
    a.q = q;
    a.o = o;
    a.lse = lse;
    a.block_table = blockTable;
    a.seqlens = seqLengths;
    a.batch = batchSize;
    if (!max_tokens(cache, maxPagesPerSeq, &a.max_seqlen)) return;
    a.num_q_heads = numQueryHeads;
    a.scale = scale;
    a.q_stride[0] = a.o_stride[0] = (int64_t)numQueryHeads * kHeadDim;
    a.q_stride[1] = a.o_stride[1] = kHeadDim;
    a.block_table_stride = maxPagesPerSeq;
    fgqa_cpp::set_last_status(fgqa_decode_blocks(&a, nullptr));
}

void LaunchKvCacheWeightsKernel(const KvCache& cache, const bf16_t* q, float scale, const float* lse, float* weights,
                                const int32_t* blockTable, const int32_t* seqLengths, int batchSize,
                                int maxPagesPerSeq, int numQueryHeads) {
    fgqa_kv_weights_args a = {};
    a.cache = as_c(cache);
    a.q = q;
    a.lse = lse;
    a.weights = weights;
    a.q_stride[0] = (int64_t)numQueryHeads * kHeadDim;
    a.q_stride[1] = kHeadDim;
    if (!max_tokens(cache, maxPagesPerSeq, &a.max_seqlen)) return;
    a.weights_stride[0] = (int64_t)cache.numKvHeads * a.max_seqlen;
    a.weights_stride[1] = a.max_seqlen;
    a.block_table = blockTable;
    a.block_table_stride = maxPagesPerSeq;
    a.seqlens = seqLengths;
    a.batch = batchSize;
    a.num_q_heads = numQueryHeads;
    a.scale = scale;
    fgqa_cpp::set_last_status(fgqa_kv_weights(&a, nullptr));
}

void LaunchKvCacheEvictKernel(const KvCache& cache, const float* weights, float* newWeights, const int32_t* blockTable,
                              const int32_t* newBlockTable, const int32_t* seqLengths, int32_t* newSeqLengths,
                              int32_t* kept, int budget, int recent, int batchSize, int maxPagesPerSeq,
                              int maxNewPagesPerSeq) {
    fgqa_kv_evict_args a = {};
    a.cache = as_c(cache);
    a.weights = weights;
    a.new_weights = newWeights;
    if (!max_tokens(cache, maxPagesPerSeq, &a.max_seqlen)) return;
    a.weights_len = a.max_seqlen;
    a.weights_stride[0] = a.new_weights_stride[0] = (int64_t)cache.numKvHeads * a.max_seqlen;
    a.weights_stride[1] = a.new_weights_stride[1] = a.max_seqlen;
    a.block_table = blockTable;
    a.new_block_table = newBlockTable;
    a.block_table_stride = maxPagesPerSeq;
    a.new_block_table_stride = maxNewPagesPerSeq;
    a.seqlens = seqLengths;
    a.new_seqlens = newSeqLengths;
    a.kept = kept;
    a.batch = batchSize;
    a.budget = budget;
    a.recent = recent;
    fgqa_cpp::set_last_status(fgqa_kv_evict(&a, nullptr));
}
