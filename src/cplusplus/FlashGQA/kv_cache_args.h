// A KvCache as the C ABI takes it, for the C++ operator entry points.
#pragma once

#include <climits>
#include <cstdint>

#include "FlashGQA/kv_cache_kernel.h"
#include "fgqa_kv.h"

namespace fgqa_cpp {

void set_last_status(int status);   // flash_gqa.cpp

constexpr int kHeadDim = 128;

// pageSize * numKvHeads * 128 stays inside 64 bits for any ints.
inline fgqa_kv_cache as_c(const KvCache& c) {
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
inline bool max_tokens(const KvCache& c, int pages, int32_t* tokens) {
    const int64_t n = pages > 0 && c.pageSize > 0 ? (int64_t)pages * c.pageSize : 0;
    if (n > INT_MAX) {
        set_last_status(FGQA_ERR_UNSUPPORTED);
        return false;
    }
    *tokens = static_cast<int32_t>(n);
    return true;
}

}  // namespace fgqa_cpp
