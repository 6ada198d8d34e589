// A paged KV cache as the kernels take it (host side).
#pragma once

#include "fgqa_kv.h"
#include "../host/kv_plan.h"

namespace fgqa {

// Index 0 is K, 1 is V; strides in bytes (the scales' in elements).
struct CacheParams {
    unsigned char* data[2];
    float* scales[2];      // or null
    float scale[2];        // of the whole cache, without block scales
    int64_t page[2], slot[2], head[2];
    int64_t scale_page[2], scale_head[2];
    int hkv, page_shift, num_pages;
};

inline CacheParams cache_params(const fgqa_kv_cache& c) {
    CacheParams p;
    const int elem = c.kv_dtype == FGQA_KV_BF16 ? 2 : 1;
    const int64_t* st[2] = {c.k_stride, c.v_stride};
    const int64_t* sc[2] = {c.k_scales_stride, c.v_scales_stride};
    void* data[2] = {c.k, c.v};
    float* scales[2] = {c.k_scales, c.v_scales};
    for (int i = 0; i < 2; ++i) {
        p.data[i] = static_cast<unsigned char*>(data[i]);
        p.scales[i] = scales[i];
        p.page[i] = st[i][0] * elem;
        p.slot[i] = st[i][1] * elem;
        p.head[i] = st[i][2] * elem;
        p.scale_page[i] = sc[i][0];
        p.scale_head[i] = sc[i][1];
    }
    p.scale[0] = c.k_scale;
    p.scale[1] = c.v_scale;
    p.hkv = c.num_kv_heads;
    p.page_shift = plan::log2_of(c.page_size);
    p.num_pages = c.num_pages;
    return p;
}

}  // namespace fgqa
