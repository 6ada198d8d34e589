// The C ABI's refusal of an eviction over its own inputs (csrc/host/kv_plan.cpp),
// built by tests/test_kv_in_place.py with g++ and AddressSanitizer +
// UndefinedBehaviorSanitizer (no recovery).
#include <stdint.h>
#include <stdio.h>
#include <string.h>

#include "kv_plan.h"

using namespace fgqa;

static void* fake(uintptr_t n) { return reinterpret_cast<void*>(0x100000 + (n << 24)); }

int main() {
    int failed = 0;
    for (int which = 0; which < 4; ++which) {
        fgqa_kv_evict_args e;
        memset(&e, 0, sizeof e);
        e.cache.k = fake(1);
        e.cache.v = fake(2);
        e.cache.kv_dtype = FGQA_KV_BF16;
        e.cache.num_kv_heads = 8;
        e.cache.head_dim = 128;
        e.cache.page_size = 16;
        e.cache.num_pages = 40;
        const int64_t st[3] = {16 * 8 * 128, 8 * 128, 128};
        for (int i = 0; i < 3; ++i) e.cache.k_stride[i] = e.cache.v_stride[i] = st[i];
        e.weights = static_cast<float*>(fake(12));
        e.new_weights = static_cast<float*>(fake(13));
        e.weights_stride[0] = e.new_weights_stride[0] = 8 * 160;
        e.weights_stride[1] = e.new_weights_stride[1] = 160;
        e.block_table = static_cast<int32_t*>(fake(7));
        e.new_block_table = static_cast<int32_t*>(fake(14));
        e.block_table_stride = 10;
        e.new_block_table_stride = 4;
        e.seqlens = static_cast<int32_t*>(fake(8));
        e.new_seqlens = static_cast<int32_t*>(fake(15));
        e.kept = static_cast<int32_t*>(fake(16));
        e.batch = 3;
        e.max_seqlen = e.weights_len = 160;
        e.budget = 64;
        if (which == 1) e.new_weights = const_cast<float*>(e.weights);
        if (which == 2) e.new_seqlens = const_cast<int32_t*>(e.seqlens);
        if (which == 3) e.kept = e.new_seqlens;
        const int want = which == 0 ? FGQA_OK : FGQA_ERR_INVALID_ARGUMENT;
        if (plan::validate_kv_evict(&e) != want) {
            ++failed;
            fprintf(stderr, "call %d: %d\n", which, plan::validate_kv_evict(&e));
        }
    }
    printf("4 checks, %d failed\n", failed);
    return failed != 0;
}
