// The eviction's max_tokens and new_tokens in the C ABI's validation
// (csrc/host/kv_plan.cpp), built by tests/test_kv_evict_tokens.py with g++ and
// AddressSanitizer + UndefinedBehaviorSanitizer (no recovery).
#include <limits.h>
#include <stdint.h>
#include <stdio.h>
#include <string.h>

#include "kv_plan.h"

using namespace fgqa;

static long g_checks = 0, g_failed = 0;

static void* fake(uintptr_t n) { return reinterpret_cast<void*>(0x100000 + (n << 24)); }

static fgqa_kv_evict_args args() {
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
    e.weights_stride[0] = e.new_weights_stride[0] = 8 * 100;
    e.weights_stride[1] = e.new_weights_stride[1] = 100;
    e.block_table = static_cast<int32_t*>(fake(7));
    e.new_block_table = static_cast<int32_t*>(fake(14));
    e.block_table_stride = 10;       // 160 tokens
    e.new_block_table_stride = 8;    // 128 tokens
    e.seqlens = static_cast<int32_t*>(fake(8));
    e.new_seqlens = static_cast<int32_t*>(fake(15));
    e.kept = static_cast<int32_t*>(fake(16));
    e.batch = 3;
    e.max_seqlen = e.weights_len = 100;
    e.budget = 128;
    return e;
}

#define EVICT(change, status)                                                              \
    do {                                                                                   \
        fgqa_kv_evict_args e = args();                                                     \
        change;                                                                            \
        ++g_checks;                                                                        \
        if (plan::validate_kv_evict(&e) != (status)) {                                     \
            ++g_failed;                                                                    \
            fprintf(stderr, "%s:%d: %s\n", __FILE__, __LINE__, #change);                   \
        }                                                                                  \
    } while (0)

int main() {
    const int OK = FGQA_OK, BAD = FGQA_ERR_INVALID_ARGUMENT, NOT = FGQA_ERR_UNSUPPORTED;
    EVICT((void)e, OK);
    EVICT(e.max_tokens = 160, OK);
    EVICT(e.max_tokens = 161, BAD);                        // past the block table's row
    EVICT(e.max_tokens = -1, BAD);
    EVICT(e.new_tokens = -1, BAD);
    EVICT(e.max_tokens = 99, OK);                          // below max_seqlen: max_seqlen
    EVICT(e.max_tokens = 160; e.budget = 129, BAD);        // past the new table's row
    EVICT(e.max_tokens = 160; e.budget = 129; e.new_tokens = 128, OK);
    EVICT(e.max_tokens = 160; e.budget = 129; e.new_tokens = 129, BAD);
    EVICT(e.budget = 129, OK);                             // no sequence is that long
    EVICT(e.max_tokens = INT_MAX; e.block_table_stride = INT_MAX, NOT);
    EVICT(e.max_seqlen = e.weights_len = 0; e.weights = e.new_weights = nullptr; e.max_tokens = 160, OK);
    EVICT(e.max_seqlen = 0; e.weights = nullptr; e.max_tokens = 160; e.block_table = nullptr, BAD);
    fgqa_kv_evict_args e = args();
    e.max_tokens = 160;
    ++g_checks;
    if (plan::evict_tokens(e) != 160 || plan::evict_most(e) != 128) ++g_failed;
    e.max_tokens = 3;
    e.new_tokens = 50;
    ++g_checks;
    if (plan::evict_tokens(e) != 100 || plan::evict_most(e) != 50) ++g_failed;
    printf("%ld checks, %ld failed\n", g_checks, g_failed);
    return g_failed != 0;
}
