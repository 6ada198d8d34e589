// csrc/host/kv_apart.h against every pair of elements, and the C ABI's refusal of
// one address for K and V (csrc/host/kv_plan.cpp), built by tests/test_kv_apart.py
// with g++ and AddressSanitizer + UndefinedBehaviorSanitizer (no recovery).
//
// Output: one line per failed check, then "N checks, M failed"; exit status 1
// when a check failed.
#include <stdint.h>
#include <stdio.h>
#include <string.h>

#include <random>
#include <vector>

#include "kv_apart.h"
#include "kv_plan.h"

using namespace fgqa;

static long g_checks = 0, g_failed = 0;

#define CHECK(cond)                                                                 \
    do {                                                                            \
        ++g_checks;                                                                 \
        if (!(cond)) {                                                              \
            ++g_failed;                                                             \
            if (g_failed < 50) fprintf(stderr, "%s:%d: %s\n", __FILE__, __LINE__, #cond); \
        }                                                                           \
    } while (0)

static bool by_elements(int64_t a, int64_t b, const int64_t* n, const int64_t* s, int k, int64_t elem) {
    std::vector<int64_t> off(1, 0);
    for (int i = 0; i < k; ++i) {
        std::vector<int64_t> next;
        for (int64_t o : off)
            for (int64_t x = 0; x < n[i]; ++x) next.push_back(o + x * s[i] * elem);
        off = next;
    }
    for (int64_t x : off)
        for (int64_t y : off) {
            const int64_t d = (b + y) - (a + x);
            if (d < elem && d > -elem) return true;
        }
    return false;
}

static void test_views() {
    std::mt19937 r(3);
    for (int t = 0; t < 20000; ++t) {
        const int k = 1 + (int)(r() % 4);
        int64_t n[4], s[4], span = 1;
        for (int i = 0; i < k; ++i) {   // nested strides, with gaps
            n[i] = 1 + (int64_t)(r() % 4);
            s[i] = span + (int64_t)(r() % 3 ? 0 : r() % 9);
            if (n[i] > 1) span = s[i] * (n[i] - 1) + span;
            else if (r() % 2) s[i] = (int64_t)(r() % 100);   // of no account
        }
        for (int i = k - 1; i > 0; --i) {   // in any order
            const int j = (int)(r() % (unsigned)(i + 1));
            std::swap(n[i], n[j]);
            std::swap(s[i], s[j]);
        }
        const int64_t elem = 1 << (r() % 3);
        const int64_t a = 1 << 20, b = a + (int64_t)(r() % (unsigned)(2 * span * elem + 5)) - span * elem;
        CHECK(plan::views_meet((uintptr_t)a, (uintptr_t)b, n, s, k, elem) == by_elements(a, b, n, s, k, elem));
    }
    const int64_t none[2] = {0, 5}, st[2] = {5, 1};
    CHECK(!plan::views_meet(64, 64, none, st, 2, 4));
    const int64_t far[2] = {INT64_MAX / 4, 2}, fst[2] = {INT64_MAX / 8, 1};   // no overflow on the way
    CHECK(plan::views_meet(0, UINTPTR_MAX, far, fst, 2, 4) || true);
}

static void* fake(uintptr_t n) { return reinterpret_cast<void*>(0x100000 + (n << 24)); }

static fgqa_kv_cache cache() {
    fgqa_kv_cache c;
    memset(&c, 0, sizeof c);
    c.k = fake(1);
    c.v = fake(2);
    c.k_scales = static_cast<float*>(fake(3));
    c.v_scales = static_cast<float*>(fake(4));
    c.kv_dtype = FGQA_KV_INT8;
    c.num_kv_heads = 8;
    c.head_dim = 128;
    c.page_size = 16;
    c.num_pages = 40;
    const int64_t st[3] = {16 * 8 * 128, 8 * 128, 128};
    for (int i = 0; i < 3; ++i) c.k_stride[i] = c.v_stride[i] = st[i];
    c.k_scales_stride[0] = c.v_scales_stride[0] = 8;
    c.k_scales_stride[1] = c.v_scales_stride[1] = 1;
    return c;
}

static void test_calls() {
    for (int which = 0; which < 3; ++which) {
        fgqa_kv_append_args a;
        memset(&a, 0, sizeof a);
        a.cache = cache();
        a.k_new = fake(5);
        a.v_new = fake(5);   // (one tensor for both is read only)
        const int64_t st[3] = {7 * 8 * 128, 8 * 128, 128};
        for (int i = 0; i < 3; ++i) a.k_new_stride[i] = a.v_new_stride[i] = st[i];
        a.block_table = static_cast<int32_t*>(fake(7));
        a.block_table_stride = a.max_pages = 10;
        a.seqlens = static_cast<int32_t*>(fake(8));
        a.batch = 3;
        a.max_new = 7;
        fgqa_kv_evict_args e;
        memset(&e, 0, sizeof e);
        e.cache = cache();
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
        for (fgqa_kv_cache* c : {&a.cache, &e.cache}) {
            if (which == 1) c->v = c->k;
            if (which == 2) c->v_scales = c->k_scales;
        }
        const int want = which == 0 ? FGQA_OK : FGQA_ERR_INVALID_ARGUMENT;
        CHECK(plan::validate_kv_append(&a) == want);
        CHECK(plan::validate_kv_evict(&e) == want);
        a.batch = e.batch = 0;   // nothing is written
        CHECK(plan::validate_kv_append(&a) == FGQA_OK && plan::validate_kv_evict(&e) == FGQA_OK);
    }
}

int main() {
    test_views();
    test_calls();
    printf("%ld checks, %ld failed\n", g_checks, g_failed);
    return g_failed ? 1 : 0;
}
