// Host-only validation of the paged KV cache's C ABI (csrc/host/kv_plan.cpp) and
// its C++ operator layer (src/cplusplus/FlashGQA/kv_cache.cpp) over a recording
// stand-in of the C ABI, built by tests/test_kv_host.py with g++ and
// AddressSanitizer + UndefinedBehaviorSanitizer (no recovery).
//
// Output: one line per failed check, then "N checks, M failed"; exit status 1
// when a check failed.
#include <limits.h>
#include <math.h>
#include <stdint.h>
#include <stdio.h>
#include <string.h>

#include <random>

#include "FlashGQA/decode_flash_gqa_kernel.h"
#include "FlashGQA/kv_cache_kernel.h"
#include "fgqa_kv.h"
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

static void* fake(uintptr_t n) { return reinterpret_cast<void*>(0x100000 + 256 * n); }

// ---------------------------------------------------------------- recording C ABI
static fgqa_kv_append_args g_append;
static fgqa_decode_blocks_args g_decode;
static fgqa_kv_weights_args g_weights;
static fgqa_kv_evict_args g_evict;
static int g_status = FGQA_OK;

namespace fgqa_cpp {
void set_last_status(int status) { g_status = status; }
}

extern "C" {
int fgqa_kv_append(const fgqa_kv_append_args* a, void*) {
    g_append = *a;
    return plan::validate_kv_append(a);
}
int fgqa_decode_blocks(const fgqa_decode_blocks_args* a, void*) {
    g_decode = *a;
    const int st = plan::validate_decode_blocks(a);
    return st != FGQA_OK ? st : plan::validate_decode_blocks_pointers(a);
}
int fgqa_kv_weights(const fgqa_kv_weights_args* a, void*) {
    g_weights = *a;
    return plan::validate_kv_weights(a);
}
int fgqa_kv_evict(const fgqa_kv_evict_args* a, void*) {
    g_evict = *a;
    return plan::validate_kv_evict(a);
}
}

// ---------------------------------------------------------------- arguments that are right
static const int kPages = 40, kPage = 16, kHeads = 8, kBatch = 3;

static fgqa_kv_cache cache(int dtype, bool blocks) {
    fgqa_kv_cache c;
    memset(&c, 0, sizeof c);
    c.k = fake(1);
    c.v = fake(2);
    if (blocks) {
        c.k_scales = static_cast<float*>(fake(3));
        c.v_scales = static_cast<float*>(fake(4));
    }
    c.kv_dtype = dtype;
    c.num_kv_heads = kHeads;
    c.head_dim = 128;
    c.page_size = kPage;
    c.num_pages = kPages;
    c.k_scale = c.v_scale = 1.f;
    const int64_t st[3] = {kPage * kHeads * 128, kHeads * 128, 128};
    for (int i = 0; i < 3; ++i) c.k_stride[i] = c.v_stride[i] = st[i];
    c.k_scales_stride[0] = c.v_scales_stride[0] = kHeads;
    c.k_scales_stride[1] = c.v_scales_stride[1] = 1;
    return c;
}

static fgqa_kv_append_args append_args(int dtype = FGQA_KV_INT8, bool blocks = true) {
    fgqa_kv_append_args a;
    memset(&a, 0, sizeof a);
    a.cache = cache(dtype, blocks);
    a.k_new = fake(5);
    a.v_new = fake(6);
    const int64_t st[3] = {7 * kHeads * 128, kHeads * 128, 128};
    for (int i = 0; i < 3; ++i) a.k_new_stride[i] = a.v_new_stride[i] = st[i];
    a.block_table = static_cast<int32_t*>(fake(7));
    a.block_table_stride = a.max_pages = 10;
    a.seqlens = static_cast<int32_t*>(fake(8));
    a.batch = kBatch;
    a.max_new = 7;
    return a;
}

static fgqa_decode_blocks_args decode_args() {
    fgqa_decode_blocks_args a;
    memset(&a, 0, sizeof a);
    a.cache = cache(FGQA_KV_FP8_E4M3, true);
    a.q = fake(9);
    a.o = fake(10);
    a.block_table = static_cast<int32_t*>(fake(7));
    a.seqlens = static_cast<int32_t*>(fake(8));
    a.batch = kBatch;
    a.max_seqlen = 160;
    a.num_q_heads = 32;
    a.scale = 0.1f;
    a.q_stride[0] = a.o_stride[0] = 32 * 128;
    a.q_stride[1] = a.o_stride[1] = 128;
    a.block_table_stride = 10;
    return a;
}

static fgqa_kv_weights_args weights_args() {
    fgqa_kv_weights_args a;
    memset(&a, 0, sizeof a);
    a.cache = cache(FGQA_KV_BF16, false);
    a.q = fake(9);
    a.lse = static_cast<float*>(fake(11));
    a.weights = static_cast<float*>(fake(12));
    a.q_stride[0] = 32 * 128;
    a.q_stride[1] = 128;
    a.weights_stride[0] = kHeads * 160;
    a.weights_stride[1] = 160;
    a.block_table = static_cast<int32_t*>(fake(7));
    a.block_table_stride = 10;
    a.seqlens = static_cast<int32_t*>(fake(8));
    a.batch = kBatch;
    a.max_seqlen = 160;
    a.num_q_heads = 32;
    a.scale = 0.1f;
    return a;
}

static fgqa_kv_evict_args evict_args() {
    fgqa_kv_evict_args a;
    memset(&a, 0, sizeof a);
    a.cache = cache(FGQA_KV_INT8, true);
    a.weights = static_cast<float*>(fake(12));
    a.new_weights = static_cast<float*>(fake(13));
    a.weights_stride[0] = a.new_weights_stride[0] = kHeads * 160;
    a.weights_stride[1] = a.new_weights_stride[1] = 160;
    a.block_table = static_cast<int32_t*>(fake(7));
    a.new_block_table = static_cast<int32_t*>(fake(14));
    a.block_table_stride = 10;
    a.new_block_table_stride = 4;
    a.seqlens = static_cast<int32_t*>(fake(8));
    a.new_seqlens = static_cast<int32_t*>(fake(15));
    a.kept = static_cast<int32_t*>(fake(16));
    a.batch = kBatch;
    a.max_seqlen = a.weights_len = 160;
    a.budget = 64;
    a.recent = 8;
    return a;
}

// A field changed: the status that comes of it.
#define APPEND(change, status)                              \
    do {                                                    \
        fgqa_kv_append_args a = append_args();              \
        change;                                             \
        CHECK(plan::validate_kv_append(&a) == (status));    \
    } while (0)
#define WEIGHTS(change, status)                             \
    do {                                                    \
        fgqa_kv_weights_args a = weights_args();            \
        change;                                             \
        CHECK(plan::validate_kv_weights(&a) == (status));   \
    } while (0)
#define EVICT(change, status)                               \
    do {                                                    \
        fgqa_kv_evict_args a = evict_args();                \
        change;                                             \
        CHECK(plan::validate_kv_evict(&a) == (status));     \
    } while (0)
#define DECODE(change, status)                              \
    do {                                                    \
        fgqa_decode_blocks_args a = decode_args();          \
        change;                                             \
        CHECK(fgqa_decode_blocks(&a, nullptr) == (status)); \
    } while (0)

static const int BAD = FGQA_ERR_INVALID_ARGUMENT, NOT = FGQA_ERR_UNSUPPORTED, OK = FGQA_OK;

static void test_cache() {
    for (int dtype = -1; dtype <= 3; ++dtype)
        for (int blocks = 0; blocks < 2; ++blocks) {
            fgqa_kv_append_args a = append_args(dtype, blocks);
            const bool ok = dtype == FGQA_KV_BF16 ? !blocks : dtype == FGQA_KV_INT8 ? blocks : dtype == FGQA_KV_FP8_E4M3;
            CHECK(plan::validate_kv_append(&a) == (ok ? OK : BAD));
        }
    APPEND(a.cache.v_scales = nullptr, BAD);
    APPEND(a.cache.num_kv_heads = 0, BAD);
    APPEND(a.cache.page_size = 0, BAD);
    APPEND(a.cache.page_size = 24, NOT);
    APPEND(a.cache.page_size = 1 << 21, NOT);
    APPEND(a.cache.head_dim = 64, NOT);
    APPEND(a.cache.head_dim = -128, BAD);
    APPEND(a.cache.num_pages = 0, BAD);
    APPEND(a.cache.num_pages = -1, BAD);
    APPEND(a.cache.k = nullptr, BAD);
    APPEND(a.cache.k = static_cast<char*>(fake(1)) + 8, NOT);
    APPEND(a.cache.v_stride[1] += 8, NOT);
    APPEND(a.cache.v_stride[1] = -128, BAD);
    APPEND(a.cache.k_stride[0] = INT64_MAX / 16 * 16, NOT);
    APPEND(a.cache.k_scales_stride[0] = -1, BAD);
    APPEND(a.cache.k_scales_stride[0] = INT64_MAX, NOT);
    APPEND(a.cache.k_scales = reinterpret_cast<float*>(0x1002), NOT);
    fgqa_kv_append_args a = append_args(FGQA_KV_FP8_E4M3, false);
    const float bad[] = {0.f, -1.f, INFINITY, NAN};
    for (float s : bad) {
        a.cache.v_scale = s;
        CHECK(plan::validate_kv_append(&a) == BAD);
    }
    a = append_args(FGQA_KV_BF16, false);   // ignored
    a.cache.v_scale = NAN;
    CHECK(plan::validate_kv_append(&a) == OK);
    a.cache.k_stride[1] += 8;               // 16 bytes of bf16
    a.cache.v_stride[1] += 8;
    CHECK(plan::validate_kv_append(&a) == OK);
}

static void test_append() {
    CHECK(plan::validate_kv_append(nullptr) == BAD);
    APPEND((void)a, OK);
    APPEND(a.batch = -1, BAD);
    APPEND(a.max_new = -1, BAD);
    APPEND(a.max_pages = -1, BAD);
    APPEND(a.block_table_stride = -1, BAD);
    APPEND(a.k_new_stride[0] = -8, BAD);
    APPEND(a.k_new_stride[0] = 4, NOT);
    APPEND(a.k_new = static_cast<char*>(fake(5)) + 2, NOT);
    APPEND(a.k_new = nullptr, BAD);
    APPEND(a.block_table = nullptr, BAD);
    APPEND(a.seqlens = nullptr, BAD);
    APPEND(a.new_lens = reinterpret_cast<int32_t*>(0x1001), NOT);
    APPEND(a.batch = 0; a.k_new = nullptr; a.cache.k = nullptr, OK);
    APPEND(a.max_new = 0; a.k_new = nullptr; a.seqlens = nullptr, OK);
    APPEND(a.max_new = INT_MAX, NOT);
    APPEND(a.max_pages = INT_MAX, NOT);
    APPEND(a.batch = INT_MAX, NOT);   // 2^31 workgroups and more
    CHECK(plan::append_pages(1, 16) == 1 && plan::append_pages(2, 16) == 2 && plan::append_pages(17, 16) == 2 &&
          plan::append_pages(18, 16) == 3 && plan::append_pages(5, 1) == 5);
}

static void test_weights() {
    CHECK(plan::validate_kv_weights(nullptr) == BAD);
    WEIGHTS((void)a, OK);
    WEIGHTS(a.cache.v = nullptr; a.cache.v_stride[0] = -3; a.cache.v_scale = NAN, OK);
    WEIGHTS(a.num_q_heads = 31, BAD);
    WEIGHTS(a.num_q_heads = 0, BAD);
    WEIGHTS(a.num_q_heads = 17 * kHeads, NOT);
    WEIGHTS(a.scale = INFINITY, BAD);
    WEIGHTS(a.max_seqlen = 161, BAD);   // past the block table's row
    WEIGHTS(a.max_seqlen = -1, BAD);
    WEIGHTS(a.weights_stride[0] = -1, BAD);
    WEIGHTS(a.weights_stride[0] = INT64_MAX, NOT);
    WEIGHTS(a.q_stride[1] = 12, NOT);
    WEIGHTS(a.q = nullptr, BAD);
    WEIGHTS(a.lse = nullptr, BAD);
    WEIGHTS(a.weights = nullptr, BAD);
    WEIGHTS(a.weights = reinterpret_cast<float*>(0x1002), NOT);
    WEIGHTS(a.batch = 0; a.q = nullptr, OK);
    WEIGHTS(a.max_seqlen = 0; a.weights = nullptr, OK);
    WEIGHTS(a.max_seqlen = INT_MAX; a.block_table_stride = INT_MAX, NOT);
    WEIGHTS(a.batch = 1 << 20; a.max_seqlen = 64 << 8; a.block_table_stride = 1 << 20, OK);   // a wave a row
    WEIGHTS(a.batch = (1 << 23) - 1, OK);
    WEIGHTS(a.batch = 1 << 23, NOT);   // 2^32 threads
    CHECK(plan::weights_waves(1, 1, 1) == 1 && plan::weights_waves(1, 1, 65) == 2 && plan::weights_waves(64, 8, 16384) == 256);
    CHECK(plan::weights_waves(64, 8, 16385) == 256 && plan::weights_waves(3, 8, 1 << 30) == (1 << 17) / 24);
    CHECK(plan::weights_waves(1 << 17, 1, 1 << 30) == 1 && plan::weights_waves(INT_MAX, INT_MAX, 1 << 30) == 1);
}

static void test_evict() {
    CHECK(plan::validate_kv_evict(nullptr) == BAD);
    EVICT((void)a, OK);
    EVICT(a.budget = 0, BAD);
    EVICT(a.recent = -1, BAD);
    EVICT(a.recent = INT_MAX, OK);
    EVICT(a.weights_len = 159, BAD);
    EVICT(a.max_seqlen = 161; a.weights_len = 161, BAD);
    EVICT(a.budget = 65, BAD);                  // past the new block table's row
    EVICT(a.budget = INT_MAX, BAD);
    EVICT(a.budget = INT_MAX; a.new_block_table_stride = 10, NOT);
    EVICT(a.budget = 1 << 30; a.new_block_table_stride = 10, OK);
    EVICT(a.weights = nullptr, BAD);
    EVICT(a.new_weights = nullptr, BAD);
    EVICT(a.kept = nullptr, BAD);
    EVICT(a.new_seqlens = nullptr, BAD);
    EVICT(a.new_block_table = nullptr, BAD);
    EVICT(a.kept = reinterpret_cast<int32_t*>(0x1002), NOT);
    EVICT(a.new_weights_stride[1] = -1, BAD);
    EVICT(a.batch = 0; a.kept = nullptr, OK);
    EVICT(a.max_seqlen = 0; a.weights = nullptr; a.block_table = nullptr; a.cache.k = nullptr, OK);
    EVICT(a.batch = INT_MAX, NOT);
    EVICT(a.batch = (1 << 19) - 1, OK);
    EVICT(a.batch = 1 << 19, NOT);                                               // rows of 1024 threads
    EVICT(a.batch = 1 << 18; a.max_seqlen = 0, OK);
    EVICT(a.batch = 1 << 18; a.budget = 1 << 20; a.weights_len = a.max_seqlen = 16 * 16;
          a.block_table_stride = a.new_block_table_stride = 1 << 20, NOT);       // 2^26 blocks of 16 rows
}

static void test_decode() {
    CHECK(plan::validate_decode_blocks(nullptr) == BAD);
    DECODE((void)a, OK);
    DECODE(a.cache.kv_dtype = FGQA_KV_INT8, OK);
    DECODE(a.cache.kv_dtype = FGQA_KV_BF16, BAD);
    DECODE(a.cache.k_scales = nullptr, BAD);
    DECODE(a.cache.v_scales_stride[1] = -1, BAD);
    DECODE(a.max_seqlen = 161, BAD);
    DECODE(a.scale = NAN, BAD);
    DECODE(a.cache.k_stride[1] += 8, NOT);
    DECODE(a.num_q_heads = 17 * kHeads, NOT);
    DECODE(a.batch = 0; a.q = nullptr; a.cache.k_scales = nullptr, OK);
    // 64 sequences of 16384 tokens, 8 heads: 128 teams of two partials of 32 rows
    // (512 + 8 bytes) each, and the sequences' prefix; 2 heads: 256 teams
    {
        fgqa_decode_blocks_args a = decode_args();
        a.batch = 64;
        a.max_seqlen = 16384;
        a.block_table_stride = 1024;
        fgqa_decode_paged_args p = plan::as_decode_paged(&a);
        plan::DecodePlan pl;
        CHECK(plan::plan_blocks(&p, 256, &pl) == OK && pl.teams == 128 && pl.least_bytes <= pl.ws_bytes);
        p.num_kv_heads = 2;
        CHECK(plan::plan_blocks(&p, 256, &pl) == OK && pl.teams == 256);
        // splits: of a length given, of the whole sequence (nothing to merge), of an even share
        p.split_tokens = 1000;
        CHECK(plan::plan_blocks(&p, 256, &pl) == OK && pl.teams == 0 && !pl.list && pl.chunk == 1024 && pl.nsplit == 16 &&
              pl.ws_bytes == (size_t)64 * 32 * 16 * 520 && pl.least_bytes == pl.ws_bytes);
        p.split_tokens = 0;
        p.batch = 8;
        p.max_seqlen = 640;
        CHECK(plan::plan_blocks(&p, 256, &pl) == OK && pl.teams == 0 && pl.nsplit == 1 && pl.ws_bytes == 0);
        p.max_seqlen = 8000;
        CHECK(plan::plan_blocks(&p, 0, &pl) == OK && pl.teams == 0 && pl.chunk == 512 && pl.nsplit == 16);
        p.max_seqlen = 0;
        CHECK(plan::plan_blocks(&p, 256, &pl) == OK);
        // more workgroups than a grid has
        p.batch = 32000;
        p.max_seqlen = 16384;
        p.split_tokens = 1;
        p.num_kv_heads = p.num_q_heads = 1 << 14;
        CHECK(plan::plan_blocks(&p, 256, &pl) == NOT);
    }
    CHECK(plan::blocks_split(1, 1, 0, 256) == 0 && plan::blocks_split(1, 1, 1, 256) == 128);
    CHECK(plan::blocks_split(1, 8, 640, 256) == 640 && plan::blocks_split(1, 8, 641, 256) == 128);
    CHECK(plan::blocks_split(64, 8, 1024, 256) == 1024 && plan::blocks_split(64, 8, 1025, 256) == 0);
    CHECK(plan::blocks_split(65, 8, 128, 256) == 0 && plan::blocks_split(64, 8, 128, 256) == 128);
    CHECK(plan::blocks_split(1, 1, 524288, 256) == 2048 && plan::blocks_split(1, 1, 524289, 256) == 0);
    CHECK(plan::blocks_split(INT_MAX, INT_MAX, INT_MAX, 256) == 0);
    // a cache without the 8-bit types of the C ABI before
    fgqa_decode_blocks_args a = decode_args();
    fgqa_decode_paged_args p = plan::as_decode_paged(&a);
    p.kv_dtype = FGQA_KV_INT8;
    CHECK(plan::validate_paged(&p) == BAD);
}

static void test_operator_layer() {
    KvCache c;
    c.k = fake(1);
    c.v = fake(2);
    c.kScales = static_cast<float*>(fake(3));
    c.vScales = static_cast<float*>(fake(4));
    c.type = KvCacheType::Int8;
    c.numPages = kPages;
    c.pageSize = kPage;
    c.numKvHeads = kHeads;
    const bf16_t* q = static_cast<const bf16_t*>(fake(5));
    bf16_t* o = static_cast<bf16_t*>(fake(6));
    const int32_t* i32 = static_cast<const int32_t*>(fake(7));
    float* f32 = static_cast<float*>(fake(12));
    LaunchKvCacheAppendKernel(c, q, q, i32, i32, nullptr, kBatch, 7, 10);
    fgqa_kv_append_args ra = append_args();
    CHECK(g_status == OK && g_append.k_new_stride[0] == 7 * kHeads * 128 && g_append.max_pages == 10 &&
          g_append.block_table_stride == 10 && g_append.new_lens == nullptr);
    CHECK(memcmp(g_append.cache.k_stride, ra.cache.k_stride, sizeof ra.cache.k_stride) == 0);
    CHECK(memcmp(g_append.cache.v_scales_stride, ra.cache.v_scales_stride, sizeof ra.cache.v_scales_stride) == 0);
    CHECK(g_append.cache.kv_dtype == FGQA_KV_INT8);
    LaunchFlashGqaBf16KernelPagedBlocks(c, q, 0.1f, o, f32, i32, i32, kBatch, 10, 32);
    CHECK(g_status == OK && g_decode.max_seqlen == 160 && g_decode.q_stride[0] == 32 * 128 && g_decode.lse == f32 &&
          g_decode.workspace == nullptr);
    LaunchKvCacheWeightsKernel(c, q, 0.1f, f32, f32 + 64, i32, i32, kBatch, 10, 32);
    CHECK(g_status == OK && g_weights.weights_stride[0] == kHeads * 160 && g_weights.max_seqlen == 160);
    LaunchKvCacheEvictKernel(c, f32, f32 + 9999, i32, i32 + 64, i32, static_cast<int32_t*>(fake(20)),
                             static_cast<int32_t*>(fake(21)), 64, 8, kBatch, 10, 4);
    CHECK(g_status == OK && g_evict.budget == 64 && g_evict.recent == 8 && g_evict.weights_len == 160 &&
          g_evict.new_block_table_stride == 4);
    // ints at their ends: refused, nothing overflows on the way
    const int ends[] = {INT_MIN, -1, 0, 1, INT_MAX};
    for (int x : ends)
        for (int y : ends)
            for (int z : ends) {
                KvCache e = c;
                e.pageSize = x;
                e.numKvHeads = y;
                e.numPages = z;
                LaunchKvCacheAppendKernel(e, q, q, i32, i32, i32, x, y, z);
                LaunchFlashGqaBf16KernelPagedBlocks(e, q, 0.1f, o, f32, i32, i32, y, z, x);
                LaunchKvCacheWeightsKernel(e, q, 0.1f, f32, f32, i32, i32, y, z, x);
                LaunchKvCacheEvictKernel(e, f32, f32, i32, i32, i32, nullptr, nullptr, x, y, z, x, y);
                ++g_checks;
            }
}

// Random fields at and around their limits: every answer is a status, and no
// arithmetic on the way overflows (the sanitizers end the program).
static void fuzz() {
    std::mt19937_64 r(1);
    auto pick = [&]() -> int64_t {
        const int64_t v[] = {0, 1, 2, 7, 8, 16, 17, 63, 64, 128, 1 << 20, 1 << 30, INT_MAX, INT_MIN, -1, INT64_MAX, INT64_MIN,
                             INT64_MAX / 2, (int64_t)1 << 40};
        return r() % 3 ? v[r() % (sizeof v / sizeof v[0])] : (int64_t)r();
    };
    for (int n = 0; n < 200000; ++n) {
        fgqa_kv_append_args a = append_args();
        fgqa_kv_weights_args w = weights_args();
        fgqa_kv_evict_args e = evict_args();
        fgqa_decode_blocks_args d = decode_args();
        fgqa_kv_cache* caches[4] = {&a.cache, &w.cache, &e.cache, &d.cache};
        for (fgqa_kv_cache* c : caches) {
            int32_t* ints[] = {&c->kv_dtype, &c->num_kv_heads, &c->page_size, &c->num_pages};
            for (int32_t* i : ints)
                if (r() % 4 == 0) *i = (int32_t)pick();
            if (r() % 4 == 0) c->k_stride[r() % 3] = (int64_t)((uint64_t)pick() * 16);
            if (r() % 4 == 0) c->v_scales_stride[r() % 2] = pick();
        }
        int32_t* ints[] = {&a.batch, &a.max_new, &a.max_pages, &w.batch, &w.max_seqlen, &w.num_q_heads, &e.batch,
                           &e.max_seqlen, &e.weights_len, &e.budget, &e.recent, &d.batch, &d.max_seqlen, &d.num_q_heads,
                           &d.split_tokens};
        for (int32_t* i : ints)
            if (r() % 3 == 0) *i = (int32_t)pick();
        int64_t* longs[] = {&a.k_new_stride[1], &a.block_table_stride, &w.q_stride[0], &w.weights_stride[1],
                            &w.block_table_stride, &e.weights_stride[0], &e.new_weights_stride[1],
                            &e.new_block_table_stride, &e.block_table_stride, &d.q_stride[1], &d.block_table_stride};
        for (int64_t* i : longs)
            if (r() % 3 == 0) *i = pick();
        CHECK(plan::validate_kv_append(&a) <= 0);
        CHECK(plan::validate_kv_weights(&w) <= 0);
        CHECK(plan::validate_kv_evict(&e) <= 0);
        CHECK(fgqa_decode_blocks(&d, nullptr) <= 0);
        if (plan::validate_kv_weights(&w) == OK && w.batch > 0 && w.max_seqlen > 0) {
            const int waves = plan::weights_waves(w.batch, w.cache.num_kv_heads, w.max_seqlen);
            CHECK(waves >= 1 && (__int128)w.batch * w.cache.num_kv_heads * waves * 64 < ((int64_t)1 << 32));
        }
    }
}

int main() {
    test_cache();
    test_append();
    test_weights();
    test_evict();
    test_decode();
    test_operator_layer();
    fuzz();
    printf("%ld checks, %ld failed\n", g_checks, g_failed);
    return g_failed ? 1 : 0;
}
