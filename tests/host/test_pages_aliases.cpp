// What forking and compacting write, at the address of something else that the call reads or
// writes, is refused whatever the sizes; what a call does not use may lie anywhere.  Built with sanitizers.
#include <cstdio>

#include "pages_plan.h"

using namespace fgqa::plan;

static int g_failed = 0;
#define CHECK(x)                                        \
    do {                                                \
        if (!(x)) {                                     \
            ++g_failed;                                 \
            std::printf("line %d: %s\n", __LINE__, #x); \
        }                                               \
    } while (0)

alignas(256) static unsigned char g_mem[4096];

static fgqa_kv_cache cache() {
    fgqa_kv_cache c = {};
    c.k = g_mem;
    c.v = g_mem + 256;
    c.kv_dtype = FGQA_KV_BF16;
    c.num_kv_heads = 2;
    c.head_dim = 128;
    c.page_size = 16;
    c.num_pages = 100;
    c.k_scale = c.v_scale = 1.f;
    const int64_t st[3] = {16 * 256, 256, 128};
    for (int i = 0; i < 3; ++i) c.k_stride[i] = c.v_stride[i] = st[i];
    return c;
}

static int32_t* ints(int at) { return reinterpret_cast<int32_t*>(g_mem + at); }

static fgqa_kv_fork_args fork_args() {
    fgqa_kv_fork_args a = {};
    a.cache = cache();
    a.block_table = ints(512);
    a.seqlens = ints(768);
    a.parents = ints(1024);
    a.new_lens = ints(1280);
    a.held = g_mem + 2304;
    a.new_block_table = ints(1536);
    a.new_seqlens = ints(1792);
    a.num_free = ints(2048);
    a.batch = 3;
    a.new_batch = 4;
    a.max_pages = a.new_max_pages = 7;
    a.block_table_stride = a.new_block_table_stride = 7;
    return a;
}

static fgqa_kv_compact_args compact_args() {
    fgqa_kv_compact_args a = {};
    a.cache = cache();
    a.block_table = ints(512);
    a.seqlens = ints(768);
    a.held = g_mem + 2304;
    a.new_block_table = ints(1536);
    a.num_used = ints(2048);
    a.batch = 3;
    a.max_pages = 7;
    a.block_table_stride = a.new_block_table_stride = 7;
    return a;
}

template <typename F>
static int fork(F&& change) {
    fgqa_kv_fork_args a = fork_args();
    change(a);
    return validate_kv_fork(&a);
}

template <typename F>
static int compact(F&& change) {
    fgqa_kv_compact_args a = compact_args();
    change(a);
    return validate_kv_compact(&a);
}

int main() {
    using F = fgqa_kv_fork_args;
    using C = fgqa_kv_compact_args;
    constexpr int kBad = FGQA_ERR_INVALID_ARGUMENT;
    CHECK(fork([](F&) {}) == FGQA_OK && compact([](C&) {}) == FGQA_OK);
    const int batches[] = {3, 0};
    for (int batch : batches) {   // (an empty old table: parents and new_lens are read all the same)
        auto of = [&](auto change) { return fork([&](F& a) { a.batch = batch; change(a); }); };
        CHECK(of([](F&) {}) == FGQA_OK);
        CHECK(of([](F& a) { a.new_seqlens = const_cast<int32_t*>(a.new_lens); }) == kBad);
        CHECK(of([](F& a) { a.new_seqlens = const_cast<int32_t*>(a.parents); }) == kBad);
        CHECK(of([](F& a) { a.new_block_table = const_cast<int32_t*>(a.new_lens); }) == kBad);
        CHECK(of([](F& a) { a.new_block_table = const_cast<int32_t*>(a.parents); }) == kBad);
        CHECK(of([](F& a) { a.num_free = const_cast<int32_t*>(a.new_lens); }) == kBad);
        CHECK(of([](F& a) { a.num_free = const_cast<int32_t*>(a.parents); }) == kBad);
        CHECK(of([](F& a) { a.num_free = a.new_seqlens; }) == kBad);
        CHECK(of([](F& a) { a.num_free = a.new_block_table; }) == kBad);
        CHECK(of([](F& a) { a.new_seqlens = a.new_block_table; }) == kBad);
        CHECK(of([](F& a) { a.held = reinterpret_cast<const uint8_t*>(a.num_free); }) == kBad);
        CHECK(of([](F& a) { a.held = reinterpret_cast<const uint8_t*>(a.new_seqlens); }) == kBad);
        CHECK(of([](F& a) { a.held = reinterpret_cast<const uint8_t*>(a.new_block_table); }) == kBad);
        // nothing is read of an old table without rows
        const int old = batch > 0 ? kBad : (int)FGQA_OK;
        CHECK(of([](F& a) { a.new_block_table = const_cast<int32_t*>(a.block_table); }) == old);
        CHECK(of([](F& a) { a.new_seqlens = const_cast<int32_t*>(a.seqlens); }) == old);
        CHECK(of([](F& a) { a.num_free = const_cast<int32_t*>(a.seqlens); }) == old);
        CHECK(of([](F& a) { a.num_free = const_cast<int32_t*>(a.block_table); }) == old);
        CHECK(of([](F& a) { a.new_seqlens = const_cast<int32_t*>(a.block_table); }) == old);
    }
    // inputs may share memory, lists that are not there are no addresses, and without new rows only held is read
    CHECK(fork([](F& a) { a.parents = a.new_lens; }) == FGQA_OK);
    CHECK(fork([](F& a) { a.parents = a.new_lens = nullptr; a.held = nullptr; a.new_batch = 3; }) == FGQA_OK);
    CHECK(fork([](F& a) { a.new_batch = 0; a.num_free = const_cast<int32_t*>(a.parents); }) == FGQA_OK);
    CHECK(fork([](F& a) { a.new_batch = 0; a.new_seqlens = a.num_free; }) == FGQA_OK);
    CHECK(fork([](F& a) { a.new_batch = 0; a.held = reinterpret_cast<const uint8_t*>(a.num_free); }) == kBad);
    CHECK(fork([](F& a) { a.new_max_pages = 0; a.new_block_table = a.num_free; }) == FGQA_OK);

    CHECK(compact([](C& a) { a.num_used = const_cast<int32_t*>(a.seqlens); }) == kBad);
    CHECK(compact([](C& a) { a.num_used = const_cast<int32_t*>(a.block_table); }) == kBad);
    CHECK(compact([](C& a) { a.num_used = a.new_block_table; }) == kBad);
    CHECK(compact([](C& a) { a.new_block_table = const_cast<int32_t*>(a.seqlens); }) == kBad);
    CHECK(compact([](C& a) { a.new_block_table = const_cast<int32_t*>(a.block_table); }) == kBad);
    CHECK(compact([](C& a) { a.held = reinterpret_cast<const uint8_t*>(a.num_used); }) == kBad);
    CHECK(compact([](C& a) { a.held = reinterpret_cast<const uint8_t*>(a.new_block_table); }) == kBad);
    CHECK(compact([](C& a) { a.batch = 0; a.num_used = const_cast<int32_t*>(a.seqlens); }) == FGQA_OK);
    CHECK(compact([](C& a) { a.max_pages = 0; a.new_block_table = a.num_used; }) == FGQA_OK);
    std::printf("%d failed\n", g_failed);
    return g_failed != 0;
}
