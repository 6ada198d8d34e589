// The host validation of include/fgqa_pages.h: each rule at its boundary, extreme sizes,
// fuzzed argument sets, and the workspaces' layout.  Built with sanitizers.
#include <climits>
#include <cstdio>
#include <random>

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
    const int kBad = FGQA_ERR_INVALID_ARGUMENT, kNot = FGQA_ERR_UNSUPPORTED;
    typedef fgqa_kv_fork_args A;
    typedef fgqa_kv_compact_args C;
    CHECK(validate_kv_fork(nullptr) == kBad);
    CHECK(validate_kv_compact(nullptr) == kBad);
    CHECK(fork([](A&) {}) == FGQA_OK);
    CHECK(compact([](C&) {}) == FGQA_OK);
    CHECK(fork([](A& a) { a.batch = -1; }) == kBad);
    CHECK(fork([](A& a) { a.new_batch = -1; }) == kBad);
    CHECK(fork([](A& a) { a.max_pages = -1; }) == kBad);
    CHECK(fork([](A& a) { a.new_block_table_stride = 6; }) == kBad);
    CHECK(fork([](A& a) { a.new_block_table_stride = 0; a.new_batch = 1; }) == FGQA_OK);
    CHECK(fork([](A& a) { a.block_table_stride = 0; }) == FGQA_OK);   // (rows that are read may be one)
    CHECK(fork([](A& a) { a.block_table_stride = INT64_MAX; }) == kNot);
    CHECK(fork([](A& a) { a.new_max_pages = 1 << 27; a.new_block_table_stride = 1 << 27; }) == kNot);
    CHECK(fork([](A& a) { a.new_max_pages = 1 << 26; a.new_block_table_stride = 1 << 26; }) == FGQA_OK);
    CHECK(fork([](A& a) { a.new_batch = 1 << 20; }) == kNot);
    CHECK(fork([](A& a) { a.new_batch = (1 << 20) - 1; }) == FGQA_OK);
    CHECK(fork([](A& a) { a.cache.num_kv_heads = 1 << 22; }) == kNot);
    CHECK(fork([](A& a) { a.cache.num_pages = 0; }) == kBad);
    CHECK(fork([](A& a) { a.cache.v = a.cache.k; }) == kBad);
    CHECK(fork([](A& a) { a.num_free = nullptr; }) == kBad);
    CHECK(fork([](A& a) { a.new_seqlens = nullptr; }) == kBad);
    CHECK(fork([](A& a) { a.new_block_table = nullptr; }) == kBad);
    CHECK(fork([](A& a) { a.new_block_table = nullptr; a.new_max_pages = 0; }) == FGQA_OK);
    CHECK(fork([](A& a) { a.seqlens = nullptr; }) == kBad);
    CHECK(fork([](A& a) { a.block_table = nullptr; }) == kBad);
    CHECK(fork([](A& a) { a.parents = nullptr; }) == kBad);            // (4 rows of 3)
    CHECK(fork([](A& a) { a.parents = nullptr; a.new_batch = 3; }) == FGQA_OK);
    CHECK(fork([](A& a) { a.new_lens = nullptr; a.held = nullptr; }) == FGQA_OK);
    CHECK(fork([](A& a) { a.parents = reinterpret_cast<int32_t*>(g_mem + 1025); }) == kNot);
    CHECK(fork([](A& a) { a.new_block_table = ints(512); }) == kBad);
    CHECK(fork([](A& a) { a.new_seqlens = ints(768); }) == kBad);
    CHECK(fork([](A& a) { a.new_batch = 0; a.new_block_table = a.new_seqlens = nullptr; }) == FGQA_OK);
    CHECK(fork([](A& a) { a.batch = 0; a.block_table = a.seqlens = nullptr; }) == FGQA_OK);
    CHECK(compact([](C& a) { a.batch = -1; }) == kBad);
    CHECK(compact([](C& a) { a.new_block_table_stride = 6; }) == kBad);
    CHECK(compact([](C& a) { a.num_used = nullptr; }) == kBad);
    CHECK(compact([](C& a) { a.new_block_table = ints(512); }) == kBad);
    CHECK(compact([](C& a) { a.seqlens = nullptr; }) == kBad);
    CHECK(compact([](C& a) { a.batch = 0; a.seqlens = nullptr; a.block_table = nullptr; }) == FGQA_OK);
    CHECK(compact([](C& a) { a.batch = 1 << 20; }) == kNot);
    CHECK(compact([](C& a) { a.cache.kv_dtype = FGQA_KV_INT8; }) == kBad);

    for (int pages : {1, 31, 32, 33, 4096, INT_MAX}) {
        fgqa_kv_fork_args a = fork_args();
        a.cache.num_pages = pages;
        const ForkLayout l = fork_layout(a);
        const int64_t words = ((int64_t)pages + 31) / 32;
        CHECK(page_words(pages) == words);
        CHECK(l.before - l.bits >= words && l.row_first - l.before >= words + 1 && l.first - l.row_first >= 4 && l.total - l.first >= 3);
        fgqa_kv_compact_args c = compact_args();
        c.cache.num_pages = pages;
        const CompactLayout m = compact_layout(c);
        CHECK(m.held - m.live >= words && m.live_before - m.held >= words && m.open_before - m.live_before >= words + 1 &&
              m.edge - m.open_before >= words + 1 && m.total > m.edge);
        CHECK(l.total % 4 == 0 && m.total % 4 == 0);
    }
    {
        fgqa_kv_compact_args c = compact_args();
        c.batch = 10;
        c.max_pages = 10;
        c.cache.num_pages = 128;   // (64 move at most, of 2^23 bytes each)
        c.cache.page_size = 4096;
        c.cache.num_kv_heads = 4;
        c.cache.kv_dtype = FGQA_KV_BF16;
        CHECK(compact_moves(c) == 64 && compact_moves_little(c) && compact_alone_ints(c) > 0);
        c.cache.num_pages = 130;
        CHECK(!compact_moves_little(c) && compact_alone_ints(c) > 0);
        c.batch = 6;
        CHECK(compact_moves(c) == 60 && compact_moves_little(c));
    }
    int alone = 0;
    std::mt19937_64 rng(11);
    const int32_t sizes[] = {0, 1, 3, 16, 128, 1 << 19, 1 << 20, INT_MAX, -1};
    auto pick = [&] { return sizes[rng() % 9]; };
    for (int i = 0; i < 200000; ++i) {
        fgqa_kv_fork_args a = fork_args();
        a.batch = pick();
        a.new_batch = pick();
        a.max_pages = pick();
        a.new_max_pages = pick();
        a.block_table_stride = (int64_t)(rng() >> (rng() % 64));
        a.new_block_table_stride = (int64_t)(rng() >> (rng() % 64));
        a.cache.num_pages = pick();
        a.cache.page_size = pick();
        if (validate_kv_fork(&a) == FGQA_OK) {
            CHECK(fork_layout(a).total > 0);
            const int64_t n = fork_alone_ints(a);
            if (n > 0) {
                ++alone;
                CHECK(n * 4 <= 61440 && n >= 2 * page_words(a.cache.num_pages) + 1 + 3 * (int64_t)a.batch + 4 * (int64_t)a.new_batch);
                CHECK((int64_t)a.batch * fork_width(a) < INT_MAX - kAloneThreads);
                CHECK((int64_t)a.new_batch * a.new_max_pages < INT_MAX - 256 * kAloneThreads);
            }
        }
        fgqa_kv_compact_args c = compact_args();
        c.batch = a.batch;
        c.max_pages = a.max_pages;
        c.new_block_table_stride = a.new_block_table_stride;
        c.cache = a.cache;
        if (validate_kv_compact(&c) == FGQA_OK) {
            CHECK(compact_layout(c).total > 0);
            const int64_t n = compact_alone_ints(c);
            if (n > 0) {
                ++alone;
                CHECK(n * 4 <= 61440 && n >= 4 * page_words(c.cache.num_pages) + 2 + c.batch);
                CHECK((int64_t)c.batch * c.max_pages < INT_MAX - 256 * kAloneThreads);
            }
        }
    }
    CHECK(alone > 100);
    std::printf("%d failed\n", g_failed);
    return g_failed != 0;
}
