// The cuts of the decode of sequences that begin alike: random lengths and groups cut as the
// planning kernel does stay within the items and rows of the plan; the validation's rules.
// Built with sanitizers.
#include <algorithm>
#include <climits>
#include <cstdio>
#include <random>
#include <vector>

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

static fgqa_decode_shared_args args() {
    fgqa_decode_shared_args a = {};
    fgqa_kv_cache& c = a.cache;
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
    a.q = g_mem;
    a.o = g_mem + 512;
    a.block_table = reinterpret_cast<int32_t*>(g_mem + 768);
    a.seqlens = reinterpret_cast<int32_t*>(g_mem + 1024);
    a.group_starts = reinterpret_cast<int32_t*>(g_mem + 1280);
    a.shared_lens = reinterpret_cast<int32_t*>(g_mem + 1536);
    a.batch = 4;
    a.max_seqlen = 160;
    a.num_q_heads = 8;
    a.num_groups = 2;
    a.scale = 0.1f;
    a.q_stride[0] = a.o_stride[0] = 1024;
    a.q_stride[1] = a.o_stride[1] = 128;
    a.block_table_stride = 10;
    return a;
}

template <typename F>
static int check(F&& change) {
    fgqa_decode_shared_args a = args();
    change(a);
    const int st = validate_decode_shared(&a);
    return st != FGQA_OK ? st : validate_decode_shared_pointers(&a);
}

int main() {
    const int kBad = FGQA_ERR_INVALID_ARGUMENT, kNot = FGQA_ERR_UNSUPPORTED;
    typedef fgqa_decode_shared_args A;
    CHECK(validate_decode_shared(nullptr) == kBad);
    CHECK(check([](A&) {}) == FGQA_OK);
    CHECK(check([](A& a) { a.num_groups = -1; }) == kBad);
    CHECK(check([](A& a) { a.num_groups = 4097; }) == kNot);
    CHECK(check([](A& a) { a.num_groups = 4096; }) == FGQA_OK);
    CHECK(check([](A& a) { a.num_groups = 0; a.group_starts = a.shared_lens = nullptr; }) == FGQA_OK);
    CHECK(check([](A& a) { a.group_starts = nullptr; }) == kBad);
    CHECK(check([](A& a) { a.shared_lens = reinterpret_cast<int32_t*>(g_mem + 2); }) == kNot);
    CHECK(check([](A& a) { a.batch = 1 << 15; }) == kNot);
    CHECK(check([](A& a) { a.batch = -1; }) == kBad);
    CHECK(check([](A& a) { a.num_q_heads = 7; }) == kBad);
    CHECK(check([](A& a) { a.num_q_heads = 34; }) == kNot);
    CHECK(check([](A& a) { a.max_seqlen = 161; }) == kBad);
    CHECK(check([](A& a) { a.q = nullptr; }) == kBad);
    CHECK(check([](A& a) { a.cache.kv_dtype = FGQA_KV_INT8; }) == kBad);
    CHECK(check([](A& a) { a.cache.k = nullptr; }) == kBad);
    CHECK(check([](A& a) { a.cache.k = nullptr; a.max_seqlen = 0; }) == FGQA_OK);
    CHECK(check([](A& a) { a.scale = 1.f / 0.f; }) == kBad);
    CHECK(check([](A& a) { a.cache.kv_dtype = FGQA_KV_FP8_E4M3; a.cache.v_scale = 1.f / 0.f; }) == kBad);

    CHECK(shared_chunk(0, 64) == 128 && shared_chunk(64 * 128, 64) == 128 && shared_chunk(64 * 128 + 1, 64) == 256);
    CHECK(shared_piece(1 << 30, 1 << 30, 64) == 1 << 30 && shared_piece((1 << 30) - 1, 1 << 29, 64) == 1 << 29);
    CHECK(shared_piece(1, 128, 64) == 64 && shared_piece(129, 128, 64) == 128 && shared_piece(1000, 384, 128) == 384);

    {
        fgqa_decode_shared_args a = args();
        float scale = 1.f;
        a.cache.num_kv_heads = 8;
        a.batch = 16;
        a.max_seqlen = 2304;
        CHECK(!shared_as_blocks(&a, 256));
        a.cache.k_scales = a.cache.v_scales = &scale;
        CHECK(shared_as_blocks(&a, 256) && shared_as_blocks(&a, 0) && !shared_as_blocks(&a, 255));
        a.max_seqlen = 2305;
        CHECK(!shared_as_blocks(&a, 256));
        a.batch = (1 << 15) - 1;
        a.max_seqlen = 1 << 30;
        CHECK(!shared_as_blocks(&a, 256));
        a.max_seqlen = 0;
        CHECK(shared_as_blocks(&a, 256));
        a.workspace = &scale;
        a.workspace_bytes = 77;
        const fgqa_decode_blocks_args b = as_decode_blocks(&a);
        CHECK(b.batch == a.batch && b.cache.k_scales == &scale && b.workspace == &scale && b.workspace_bytes == 77);
    }

    std::mt19937_64 rng(5);
    auto some = [&](int64_t n) { return (int64_t)(rng() % (uint64_t)n); };
    for (int turn = 0; turn < 20000; ++turn) {
        fgqa_decode_shared_args a = args();
        const int heads[] = {1, 2, 3, 8, 40};
        a.cache.num_kv_heads = heads[some(5)];
        const int group = 1 + (int)some(16);
        a.num_q_heads = a.cache.num_kv_heads * group;
        a.batch = 1 + (int)some(turn % 10 ? 40 : 400);
        a.num_groups = (int)some(2 * a.batch);
        const int cus = turn % 3 ? 256 : 1 + (int)some(300);
        SharedPlan pl;
        CHECK(plan_decode_shared(&a, cus, &pl) == FGQA_OK);
        // disjoint groups in order; what each shares is at most its shortest sequence
        const int64_t longest = (int64_t)1 << some(22);
        std::vector<int64_t> len(a.batch);
        for (int64_t& n : len) n = some(longest + 1);
        std::vector<int> cut(a.num_groups + 1);
        for (int& c : cut) c = (int)some(a.batch + 1);
        std::sort(cut.begin(), cut.end());
        std::vector<int64_t> left = len, shared(a.num_groups, 0);
        int64_t total = 0;
        for (int g = 0; g < a.num_groups; ++g) {
            if (cut[g + 1] - cut[g] < 2) continue;
            int64_t n = INT64_MAX;
            for (int b = cut[g]; b < cut[g + 1]; ++b) n = std::min(n, len[b]);
            n = n / 16 * 16;
            if (n < kSharedChunk) continue;
            shared[g] = n;
            total += n * (((int64_t)(cut[g + 1] - cut[g]) * group + kSharedRows - 1) / kSharedRows);
            for (int b = cut[g]; b < cut[g + 1]; ++b) left[b] -= n;
        }
        for (int64_t n : left) total += n;
        const int chunk = (int)std::min<int64_t>(shared_chunk(total, pl.slots), 1 << 30);
        int64_t items = 0, rows = 0;
        for (int g = 0; g < a.num_groups; ++g) {
            if (shared[g] == 0) continue;
            const int64_t piece = shared_piece((int)shared[g], chunk, 64), pieces = (shared[g] + piece - 1) / piece;
            const int64_t r = (int64_t)(cut[g + 1] - cut[g]) * group;
            CHECK(piece <= chunk && piece % 64 == 0);
            items += pieces * ((r + kSharedRows - 1) / kSharedRows);
            rows += pieces * a.cache.num_kv_heads * r;
        }
        for (int64_t n : left) {
            if (n == 0) continue;
            const int64_t piece = shared_piece((int)n, chunk, kSharedChunk), pieces = (n + piece - 1) / piece;
            CHECK(piece <= chunk && piece % kSharedChunk == 0);
            items += pieces;
            rows += pieces * a.cache.num_kv_heads * group;
        }
        CHECK(items <= pl.max_items);
        CHECK(rows <= pl.max_rows);
        CHECK(pl.part_ml_off >= (size_t)pl.max_rows * 512 && pl.items_off >= pl.part_ml_off + (size_t)pl.max_rows * 8 &&
              pl.seqs_off >= pl.items_off + (size_t)pl.max_items * 32 && pl.count_off >= pl.seqs_off + (size_t)a.batch * 32 &&
              pl.total > pl.count_off);
    }
    for (int i = 0; i < 100000; ++i) {
        fgqa_decode_shared_args a = args();
        const int32_t sizes[] = {0, 1, 3, 16, 128, 32767, 1 << 20, INT_MAX, -1};
        a.batch = sizes[some(9)];
        a.num_groups = sizes[some(9)];
        a.num_q_heads = sizes[some(9)];
        a.cache.num_kv_heads = sizes[some(9)];
        a.max_seqlen = sizes[some(9)];
        a.block_table_stride = (int64_t)(rng() >> some(64));
        SharedPlan pl;
        if (validate_decode_shared(&a) == FGQA_OK) {
            const int st = plan_decode_shared(&a, 256, &pl);
            CHECK(st == FGQA_OK || st == kNot);
        }
    }
    std::printf("%d failed\n", g_failed);
    return g_failed != 0;
}
