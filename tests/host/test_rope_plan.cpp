// The host validation of include/fgqa_rope.h: every rule at its boundary, extreme
// sizes, fuzzed argument sets, and the test of blocks that share memory against a
// search of all pairs.  Built with sanitizers.
#include <climits>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "kv_apart.h"
#include "rope_plan.h"

using namespace fgqa::plan;

static int g_failed = 0;
#define CHECK(x)                                             \
    do {                                                     \
        if (!(x)) {                                          \
            ++g_failed;                                      \
            std::printf("line %d: %s\n", __LINE__, #x);      \
        }                                                    \
    } while (0)

alignas(256) static unsigned char g_mem[4096];

static fgqa_rope_args forward_args() {
    fgqa_rope_args a = {};
    a.q = g_mem;
    a.k = g_mem + 256;
    a.q_out = g_mem + 512;
    a.k_out = g_mem + 768;
    a.positions = g_mem + 1024;
    a.inv_freq = reinterpret_cast<float*>(g_mem + 1280);
    a.q_weight = g_mem + 1536;
    a.k_weight = g_mem + 1792;
    a.num_axes = 1;
    a.batch = 2;
    a.seqlen = 5;
    a.num_q_heads = 8;
    a.num_kv_heads = 2;
    a.head_dim = a.rotary_dim = 128;
    a.eps = 1e-6f;
    const int64_t q[3] = {5 * 1024, 1024, 128}, k[3] = {5 * 256, 256, 128}, pos[3] = {10, 5, 1};
    for (int i = 0; i < 3; ++i) {
        a.q_stride[i] = a.q_out_stride[i] = q[i];
        a.k_stride[i] = a.k_out_stride[i] = k[i];
        a.positions_stride[i] = pos[i];
    }
    return a;
}

static fgqa_rope_backward_args backward_args() {
    fgqa_rope_backward_args a = {};
    a.fwd = forward_args();
    a.grad_q_out = g_mem + 2048;
    a.grad_k_out = g_mem + 2304;
    a.grad_q = g_mem + 2560;
    a.grad_k = g_mem + 2816;
    a.grad_q_weight = reinterpret_cast<float*>(g_mem + 3584);
    a.grad_k_weight = reinterpret_cast<float*>(g_mem + 3840);
    for (int i = 0; i < 3; ++i) {
        a.grad_q_out_stride[i] = a.grad_q_stride[i] = a.fwd.q_stride[i];
        a.grad_k_out_stride[i] = a.grad_k_stride[i] = a.fwd.k_stride[i];
    }
    return a;
}

template <typename F>
static int forward(F&& change) {
    fgqa_rope_args a = forward_args();
    change(a);
    return validate_rope(&a);
}
template <typename F>
static int backward(F&& change) {
    fgqa_rope_backward_args a = backward_args();
    change(a);
    return validate_rope_backward(&a);
}

// blocks_meet by all pairs
static bool all_pairs(int64_t a, int64_t la, int64_t b, int64_t lb, int64_t n0, int64_t s0, int64_t n1, int64_t s1) {
    for (int64_t i = 0; i < n0; ++i)
        for (int64_t j = 0; j < n1; ++j)
            for (int64_t k = 0; k < n0; ++k)
                for (int64_t l = 0; l < n1; ++l) {
                    const int64_t x = a + i * s0 + j * s1, y = b + k * s0 + l * s1;
                    if (x < y + lb && y < x + la) return true;
                }
    return false;
}

int main() {
    const int kBad = FGQA_ERR_INVALID_ARGUMENT, kNot = FGQA_ERR_UNSUPPORTED;
    typedef fgqa_rope_args A;
    typedef fgqa_rope_backward_args G;
    CHECK(validate_rope(nullptr) == kBad);
    CHECK(validate_rope_backward(nullptr) == kBad);
    CHECK(forward([](A&) {}) == FGQA_OK);
    CHECK(forward([](A& a) { a.batch = -1; }) == kBad);
    CHECK(forward([](A& a) { a.seqlen = -1; }) == kBad);
    CHECK(forward([](A& a) { a.num_q_heads = 0; }) == kBad);
    CHECK(forward([](A& a) { a.num_kv_heads = 0; }) == kBad);
    CHECK(forward([](A& a) { a.num_axes = 0; }) == kBad);
    CHECK(forward([](A& a) { a.rotary_dim = 144; }) == kBad);
    CHECK(forward([](A& a) { a.rotary_dim = 120; }) == kNot);
    CHECK(forward([](A& a) { a.rotary_dim = 0; a.positions = nullptr; a.inv_freq = nullptr; }) == FGQA_OK);
    CHECK(forward([](A& a) { a.head_dim = 136; }) == kNot);
    CHECK(forward([](A& a) { a.head_dim = 272; }) == kNot);
    CHECK(forward([](A& a) { a.head_dim = 256; }) == FGQA_OK);
    CHECK(forward([](A& a) { a.eps = -1.f; }) == kBad);
    CHECK(forward([](A& a) { a.eps = 1.f / 0.f; }) == kBad);
    CHECK(forward([](A& a) { a.eps = 0.f; }) == FGQA_OK);
    CHECK(forward([](A& a) { a.k_weight = nullptr; }) == kBad);
    CHECK(forward([](A& a) { a.q_weight = a.k_weight = nullptr; }) == FGQA_OK);
    CHECK(forward([](A& a) { a.q_weight = g_mem + 1; }) == kNot);
    CHECK(forward([](A& a) { a.q_weight = g_mem + 2; }) == kNot);
    CHECK(forward([](A& a) { a.q_weight = g_mem + 2; a.weights_bf16 = 1; }) == FGQA_OK);
    CHECK(forward([](A& a) { a.q = nullptr; }) == kBad);
    CHECK(forward([](A& a) { a.k_out = nullptr; }) == kBad);
    CHECK(forward([](A& a) { a.q = g_mem + 8; }) == kNot);
    CHECK(forward([](A& a) { a.q_stride[1] = 1028; }) == kNot);
    CHECK(forward([](A& a) { a.k_out_stride[2] = -128; }) == kBad);
    CHECK(forward([](A& a) { a.q_stride[0] = INT64_MAX; a.q_stride[1] = INT64_MAX; }) == kNot);
    CHECK(forward([](A& a) { a.positions = nullptr; }) == kBad);
    CHECK(forward([](A& a) { a.inv_freq = nullptr; }) == kBad);
    CHECK(forward([](A& a) { a.positions = g_mem + 2; }) == kNot);
    CHECK(forward([](A& a) { a.positions = g_mem + 4; }) == FGQA_OK);
    CHECK(forward([](A& a) { a.positions = g_mem + 4; a.positions_int64 = 1; }) == kNot);
    CHECK(forward([](A& a) { a.positions_stride[1] = -1; }) == kBad);
    CHECK(forward([](A& a) { a.positions_stride[2] = INT64_MAX; }) == kNot);
    CHECK(forward([](A& a) { a.axes = reinterpret_cast<int32_t*>(g_mem + 1); }) == kNot);
    CHECK(forward([](A& a) { a.q_out = const_cast<void*>(a.q); }) == FGQA_OK);
    CHECK(forward([](A& a) { a.q_out = const_cast<void*>(a.q); a.q_out_stride[0] += 8; }) == kBad);
    CHECK(forward([](A& a) { a.q_out = const_cast<void*>(a.k); }) == kBad);
    CHECK(forward([](A& a) { a.k_out = a.q_out; }) == kBad);
    CHECK(forward([](A& a) { a.batch = 0; a.q = nullptr; }) == FGQA_OK);
    CHECK(forward([](A& a) { a.batch = INT_MAX; a.seqlen = INT_MAX; }) == kNot);
    // 2^31 rows, and 2^32 threads, are one too many
    CHECK(forward([](A& a) { a.batch = 1 << 15; a.seqlen = 1 << 10; a.num_q_heads = 62; a.head_dim = a.rotary_dim = 64; }) == kNot);
    CHECK(forward([](A& a) { a.batch = 1 << 15; a.seqlen = 1 << 10; a.num_q_heads = 13; a.head_dim = a.rotary_dim = 128; }) == FGQA_OK);
    CHECK(forward([](A& a) { a.batch = 1 << 15; a.seqlen = 1 << 10; a.num_q_heads = 14; a.head_dim = a.rotary_dim = 128; }) == kNot);

    CHECK(backward([](G&) {}) == FGQA_OK);
    CHECK(backward([](G& g) { g.grad_q_weight = nullptr; }) == kBad);
    CHECK(backward([](G& g) { g.grad_k_weight = g.grad_q_weight; }) == kBad);
    CHECK(backward([](G& g) { g.grad_k_weight = reinterpret_cast<float*>(g_mem + 2); }) == kNot);
    CHECK(backward([](G& g) { g.grad_q = nullptr; }) == kBad);
    CHECK(backward([](G& g) { g.fwd.q = nullptr; }) == kBad);
    CHECK(backward([](G& g) { g.fwd.q = g.fwd.k = nullptr; g.fwd.q_weight = g.fwd.k_weight = nullptr; }) == FGQA_OK);
    CHECK(backward([](G& g) { g.fwd.q_out = g.fwd.k_out = nullptr; }) == FGQA_OK);
    CHECK(backward([](G& g) { g.grad_q_stride[2] = 4; }) == kNot);
    CHECK(backward([](G& g) { g.fwd.k_stride[2] = 4; }) == kNot);
    CHECK(backward([](G& g) { g.grad_q = const_cast<void*>(g.grad_q_out); }) == FGQA_OK);
    CHECK(backward([](G& g) { g.grad_q = const_cast<void*>(g.grad_q_out); g.grad_q_stride[1] += 8; }) == kBad);
    CHECK(backward([](G& g) { g.grad_q = const_cast<void*>(g.fwd.q); }) == kBad);
    CHECK(backward([](G& g) { g.grad_k = const_cast<void*>(g.grad_q_out); }) == kBad);
    CHECK(backward([](G& g) { g.fwd.seqlen = 0; g.grad_q = nullptr; }) == FGQA_OK);
    CHECK(backward([](G& g) { g.fwd.seqlen = 0; g.grad_q_weight = nullptr; }) == kBad);

    // every row of the plan's items has a place, and its workspace holds its workgroups' sums
    for (int64_t tokens : {1, 3, 31, 32, 33, 1000, 100000})
        for (int heads : {1, 2, 7, 128}) {
            fgqa_rope_args a = forward_args();
            a.batch = 1;
            a.seqlen = (int)tokens;
            a.num_q_heads = heads;
            const RopeGradPlan p = rope_grad_plan(a);
            CHECK(p.blocks[0] >= 1 && p.blocks[1] >= 1 && p.blocks[0] + p.blocks[1] <= 1026);
            CHECK(p.ws_bytes == (size_t)(p.blocks[0] + p.blocks[1]) * 128 * 4);
        }
    {
        fgqa_rope_args a = forward_args();   // 10 heads of 128
        a.batch = 1;
        a.seqlen = 52428;
        CHECK(!rope_streams(a, 2) && rope_streams(a, 3) && rope_heads_per(a) == 4);
        a.seqlen = 52429;
        CHECK(rope_streams(a, 2));
    }
    std::mt19937_64 rng(7);
    const int64_t sizes[] = {0, 1, 2, 5, 127, 128, 4096, INT_MAX, -1};
    auto pick = [&] { return (int32_t)sizes[rng() % 9]; };
    for (int i = 0; i < 200000; ++i) {
        fgqa_rope_backward_args g = backward_args();
        g.fwd.batch = pick();
        g.fwd.seqlen = pick();
        g.fwd.num_q_heads = pick();
        g.fwd.num_kv_heads = pick();
        g.fwd.head_dim = pick();
        g.fwd.rotary_dim = pick();
        g.fwd.num_axes = pick();
        for (int j = 0; j < 3; ++j) {
            g.fwd.q_stride[j] = (int64_t)(rng() >> (rng() % 64));
            g.grad_k_stride[j] = (int64_t)(rng() >> (rng() % 64));
            g.fwd.positions_stride[j] = (int64_t)(rng() >> (rng() % 64));
        }
        validate_rope(&g.fwd);
        if (validate_rope_backward(&g) == FGQA_OK && g.fwd.batch > 0 && g.fwd.seqlen > 0) {
            CHECK(rope_grad_plan(g.fwd).ws_bytes > 0);
            CHECK(rope_heads_per(g.fwd) > 0);
        }
    }

    // blocks: exact where the strides nest, never false where any two meet
    for (int i = 0; i < 200000; ++i) {
        auto some = [&](int n) { return (int64_t)(rng() % n); };
        const int64_t n0 = 1 + some(4), n1 = 1 + some(4), la = 1 + some(12), lb = 1 + some(12);
        const bool nested = some(4) != 0;
        const int64_t s1 = nested ? la + lb + some(20) : some(30), s0 = nested ? n1 * s1 + some(40) : some(60);
        const int64_t a = 1000, b = 1000 + some(2 * (n0 * s0 + n1 * s1) + 40) - (n0 * s0 + n1 * s1) - 20;
        const bool swap = some(2) != 0;
        const bool got = swap ? blocks_meet(a, la, b, lb, n1, s1, n0, s0) : blocks_meet(a, la, b, lb, n0, s0, n1, s1);
        const bool want = all_pairs(a, la, b, lb, n0, s0, n1, s1);
        CHECK(nested ? got == want : got || !want);
    }
    CHECK(blocks_meet(0, 10, (uintptr_t)1 << 62, 10, INT_MAX, INT64_MAX / INT_MAX, INT_MAX, 1));
    CHECK(!blocks_meet(0, 10, 20, 10, 0, 1, 1, 1));
    std::printf("%d failed\n", g_failed);
    return g_failed != 0;
}
