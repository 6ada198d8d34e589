// The norm and rotation's items: every head of a token in one slice, none in two, and as many
// workgroups as the plan has room for.  Built with sanitizers.
#include <climits>
#include <cstdio>

#include "rope_plan.h"

using namespace fgqa::plan;

static int g_failed = 0;
#define CHECK(x)                                        \
    do {                                                \
        if (!(x)) {                                     \
            ++g_failed;                                 \
            std::printf("line %d: %s\n", __LINE__, #x); \
        }                                               \
    } while (0)

// What a slice of a token's heads does not take the next one does, and the last is not empty.
static bool covers(const RopeSlices& s, int heads, int most) {
    return s.per >= 1 && s.per <= most && s.count >= 1 && (int64_t)s.per * s.count >= heads && (int64_t)s.per * (s.count - 1) < heads;
}

int main() {
    const int all_heads[] = {1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 28, 31, 32, 33, 64, 127, 128, 1000};
    const int all_most[] = {1, 2, 4, 8};
    for (int heads : all_heads)
        for (int most : all_most) CHECK(covers(rope_slices(heads, most), heads, most));

    const int all_tokens[] = {1, 3, 31, 32, 33, 1000, 4501, 100000};
    const int all_dims[] = {16, 64, 80, 128, 176, 256};
    for (int tokens : all_tokens)
        for (int hq : all_heads)
            for (int hkv : all_heads)
                for (int dim : all_dims) {
                    fgqa_rope_args a = {};
                    a.batch = 1;
                    a.seqlen = tokens;
                    a.num_q_heads = hq;
                    a.num_kv_heads = hkv;
                    a.head_dim = a.rotary_dim = dim;
                    const int per = rope_heads_per(a);
                    CHECK(per == 1 || per == 4);
                    const RopeGradPlan p = rope_grad_plan(a);
                    CHECK(covers(p.slices[0], hq, 8) && covers(p.slices[1], hkv, 8));
                    CHECK(p.blocks[0] >= 1 && p.blocks[1] >= 1 && p.blocks[0] + p.blocks[1] <= 768);
                    // no workgroup without an item
                    const int64_t groups = kRopeThreads / rope_row_lanes(dim);
                    const int heads[] = {hq, hkv};
                    for (int i = 0; i < 2; ++i) {
                        const int64_t items = (int64_t)tokens * p.slices[i].count;
                        CHECK(((int64_t)p.blocks[i] - 1) * groups < items && heads[i] > 0);
                    }
                    CHECK(p.ws_bytes == (size_t)(p.blocks[0] + p.blocks[1]) * (size_t)dim * 4);
                }
    std::printf("%d failed\n", g_failed);
    return g_failed != 0;
}
