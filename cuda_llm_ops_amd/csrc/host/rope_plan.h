// Host-only argument validation of include/fgqa_rope.h, apart from HIP like
// fgqa_plan.h, so that the CPU tests build it with sanitizers.
#pragma once

#include "fgqa_plan.h"
#include "fgqa_rope.h"

namespace fgqa {
namespace plan {

constexpr int kRopeMaxHeadDim = 256;
constexpr int kRopeThreads = 256;

// Lanes of a row, 16 elements each: the power of two from 4 that holds head_dim.
constexpr int rope_row_lanes(int head_dim) { return head_dim <= 64 ? 4 : head_dim <= 128 ? 8 : 16; }

// An item is up to `per` heads' rows of one token, `count` items a token.
struct RopeSlices {
    int per, count;
};

// Even slices of at most `most` heads.
inline RopeSlices rope_slices(int heads, int most) {
    const int count = (int)ceil_div(heads, most);
    return {(int)ceil_div(heads, count), count};
}

// Heads that a lane group of the forward takes: 4 (1 where that leaves fewer than kRopeWaves waves).
int rope_heads_per(const fgqa_rope_args& a);

// Whether the rows, read and written `passes` times, are more than the caches hold.
bool rope_streams(const fgqa_rope_args& a, int passes);

// Backward with weights: Q's and K's items, walked by at most kRopeGradBlocks
// workgroups that are shared out in proportion to their heads.
struct RopeGradPlan {
    RopeSlices slices[2];
    int blocks[2];
    size_t ws_bytes;   // fp32 [blocks[0] + blocks[1], head_dim]
};
RopeGradPlan rope_grad_plan(const fgqa_rope_args& a);

// The sizes that both directions use.
int validate_rope_sizes(const fgqa_rope_args& a);

// Sizes and addresses of a call; FGQA_OK with batch or seqlen zero, where no address is looked at.
int validate_rope(const fgqa_rope_args* a);
int validate_rope_backward(const fgqa_rope_backward_args* a);

}  // namespace plan
}  // namespace fgqa
