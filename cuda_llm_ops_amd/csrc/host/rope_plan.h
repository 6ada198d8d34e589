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

// Items of one tensor: a lane group takes up to heads_per rows of one token.
inline int64_t rope_items(int64_t tokens, int heads, int heads_per) { return tokens * ceil_div(heads, heads_per); }

// Heads of an item: 4 (1 where that leaves fewer than kRopeFullWaves waves).
int rope_heads_per(const fgqa_rope_args& a);

// Workgroups of the backward with weights, for Q and for K: the items shared out over
// at most kRopeGradBlocks, in proportion.
struct RopeGradPlan {
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
