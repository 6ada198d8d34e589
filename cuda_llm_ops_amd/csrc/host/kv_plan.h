// Host-only argument validation of the paged KV cache's C ABI (include/fgqa_kv.h),
// apart from HIP like fgqa_plan.h, so that the CPU tests build it with sanitizers.
#pragma once

#include "fgqa_kv.h"
#include "fgqa_plan.h"

namespace fgqa {
namespace plan {

// Sizes and addresses of a call; FGQA_OK with batch (or what it would write)
// zero, where nothing is launched and no address is looked at.
int validate_kv_append(const fgqa_kv_append_args* a);
int validate_kv_weights(const fgqa_kv_weights_args* a);
int validate_kv_evict(const fgqa_kv_evict_args* a);

// The block-scaled decode's cache and scales; then what fgqa_decode_paged
// checks, on its arguments for the same call (an e4m3 cache: the same element size).
int validate_decode_blocks(const fgqa_decode_blocks_args* a);
int validate_decode_blocks_pointers(const fgqa_decode_blocks_args* a);
fgqa_decode_paged_args as_decode_paged(const fgqa_decode_blocks_args* a);

// Heads' items that the chip holds at once in the block-scaled decode: 256 CUs
// times 4 heads of 2 waves, or 2 of 4.
constexpr int block_item_slots(int num_kv_heads) { return num_kv_heads % 4 == 0 ? 1024 : kDecodeItemSlots; }

// Tokens per split of a block-scaled decode without a given length on a device of
// `cus` CUs, or 0: the batch shared out evenly over teams.
int blocks_split(int64_t batch, int64_t num_kv_heads, int64_t max_seqlen, int cus);

// The plan of a block-scaled decode on a device of `cus` CUs (0, unknown: 256, what
// the teams are made for): splits of the given length or of blocks_split() (teams
// 0, no work list), or teams, which become splits where the workspace holds only
// those (fit_workspace).
int plan_blocks(const fgqa_decode_paged_args* a, int cus, DecodePlan* plan);

inline int log2_of(int power_of_two) {
    int shift = 0;
    while ((1 << shift) < power_of_two) ++shift;
    return shift;
}

// Tokens an eviction leaves of the longest sequence at most, and its longest length.
inline int evict_tokens(const fgqa_kv_evict_args& a) { return a.max_tokens > a.max_seqlen ? a.max_tokens : a.max_seqlen; }
inline int evict_most(const fgqa_kv_evict_args& a) {
    return a.new_tokens > 0 && a.new_tokens < a.budget ? a.new_tokens : a.budget;
}

// Most pages of one sequence that `max_new` tokens in a row touch.
inline int64_t append_pages(int64_t max_new, int64_t page_size) { return (max_new + page_size - 2) / page_size + 1; }

constexpr int kWeightsTokens = 64;   // of a wave's item in the weights kernel

// Waves of one (sequence, KV head) in the weights kernel, each of which takes every
// so many-th item: one an item, but kWeightsWaves in all (where a batch needs no
// more than one each).  What decides is a capacity far above the lengths, whose
// empty waves only end: 64 sequences of up to 2048 tokens, 8 heads, take 17 us with
// max_seqlen 2048; with 131072 they took 100 at an item a wave and take 25 so.
constexpr int64_t kWeightsWaves = 1 << 17;
inline int weights_waves(int64_t batch, int64_t num_kv_heads, int64_t max_seqlen) {
    const int64_t items = ceil_div(max_seqlen, kWeightsTokens), rows = batch * num_kv_heads;
    const int64_t most = rows >= kWeightsWaves ? 1 : kWeightsWaves / rows;
    return (int)(items < most ? items : most);
}

// A block of the append and the eviction is a wave's, or a workgroup's of 4.
constexpr int kWavePageRows = 64;

}  // namespace plan
}  // namespace fgqa
