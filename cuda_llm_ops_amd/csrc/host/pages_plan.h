// Host-only argument validation and workspace layout of include/fgqa_pages.h, apart
// from HIP like fgqa_plan.h, so that the CPU tests build it with sanitizers.
#pragma once

#include "fgqa_pages.h"
#include "fgqa_plan.h"

namespace fgqa {
namespace plan {

// 32 pages a word.
inline int64_t page_words(int num_pages) { return ceil_div(num_pages, 32); }

// int32 offsets into the workspaces.
struct ForkLayout {
    int64_t bits;        // [words]: pages in use
    int64_t before;      // [words + 1]: free pages before each word
    int64_t row_first;   // [new_batch]: fresh pages of the rows before each
    int64_t first;       // [batch]: the first new row of each old one
    int64_t total;
};
ForkLayout fork_layout(const fgqa_kv_fork_args& a);

struct CompactLayout {
    int64_t live, held;                // [words] each
    int64_t live_before, open_before;  // [words + 1]: pages in use, and pages not held, before each word
    int64_t edge;                      // [1]: the first page past the kept range
    int64_t total;
};
CompactLayout compact_layout(const fgqa_kv_compact_args& a);

// int32 of LDS of a workgroup that plans for itself; 0 where the call's sizes are too large
// for that (the general form, with a workspace).
constexpr int kAloneThreads = 1024;
int fork_alone_ints(const fgqa_kv_fork_args& a);
int compact_alone_ints(const fgqa_kv_compact_args& a);
// Pages that can move: at most half of all, and no more than the table has cells.
inline int64_t compact_moves(const fgqa_kv_compact_args& a) {
    const int64_t cells = (int64_t)a.batch * a.max_pages;
    return cells < a.cache.num_pages / 2 ? cells : a.cache.num_pages / 2;
}
// Whether workgroups that plan for themselves move them: smaller ones copy large amounts faster.
bool compact_moves_little(const fgqa_kv_compact_args& a);
// Cells of an old row that a new one can hold.
inline int fork_width(const fgqa_kv_fork_args& a) { return a.max_pages < a.new_max_pages ? a.max_pages : a.new_max_pages; }

// FGQA_OK with new_batch 0 too (num_free is still written); a cache without pages is refused.
int validate_kv_fork(const fgqa_kv_fork_args* a);
int validate_kv_compact(const fgqa_kv_compact_args* a);
// The sizes alone, which the workspace follows from.
int validate_kv_fork_sizes(const fgqa_kv_fork_args* a);
int validate_kv_compact_sizes(const fgqa_kv_compact_args* a);

// ---------------------------------------------------------------- decode of sequences that begin alike
constexpr int kSharedRows = 128;       // query rows (sequences times heads of a KV head) of a workgroup
constexpr int kSharedMaxGroups = 4096;
constexpr int kSharedChunk = 128;      // tokens that the work is cut in multiples of

// Tokens of a cut, of `total` of all row tiles and sequences.
constexpr int64_t shared_chunk(int64_t total, int slots) {
    const int64_t even = (total + slots - 1) / slots;
    const int64_t c = (even + kSharedChunk - 1) / kSharedChunk * kSharedChunk;
    return c < kSharedChunk ? kSharedChunk : c;
}
// What a range of n > 0 tokens is cut into: equal pieces of a multiple of `step` that are
// at most a chunk (a multiple of step, and 2^30 at most).
constexpr int shared_piece(int n, int chunk, int step) {
    const int pieces = (int)(((uint32_t)n + (uint32_t)chunk - 1) / (uint32_t)chunk);
    const uint32_t even = ((uint32_t)n + (uint32_t)pieces - 1) / (uint32_t)pieces;
    return (int)((even + (uint32_t)step - 1) / (uint32_t)step * (uint32_t)step);
}

// Sizes that a call's kernels and workspace are bounded by, whatever the lengths.
struct SharedPlan {
    int slots;             // workgroups of one KV head that run at once
    int max_items;         // of one KV head
    int64_t max_rows;      // of partials
    size_t part_ml_off, items_off, seqs_off, count_off, total;   // bytes; partial O at 0
};
constexpr int kSharedItemInts = 8, kSharedSeqInts = 8;
// The call without its groups, over a cache with block scales.
fgqa_decode_blocks_args as_decode_blocks(const fgqa_decode_shared_args* a);
// Whether a call is that one: with few tokens its launch and chain of loads cost more than
// reading what is shared once for each sequence.
bool shared_as_blocks(const fgqa_decode_shared_args* a, int cus);
// What the decode checks of its arguments, an e4m3 cache of the same sizes for int8.
fgqa_decode_paged_args as_decode_paged(const fgqa_decode_shared_args* a);
int validate_decode_shared(const fgqa_decode_shared_args* a);
int validate_decode_shared_pointers(const fgqa_decode_shared_args* a);
int plan_decode_shared(const fgqa_decode_shared_args* a, int cus, SharedPlan* plan);

}  // namespace plan
}  // namespace fgqa
