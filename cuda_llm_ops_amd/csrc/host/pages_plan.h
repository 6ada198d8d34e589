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

// FGQA_OK with new_batch 0 too (num_free is still written); a cache without pages is refused.
int validate_kv_fork(const fgqa_kv_fork_args* a);
int validate_kv_compact(const fgqa_kv_compact_args* a);
// The sizes alone, which the workspace follows from.
int validate_kv_fork_sizes(const fgqa_kv_fork_args* a);
int validate_kv_compact_sizes(const fgqa_kv_compact_args* a);

}  // namespace plan
}  // namespace fgqa
