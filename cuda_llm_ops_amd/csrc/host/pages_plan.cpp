// Host-only argument validation of include/fgqa_pages.h (see pages_plan.h).
// Products of caller-supplied sizes are formed in 128 bits.
#include "pages_plan.h"

#include <initializer_list>

#include "kv_plan.h"

namespace fgqa {
namespace plan {

namespace {
typedef __int128 i128;

bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

int64_t round4(int64_t n) { return ceil_div(n, 4) * 4; }

// A table of n rows of `pages` cells.
int check_table(int n, int pages, int64_t stride, int page_size) {
    if (n < 0 || pages < 0 || stride < 0) return FGQA_ERR_INVALID_ARGUMENT;
    if ((i128)pages * page_size > kMaxTokens) return FGQA_ERR_UNSUPPORTED;
    if ((i128)n * stride + pages >= ((i128)1 << 60)) return FGQA_ERR_UNSUPPORTED;
    return FGQA_OK;
}

// (a table that is written: its rows lie apart)
bool rows_apart(int n, int pages, int64_t stride) { return n <= 1 || stride >= pages; }

// Rows of a launch of up to 16 workgroups each.
bool grid_ok(int64_t rows) { return rows < ((int64_t)1 << 20); }

// A page's 16-byte pieces are counted in 32 bits.
bool pages_ok(const fgqa_kv_cache& c) { return (i128)c.page_size * c.num_kv_heads * 16 < ((i128)1 << 30); }
}  // namespace

ForkLayout fork_layout(const fgqa_kv_fork_args& a) {
    ForkLayout l;
    const int64_t words = page_words(a.cache.num_pages);
    l.bits = 0;
    l.before = l.bits + round4(words);
    l.row_first = l.before + round4(words + 1);
    l.first = l.row_first + round4(a.new_batch);
    l.total = l.first + round4(a.batch);
    return l;
}

CompactLayout compact_layout(const fgqa_kv_compact_args& a) {
    CompactLayout l;
    const int64_t words = page_words(a.cache.num_pages);
    l.live = 0;
    l.held = l.live + round4(words);
    l.live_before = l.held + round4(words);
    l.open_before = l.live_before + round4(words + 1);
    l.edge = l.open_before + round4(words + 1);
    l.total = l.edge + 4;
    return l;
}

int validate_kv_fork_sizes(const fgqa_kv_fork_args* a) {
    if (a == nullptr) return FGQA_ERR_INVALID_ARGUMENT;
    int st = validate_cache(a->cache, true, false);
    if (st != FGQA_OK) return st;
    st = check_table(a->batch, a->max_pages, a->block_table_stride, a->cache.page_size);
    if (st == FGQA_OK) st = check_table(a->new_batch, a->new_max_pages, a->new_block_table_stride, a->cache.page_size);
    if (st != FGQA_OK) return st;
    if (!rows_apart(a->new_batch, a->new_max_pages, a->new_block_table_stride)) return FGQA_ERR_INVALID_ARGUMENT;
    return grid_ok(a->new_batch) && grid_ok(a->batch) && pages_ok(a->cache) ? FGQA_OK : FGQA_ERR_UNSUPPORTED;
}

int validate_kv_fork(const fgqa_kv_fork_args* a) {
    int st = validate_kv_fork_sizes(a);
    if (st != FGQA_OK) return st;
    st = validate_cache_pointers(a->cache, true);
    if (st != FGQA_OK) return st;
    if (!written_apart(a->cache) || a->num_free == nullptr) return FGQA_ERR_INVALID_ARGUMENT;
    const bool rows = a->new_batch > 0;
    if (rows && a->new_seqlens == nullptr) return FGQA_ERR_INVALID_ARGUMENT;
    if (rows && a->new_max_pages > 0 && a->new_block_table == nullptr) return FGQA_ERR_INVALID_ARGUMENT;
    if (rows && a->batch > 0 && a->seqlens == nullptr) return FGQA_ERR_INVALID_ARGUMENT;
    if (rows && a->batch > 0 && a->max_pages > 0 && a->block_table == nullptr) return FGQA_ERR_INVALID_ARGUMENT;
    // (without a list, row i goes on from row i: one is there for each)
    if (a->parents == nullptr && a->new_batch > a->batch) return FGQA_ERR_INVALID_ARGUMENT;
    for (const void* p : {(const void*)a->block_table, (const void*)a->seqlens, (const void*)a->parents,
                          (const void*)a->new_lens, (const void*)a->new_block_table, (const void*)a->new_seqlens,
                          (const void*)a->num_free})
        if (!aligned4(p)) return FGQA_ERR_UNSUPPORTED;
    if (rows && (a->new_block_table == a->block_table || a->new_seqlens == a->seqlens || a->new_seqlens == a->new_lens ||
                 a->new_seqlens == a->parents))
        if (a->batch > 0) return FGQA_ERR_INVALID_ARGUMENT;
    return FGQA_OK;
}

int validate_kv_compact_sizes(const fgqa_kv_compact_args* a) {
    if (a == nullptr) return FGQA_ERR_INVALID_ARGUMENT;
    int st = validate_cache(a->cache, true, false);
    if (st != FGQA_OK) return st;
    st = check_table(a->batch, a->max_pages, a->block_table_stride, a->cache.page_size);
    if (st == FGQA_OK) st = check_table(a->batch, a->max_pages, a->new_block_table_stride, a->cache.page_size);
    if (st != FGQA_OK) return st;
    if (!rows_apart(a->batch, a->max_pages, a->new_block_table_stride)) return FGQA_ERR_INVALID_ARGUMENT;
    return grid_ok(a->batch) && pages_ok(a->cache) ? FGQA_OK : FGQA_ERR_UNSUPPORTED;
}

int validate_kv_compact(const fgqa_kv_compact_args* a) {
    int st = validate_kv_compact_sizes(a);
    if (st != FGQA_OK) return st;
    st = validate_cache_pointers(a->cache, true);
    if (st != FGQA_OK) return st;
    if (!written_apart(a->cache) || a->num_used == nullptr) return FGQA_ERR_INVALID_ARGUMENT;
    if (a->batch > 0 && a->seqlens == nullptr) return FGQA_ERR_INVALID_ARGUMENT;
    if (a->batch > 0 && a->max_pages > 0 &&
        (a->block_table == nullptr || a->new_block_table == nullptr || a->new_block_table == a->block_table))
        return FGQA_ERR_INVALID_ARGUMENT;
    for (const void* p : {(const void*)a->block_table, (const void*)a->seqlens, (const void*)a->new_block_table,
                          (const void*)a->num_used})
        if (!aligned4(p)) return FGQA_ERR_UNSUPPORTED;
    return FGQA_OK;
}

}  // namespace plan
}  // namespace fgqa
