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

// An address, and whether the call uses it.
struct Used {
    const void* at;
    bool used;
};

// Each output is at an address of its own (workgroups that plan for themselves would read what others write).
template <size_t kOut, size_t kIn>
bool outputs_apart(const Used (&out)[kOut], const Used (&in)[kIn]) {
    for (size_t i = 0; i < kOut; ++i) {
        if (!out[i].used) continue;
        for (size_t j = 0; j < i; ++j)
            if (out[j].used && out[i].at == out[j].at) return false;
        for (const Used& x : in)
            if (x.used && x.at == out[i].at) return false;
    }
    return true;
}

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

namespace {
// A table that a workgroup of kAloneThreads reads in passing, and LDS for its rows and bits
// that any kernel has.  Planning in each workgroup and in launches of its own took, on
// tables of n cells: fork 8.4 and 17.5 us (n = 2,016), 18 and 21 (n = 32,256), compact 9.6
// and 16.4, 18 and 24.
constexpr int64_t kAloneCells = 32768, kAloneInts = 15360;
}  // namespace

int fork_alone_ints(const fgqa_kv_fork_args& a) {
    const int64_t ints = 2 * page_words(a.cache.num_pages) + 1 + 3 * (int64_t)a.batch + 4 * (int64_t)a.new_batch;
    const bool small = (int64_t)a.batch * fork_width(a) <= kAloneCells && (int64_t)a.new_batch * a.new_max_pages < ((int64_t)1 << 30);
    return small && ints <= kAloneInts ? (int)ints : 0;
}

int compact_alone_ints(const fgqa_kv_compact_args& a) {
    const int64_t ints = 4 * page_words(a.cache.num_pages) + 2 + a.batch;
    return (int64_t)a.batch * a.max_pages <= kAloneCells && ints <= kAloneInts ? (int)ints : 0;
}

bool compact_moves_little(const fgqa_kv_compact_args& a) {
    // Bytes of the pages: with 1.2 GB workgroups of 256 threads take 160 us and 1024 threads, which plan too, 176.
    constexpr int64_t kAloneMoves = (int64_t)1 << 29;
    const int64_t page = (int64_t)a.cache.page_size * a.cache.num_kv_heads * (a.cache.kv_dtype == FGQA_KV_BF16 ? 512 : 256);
    return compact_moves(a) <= kAloneMoves / page;
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
    const bool old = rows && a->batch > 0, cells = rows && a->new_max_pages > 0;
    const Used out[] = {{a->num_free, true}, {a->new_seqlens, rows}, {a->new_block_table, cells}};
    const Used in[] = {{a->seqlens, old}, {a->block_table, old}, {a->parents, rows}, {a->new_lens, rows}, {a->held, true}};
    return outputs_apart(out, in) ? FGQA_OK : FGQA_ERR_INVALID_ARGUMENT;
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
    const bool cells = a->batch > 0 && a->max_pages > 0;
    if (cells && (a->block_table == nullptr || a->new_block_table == nullptr)) return FGQA_ERR_INVALID_ARGUMENT;
    const Used out[] = {{a->num_used, true}, {a->new_block_table, cells}};
    const Used in[] = {{a->seqlens, a->batch > 0}, {a->block_table, cells}, {a->held, true}};
    if (!outputs_apart(out, in)) return FGQA_ERR_INVALID_ARGUMENT;
    for (const void* p : {(const void*)a->block_table, (const void*)a->seqlens, (const void*)a->new_block_table,
                          (const void*)a->num_used})
        if (!aligned4(p)) return FGQA_ERR_UNSUPPORTED;
    return FGQA_OK;
}

fgqa_decode_blocks_args as_decode_blocks(const fgqa_decode_shared_args* a) {
    fgqa_decode_blocks_args b = {};
    b.cache = a->cache;
    b.q = a->q;
    b.o = a->o;
    b.lse = a->lse;
    b.block_table = a->block_table;
    b.seqlens = a->seqlens;
    b.batch = a->batch;
    b.max_seqlen = a->max_seqlen;
    b.num_q_heads = a->num_q_heads;
    b.scale = a->scale;
    for (int i = 0; i < 2; ++i) {
        b.q_stride[i] = a->q_stride[i];
        b.o_stride[i] = a->o_stride[i];
    }
    b.block_table_stride = a->block_table_stride;
    b.workspace = a->workspace;
    b.workspace_bytes = a->workspace_bytes;
    return b;
}

bool shared_as_blocks(const fgqa_decode_shared_args* a, int cus) {
    // Tokens of a KV head for each CU, of sequences as long as they may be.  Each on their own and together, e4m3
    // to int8: 33,600 tokens of all KV heads 13.2 and 16.7 to 17.5 us (8 samples), 134,000 14 and 19.3 to 19.9, 282,000 17 to
    // 18.9 and 22.6 to 23.1, 352,000 17.7 to 19.9 and 23.3 to 23.7, 422,000 (24 samples) 18.3 to 35.2 and 28.5 to 26.6,
    // 480,000 20.5 to 23.6 and 23.6 to 24.5, 550,000 31.8 to 36 and 27.2 to 27.7: the rule ends where the first are always less.
    // (Without block scales the decode on their own takes longer from the start: 23.1 and 13.8.)
    constexpr int64_t kAloneTokens = 1152;
    return a->cache.k_scales != nullptr &&
           (i128)a->batch * a->cache.num_kv_heads * a->max_seqlen <= (i128)kAloneTokens * (cus > 0 ? cus : 256);
}

fgqa_decode_paged_args as_decode_paged(const fgqa_decode_shared_args* a) {
    const fgqa_decode_blocks_args b = as_decode_blocks(a);
    fgqa_decode_paged_args p = as_decode_paged(&b);
    if (a->cache.kv_dtype == FGQA_KV_BF16) p.kv_dtype = FGQA_KV_BF16;
    if (a->cache.kv_dtype == FGQA_KV_FP8_E4M3 && a->cache.k_scales == nullptr) {
        p.k_scale = a->cache.k_scale;
        p.v_scale = a->cache.v_scale;
    }
    return p;
}

int validate_decode_shared(const fgqa_decode_shared_args* a) {
    if (a == nullptr) return FGQA_ERR_INVALID_ARGUMENT;
    int st = validate_cache(a->cache, true, false);
    if (st != FGQA_OK) return st;
    const fgqa_decode_paged_args p = as_decode_paged(a);
    st = validate_paged(&p);
    if (st != FGQA_OK) return st;
    if (a->num_groups < 0) return FGQA_ERR_INVALID_ARGUMENT;
    // (the merge's grid has a row for each sequence)
    return a->num_groups <= kSharedMaxGroups && a->batch < (1 << 15) ? FGQA_OK : FGQA_ERR_UNSUPPORTED;
}

int validate_decode_shared_pointers(const fgqa_decode_shared_args* a) {
    const fgqa_decode_paged_args p = as_decode_paged(a);
    int st = validate_paged_pointers(&p);
    if (st != FGQA_OK || a->batch == 0) return st;
    if (a->num_groups > 0) {
        if (a->group_starts == nullptr || a->shared_lens == nullptr) return FGQA_ERR_INVALID_ARGUMENT;
        if (!aligned4(a->group_starts) || !aligned4(a->shared_lens)) return FGQA_ERR_UNSUPPORTED;
    }
    return a->max_seqlen == 0 ? FGQA_OK : validate_cache_pointers(a->cache, true);
}

// With C tokens a chunk, C >= (all rows of tiles' and sequences' tokens) / slots, the items of one
// KV head are at most slots + tiles + sequences (each cut leaves one rest), and their
// rows of partials, at most 128 (and the batch's) a tile's chunk and the group's a sequence's.
int plan_decode_shared(const fgqa_decode_shared_args* a, int cus, SharedPlan* plan) {
    if (cus <= 0) cus = 256;
    const int64_t hkv = a->cache.num_kv_heads, group = a->num_q_heads / hkv;
    const int64_t rows = (int64_t)a->batch * group;   // of one KV head
    const int64_t tiles = rows / kSharedRows + (a->num_groups < a->batch ? a->num_groups : a->batch);
    const int64_t slots = ceil_div(2 * (int64_t)cus, hkv);
    const int64_t items = slots + tiles + a->batch;
    if ((i128)items * hkv >= ((i128)1 << 24)) return FGQA_ERR_UNSUPPORTED;
    plan->slots = (int)slots;
    plan->max_items = (int)items;
    plan->max_rows = hkv * (slots * (rows < kSharedRows ? (rows > group ? rows : group) : kSharedRows) + 2 * rows);
    if (plan->max_rows >= ((int64_t)1 << 31)) return FGQA_ERR_UNSUPPORTED;
    auto round = [](size_t n) { return (n + 255) / 256 * 256; };
    plan->part_ml_off = round((size_t)plan->max_rows * kHeadDim * 4);
    plan->items_off = plan->part_ml_off + round((size_t)plan->max_rows * 2 * 4);
    plan->seqs_off = plan->items_off + round((size_t)items * kSharedItemInts * 4);
    plan->count_off = plan->seqs_off + round((size_t)a->batch * kSharedSeqInts * 4);
    plan->total = plan->count_off + 256;
    return FGQA_OK;
}

}  // namespace plan
}  // namespace fgqa
