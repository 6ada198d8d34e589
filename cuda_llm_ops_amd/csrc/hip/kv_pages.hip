// Forking and freeing the sequences of a paged KV cache, and moving the pages in use
// together (include/fgqa_pages.h).
//
// Which pages are in use is worked out anew for each call from the block table, as one bit a
// page; a free page's number is found from the bits and a running count of them by words
// (a search over the words, then over one word's bits).  So there is no list of free
// pages to keep, and equal tables give equal results.
#include <algorithm>

#include "fgqa_device.h"
#include "fgqa_internal.h"
#include "kv_cache_params.h"
#include "../host/pages_plan.h"

namespace fgqa {
namespace {

constexpr int kThreads = 256;
constexpr int kScanThreads = 1024;
constexpr int kWordsPerScan = 4;   // of a thread

// A page's rows as 16-byte pieces, and how many slots of it are copied.
struct CopyShape {
    int piece_log2;     // pieces of a row: 8 or 16
    FastDiv div_heads;
};

// Slots [0, slots) of page src to page dst, K and V and their scales: pieces first,
// first + step, ... of all.
__device__ __forceinline__ void copy_slots(const CacheParams& c, const CopyShape& sh, int src, int dst, int slots, int first,
                                           int step) {
    const int total = (slots * c.hkv) << sh.piece_log2;   // (a page's bytes / 16 stay below 2^31)
    constexpr int kAhead = 4;
    for (int x0 = first; x0 < total; x0 += kAhead * step) {
        u32x4_t v[kAhead][2];
        int64_t at[kAhead][2];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int x = min(x0 + i * step, total - 1);   // (past the end: the last piece again)
            const int row = x >> sh.piece_log2;
            const int slot = fast_div(row, sh.div_heads);
            const int h = row - slot * c.hkv;
#pragma unroll
            for (int kv = 0; kv < 2; ++kv) {
                at[i][kv] = slot * c.slot[kv] + h * c.head[kv] + 16 * (x & ((1 << sh.piece_log2) - 1));
                v[i][kv] = *reinterpret_cast<const u32x4_t*>(c.data[kv] + src * c.page[kv] + at[i][kv]);
            }
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
#pragma unroll
            for (int kv = 0; kv < 2; ++kv)
                if (x0 + i * step < total) *reinterpret_cast<u32x4_t*>(c.data[kv] + dst * c.page[kv] + at[i][kv]) = v[i][kv];
    }
    if (c.scales[0] != nullptr) {
        for (int h = first; h < c.hkv; h += step)
#pragma unroll
            for (int kv = 0; kv < 2; ++kv) {
                float* s = c.scales[kv] + h * c.scale_head[kv];
                s[dst * c.scale_page[kv]] = s[src * c.scale_page[kv]];
            }
    }
}

// The last index w of words' counts (before[0] = 0, ascending, n + 1 of them) with before[w] <= k < before[n].
template <typename F>
__device__ __forceinline__ int word_of(int n, int k, F&& before) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (before(mid) <= k) lo = mid;
        else hi = mid;
    }
    return lo;
}

// The place of the k-th set bit (k < the number of them).
__device__ __forceinline__ int bit_of(uint32_t bits, int k) {
    for (int i = 0; i < k; ++i) bits &= bits - 1;
    return __builtin_ctz(bits);
}

// The pages of word w that there are.
__device__ __forceinline__ uint32_t word_mask(int w, int num_pages) {
    const int left = num_pages - 32 * w;
    return left >= 32 ? 0xffffffffu : (1u << left) - 1;
}

// held[32w .. 32w + 31] as bits.
__device__ __forceinline__ uint32_t held_word(const uint8_t* held, int w, int num_pages) {
    uint32_t bits = 0;
    if (held != nullptr) {
        const int n = min(32, num_pages - 32 * w);
        for (int i = 0; i < n; ++i) bits |= (held[(int64_t)32 * w + i] != 0 ? 1u : 0u) << i;
    }
    return bits;
}

// before[w]: the sum of count(0 .. w - 1), for w <= words; a workgroup.
template <typename F>
__device__ __forceinline__ int scan_words(int words, int32_t* before, int* s_wave, F&& count) {
    int carry = 0;
    for (int w0 = 0; w0 < words; w0 += kScanThreads * kWordsPerScan) {
        int n[kWordsPerScan], sum = 0, total;
#pragma unroll
        for (int i = 0; i < kWordsPerScan; ++i) {
            const int w = w0 + (int)threadIdx.x * kWordsPerScan + i;
            n[i] = w < words ? count(w) : 0;
            sum += n[i];
        }
        int at = carry + block_exclusive_scan<kScanThreads, true>(sum, s_wave, &total);
#pragma unroll
        for (int i = 0; i < kWordsPerScan; ++i) {
            const int w = w0 + (int)threadIdx.x * kWordsPerScan + i;
            if (w < words) before[w] = at;
            at += n[i];
        }
        carry += total;
    }
    if (threadIdx.x == 0) before[words] = carry;
    return carry;
}

// ---------------------------------------------------------------- fork
struct ForkParams {
    CacheParams c;
    CopyShape shape;
    const int32_t* table;
    const int32_t* seqlens;
    const int32_t* parents;
    const int32_t* new_lens;
    const uint8_t* held;
    int32_t* new_table;
    int32_t* new_seqlens;
    int32_t* num_free;
    int64_t stride, new_stride;
    int batch, new_batch, new_max_pages, max_tokens;   // max_tokens: of an old row that a new one can hold
    int words;
    uint32_t* bits;
    int32_t* before;
    int32_t* row_first;
    int32_t* first;
};

// What a new row takes from its old one.
struct ForkRow {
    int p, len, full, part;
    bool there;         // an old row
};
__device__ __forceinline__ ForkRow fork_row(const ForkParams& p, int i) {
    ForkRow r;
    r.p = p.parents != nullptr ? p.parents[i] : i;
    r.there = r.p >= 0 && r.p < p.batch;
    r.len = r.there ? min(max(p.seqlens[r.p], 0), p.max_tokens) : 0;
    r.full = r.len >> p.c.page_shift;
    r.part = r.len & ((1 << p.c.page_shift) - 1);
    return r;
}
__device__ __forceinline__ bool is_page(const CacheParams& c, int page) { return page >= 0 && page < c.num_pages; }

// The partly filled page of a row (its cell r.full), and whether the row keeps it.
__device__ __forceinline__ bool keeps_last(const ForkParams& p, const ForkRow& r, int i, const int32_t* first, int* page) {
    *page = p.table[r.p * p.stride + r.full];
    if (!is_page(p.c, *page)) return true;
    return first[r.p] == i && (p.held == nullptr || p.held[*page] == 0);
}

// Pages of its own that row i wants; *kept: cells before them.
__device__ __forceinline__ int fresh_pages(const ForkParams& p, const ForkRow& r, int i, const int32_t* first, int* kept) {
    int page;
    *kept = r.full + (r.part > 0 && keeps_last(p, r, i, first, &page) ? 1 : 0);
    const int64_t more = p.new_lens != nullptr ? max(p.new_lens[i], 0) : 0;
    const int64_t cells = (r.len + more + (1 << p.c.page_shift) - 1) >> p.c.page_shift;
    return (int)min(cells, (int64_t)p.new_max_pages) - *kept;
}

__global__ __launch_bounds__(kThreads) void fork_clear_kernel(ForkParams p) {
    const int64_t at = (int64_t)blockIdx.x * kThreads + threadIdx.x, step = (int64_t)gridDim.x * kThreads;
    for (int64_t w = at; w < p.words; w += step) p.bits[w] = held_word(p.held, (int)w, p.c.num_pages);
    for (int64_t b = at; b < p.batch; b += step) p.first[b] = INT32_MAX;
}

// The pages that new rows have from old ones, and each old row's first new one.
__global__ __launch_bounds__(kThreads) void fork_mark_kernel(ForkParams p) {
    const int i = blockIdx.x;
    const ForkRow r = fork_row(p, i);
    if (!r.there) return;
    if (blockIdx.y == 0 && threadIdx.x == 0) atomicMin(&p.first[r.p], i);
    const int cells = r.full + (r.part > 0 ? 1 : 0);
    for (int j = blockIdx.y * kThreads + threadIdx.x; j < cells; j += gridDim.y * kThreads) {
        const int page = p.table[r.p * p.stride + j];
        if (is_page(p.c, page)) atomicOr(&p.bits[page >> 5], 1u << (page & 31));
        if (j < r.full) p.new_table[i * p.new_stride + j] = page;
    }
}

// Counts of free pages by words and of fresh ones by rows.
__global__ __launch_bounds__(kScanThreads) void fork_scan_kernel(ForkParams p) {
    __shared__ int s_wave[kScanThreads / kWave];
    const int free_pages = scan_words(p.words, p.before, s_wave,
                                      [&](int w) { return __popc(~p.bits[w] & word_mask(w, p.c.num_pages)); });
    __shared__ int64_t s_wave64[kScanThreads / kWave];
    int64_t wanted = 0;   // (rows times cells can pass 2^31)
    for (int i0 = 0; i0 < p.new_batch; i0 += kScanThreads) {
        const int i = i0 + (int)threadIdx.x;
        int kept;
        int64_t total;
        const int64_t n = i < p.new_batch ? fresh_pages(p, fork_row(p, i), i, p.first, &kept) : 0;
        const int64_t at = block_exclusive_scan<kScanThreads, true>(n, s_wave64, &total);
        if (i < p.new_batch) p.row_first[i] = (int)min(wanted + at, (int64_t)INT32_MAX);
        wanted += total;
    }
    if (threadIdx.x == 0) *p.num_free = (int)max((int64_t)free_pages - wanted, (int64_t)INT32_MIN);
}

// The rows' other cells, and the copies of partly filled pages.
__global__ __launch_bounds__(kThreads) void fork_fill_kernel(ForkParams p) {
    const int i = blockIdx.x;
    const ForkRow r = fork_row(p, i);
    int kept;
    const int fresh = fresh_pages(p, r, i, p.first, &kept);
    const int first = p.row_first[i], free_pages = p.before[p.words];
    auto fresh_page = [&](int n) {
        if (n >= free_pages - first) return -1;
        const int k = first + n;
        const int w = word_of(p.words, k, [&](int x) { return p.before[x]; });
        return 32 * w + bit_of(~p.bits[w] & word_mask(w, p.c.num_pages), k - p.before[w]);
    };
    const int at = blockIdx.y * kThreads + threadIdx.x, step = gridDim.y * kThreads;
    for (int j = r.full + at; j < p.new_max_pages; j += step)
        p.new_table[i * p.new_stride + j] = j < kept ? p.table[r.p * p.stride + j] : j - kept < fresh ? fresh_page(j - kept) : -1;
    const bool copied = r.part > 0 && kept == r.full;
    const int dst = copied ? fresh_page(0) : -1;
    if (at == 0) p.new_seqlens[i] = copied && dst < 0 ? r.full << p.c.page_shift : r.len;
    if (dst >= 0) copy_slots(p.c, p.shape, p.table[r.p * p.stride + r.full], dst, r.part, at, step);
}

// ---------------------------------------------------------------- compact
struct CompactParams {
    CacheParams c;
    CopyShape shape;
    const int32_t* table;
    const int32_t* seqlens;
    const uint8_t* held;
    int32_t* new_table;
    int32_t* num_used;
    int64_t stride, new_stride;
    int batch, max_pages, max_tokens;
    int words, slices, table_blocks;
    uint32_t* live;
    uint32_t* held_bits;
    int32_t* live_before;
    int32_t* open_before;
    int32_t* edge;
};

__device__ __forceinline__ int compact_cells(const CompactParams& p, int b) {
    const int len = min(max(p.seqlens[b], 0), p.max_tokens);
    return (int)(((int64_t)len + (1 << p.c.page_shift) - 1) >> p.c.page_shift);
}

__global__ __launch_bounds__(kThreads) void compact_clear_kernel(CompactParams p) {
    for (int64_t w = (int64_t)blockIdx.x * kThreads + threadIdx.x; w < p.words; w += (int64_t)gridDim.x * kThreads) {
        p.live[w] = 0;
        p.held_bits[w] = held_word(p.held, (int)w, p.c.num_pages);
    }
}

__global__ __launch_bounds__(kThreads) void compact_mark_kernel(CompactParams p) {
    const int b = blockIdx.x, cells = compact_cells(p, b);
    for (int j = blockIdx.y * kThreads + threadIdx.x; j < cells; j += gridDim.y * kThreads) {
        const int page = p.table[b * p.stride + j];
        if (is_page(p.c, page)) atomicOr(&p.live[page >> 5], 1u << (page & 31));
    }
}

// (held pages are not counted as live: they stay)
__device__ __forceinline__ uint32_t live_word(const CompactParams& p, int w) { return p.live[w] & ~p.held_bits[w]; }
__device__ __forceinline__ uint32_t open_word(const CompactParams& p, int w) {
    return ~p.held_bits[w] & word_mask(w, p.c.num_pages);
}

// Counts by words; the edge, behind the first L pages that are not held (L: live ones).
__global__ __launch_bounds__(kScanThreads) void compact_scan_kernel(CompactParams p) {
    __shared__ int s_wave[kScanThreads / kWave];
    __shared__ int s_last;
    if (threadIdx.x == 0) s_last = -1;
    const int live = scan_words(p.words, p.live_before, s_wave, [&](int w) { return __popc(live_word(p, w)); });
    scan_words(p.words, p.open_before, s_wave, [&](int w) { return __popc(open_word(p, w)); });
    __syncthreads();
    for (int w = threadIdx.x; w < p.words; w += kScanThreads) {
        if (p.held_bits[w] != 0) atomicMax(&s_last, 32 * w + 31 - __builtin_clz(p.held_bits[w]));
        const int n = live - 1 - p.open_before[w];
        if (live > 0 && n >= 0 && n < __popc(open_word(p, w))) {   // (one word's)
            *p.edge = 32 * w + bit_of(open_word(p, w), n) + 1;
            atomicMax(&s_last, 32 * w + bit_of(open_word(p, w), n));
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        if (live == 0) *p.edge = 0;
        *p.num_used = s_last + 1;
    }
}

// Live pages before page x.
__device__ __forceinline__ int live_rank(const CompactParams& p, int x) {
    if (x >= 32 * p.words) return p.live_before[p.words];
    return p.live_before[x >> 5] + __popc(live_word(p, x >> 5) & ((1u << (x & 31)) - 1));
}

// The t-th page before the edge that is neither held nor live.
__device__ __forceinline__ int hole(const CompactParams& p, int t) {
    const int w = word_of(p.words, t, [&](int x) { return p.open_before[x] - p.live_before[x]; });
    return 32 * w + bit_of(open_word(p, w) & ~p.live[w], t - (p.open_before[w] - p.live_before[w]));
}

// Workgroups up to table_blocks renumber the table; the others copy, a slice of a page at a time.
__global__ __launch_bounds__(kThreads) void compact_move_kernel(CompactParams p) {
    const int edge = *p.edge;
    const int stay = live_rank(p, edge), live = p.live_before[p.words];
    if ((int)blockIdx.x < p.table_blocks) {
        const int64_t cells = (int64_t)p.batch * p.max_pages;
        for (int64_t x = (int64_t)blockIdx.x * kThreads + threadIdx.x; x < cells; x += (int64_t)p.table_blocks * kThreads) {
            const int b = (int)(x / p.max_pages), j = (int)(x - (int64_t)b * p.max_pages);
            int page = -1;
            if (j < compact_cells(p, b)) {
                page = p.table[b * p.stride + j];
                if (is_page(p.c, page) && page >= edge && !((p.held_bits[page >> 5] >> (page & 31)) & 1))
                    page = hole(p, live_rank(p, page) - stay);
            }
            p.new_table[b * p.new_stride + j] = page;
        }
        return;
    }
    const int64_t tasks = (int64_t)(live - stay) * p.slices;
    for (int64_t t = (int)blockIdx.x - p.table_blocks; t < tasks; t += gridDim.x - p.table_blocks) {
        const int mover = (int)(t / p.slices), slice = (int)(t - (int64_t)mover * p.slices);
        const int w = word_of(p.words, stay + mover, [&](int x) { return p.live_before[x]; });
        const int src = 32 * w + bit_of(live_word(p, w), stay + mover - p.live_before[w]);
        copy_slots(p.c, p.shape, src, hole(p, mover), 1 << p.c.page_shift, slice * kThreads + threadIdx.x, p.slices * kThreads);
    }
}

CopyShape copy_shape(const fgqa_kv_cache& c) {
    return CopyShape{c.kv_dtype == FGQA_KV_BF16 ? 4 : 3, make_fast_div(c.num_kv_heads)};
}

// 16-byte pieces of a page of K.
int64_t page_pieces(const fgqa_kv_cache& c) { return ((int64_t)c.page_size * c.num_kv_heads) << copy_shape(c).piece_log2; }

// The workspace of a call (NULL and 0: the library's, whose lock is then held).
int take_workspace(void* given, size_t given_bytes, size_t bytes, std::unique_lock<std::mutex>* lock, void** ws) {
    *ws = given;
    if (given == nullptr && given_bytes == 0) {
        *lock = workspace_lock();
        int st = FGQA_OK;
        *ws = internal_workspace(bytes, &st);
        return st;
    }
    if (given == nullptr || given_bytes < bytes) return FGQA_ERR_WORKSPACE;
    return aligned16(given) ? FGQA_OK : FGQA_ERR_UNSUPPORTED;
}

unsigned blocks_for(int64_t n, int64_t most) { return (unsigned)std::max<int64_t>(1, std::min(ceil_div(n, kThreads), most)); }

}  // namespace
}  // namespace fgqa

using namespace fgqa;

extern "C" int fgqa_kv_fork_workspace_bytes(const fgqa_kv_fork_args* a, size_t* bytes) {
    const int st = plan::validate_kv_fork_sizes(a);
    if (st != FGQA_OK || bytes == nullptr) return st != FGQA_OK ? st : FGQA_ERR_INVALID_ARGUMENT;
    *bytes = (size_t)plan::fork_layout(*a).total * 4;
    return FGQA_OK;
}

extern "C" int fgqa_kv_fork(const fgqa_kv_fork_args* a, void* stream) {
    int st = plan::validate_kv_fork(a);
    if (st != FGQA_OK) return st;
    const plan::ForkLayout l = plan::fork_layout(*a);
    std::unique_lock<std::mutex> lock;
    void* ws = nullptr;
    st = take_workspace(a->workspace, a->workspace_bytes, (size_t)l.total * 4, &lock, &ws);
    if (st != FGQA_OK) return st;
    int32_t* w = static_cast<int32_t*>(ws);
    ForkParams p;
    p.c = cache_params(a->cache);
    p.shape = copy_shape(a->cache);
    p.table = a->block_table;
    p.seqlens = a->seqlens;
    p.parents = a->parents;
    p.new_lens = a->new_lens;
    p.held = a->held;
    p.new_table = a->new_block_table;
    p.new_seqlens = a->new_seqlens;
    p.num_free = a->num_free;
    p.stride = a->block_table_stride;
    p.new_stride = a->new_block_table_stride;
    p.batch = a->batch;
    p.new_batch = a->new_batch;
    p.new_max_pages = a->new_max_pages;
    p.max_tokens = std::min(a->max_pages, a->new_max_pages) * a->cache.page_size;
    p.words = (int)plan::page_words(a->cache.num_pages);
    p.bits = reinterpret_cast<uint32_t*>(w + l.bits);
    p.before = w + l.before;
    p.row_first = w + l.row_first;
    p.first = w + l.first;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const unsigned rows = (unsigned)a->new_batch;
    const unsigned cells = blocks_for(a->new_max_pages, 16);
    hipLaunchKernelGGL(fork_clear_kernel, dim3(blocks_for(std::max<int64_t>(p.words, a->batch), 1024)), dim3(kThreads), 0, s, p);
    if (rows > 0) hipLaunchKernelGGL(fork_mark_kernel, dim3(rows, cells), dim3(kThreads), 0, s, p);
    hipLaunchKernelGGL(fork_scan_kernel, dim3(1), dim3(kScanThreads), 0, s, p);
    // slices of a row that fill the chip, with pieces for each thread of them
    const int64_t slices = std::min<int64_t>(ceil_div(2048, std::max(1u, rows)), ceil_div(page_pieces(a->cache), kThreads));
    if (rows > 0)
        hipLaunchKernelGGL(fork_fill_kernel, dim3(rows, (unsigned)std::max<int64_t>(cells, slices)), dim3(kThreads), 0, s, p);
    return hipGetLastError() == hipSuccess ? FGQA_OK : FGQA_ERR_HIP;
}

extern "C" int fgqa_kv_compact_workspace_bytes(const fgqa_kv_compact_args* a, size_t* bytes) {
    const int st = plan::validate_kv_compact_sizes(a);
    if (st != FGQA_OK || bytes == nullptr) return st != FGQA_OK ? st : FGQA_ERR_INVALID_ARGUMENT;
    *bytes = (size_t)plan::compact_layout(*a).total * 4;
    return FGQA_OK;
}

extern "C" int fgqa_kv_compact(const fgqa_kv_compact_args* a, void* stream) {
    int st = plan::validate_kv_compact(a);
    if (st != FGQA_OK) return st;
    const plan::CompactLayout l = plan::compact_layout(*a);
    std::unique_lock<std::mutex> lock;
    void* ws = nullptr;
    st = take_workspace(a->workspace, a->workspace_bytes, (size_t)l.total * 4, &lock, &ws);
    if (st != FGQA_OK) return st;
    int32_t* w = static_cast<int32_t*>(ws);
    CompactParams p;
    p.c = cache_params(a->cache);
    p.shape = copy_shape(a->cache);
    p.table = a->block_table;
    p.seqlens = a->seqlens;
    p.held = a->held;
    p.new_table = a->new_block_table;
    p.num_used = a->num_used;
    p.stride = a->block_table_stride;
    p.new_stride = a->new_block_table_stride;
    p.batch = a->batch;
    p.max_pages = a->max_pages;
    p.max_tokens = a->max_pages * a->cache.page_size;
    p.words = (int)plan::page_words(a->cache.num_pages);
    p.live = reinterpret_cast<uint32_t*>(w + l.live);
    p.held_bits = reinterpret_cast<uint32_t*>(w + l.held);
    p.live_before = w + l.live_before;
    p.open_before = w + l.open_before;
    p.edge = w + l.edge;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const int64_t cells = (int64_t)a->batch * a->max_pages;
    hipLaunchKernelGGL(compact_clear_kernel, dim3(blocks_for(p.words, 1024)), dim3(kThreads), 0, s, p);
    if (cells > 0)
        hipLaunchKernelGGL(compact_mark_kernel, dim3((unsigned)a->batch, blocks_for(a->max_pages, 16)), dim3(kThreads), 0, s, p);
    hipLaunchKernelGGL(compact_scan_kernel, dim3(1), dim3(kScanThreads), 0, s, p);
    if (cells > 0) {
        // (at most half of the pages move, and no more than the table has cells)
        const int64_t pieces = page_pieces(a->cache), moves = std::min<int64_t>(a->cache.num_pages / 2, cells);
        p.slices = (int)std::max<int64_t>(1, std::min<int64_t>(pieces / (4 * kThreads), 16));
        p.table_blocks = (int)blocks_for(cells, 256);
        const int64_t copy_blocks = std::min<int64_t>(moves * p.slices, 4096);
        hipLaunchKernelGGL(compact_move_kernel, dim3((unsigned)(p.table_blocks + copy_blocks)), dim3(kThreads), 0, s, p);
    }
    return hipGetLastError() == hipSuccess ? FGQA_OK : FGQA_ERR_HIP;
}
