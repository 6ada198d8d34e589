// Forking and freeing the sequences of a paged KV cache, and moving the pages in use
// together (include/fgqa_pages.h).
//
// Which pages are in use is worked out anew for each call from the block table, as one bit a
// page; a free page's number is found from the bits and a running count of them by words
// (a search over the words, then over one word's bits).  So there is no list of free
// pages to keep, and equal tables give equal results.
//
// With tables that one workgroup reads in passing, a call is one launch: each
// workgroup works the bits and counts out for itself, in LDS, and then takes its share of
// cells and copies.  Larger ones do that once, in three launches before the last (one, if
// only the pages that may move are many).
//
// Small calls are bound by one launch and the chain behind it (lengths, table, bits,
// counts, copies): 16 beams of up to 700 tokens forked 6.6 us, a cache of 8 sequences made
// compact 7.9 us (18.2 and 17.1 us with four launches).  Large ones are bound by the pages'
// bytes: 256 samples of 16 prompts of 8000 tokens 12 us (38 MB read and written; 40 us in
// four launches, their threads after the free pages through the L2), 48 conversations of
// 8000 tokens of bf16 155 us, the copies at 5.7 TB/s.  A page's pieces are dealt out to
// threads a slice's width apart: consecutive ones took 11 us more.
#include <algorithm>

#include "fgqa_device.h"
#include "fgqa_internal.h"
#include "kv_cache_params.h"
#include "../host/pages_plan.h"

namespace fgqa {
namespace {

constexpr int kThreads = 256;
constexpr int kScanThreads = plan::kAloneThreads;
constexpr int kWordsPerScan = 4;   // of a thread

// A page's rows as 16-byte pieces, and how many slots of it are copied.
struct CopyShape {
    int piece_log2;     // pieces of a row: 8 or 16
    FastDiv div_heads;
};

constexpr int kAhead = 4;   // pieces of K and of V that a thread has in flight

// Slots [0, slots) of page src to page dst, K and V and their scales: 16-byte pieces first,
// first + step, ... of all.  kStream: past the caches.
template <bool kStream = false>
__device__ __forceinline__ void copy_slots(const CacheParams& c, const CopyShape& sh, int src, int dst, int slots, int first,
                                           int step) {
    const int total = (slots * c.hkv) << sh.piece_log2;   // (a page's bytes / 16 stay below 2^31)
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
                const u32x4_t* from = reinterpret_cast<const u32x4_t*>(c.data[kv] + src * c.page[kv] + at[i][kv]);
                if constexpr (kStream) v[i][kv] = __builtin_nontemporal_load(from);
                else v[i][kv] = *from;
            }
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
#pragma unroll
            for (int kv = 0; kv < 2; ++kv)
                if (x0 + i * step < total) {
                    u32x4_t* to = reinterpret_cast<u32x4_t*>(c.data[kv] + dst * c.page[kv] + at[i][kv]);
                    if constexpr (kStream) __builtin_nontemporal_store(v[i][kv], to);
                    else *to = v[i][kv];
                }
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

typedef uint32_t u32x4b_t __attribute__((ext_vector_type(4), aligned(1)));

// held[32w .. 32w + 31] as bits.
__device__ __forceinline__ uint32_t held_word(const uint8_t* held, int w, int num_pages) {
    if (held == nullptr) return 0;
    const uint8_t* src = held + (int64_t)32 * w;
    const int n = min(32, num_pages - 32 * w);
    uint32_t bits = 0;
    if (n == 32) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const u32x4b_t x = *reinterpret_cast<const u32x4b_t*>(src + 16 * i);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                // bytes other than 0 have their top bits in m, which the product brings together
                const uint32_t m = ((((x[j] & 0x7f7f7f7fu) + 0x7f7f7f7fu) | x[j]) & 0x80808080u) >> 7;
                bits |= ((m * 0x01020408u) >> 24 & 15u) << (16 * i + 4 * j);
            }
        }
    } else {
        for (int i = 0; i < n; ++i) bits |= (src[i] != 0 ? 1u : 0u) << i;
    }
    return bits;
}

// store(w, the sum of count(0 .. w - 1)), for w <= words; the sum of all.  A workgroup.
template <typename T, typename Count, typename Store>
__device__ __forceinline__ T scan_words(int words, T* s_wave, Count&& count, Store&& store) {
    T carry = 0;
    for (int w0 = 0; w0 < words; w0 += kScanThreads * kWordsPerScan) {
        T n[kWordsPerScan], sum = 0, total;
#pragma unroll
        for (int i = 0; i < kWordsPerScan; ++i) {
            const int w = w0 + (int)threadIdx.x * kWordsPerScan + i;
            n[i] = w < words ? count(w) : 0;
            sum += n[i];
        }
        T at = carry + block_exclusive_scan<kScanThreads, true>(sum, s_wave, &total);
#pragma unroll
        for (int i = 0; i < kWordsPerScan; ++i) {
            const int w = w0 + (int)threadIdx.x * kWordsPerScan + i;
            if (w < words) store(w, at);
            at += n[i];
        }
        carry += total;
    }
    if (threadIdx.x == 0) store(words, carry);
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
__device__ __forceinline__ ForkRow fork_row(const ForkParams& p, int old, const int32_t* lens) {   // old: -1, or a row
    ForkRow r;
    r.p = old;
    r.there = old >= 0;
    r.len = r.there ? lens[old] : 0;
    r.full = r.len >> p.c.page_shift;
    r.part = r.len & ((1 << p.c.page_shift) - 1);
    return r;
}
__device__ __forceinline__ bool is_page(const CacheParams& c, int page) { return page >= 0 && page < c.num_pages; }

// Pages of its own that row i wants; *kept: cells before them.  last: the old row's partly filled page (its
// cell r.full), which its first new row keeps.
__device__ __forceinline__ int fresh_pages(const ForkParams& p, const ForkRow& r, int i, int first, int last, int* kept) {
    const bool keeps = !is_page(p.c, last) || (first == i && (p.held == nullptr || p.held[last] == 0));
    *kept = r.full + (r.part > 0 && keeps ? 1 : 0);
    const int64_t more = p.new_lens != nullptr ? max(p.new_lens[i], 0) : 0;
    const int64_t cells = (r.len + more + (1 << p.c.page_shift) - 1) >> p.c.page_shift;
    return (int)min(cells, (int64_t)p.new_max_pages) - *kept;
}
__device__ __forceinline__ int fresh_pages(const ForkParams& p, const ForkRow& r, int i, int* kept) {
    const bool part = r.part > 0;   // (of an old row, then)
    return fresh_pages(p, r, i, part ? p.first[r.p] : -1, part ? p.table[r.p * p.stride + r.full] : -1, kept);
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

// Counts of free pages by words and of fresh ones by rows (fresh(i, &cells kept) has a row's, row(i, fresh
// pages, those of rows before it, cells kept) takes them); the free pages that are left.  A workgroup.
template <typename Fresh, typename Row>
__device__ __forceinline__ int fork_scan(const ForkParams& p, const uint32_t* bits, int32_t* before, Fresh&& fresh, Row&& row) {
    __shared__ int s_wave[kScanThreads / kWave];
    const int free_pages = scan_words(
        p.words, s_wave, [&](int w) { return __popc(~bits[w] & word_mask(w, p.c.num_pages)); }, [&](int w, int n) { before[w] = n; });
    __shared__ int64_t s_wave64[kScanThreads / kWave];
    int64_t wanted = 0;   // (rows times cells can pass 2^31)
    for (int i0 = 0; i0 < p.new_batch; i0 += kScanThreads) {
        const int i = i0 + (int)threadIdx.x;
        int kept = 0;
        int64_t total;
        const int64_t n = i < p.new_batch ? fresh(i, &kept) : 0;
        const int64_t at = block_exclusive_scan<kScanThreads, true>(n, s_wave64, &total);
        if (i < p.new_batch) row(i, (int)n, (int)min(wanted + at, (int64_t)INT32_MAX), kept);
        wanted += total;
    }
    return (int)max((int64_t)free_pages - wanted, (int64_t)INT32_MIN);
}

__global__ __launch_bounds__(kScanThreads) void fork_scan_kernel(ForkParams p) {
    const int left = fork_scan(
        p, p.bits, p.before, [&](int i, int* kept) { return fresh_pages(p, fork_row(p, i), i, kept); },
        [&](int i, int, int at, int) { p.row_first[i] = at; });
    if (threadIdx.x == 0) *p.num_free = left;
}

// The k-th free page.
__device__ __forceinline__ int free_page(const ForkParams& p, const uint32_t* bits, const int32_t* before, int k) {
    const int w = word_of(p.words, k, [&](int x) { return before[x]; });
    return 32 * w + bit_of(~bits[w] & word_mask(w, p.c.num_pages), k - before[w]);
}

// The rows' other cells, and the copies of partly filled pages.
__global__ __launch_bounds__(kThreads) void fork_fill_kernel(ForkParams p) {
    const int i = blockIdx.x;
    const ForkRow r = fork_row(p, i);
    int kept;
    const int fresh = fresh_pages(p, r, i, &kept);
    const int first = p.row_first[i], free_pages = p.before[p.words];
    auto fresh_page = [&](int n) { return n < free_pages - first ? free_page(p, p.bits, p.before, first + n) : -1; };
    const int at = blockIdx.y * kThreads + threadIdx.x, step = gridDim.y * kThreads;
    for (int j = r.full + at; j < p.new_max_pages; j += step)
        p.new_table[i * p.new_stride + j] = j < kept ? p.table[r.p * p.stride + j] : j - kept < fresh ? fresh_page(j - kept) : -1;
    const bool copied = r.part > 0 && kept == r.full;
    const int dst = copied ? fresh_page(0) : -1;
    if (at == 0) p.new_seqlens[i] = copied && dst < 0 ? r.full << p.c.page_shift : r.len;
    if (dst >= 0) copy_slots(p.c, p.shape, p.table[r.p * p.stride + r.full], dst, r.part, at, step);
}

// The cells of a table of `cells` = rows x width, x = threadIdx.x, + kScanThreads, ...:
// use(row, column, entry) for each.  begin() reads the first kCellsAhead rounds, so that they are under way together with
// what else a kernel reads first.  (Columns past a sequence's cells are read and not used.)
constexpr int kCellsAhead = 4;
struct TableCells {
    const int32_t* table;
    int64_t stride;
    FastDiv div_width;
    int width, cells;
    int ahead[kCellsAhead];

    __device__ __forceinline__ int entry(int x) const {
        const int b = fast_div(x, div_width);
        return table[b * stride + (x - b * width)];
    }
    __device__ __forceinline__ void begin() {
#pragma unroll
        for (int i = 0; i < kCellsAhead; ++i) {
            const int x = (int)threadIdx.x + i * kScanThreads;
            ahead[i] = x < cells ? entry(x) : -1;
        }
    }
    template <typename F>
    __device__ __forceinline__ void each(F&& use) const {
#pragma unroll
        for (int i = 0; i < kCellsAhead; ++i) {
            const int x = (int)threadIdx.x + i * kScanThreads;
            const int b = fast_div(min(x, max(cells - 1, 0)), div_width);
            if (x < cells) use(b, x - b * width, ahead[i]);
        }
#pragma unroll 4
        for (int x = (int)threadIdx.x + kCellsAhead * kScanThreads; x < cells; x += kScanThreads) {
            const int b = fast_div(x, div_width);
            use(b, x - b * width, entry(x));
        }
    }
};

// All of it, each workgroup planning for itself.  LDS: plan::fork_alone_ints.
__global__ __launch_bounds__(kScanThreads) void fork_alone_kernel(ForkParams p, FastDiv div_width, int width, FastDiv div_new_width,
                                                                  int slices) {
    extern __shared__ int32_t smem[];
    uint32_t* bits = reinterpret_cast<uint32_t*>(smem);
    int32_t* before = smem + p.words;
    int32_t* first = before + p.words + 1;   // [batch]
    int32_t* lens = first + p.batch;         // [batch]
    int32_t* last = lens + p.batch;          // [batch]: their partly filled pages
    int32_t* row = last + p.batch;           // [new_batch][4]: old row, fresh pages, those of rows before it, cells kept
    const int tid = threadIdx.x;
    auto parent_of = [&](int i) { return p.parents != nullptr ? p.parents[i] : i; };
    TableCells old{p.table, p.stride, div_width, width, p.batch * width};
    old.begin();
    const int parent0 = tid < p.new_batch ? parent_of(tid) : -1;
    for (int w = tid; w < p.words; w += kScanThreads) bits[w] = held_word(p.held, w, p.c.num_pages);
    for (int b = tid; b < p.batch; b += kScanThreads) {
        first[b] = INT32_MAX;
        lens[b] = min(max(p.seqlens[b], 0), p.max_tokens);
    }
    __syncthreads();
    for (int i = tid; i < p.new_batch; i += kScanThreads) {
        const int parent = i == tid ? parent0 : parent_of(i);
        const bool there = parent >= 0 && parent < p.batch;
        row[4 * i] = there ? parent : -1;
        if (there) atomicMin(&first[parent], i);
    }
    __syncthreads();
    old.each([&](int b, int j, int page) {
        if (j <= (lens[b] - 1) >> p.c.page_shift && first[b] != INT32_MAX) {
            if (is_page(p.c, page)) atomicOr(&bits[page >> 5], 1u << (page & 31));
            if (j == lens[b] >> p.c.page_shift) last[b] = page;
        }
    });
    __syncthreads();
    const int left = fork_scan(
        p, bits, before,
        [&](int i, int* kept) {
            const ForkRow r = fork_row(p, row[4 * i], lens);
            const bool part = r.part > 0;
            return fresh_pages(p, r, i, part ? first[r.p] : -1, part ? last[r.p] : -1, kept);
        },
        [&](int i, int n, int at, int kept) {
            row[4 * i + 1] = n;
            row[4 * i + 2] = at;
            row[4 * i + 3] = kept;
        });
    if (blockIdx.x == 0 && tid == 0) *p.num_free = left;
    __syncthreads();
    const int free_pages = before[p.words];
    auto fresh_page = [&](int at, int n) { return n < free_pages - at ? free_page(p, bits, before, at + n) : -1; };

    // slices of the copied pages, one to a wave
    const int lane = tid % kWave, waves = gridDim.x * (kScanThreads / kWave);
    for (int64_t t = (tid / kWave) * gridDim.x + blockIdx.x; t < (int64_t)p.new_batch * slices; t += waves) {
        const int i = (int)(t / slices), slice = (int)(t - (int64_t)i * slices);
        const ForkRow r = fork_row(p, row[4 * i], lens);
        const bool copied = r.part > 0 && row[4 * i + 3] == r.full;
        const int dst = copied ? fresh_page(row[4 * i + 2], 0) : -1;
        if (slice == 0 && lane == 0) p.new_seqlens[i] = copied && dst < 0 ? r.full << p.c.page_shift : r.len;
        if (dst >= 0) copy_slots(p.c, p.shape, last[r.p], dst, r.part, slice * kWave + lane, slices * kWave);
    }
    const int cells = p.new_batch * p.new_max_pages;
    for (int x = blockIdx.x * kScanThreads + tid; x < cells; x += gridDim.x * kScanThreads) {
        const int i = fast_div(x, div_new_width), j = x - i * p.new_max_pages;
        const int fresh = row[4 * i + 1], kept = row[4 * i + 3];
        p.new_table[i * p.new_stride + j] = j < kept          ? p.table[row[4 * i] * p.stride + j]
                                            : j - kept < fresh ? fresh_page(row[4 * i + 2], j - kept)
                                                               : -1;
    }
}

// ---------------------------------------------------------------- compact
// The pages' bits and counts by words.
struct PageWords {
    int words, num_pages;
    uint32_t* live;
    uint32_t* held;
    int32_t* live_before;
    int32_t* open_before;
};

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
    int slices, table_blocks;
    PageWords words;
    int32_t* edge;
};

__device__ __forceinline__ int compact_cells(const CompactParams& p, int b) {
    const int len = min(max(p.seqlens[b], 0), p.max_tokens);
    return (int)(((int64_t)len + (1 << p.c.page_shift) - 1) >> p.c.page_shift);
}

__global__ __launch_bounds__(kThreads) void compact_clear_kernel(CompactParams p) {
    for (int64_t w = (int64_t)blockIdx.x * kThreads + threadIdx.x; w < p.words.words; w += (int64_t)gridDim.x * kThreads) {
        p.words.live[w] = 0;
        p.words.held[w] = held_word(p.held, (int)w, p.c.num_pages);
    }
}

__global__ __launch_bounds__(kThreads) void compact_mark_kernel(CompactParams p) {
    const int b = blockIdx.x, cells = compact_cells(p, b);
    for (int j = blockIdx.y * kThreads + threadIdx.x; j < cells; j += gridDim.y * kThreads) {
        const int page = p.table[b * p.stride + j];
        if (is_page(p.c, page)) atomicOr(&p.words.live[page >> 5], 1u << (page & 31));
    }
}

// (held pages are not counted as live: they stay)
__device__ __forceinline__ uint32_t live_word(const PageWords& s, int w) { return s.live[w] & ~s.held[w]; }
__device__ __forceinline__ uint32_t open_word(const PageWords& s, int w) { return ~s.held[w] & word_mask(w, s.num_pages); }

// Counts by words; *edge, behind the first L pages that are not held (L: live ones); how many
// pages are in use or held up to the last such one.  A workgroup.
__device__ __forceinline__ int compact_scan(const PageWords& s, int32_t* edge) {
    __shared__ int64_t s_wave[kScanThreads / kWave];
    __shared__ int s_last;
    if (threadIdx.x == 0) s_last = -1;
    const int live = (int)scan_words(
        s.words, s_wave, [&](int w) { return (int64_t)__popc(open_word(s, w)) << 32 | __popc(live_word(s, w)); },
        [&](int w, int64_t n) {
            s.live_before[w] = (int)n;   // (counts stay below 2^31)
            s.open_before[w] = (int)(n >> 32);
        });
    __syncthreads();
    for (int w = threadIdx.x; w < s.words; w += kScanThreads) {
        if (s.held[w] != 0) atomicMax(&s_last, 32 * w + 31 - __builtin_clz(s.held[w]));
        const int n = live - 1 - s.open_before[w];
        if (live > 0 && n >= 0 && n < __popc(open_word(s, w))) {   // (one word's)
            *edge = 32 * w + bit_of(open_word(s, w), n) + 1;
            atomicMax(&s_last, 32 * w + bit_of(open_word(s, w), n));
        }
    }
    if (threadIdx.x == 0 && live == 0) *edge = 0;
    __syncthreads();
    return s_last + 1;
}

__global__ __launch_bounds__(kScanThreads) void compact_scan_kernel(CompactParams p) {
    const int used = compact_scan(p.words, p.edge);
    if (threadIdx.x == 0) *p.num_used = used;
}

// Live pages before page x.
__device__ __forceinline__ int live_rank(const PageWords& s, int x) {
    if (x >= 32 * s.words) return s.live_before[s.words];
    return s.live_before[x >> 5] + __popc(live_word(s, x >> 5) & ((1u << (x & 31)) - 1));
}

// The t-th page before the edge that is neither held nor live.
__device__ __forceinline__ int hole(const PageWords& s, int t) {
    const int w = word_of(s.words, t, [&](int x) { return s.open_before[x] - s.live_before[x]; });
    return 32 * w + bit_of(open_word(s, w) & ~s.live[w], t - (s.open_before[w] - s.live_before[w]));
}

// The new number of page `page` of the old table.
__device__ __forceinline__ int moved_to(const CompactParams& p, const PageWords& s, int page, int edge, int stay) {
    if (!is_page(p.c, page) || page < edge || ((s.held[page >> 5] >> (page & 31)) & 1)) return page;
    return hole(s, live_rank(s, page) - stay);
}

// Slice t % slices of the page that is the (t / slices)-th to move, by `threads` threads.
template <bool kStream>
__device__ __forceinline__ void move_slice(const CompactParams& p, const PageWords& s, int64_t t, int stay, int thread, int threads) {
    const int mover = (int)(t / p.slices), slice = (int)(t - (int64_t)mover * p.slices);
    const int w = word_of(s.words, stay + mover, [&](int x) { return s.live_before[x]; });
    const int src = 32 * w + bit_of(live_word(s, w), stay + mover - s.live_before[w]);
    copy_slots<kStream>(p.c, p.shape, src, hole(s, mover), 1 << p.c.page_shift, slice * threads + thread, p.slices * threads);
}

// Workgroups up to table_blocks renumber the table; the others copy, a slice of a page at a time (with kStream,
// where many bytes may move, past the caches: 155 us where 166).
template <bool kStream>
__global__ __launch_bounds__(kThreads) void compact_move_kernel(CompactParams p) {
    const PageWords& s = p.words;
    const int edge = *p.edge;
    const int stay = live_rank(s, edge), live = s.live_before[s.words];
    if ((int)blockIdx.x < p.table_blocks) {
        const int64_t cells = (int64_t)p.batch * p.max_pages;
        for (int64_t x = (int64_t)blockIdx.x * kThreads + threadIdx.x; x < cells; x += (int64_t)p.table_blocks * kThreads) {
            const int b = (int)(x / p.max_pages), j = (int)(x - (int64_t)b * p.max_pages);
            p.new_table[b * p.new_stride + j] =
                j < compact_cells(p, b) ? moved_to(p, s, p.table[b * p.stride + j], edge, stay) : -1;
        }
        return;
    }
    const int64_t tasks = (int64_t)(live - stay) * p.slices;
    for (int64_t t = (int)blockIdx.x - p.table_blocks; t < tasks; t += gridDim.x - p.table_blocks)
        move_slice<kStream>(p, s, t, stay, threadIdx.x, kThreads);
}

// All of it, each workgroup planning for itself.  LDS: plan::compact_alone_ints.  kPlan: the words and the edge
// alone, to memory, by one workgroup.
template <bool kPlan>
__global__ __launch_bounds__(kScanThreads) void compact_alone_kernel(CompactParams p, FastDiv div_width) {
    extern __shared__ int32_t smem[];
    __shared__ int32_t s_edge;
    PageWords s = p.words;
    s.live = reinterpret_cast<uint32_t*>(smem);
    s.held = s.live + s.words;
    s.live_before = smem + 2 * s.words;
    s.open_before = s.live_before + s.words + 1;
    int32_t* cells_of = s.open_before + s.words + 1;   // [batch]
    const int tid = threadIdx.x;
    const int cells = p.batch * p.max_pages;
    TableCells old{p.table, p.stride, div_width, p.max_pages, cells};
    old.begin();
    for (int w = tid; w < s.words; w += kScanThreads) {
        s.live[w] = 0;
        s.held[w] = held_word(p.held, w, p.c.num_pages);
    }
    for (int b = tid; b < p.batch; b += kScanThreads) cells_of[b] = compact_cells(p, b);
    __syncthreads();
    old.each([&](int b, int j, int page) {
        if (j < cells_of[b] && is_page(p.c, page)) atomicOr(&s.live[page >> 5], 1u << (page & 31));
    });
    __syncthreads();
    const int used = compact_scan(s, &s_edge);
    if (blockIdx.x == 0 && tid == 0) *p.num_used = used;
    const int edge = s_edge;
    if constexpr (kPlan) {
        for (int w = tid; w <= s.words; w += kScanThreads) {
            if (w < s.words) {
                p.words.live[w] = s.live[w];
                p.words.held[w] = s.held[w];
            }
            p.words.live_before[w] = s.live_before[w];
            p.words.open_before[w] = s.open_before[w];
        }
        if (tid == 0) *p.edge = edge;
        return;
    }
    const int stay = live_rank(s, edge);
    const int64_t tasks = (int64_t)(s.live_before[s.words] - stay) * p.slices;
    const int waves = gridDim.x * (kScanThreads / kWave);
    for (int64_t t = (tid / kWave) * gridDim.x + blockIdx.x; t < tasks; t += waves)   // (a wave's)
        move_slice<false>(p, s, t, stay, tid % kWave, kWave);
    for (int x = blockIdx.x * kScanThreads + tid; x < cells; x += gridDim.x * kScanThreads) {
        const int b = fast_div(x, div_width), j = x - b * p.max_pages;
        p.new_table[b * p.new_stride + j] = j < cells_of[b] ? moved_to(p, s, p.table[b * p.stride + j], edge, stay) : -1;
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

// Workgroups that plan for themselves: 4 waves' slices or 1024 cells each, and at most `most`.
unsigned alone_blocks(int64_t slices, int64_t cells, int64_t most) {
    const int64_t n = std::max(ceil_div(slices, 4), ceil_div(cells, kScanThreads));
    return (unsigned)std::max<int64_t>(1, std::min(n, most));
}

}  // namespace
}  // namespace fgqa

using namespace fgqa;

extern "C" int fgqa_kv_fork_workspace_bytes(const fgqa_kv_fork_args* a, size_t* bytes) {
    const int st = plan::validate_kv_fork_sizes(a);
    if (st != FGQA_OK || bytes == nullptr) return st != FGQA_OK ? st : FGQA_ERR_INVALID_ARGUMENT;
    *bytes = plan::fork_alone_ints(*a) > 0 ? 0 : (size_t)plan::fork_layout(*a).total * 4;
    return FGQA_OK;
}

extern "C" int fgqa_kv_fork(const fgqa_kv_fork_args* a, void* stream) {
    int st = plan::validate_kv_fork(a);
    if (st != FGQA_OK) return st;
    ForkParams p = {};
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
    p.batch = a->new_batch > 0 ? a->batch : 0;   // (with no new row the old ones are not read, and may be NULL)
    p.new_batch = a->new_batch;
    p.new_max_pages = a->new_max_pages;
    p.max_tokens = std::min(a->max_pages, a->new_max_pages) * a->cache.page_size;
    p.words = (int)plan::page_words(a->cache.num_pages);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const int alone = plan::fork_alone_ints(*a);
    if (alone > 0) {
        const int width = plan::fork_width(*a);
        const int slices = (int)ceil_div(page_pieces(a->cache), kAhead * kWave);
        const int64_t cells = (int64_t)a->new_batch * a->new_max_pages;
        hipLaunchKernelGGL(fork_alone_kernel, dim3(alone_blocks((int64_t)a->new_batch * slices, cells, 256)), dim3(kScanThreads), (size_t)alone * 4, s, p,
                           make_fast_div(std::max(width, 1)), width, make_fast_div(std::max(a->new_max_pages, 1)), slices);
        return hipGetLastError() == hipSuccess ? FGQA_OK : FGQA_ERR_HIP;
    }
    const plan::ForkLayout l = plan::fork_layout(*a);
    std::unique_lock<std::mutex> lock;
    void* ws = nullptr;
    st = take_workspace(a->workspace, a->workspace_bytes, (size_t)l.total * 4, &lock, &ws);
    if (st != FGQA_OK) return st;
    int32_t* w = static_cast<int32_t*>(ws);
    p.bits = reinterpret_cast<uint32_t*>(w + l.bits);
    p.before = w + l.before;
    p.row_first = w + l.row_first;
    p.first = w + l.first;
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
    const bool none = plan::compact_alone_ints(*a) > 0 && plan::compact_moves_little(*a);
    *bytes = none ? 0 : (size_t)plan::compact_layout(*a).total * 4;
    return FGQA_OK;
}

extern "C" int fgqa_kv_compact(const fgqa_kv_compact_args* a, void* stream) {
    int st = plan::validate_kv_compact(a);
    if (st != FGQA_OK) return st;
    CompactParams p = {};
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
    p.words.words = (int)plan::page_words(a->cache.num_pages);
    p.words.num_pages = a->cache.num_pages;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const int64_t cells = (int64_t)a->batch * a->max_pages;
    const int64_t pieces = page_pieces(a->cache), moves = plan::compact_moves(*a);
    const int alone = plan::compact_alone_ints(*a);
    if (alone > 0 && plan::compact_moves_little(*a)) {
        p.slices = (int)ceil_div(pieces, kAhead * kWave);
        hipLaunchKernelGGL(compact_alone_kernel<false>, dim3(alone_blocks(moves * p.slices, cells, 256)), dim3(kScanThreads), (size_t)alone * 4, s, p,
                           make_fast_div(std::max(a->max_pages, 1)));
        return hipGetLastError() == hipSuccess ? FGQA_OK : FGQA_ERR_HIP;
    }
    const plan::CompactLayout l = plan::compact_layout(*a);
    std::unique_lock<std::mutex> lock;
    void* ws = nullptr;
    st = take_workspace(a->workspace, a->workspace_bytes, (size_t)l.total * 4, &lock, &ws);
    if (st != FGQA_OK) return st;
    int32_t* w = static_cast<int32_t*>(ws);
    p.words.live = reinterpret_cast<uint32_t*>(w + l.live);
    p.words.held = reinterpret_cast<uint32_t*>(w + l.held);
    p.words.live_before = w + l.live_before;
    p.words.open_before = w + l.open_before;
    p.edge = w + l.edge;
    if (alone > 0) {
        hipLaunchKernelGGL(compact_alone_kernel<true>, dim3(1), dim3(kScanThreads), (size_t)alone * 4, s, p,
                           make_fast_div(std::max(a->max_pages, 1)));
    } else {
        hipLaunchKernelGGL(compact_clear_kernel, dim3(blocks_for(p.words.words, 1024)), dim3(kThreads), 0, s, p);
        if (cells > 0)
            hipLaunchKernelGGL(compact_mark_kernel, dim3((unsigned)a->batch, blocks_for(a->max_pages, 16)), dim3(kThreads), 0, s, p);
        hipLaunchKernelGGL(compact_scan_kernel, dim3(1), dim3(kScanThreads), 0, s, p);
    }
    if (cells > 0) {
        p.slices = (int)std::max<int64_t>(1, std::min<int64_t>(pieces / (kAhead * kThreads), 16));
        p.table_blocks = (int)blocks_for(cells, 256);
        const int64_t copy_blocks = std::min<int64_t>(moves * p.slices, 4096);
        const dim3 grid((unsigned)(p.table_blocks + copy_blocks));
        if (plan::compact_moves_little(*a)) hipLaunchKernelGGL(compact_move_kernel<false>, grid, dim3(kThreads), 0, s, p);
        else hipLaunchKernelGGL(compact_move_kernel<true>, grid, dim3(kThreads), 0, s, p);
    }
    return hipGetLastError() == hipSuccess ? FGQA_OK : FGQA_ERR_HIP;
}
