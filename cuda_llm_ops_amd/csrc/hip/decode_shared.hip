// Single-token attention for sequences that begin alike (fgqa_decode_shared).
//
// With the tokens that a group of sequences shares, P, and each one's own, T,
//   O = (e^{m_P - m} l_P o_P + e^{m_T - m} l_T o_T) / (e^{m_P - m} l_P + e^{m_T - m} l_T):
// a sequence's partials over P and T merge as those of a split decode do.  Over T the
// item of the paged decode runs as it is.  Over P the queries of all the group's
// sequences and of a KV head's query heads are rows of one matrix, 128 of them a workgroup:
// S^T = K Q^T and O^T += V^T P^T on 32x32x16 MFMAs, 32 rows a wave, each K and V row read
// once from memory for all of them, widened to bf16 and staged in LDS for the four waves.
//
// One planning workgroup finds the groups and cuts all work into pieces of about equal
// token counts that fill the chip; one launch runs them; one merges the partials.
#include <algorithm>
#include <type_traits>

#include "decode_item.h"
#include "fgqa_device.h"
#include "fgqa_internal.h"
#include "../host/pages_plan.h"

namespace fgqa {
namespace {

constexpr int kThreads = 256;
constexpr int kTile = 64;             // shared tokens of a step
constexpr int kPlanThreads = 1024;

// What runs on one workgroup for each KV head.
struct Item {
    int b;        // a sequence, or the first of a group
    int t0, t1;   // tokens
    int slot;     // row of the partials of KV head 0 (whole: -1)
    int rows;     // 0: a sequence's own tokens; else query rows, from row0 of the group
    int row0;
    int stride;   // rows of partials from one KV head to the next
    int table;    // the sequence whose block table row is read
};
static_assert(sizeof(Item) == 4 * plan::kSharedItemInts, "item");

// A sequence's partials: n_shared at shared + i * step, then n_own at own + i * hkv * group; rows of KV head 0's
// first query head (further KV heads `head` and `group` rows on).
struct Seq {
    int shared, step, head, n_shared;
    int own, n_own;
    int whole;    // written already
    int pad;
};
static_assert(sizeof(Seq) == 4 * plan::kSharedSeqInts, "sequence");

struct SharedParams {
    DecodeParams d;
    const int32_t* group_starts;
    const int32_t* shared_lens;
    int num_groups, slots;
    FastDiv div_group, div_hkv;
    Item* items;
    Seq* seqs;
    int32_t* count;
};

// ---------------------------------------------------------------- plan
// The group of sequence b (starts ascending), or -1.
__device__ __forceinline__ int group_of(const int* starts, int n, int b) {
    if (n == 0 || b < starts[0] || b >= starts[n]) return -1;
    int lo = 0, hi = n;   // starts[lo] <= b < starts[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (starts[mid] <= b) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Latency bounds it: a few dependent loads and scans of one workgroup.
__global__ __launch_bounds__(kPlanThreads) void shared_plan_kernel(SharedParams p) {
    __shared__ int s_start[plan::kSharedMaxGroups + 1];
    __shared__ int s_len[plan::kSharedMaxGroups];     // shortest of its sequences, then what is shared
    __shared__ int s_first[plan::kSharedMaxGroups];   // its first sequence with tokens
    __shared__ int s_more[plan::kSharedMaxGroups];    // its last one
    __shared__ int64_t s_wave64[kPlanThreads / kWave];
    __shared__ int s_wave[kPlanThreads / kWave];
    const int tid = threadIdx.x, n = p.num_groups, batch = p.d.batch, group = p.d.group, hkv = p.d.hkv;
    for (int i = tid; i <= n; i += kPlanThreads) {
        s_start[i] = n > 0 ? min(max(p.group_starts[i], 0), batch) : 0;
        if (i < n) {
            s_len[i] = s_first[i] = INT32_MAX;
            s_more[i] = -1;
        }
    }
    __syncthreads();
    // each start at least the one before it
    for (int d = 1; d <= n; d *= 2) {
        int v[plan::kSharedMaxGroups / kPlanThreads + 1];
        int k = 0;
        for (int i = tid; i <= n; i += kPlanThreads) v[k++] = max(s_start[i], i >= d ? s_start[i - d] : 0);
        __syncthreads();
        k = 0;
        for (int i = tid; i <= n; i += kPlanThreads) s_start[i] = v[k++];
        __syncthreads();
    }
    for (int b = tid; b < batch; b += kPlanThreads) {
        const int len = clamp_len(p.d, b), g = group_of(s_start, n, b);
        if (g < 0 || len == 0) continue;
        atomicMin(&s_len[g], len);
        atomicMin(&s_first[g], b);
        atomicMax(&s_more[g], b);
    }
    __syncthreads();
    int64_t sum = 0, total;
    auto tiles_of = [&](int g) {
        return (int)(((int64_t)(s_start[g + 1] - s_start[g]) * group + plan::kSharedRows - 1) / plan::kSharedRows);
    };
    for (int g = tid; g < n; g += kPlanThreads) {
        // (one sequence shares with none)
        int len = s_more[g] > s_first[g] ? min(s_len[g], p.shared_lens[g]) : 0;
        len = max(len, 0) >> p.d.page_shift << p.d.page_shift;
        s_len[g] = len < plan::kSharedChunk ? 0 : len;
        sum += (int64_t)tiles_of(g) * s_len[g];
    }
    __syncthreads();
    for (int b = tid; b < batch; b += kPlanThreads) {
        const int g = group_of(s_start, n, b), len = clamp_len(p.d, b);
        if (len > 0) sum += len - (g < 0 ? 0 : s_len[g]);
    }
    block_exclusive_scan<kPlanThreads, true>(sum, s_wave64, &total);
    const int64_t chunk = plan::shared_chunk(total, p.slots);
    int item = 0, row = 0;   // so far
    for (int g0 = 0; g0 < n; g0 += kPlanThreads) {
        const int g = g0 + tid;
        const int len = g < n ? s_len[g] : 0, tiles = len > 0 ? tiles_of(g) : 0;
        const int rows = len > 0 ? (s_start[g + 1] - s_start[g]) * group : 0;
        const int piece = len > 0 ? (int)plan::shared_piece(len, chunk, kTile) : 1, pieces = (len + piece - 1) / piece;
        int all_items, all_rows;
        int at = item + block_exclusive_scan<kPlanThreads, true>(pieces * tiles, s_wave, &all_items);
        const int base = row + block_exclusive_scan<kPlanThreads, true>(pieces * hkv * rows, s_wave, &all_rows);
        for (int i = 0; i < pieces; ++i)
            for (int t = 0; t < tiles; ++t) {
                Item it;
                it.b = s_start[g];
                it.table = s_first[g];
                it.t0 = i * piece;
                it.t1 = min(len, it.t0 + piece);
                it.row0 = t * plan::kSharedRows;
                it.rows = min(plan::kSharedRows, rows - it.row0);
                it.slot = base + i * hkv * rows + it.row0;
                it.stride = rows;
                p.items[at++] = it;
            }
        if (g < n) {
            s_first[g] = base;      // (the first sequence is not needed any more)
            s_more[g] = pieces;
        }
        item += all_items;
        row += all_rows;
    }
    __syncthreads();
    for (int b0 = 0; b0 < batch; b0 += kPlanThreads) {
        const int b = b0 + tid;
        const bool here = b < batch;
        const int g = here ? group_of(s_start, n, b) : -1, len = here ? clamp_len(p.d, b) : 0;
        const int begin = g < 0 || len == 0 ? 0 : s_len[g], left = len - begin;
        const int piece = left > 0 ? (int)plan::shared_piece(left, chunk, plan::kSharedChunk) : 1, pieces = (left + piece - 1) / piece;
        const bool whole = begin == 0 && pieces == 1;
        int all_items, all_rows;
        int at = item + block_exclusive_scan<kPlanThreads, true>(pieces, s_wave, &all_items);
        const int base = row + block_exclusive_scan<kPlanThreads, true>(whole ? 0 : pieces * hkv * group, s_wave, &all_rows);
        for (int i = 0; i < pieces; ++i) {
            Item it;
            it.b = it.table = b;
            it.t0 = begin + i * piece;
            it.t1 = min(len, it.t0 + piece);
            it.slot = whole ? -1 : base + i * hkv * group;
            it.rows = it.row0 = 0;
            it.stride = group;
            p.items[at++] = it;
        }
        if (here) {
            Seq s;
            s.n_shared = begin > 0 ? s_more[g] : 0;
            s.head = begin > 0 ? (s_start[g + 1] - s_start[g]) * group : 0;
            s.step = hkv * s.head;
            s.shared = begin > 0 ? s_first[g] + (b - s_start[g]) * group : 0;
            s.own = base;
            s.n_own = pieces;
            s.whole = whole;
            s.pad = 0;
            p.seqs[b] = s;
        }
        item += all_items;
        row += all_rows;
    }
    if (tid == 0) *p.count = item;
}

// ---------------------------------------------------------------- shared tokens
constexpr int kTileBytes = kTile * kHeadDim * 2;
constexpr int kBufBytes = 2 * kTileBytes + 2 * kTile * 4;   // K, V, their scales
constexpr int kSharedSmem = 2 * kBufBytes;

// Loads of a tile: 16 bytes of a row each, bf16 rows by 16 threads, rows of codes by 8.
template <int kKv>
struct TileShape {
    static constexpr bool bf16 = kKv == kKvPagedBf16;
    static constexpr bool blocks = kKv >= kKvBlocksFp8;
    static constexpr int row_threads = bf16 ? 16 : 8;
    static constexpr int rows = kThreads / row_threads;   // of one load
    static constexpr int loads = kTile / rows;
};

template <int kKv>
__device__ __forceinline__ void shared_item(const SharedParams& sp, unsigned char* smem, const Item& it, int kvh) {
    using T = TileShape<kKv>;
    const DecodeParams& p = sp.d;
    const int tid = threadIdx.x, lane = tid & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int l32 = lane & 31, half = lane >> 5;
    const bool active = 32 * wave < it.rows;   // (other waves only load)

    // Q^T as the B operand: lane holds Q[row l32][16 ks + 8 half .. +7]
    bf16x8_t qop[8];
    {
        const int row = it.row0 + min(32 * wave + l32, it.rows - 1);
        const int seq = fast_div(row, sp.div_group);
        const __bf16* q = p.q + (it.b + seq) * p.q_sb + (int64_t)(kvh * p.group + row - seq * p.group) * p.q_sh + 8 * half;
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) qop[ks] = as_bf16x8(*reinterpret_cast<const u32x4_t*>(q + 16 * ks));
    }
    float m_run = -INFINITY, l_run = 0.f;   // l: this lane's share
    f32x16_t oacc[4];
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) oacc[db][i] = 0.f;

    constexpr int kElem = T::bf16 ? 2 : 1;
    const unsigned char* kbase = reinterpret_cast<const unsigned char*>(p.k) + kvh * p.k_sh * kElem;
    const unsigned char* vbase = reinterpret_cast<const unsigned char*>(p.v) + kvh * p.v_sh * kElem;
    const int32_t* bt = p.block_table + (int64_t)it.table * p.bt_stride;
    const int pmask = (1 << p.page_shift) - 1;
    const int lrow = tid / T::row_threads, chunk = tid % T::row_threads;
    const int tiles = (it.t1 - it.t0 + kTile - 1) / kTile;
    u32x4_t kreg[T::loads], vreg[T::loads];
    [[maybe_unused]] float ksreg[T::loads], vsreg[T::loads];
    int pg[T::loads];
    // Tokens past the end read the last one again (their scores are masked; the rows are numbers).
    auto token = [&](int j, int i) { return min(it.t0 + j * kTile + lrow + i * T::rows, it.t1 - 1); };
    auto fetch_pages = [&](int j) {
#pragma unroll
        for (int i = 0; i < T::loads; ++i) pg[i] = bt[token(j, i) >> p.page_shift];
    };
    // The table's entries are loaded a tile before they are used, ahead of the rows between.
    auto load = [&](int j, bool more) {
        int64_t page[T::loads];
#pragma unroll
        for (int i = 0; i < T::loads; ++i) page[i] = min(max(pg[i], 0), p.num_pages - 1);
        if (more) fetch_pages(j + 1);
#pragma unroll
        for (int i = 0; i < T::loads; ++i) {
            const int64_t slot = token(j, i) & pmask;
            kreg[i] = *reinterpret_cast<const u32x4_t*>(kbase + (page[i] * p.k_sb + slot * p.k_ss) * kElem + chunk * 16);
            vreg[i] = *reinterpret_cast<const u32x4_t*>(vbase + (page[i] * p.v_sb + slot * p.v_ss) * kElem + chunk * 16);
            if constexpr (T::blocks) {
                ksreg[i] = p.k_scales[page[i] * p.ks_sp + kvh * p.ks_sh];
                vsreg[i] = p.v_scales[page[i] * p.vs_sp + kvh * p.vs_sh];
            }
        }
    };
    // K's 16-byte piece c of row r lies at piece c ^ (r % 16), V's at c ^ 4 (r % 4): reads and
    // writes then spread over all banks.
    auto stage = [&](unsigned char* buf) {
        __bf16* kl = reinterpret_cast<__bf16*>(buf);
        __bf16* vl = kl + kTile * kHeadDim;
        float* sl = reinterpret_cast<float*>(buf + 2 * kTileBytes);
#pragma unroll
        for (int i = 0; i < T::loads; ++i) {
            const int r = lrow + i * T::rows;
            __bf16* kr = kl + r * kHeadDim;
            __bf16* vr = vl + r * kHeadDim;
            if constexpr (T::bf16) {
                *reinterpret_cast<u32x4_t*>(kr + 8 * (chunk ^ (r & 15))) = kreg[i];
                *reinterpret_cast<u32x4_t*>(vr + 8 * (chunk ^ (4 * (r & 3)))) = vreg[i];
            } else {
                constexpr int kCode = kKv == kKvBlocksInt8 ? kCodeInt8 : kCodeFp8;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int c = 2 * chunk + h;
                    *reinterpret_cast<bf16x8_t*>(kr + 8 * (c ^ (r & 15))) = codes_to_bf16<kCode>(kreg[i][2 * h], kreg[i][2 * h + 1]);
                    *reinterpret_cast<bf16x8_t*>(vr + 8 * (c ^ (4 * (r & 3)))) = codes_to_bf16<kCode>(vreg[i][2 * h], vreg[i][2 * h + 1]);
                }
                if constexpr (T::blocks) {
                    if (chunk == 0) {
                        sl[r] = ksreg[i] * p.scale_log2;
                        sl[kTile + r] = vsreg[i];
                    }
                }
            }
        }
    };

    auto compute = [&](const unsigned char* buf, int j) {
        const __bf16* kl = reinterpret_cast<const __bf16*>(buf);
        const __bf16* vl = kl + kTile * kHeadDim;
        const float* sl = reinterpret_cast<const float*>(buf + 2 * kTileBytes);
        // S^T: register i of block tb is token 32 tb + 8 (i / 4) + 4 half + i % 4, of row l32
        f32x16_t s[2];
#pragma unroll
        for (int tb = 0; tb < 2; ++tb) {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[tb][i] = 0.f;
#pragma unroll
            for (int ks = 0; ks < 8; ++ks) {
                const bf16x8_t ka =
                    *reinterpret_cast<const bf16x8_t*>(kl + (32 * tb + l32) * kHeadDim + 8 * ((2 * ks + half) ^ (l32 & 15)));
                s[tb] = mfma32(ka, qop[ks], s[tb]);
            }
        }
        float top = -INFINITY;
#pragma unroll
        for (int tb = 0; tb < 2; ++tb)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                [[maybe_unused]] f32x4_t ks4;
                if constexpr (T::blocks) ks4 = *reinterpret_cast<const f32x4_t*>(sl + 32 * tb + 8 * q + 4 * half);
#pragma unroll
                for (int i = 0; i < 4; ++i) s[tb][4 * q + i] *= T::blocks ? ks4[i] : p.scale_log2;
            }
        const int left = it.t1 - (it.t0 + j * kTile);
        if (left < kTile) {
#pragma unroll
            for (int tb = 0; tb < 2; ++tb)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (32 * tb + 8 * (i / 4) + 4 * half + i % 4 >= left) s[tb][i] = -INFINITY;
        }
#pragma unroll
        for (int tb = 0; tb < 2; ++tb)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, s[tb][i]);
        top = half_max(top);
        // The maximum moves only where it is exceeded by more than 2^8 (P is at most 2^8 then).
        if (__any(top > m_run + 8.f)) {
            const float m_new = fmaxf(m_run, top);
            const float alpha = fast_exp2(m_run - (m_new == -INFINITY ? 0.f : m_new));
            m_run = m_new;
            l_run *= alpha;
#pragma unroll
            for (int db = 0; db < 4; ++db) oacc[db] *= alpha;
        }
        const float m_sub = m_run == -INFINITY ? 0.f : m_run;
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int tb = 0; tb < 2; ++tb)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[tb][i] = fast_exp2(s[tb][i] - m_sub);
                sum[i & 1] += s[tb][i];
            }
        l_run += sum[0] + sum[1];
        // V^T as the A operand: lane holds column 32 db + l32 of the tokens whose P it holds
        const int l16 = lane & 15;
#pragma unroll
        for (int tb = 0; tb < 2; ++tb)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                bf16x8_t pop;
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    [[maybe_unused]] f32x4_t vs4;
                    if constexpr (T::blocks)
                        vs4 = *reinterpret_cast<const f32x4_t*>(sl + kTile + 32 * tb + 16 * h + 8 * q + 4 * half);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float x = s[tb][8 * h + 4 * q + i];
                        pop[4 * q + i] = (__bf16)(T::blocks ? x * vs4[i] : x);
                    }
                }
                // rows 32 tb + 16 h + 4 half + {0..3} and 8 more; lane l16 / 4 of its 16 names the row
                const int row = 32 * tb + 16 * h + 4 * half + (l16 >> 2);
#pragma unroll
                for (int db = 0; db < 4; ++db) {
                    // columns 32 db + 16 (l32 / 16) + 4 (l16 % 4) .. +3: half a 16-byte piece
                    const int c = 4 * db + 2 * (l32 >> 4) + ((l16 & 3) >> 1);
                    const __bf16* src = vl + row * kHeadDim + 8 * (c ^ (4 * (row & 3))) + 4 * (l16 & 1);
                    const bf16x4_t lo = lds_read_tr16(src);
                    const bf16x4_t hi = lds_read_tr16(src + 8 * kHeadDim);
                    oacc[db] = mfma32(__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7), pop, oacc[db]);
                }
            }
    };

    fetch_pages(0);
    load(0, tiles > 1);
    for (int j = 0; j < tiles; ++j) {
        unsigned char* buf = smem + (j & 1) * kBufBytes;
        stage(buf);
        if (j + 1 < tiles) load(j + 1, j + 2 < tiles);
        __syncthreads();   // (the buffer before this one is written again only after the next barrier)
        if (active) compute(buf, j);
    }

    if (!active) return;
    l_run = half_sum(l_run);
    if (32 * wave + l32 < it.rows) {
        const int64_t slot = it.slot + (int64_t)kvh * it.stride + 32 * wave + l32;
        float* po = p.part_o + slot * kHeadDim + 4 * half;
#pragma unroll
        for (int db = 0; db < 4; ++db)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const f32x4_t o = {oacc[db][4 * q], oacc[db][4 * q + 1], oacc[db][4 * q + 2], oacc[db][4 * q + 3]};
                *reinterpret_cast<f32x4_t*>(po + 32 * db + 8 * q) = T::blocks ? o : o * p.v_scale;
            }
        if (half == 0) {
            p.part_ml[slot * 2] = m_run;
            p.part_ml[slot * 2 + 1] = l_run;
        }
    }
}

constexpr int max_int(int a, int b) { return a > b ? a : b; }

template <int kKv, int kSeg>
__global__ __launch_bounds__(kThreads, 2) void decode_shared_kernel(SharedParams p) {
    __shared__ __attribute__((aligned(16))) unsigned char smem[max_int(kSharedSmem, kDecItemSmem<kKv, kDecWaves>)];
    const int at = fast_div((int)blockIdx.x, p.div_hkv);
    const int kvh = (int)blockIdx.x - at * p.d.hkv;
    const Item it = p.items[at];   // (there is room for every workgroup's)
    if (at >= *p.count) return;
    if (it.rows > 0) {
        shared_item<kKv>(p, smem, it, kvh);
    } else {
        const bool whole = it.slot < 0;
        dec_item_of<kKv, kSeg, kDecWaves, true>(p.d, smem, it.t0, it.t1, kvh, it.b, threadIdx.x, whole,
                                                whole ? 0 : it.slot + (int64_t)kvh * it.stride);
    }
}

// ---------------------------------------------------------------- merge
// As decode_combine_kernel: 16 lanes of 8 columns for each of 16 / kWays query heads,
// kWays ways over a sequence's partials.
template <int kWays>
__global__ __launch_bounds__(kThreads) void shared_merge_kernel(SharedParams sp) {
    const DecodeParams& p = sp.d;
    constexpr int kHeads = 16 / kWays;
    __shared__ float s_part[kWays * kHeads * 160];
    const int b = blockIdx.y;
    const Seq s = sp.seqs[b];
    if (s.whole) return;
    const int d16 = threadIdx.x & 15;
    const int way = (threadIdx.x >> 4) / kHeads, hl = (threadIdx.x >> 4) % kHeads;
    const int qh_raw = blockIdx.x * kHeads + hl, qh = min(qh_raw, p.hq - 1);
    const int kvh = fast_div(qh, sp.div_group), h = qh - kvh * p.group;
    const int n = s.n_shared + s.n_own;
    const bool store = way == 0 && qh_raw < p.hq;
    __bf16* out = p.o + b * p.o_sb + qh * p.o_sh + 8 * d16;
    if (n == 0) {
        bf16x8_t z;
#pragma unroll
        for (int j = 0; j < 8; ++j) z[j] = (__bf16)0.f;
        if (store) *reinterpret_cast<bf16x8_t*>(out) = z;
        if (store && p.lse != nullptr && d16 == 0) p.lse[(int64_t)b * p.hq + qh] = -INFINITY;
        return;
    }
    auto row_of = [&](int i) {
        i = min(i, n - 1);
        return i < s.n_shared ? (int64_t)s.shared + (int64_t)i * s.step + kvh * s.head + h
                              : (int64_t)s.own + ((int64_t)(i - s.n_shared) * p.hkv + kvh) * p.group + h;
    };
    constexpr int kBatch = 4;
    float M = -INFINITY, L = 0.f;
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    auto merge = [&](float m, float l, const float* o, bool valid) {
        const float m_new = fmaxf(M, valid ? m : -INFINITY);
        const float m_sub = m_new == -INFINITY ? 0.f : m_new;
        const float c0 = fast_exp2(M - m_sub), c1 = fast_exp2(m - m_sub);
        M = m_new;
        L = valid ? c0 * L + c1 * l : L;
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] = valid ? c0 * acc[j] + c1 * o[j] : acc[j];
    };
    for (int i0 = way; i0 < n; i0 += kBatch * kWays) {
        float ms[kBatch], ls[kBatch];
        f32x4_t a[kBatch][2];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int64_t row = row_of(i0 + i * kWays);
            ms[i] = p.part_ml[2 * row];
            ls[i] = p.part_ml[2 * row + 1];
            a[i][0] = *reinterpret_cast<const f32x4_t*>(p.part_o + row * kHeadDim + 8 * d16);
            a[i][1] = *reinterpret_cast<const f32x4_t*>(p.part_o + row * kHeadDim + 8 * d16 + 4);
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const float o[8] = {a[i][0][0], a[i][0][1], a[i][0][2], a[i][0][3], a[i][1][0], a[i][1][1], a[i][1][2], a[i][1][3]};
            merge(ms[i], ls[i], o, i0 + i * kWays < n);
        }
    }
    if constexpr (kWays > 1) {
        float* mine = s_part + (way * kHeads + hl) * 160 + d16;
#pragma unroll
        for (int j = 0; j < 8; ++j) mine[16 * j] = acc[j];
        mine[128] = M;
        mine[144] = L;
        __syncthreads();
        if (way != 0) return;
        for (int w = 1; w < min(kWays, n); ++w) {
            const float* o = s_part + (w * kHeads + hl) * 160 + d16;
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = o[16 * j];
            merge(o[128], o[144], v, true);
        }
    }
    if (!store) return;
    const float inv = 1.f / L;
    bf16x8_t r;
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = (__bf16)(acc[j] * inv);
    *reinterpret_cast<bf16x8_t*>(out) = r;
    if (p.lse != nullptr && d16 == 0) p.lse[(int64_t)b * p.hq + qh] = M * kLn2 + logf(L);
}

// Page segments as the paged decode takes them (decode_item.h).
int page_segment(const fgqa_kv_cache& c) {
    const int64_t most = std::max(c.k_stride[1], c.v_stride[1]);
    if ((int64_t)c.page_size * most * 2 >= ((int64_t)1 << 31)) return 0;
    const int least = c.kv_dtype == FGQA_KV_BF16 ? 4 : 8;
    return c.page_size >= 32 ? 32 : c.page_size >= least ? c.page_size : 0;
}

template <int kKv>
void launch_shared(const SharedParams& p, int seg, unsigned grid, hipStream_t s) {
    auto launch = [&](auto segment) {
        hipLaunchKernelGGL((decode_shared_kernel<kKv, decltype(segment)::value>), dim3(grid), dim3(kThreads), 0, s, p);
    };
    if (seg == 32) launch(std::integral_constant<int, 32>{});
    else if (seg == 16) launch(std::integral_constant<int, 16>{});
    else if (seg == 8) launch(std::integral_constant<int, 8>{});
    else if constexpr (kKv == kKvPagedBf16) {
        if (seg == 4) launch(std::integral_constant<int, 4>{});
        else launch(std::integral_constant<int, 0>{});
    } else launch(std::integral_constant<int, 0>{});
}

}  // namespace
}  // namespace fgqa

using namespace fgqa;

extern "C" int fgqa_decode_shared_workspace_bytes(const fgqa_decode_shared_args* a, size_t* bytes) {
    int st = plan::validate_decode_shared(a);
    if (st != FGQA_OK || bytes == nullptr) return st != FGQA_OK ? st : FGQA_ERR_INVALID_ARGUMENT;
    plan::SharedPlan pl;
    st = plan::plan_decode_shared(a, device_cu_count(), &pl);
    if (st != FGQA_OK) return st;
    *bytes = pl.total;
    return FGQA_OK;
}

extern "C" int fgqa_decode_shared(const fgqa_decode_shared_args* a, void* stream) {
    int st = plan::validate_decode_shared(a);
    if (st == FGQA_OK) st = plan::validate_decode_shared_pointers(a);
    if (st != FGQA_OK) return st;
    if (a->batch == 0) return FGQA_OK;
    plan::SharedPlan pl;
    st = plan::plan_decode_shared(a, device_cu_count(), &pl);
    if (st != FGQA_OK) return st;
    std::unique_lock<std::mutex> lock;
    char* ws = static_cast<char*>(a->workspace);
    if (ws == nullptr && a->workspace_bytes == 0) {
        lock = workspace_lock();
        ws = static_cast<char*>(internal_workspace(pl.total, &st));
        if (st != FGQA_OK) return st;
    } else if (ws == nullptr || a->workspace_bytes < pl.total) {
        return FGQA_ERR_WORKSPACE;
    } else if ((reinterpret_cast<uintptr_t>(ws) & 255u) != 0) {
        return FGQA_ERR_UNSUPPORTED;
    }

    const fgqa_kv_cache& c = a->cache;
    SharedParams p = {};
    DecodeParams& d = p.d;
    d.q = static_cast<const __bf16*>(a->q);
    d.k = static_cast<const __bf16*>(c.k);
    d.v = static_cast<const __bf16*>(c.v);
    d.o = static_cast<__bf16*>(a->o);
    d.lse = a->lse;
    d.seqlens = a->seqlens;
    d.part_o = reinterpret_cast<float*>(ws);
    d.part_ml = reinterpret_cast<float*>(ws + pl.part_ml_off);
    d.q_sb = a->q_stride[0];
    d.q_sh = a->q_stride[1];
    d.o_sb = a->o_stride[0];
    d.o_sh = a->o_stride[1];
    d.k_sb = c.k_stride[0];
    d.k_ss = c.k_stride[1];
    d.k_sh = c.k_stride[2];
    d.v_sb = c.v_stride[0];
    d.v_ss = c.v_stride[1];
    d.v_sh = c.v_stride[2];
    d.batch = a->batch;
    d.max_seqlen = a->max_seqlen;
    d.hq = a->num_q_heads;
    d.hkv = c.num_kv_heads;
    d.group = d.hq / d.hkv;
    const bool blocks = c.k_scales != nullptr, whole = c.kv_dtype == FGQA_KV_FP8_E4M3 && !blocks;
    d.scale_log2 = a->scale * (whole ? c.k_scale : 1.f) * kLog2e;
    d.v_scale = whole ? c.v_scale : 1.f;
    d.block_table = a->block_table;
    d.bt_stride = a->block_table_stride;
    d.page_shift = plan::log2_of(c.page_size);
    d.num_pages = c.num_pages;
    if (blocks) {
        d.k_scales = c.k_scales;
        d.v_scales = c.v_scales;
        d.ks_sp = c.k_scales_stride[0];
        d.ks_sh = c.k_scales_stride[1];
        d.vs_sp = c.v_scales_stride[0];
        d.vs_sh = c.v_scales_stride[1];
    }
    p.group_starts = a->group_starts;
    p.shared_lens = a->shared_lens;
    p.num_groups = a->num_groups;
    p.slots = pl.slots;
    p.div_group = make_fast_div(d.group);
    p.div_hkv = make_fast_div(d.hkv);
    p.items = reinterpret_cast<Item*>(ws + pl.items_off);
    p.seqs = reinterpret_cast<Seq*>(ws + pl.seqs_off);
    p.count = reinterpret_cast<int32_t*>(ws + pl.count_off);

    const hipStream_t s = static_cast<hipStream_t>(stream);
    hipLaunchKernelGGL(shared_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, p);
    if (a->max_seqlen > 0) {
        const unsigned grid = (unsigned)(pl.max_items * d.hkv);
        const int seg = page_segment(c);
        if (c.kv_dtype == FGQA_KV_BF16) launch_shared<kKvPagedBf16>(p, seg, grid, s);
        else if (c.kv_dtype == FGQA_KV_INT8) launch_shared<kKvBlocksInt8>(p, seg, grid, s);
        else if (blocks) launch_shared<kKvBlocksFp8>(p, seg, grid, s);
        else launch_shared<kKvPagedFp8>(p, seg, grid, s);
    }
    hipLaunchKernelGGL(shared_merge_kernel<4>, dim3((unsigned)((d.hq + 3) / 4), (unsigned)d.batch), dim3(kThreads), 0, s, p);
    return hipGetLastError() == hipSuccess ? FGQA_OK : FGQA_ERR_HIP;
}
