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
// A plan finds the groups and cuts all work into pieces of about equal token counts that
// fill the chip; one launch runs them; one merges the partials.  The running launch's
// workgroups plan for themselves up to 256 sequences: 4 samples of a prompt of 1000 tokens
// of bf16, 8 KV heads, took 14.5 us, with the plan in a launch of its own 18.2 (128 of 8000,
// one KV head: 34.3 and 64.4; 4 prompts of 8000 tokens of e4m3, 16 samples each: 55.6 and
// 57.4; 128 questions to one document of 32,768 of bf16: 208 and 209, of e4m3: 276 and 283).
#include <algorithm>
#include <type_traits>

#include "decode_item.h"
#include "fgqa_device.h"
#include "fgqa_internal.h"
#include "../host/pages_plan.h"

namespace fgqa {
namespace {

constexpr int kThreads = 256;
constexpr int kPlanThreads = 1024;       // of a planning workgroup of its own
constexpr int kTile = 64, kBlock = 32;   // shared tokens of a barrier, and of a step

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
    float scale_log2;    // shared tokens of caches without block scales: not negative, Q negated instead
    uint32_t q_sign;
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

// A workgroup of kN threads plans all work: items(first, n, item) has a range of items,
// of which item(i) makes one; seqs(b, s) a sequence's partials.  The number of items.
//
// Latency bounds it: a few dependent loads, barriers and scans, with a thread for each
// group and sequence as far as they go.  Where 256 threads go that far each workgroup of the
// decode plans for itself and makes its own item: a launch less.
template <int kN, typename Items, typename Seqs>
__device__ __forceinline__ int shared_plan(const SharedParams& p, Items&& items, Seqs&& seqs) {
    constexpr int kGroups = kN == kThreads ? kThreads : plan::kSharedMaxGroups;
    __shared__ int s_start[kGroups + 1];
    __shared__ int s_len[kGroups];     // shortest of its sequences, then what is shared
    __shared__ int s_first[kGroups];   // its first sequence with tokens, then its first row of partials
    __shared__ int s_count[kGroups];   // its sequences with tokens, then its pieces
    __shared__ int64_t s_wave[kN / kWave];
    const int tid = threadIdx.x, n = p.num_groups, batch = p.d.batch, group = p.d.group, hkv = p.d.hkv;
    // (these loads are under way together)
    const int len0 = tid < batch ? clamp_len(p.d, tid) : 0;
    const int shared0 = tid < n ? p.shared_lens[tid] : 0;
    for (int i = tid; i <= n; i += kN) {
        s_start[i] = n > 0 ? min(max(p.group_starts[i], 0), batch) : 0;
        if (i < n) {
            s_len[i] = s_first[i] = INT32_MAX;
            s_count[i] = 0;
        }
    }
    __syncthreads();
    int falls = 0;
    for (int i = tid; i < n; i += kN) falls |= s_start[i + 1] < s_start[i];
    if (__syncthreads_or(falls)) {   // each start at least the one before it
        for (int d = 1; d <= n; d *= 2) {
            int v[kGroups / kN + 1];
            int k = 0;
            for (int i = tid; i <= n; i += kN) v[k++] = max(s_start[i], i >= d ? s_start[i - d] : 0);
            __syncthreads();
            k = 0;
            for (int i = tid; i <= n; i += kN) s_start[i] = v[k++];
            __syncthreads();
        }
    }
    int64_t sum = 0, total;
    for (int b = tid; b < batch; b += kN) {
        const int len = b == tid ? len0 : clamp_len(p.d, b), g = group_of(s_start, n, b);
        sum += len;
        if (g < 0 || len == 0) continue;
        atomicMin(&s_len[g], len);
        atomicMin(&s_first[g], b);
        atomicAdd(&s_count[g], 1);
    }
    __syncthreads();
    auto rows_of = [&](int g) { return (s_start[g + 1] - s_start[g]) * group; };
    auto tiles_of = [&](int g) { return (rows_of(g) + plan::kSharedRows - 1) / plan::kSharedRows; };
    for (int g = tid; g < n; g += kN) {
        // (one sequence shares with none)
        int len = s_count[g] > 1 ? min(s_len[g], g == tid ? shared0 : p.shared_lens[g]) : 0;
        len = max(len, 0) >> p.d.page_shift << p.d.page_shift;
        if (len < plan::kSharedChunk) len = 0;
        s_len[g] = len;
        sum += (int64_t)(tiles_of(g) - s_count[g]) * len;   // in the tiles instead of each sequence
    }
    block_exclusive_scan<kN, true>(sum, s_wave, &total);
    const int chunk = (int)min(plan::shared_chunk(total, p.slots), (int64_t)1 << 30);   // (longer than any sequence)
    // Offsets of items, and, 32 bits up, of rows.
    int64_t at = 0;
    for (int g0 = 0; g0 < n; g0 += kN) {
        const int g = g0 + tid;
        const int len = g < n ? s_len[g] : 0, tiles = len > 0 ? tiles_of(g) : 0, rows = len > 0 ? rows_of(g) : 0;
        const int piece = len > 0 ? plan::shared_piece(len, chunk, kTile) : 1, pieces = (len + piece - 1) / piece;
        int64_t all;
        const int64_t mine = at + block_exclusive_scan<kN, true>(
                                      ((int64_t)pieces * hkv * rows << 32) + pieces * tiles, s_wave, &all);
        const int base = (int)(mine >> 32);
        items((int)(mine & 0xffffffff), pieces * tiles, [&](int i) {
            const int t = i % tiles;
            i /= tiles;
            Item it;
            it.b = s_start[g];
            it.table = s_first[g];
            it.t0 = i * piece;
            it.t1 = min(len, it.t0 + piece);
            it.row0 = t * plan::kSharedRows;
            it.rows = min(plan::kSharedRows, rows - it.row0);
            it.slot = base + i * hkv * rows + it.row0;
            it.stride = rows;
            return it;
        });
        if (g < n) {
            s_first[g] = base;
            s_count[g] = pieces;
        }
        at += all;
    }
    __syncthreads();
    for (int b0 = 0; b0 < batch; b0 += kN) {
        const int b = b0 + tid;
        const bool here = b < batch;
        const int g = here ? group_of(s_start, n, b) : -1, len = b == tid ? len0 : here ? clamp_len(p.d, b) : 0;
        const int begin = g < 0 || len == 0 ? 0 : s_len[g], left = len - begin;
        const int piece = left > 0 ? plan::shared_piece(left, chunk, plan::kSharedChunk) : 1, pieces = (left + piece - 1) / piece;
        const bool whole = begin == 0 && pieces == 1;
        int64_t all;
        const int64_t mine = at + block_exclusive_scan<kN, true>(
                                      ((int64_t)(whole ? 0 : pieces * hkv * group) << 32) + pieces, s_wave, &all);
        const int base = (int)(mine >> 32);
        items((int)(mine & 0xffffffff), pieces, [&](int i) {
            Item it;
            it.b = it.table = b;
            it.t0 = begin + i * piece;
            it.t1 = min(len, it.t0 + piece);
            it.slot = whole ? -1 : base + i * hkv * group;
            it.rows = it.row0 = 0;
            it.stride = group;
            return it;
        });
        if (here) {
            Seq s;
            s.n_shared = begin > 0 ? s_count[g] : 0;
            s.head = begin > 0 ? rows_of(g) : 0;
            s.step = hkv * s.head;
            s.shared = begin > 0 ? s_first[g] + (b - s_start[g]) * group : 0;
            s.own = base;
            s.n_own = pieces;
            s.whole = whole;
            s.pad = 0;
            seqs(b, s);
        }
        at += all;
    }
    return (int)(at & 0xffffffff);
}

__global__ __launch_bounds__(kPlanThreads) void shared_plan_kernel(SharedParams p) {
    const int count = shared_plan<kPlanThreads>(
        p,
        [&](int first, int n, auto&& item) {
            for (int i = 0; i < n; ++i) p.items[first + i] = item(i);
        },
        [&](int b, const Seq& s) { p.seqs[b] = s; });
    if (threadIdx.x == 0) *p.count = count;
}

// ---------------------------------------------------------------- shared tokens
// LDS rows are 256 bytes of bf16.  K's 16-byte piece c of row r lies at piece c ^ (r % 16), V's at
// c ^ 4 (r % 4): b128 reads of a piece of 16 rows, transposed reads of 64 bytes of 4 rows, and
// writes of whole rows then fall on all banks.
constexpr int kTileBytes = kTile * kHeadDim * 2;
constexpr int kSharedSmem = 4 * kTileBytes + 4 * kTile * 4;   // K and V of two tiles, their scales

// Loads of a tile: 16 bytes of a row each, bf16 rows by 16 threads, rows of codes by 8.
template <int kKv>
struct TileShape {
    static constexpr bool bf16 = kKv == kKvPagedBf16;
    static constexpr bool blocks = kKv >= kKvBlocksFp8;
    static constexpr int row_threads = bf16 ? 16 : 8;
    static constexpr int rows = kThreads / row_threads;   // of one load
    static constexpr int wave_rows = kWave / row_threads;
    static constexpr int loads = kTile / rows;
};

// Four scores times their tokens' scales.
__device__ __forceinline__ void scale4(f32x16_t& s, int q, f32x4_t by) {
#pragma unroll
    for (int i = 0; i < 4; ++i) s[4 * q + i] *= by[i];
}

// f(integral_constant<int, 0>), ..., f(integral_constant<int, N - 1>)
template <int N, int I = 0, typename F>
__device__ __forceinline__ void static_for(F&& f) {
    if constexpr (I < N) {
        f(std::integral_constant<int, I>{});
        static_for<N, I + 1>(f);
    }
}

// Tokens [it.t0, it.t1) of up to 128 query rows of one KV head.
// kUni: the rows of a wave's load lie in one page (pages of at least 4 rows of bf16, 8 of codes, whose
// bytes stay below 2^31), read through a buffer resource that ends at the last token (rows past
// it are zeros); the wave's pages come 64 loads at a time from one vector load of the table.
// kFlat: 32 tokens of a block-scaled cache lie in one page, so that a step's scores have one factor, as they
// have without block scales, and its P one too (128 questions to 32,768 tokens of e4m3: 276 us, with a
// factor for each token 281).
template <int kKv, int kSeg>
__device__ __forceinline__ void shared_item(const SharedParams& sp, unsigned char* smem, const Item& it, int kvh) {
    using T = TileShape<kKv>;
    constexpr bool kUni = kSeg > 0, kFlat = T::blocks && kSeg >= kBlock, kScaled = T::blocks && !kFlat;
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
        for (int ks = 0; ks < 8; ++ks) {
            const u32x4_t x = *reinterpret_cast<const u32x4_t*>(q + 16 * ks);
            qop[ks] = as_bf16x8(kScaled ? x : x ^ sp.q_sign);
        }
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
    const float* kscales = T::blocks ? p.k_scales + kvh * p.ks_sh : nullptr;
    const float* vscales = T::blocks ? p.v_scales + kvh * p.vs_sh : nullptr;
    const int32_t* bt = p.block_table + (int64_t)it.table * p.bt_stride;
    const int pmask = (1 << p.page_shift) - 1;
    const int lrow = tid / T::row_threads, chunk = tid % T::row_threads;
    const int t0 = __builtin_amdgcn_readfirstlane(it.t0), t1 = __builtin_amdgcn_readfirstlane(it.t1);
    const int tiles = (t1 - t0 + kTile - 1) / kTile;
    // bf16 rows go straight to LDS; codes pass through registers, where they are widened
    constexpr bool kDma = kUni && T::bf16;
    [[maybe_unused]] u32x4_t kreg[T::loads], vreg[T::loads];
    [[maybe_unused]] float ksreg[T::loads], vsreg[T::loads];
    [[maybe_unused]] const uint32_t kss = (uint32_t)(p.k_ss * kElem), vss = (uint32_t)(p.v_ss * kElem);   // (kUni: below 2^31)
    // (straight to LDS: lane l fills piece l % 16 of row l / 16 of the wave's four)
    const int lane_row = lane / T::row_threads;
    [[maybe_unused]] const uint32_t koff =
        (uint32_t)lane_row * kss + 16 * (kDma ? chunk ^ (T::wave_rows * wave + lane_row) : chunk);
    [[maybe_unused]] const uint32_t voff = (uint32_t)lane_row * vss + 16 * (kDma ? chunk ^ (4 * lane_row) : chunk);
    [[maybe_unused]] const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)smem +
                                           (uint32_t)(wave * T::wave_rows * kHeadDim * 2);
    // The scores run one block of 32 tokens ahead of P.V, so K's tile j is tokens 64 j + 32 .. 64 j + 95 (from -1
    // on, for the first block) and V's 64 j .. 64 j + 63: a step reads one of each.
    // kUni: lane l holds the addresses of the first rows of the wave's loads pt_first + l (load i of tile j being
    // (j + 1) * loads + i), the bytes of V's rows before the end (rows past it are zeros; K's may be any, in a page
    // all the same), and their scales.  A load then takes a few scalar instructions, not thirty.
    [[maybe_unused]] int pt_first = -kWave;
    [[maybe_unused]] uint32_t pt_k[2] = {0u, 0u}, pt_v[2] = {0u, 0u}, pt_vbytes = 0u;
    [[maybe_unused]] float pt_ks = 0.f, pt_vs = 0.f;
    [[maybe_unused]] auto pt_load = [&](int first) {
        const int n = first + lane;
        const int tok_v = t0 + (n / T::loads - 1) * kTile + (n % T::loads) * T::rows + wave * T::wave_rows;
        const int tok_k = max(tok_v + kBlock, t0);
        const int page_k = min(max(bt[min(tok_k, t1 - 1) >> p.page_shift], 0), p.num_pages - 1);
        const int page_v = min(max(bt[min(max(tok_v, t0), t1 - 1) >> p.page_shift], 0), p.num_pages - 1);
        const uint64_t k = reinterpret_cast<uint64_t>(kbase + page_k * p.k_sb * kElem + (int64_t)(tok_k & pmask) * kss);
        const uint64_t v = reinterpret_cast<uint64_t>(vbase + page_v * p.v_sb * kElem + (int64_t)(tok_v & pmask) * vss);
        pt_k[0] = (uint32_t)k;
        pt_k[1] = (uint32_t)(k >> 32);
        pt_v[0] = (uint32_t)v;
        pt_v[1] = (uint32_t)(v >> 32);
        const int rows = min(T::wave_rows, t1 - tok_v);
        pt_vbytes = rows > 0 ? (uint32_t)(rows - 1) * vss + kHeadDim * kElem : 0u;
        if constexpr (T::blocks) {
            pt_ks = kscales[page_k * p.ks_sp];
            pt_vs = vscales[page_v * p.vs_sp];
        }
        pt_first = first;
    };
    // else each row's page is looked up.  Tokens past the end read the last one again (their scores are masked;
    // the rows are numbers).
    [[maybe_unused]] auto load_rows = [&](int first, const unsigned char* base, int64_t page_bytes, int64_t row_bytes,
                                          [[maybe_unused]] const float* scales, [[maybe_unused]] int64_t scale_page,
                                          u32x4_t (&reg)[T::loads], [[maybe_unused]] float (&sreg)[T::loads]) {
#pragma unroll
        for (int i = 0; i < T::loads; ++i) {
            const int tok = min(max(first + lrow + i * T::rows, t0), t1 - 1);
            const int64_t page = min(max(bt[tok >> p.page_shift], 0), p.num_pages - 1);
            reg[i] = *reinterpret_cast<const u32x4_t*>(base + page * page_bytes + (tok & pmask) * row_bytes + chunk * 16);
            if constexpr (T::blocks) sreg[i] = scales[page * scale_page];
        }
    };
    // The loads of one cache's tile j: kUni, to registers or (kDma) to `lds`; else to registers.
    [[maybe_unused]] auto load_uni = [&](int j, const uint32_t (&at)[2], bool v, uint32_t off, [[maybe_unused]] u32x4_t (&reg)[T::loads],
                                         [[maybe_unused]] uint32_t lds) {
        const int first = (j + 1) * T::loads - pt_first;
        [[maybe_unused]] __amdgpu_buffer_rsrc_t rs[T::loads];
#pragma unroll
        for (int i = 0; i < T::loads; ++i) {
            const uint64_t base = (uint64_t)__builtin_amdgcn_readlane(at[1], first + i) << 32 |
                                  (uint32_t)__builtin_amdgcn_readlane(at[0], first + i);
            const uint32_t bytes = v ? __builtin_amdgcn_readlane(pt_vbytes, first + i)
                                     : (uint32_t)(T::wave_rows - 1) * kss + kHeadDim * kElem;
            const __amdgpu_buffer_rsrc_t r = make_rsrc(reinterpret_cast<const void*>(base), bytes);
            if constexpr (kDma) rs[i] = r;
            else reg[i] = buf_load16(r, off);
        }
        if constexpr (kDma) {
            lds_load_settle(rs);
            static_for<T::loads>([&](auto ic) {
                constexpr int i = decltype(ic)::value;
                lds_load16<i * T::rows * kHeadDim * 2>(lds, off, rs[i]);
            });
        }
    };
    auto load = [&](int j) {
        if constexpr (kUni) {
            if ((j + 2) * T::loads > pt_first + kWave) pt_load((j + 1) * T::loads);
            load_uni(j, pt_k, false, koff, kreg, lds0 + (j & 1) * kTileBytes);
            load_uni(j, pt_v, true, voff, vreg, lds0 + (2 + (j & 1)) * kTileBytes);
        } else {
            load_rows(t0 + j * kTile + kBlock, kbase, p.k_sb * kElem, p.k_ss * kElem, kscales, p.ks_sp, kreg, ksreg);
            load_rows(t0 + j * kTile, vbase, p.v_sb * kElem, p.v_ss * kElem, vscales, p.vs_sp, vreg, vsreg);
        }
    };
    float* const scale_lds = reinterpret_cast<float*>(smem + 4 * kTileBytes);   // K's of two tiles, V's
    // Registers to buffer `at` (K: 0 and 1, V: 2 and 3).
    [[maybe_unused]] auto stage_one = [&](int j, int at, const u32x4_t (&reg)[T::loads], [[maybe_unused]] const float (&sreg)[T::loads],
                                      [[maybe_unused]] float pt_scale, [[maybe_unused]] float factor) {
        const int turn = at < 2 ? lrow & 15 : 4 * (lrow & 3);   // (rows 16 on turn alike)
        __bf16* d = reinterpret_cast<__bf16*>(smem + at * kTileBytes) + lrow * kHeadDim;
#pragma unroll
        for (int i = 0; i < T::loads; ++i) {
            __bf16* r = d + i * T::rows * kHeadDim;
            if constexpr (T::bf16) {
                *reinterpret_cast<u32x4_t*>(r + 8 * (chunk ^ turn)) = reg[i];
            } else {
                constexpr int kCode = kKv == kKvBlocksInt8 ? kCodeInt8 : kCodeFp8;
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    *reinterpret_cast<bf16x8_t*>(r + 8 * ((2 * chunk + h) ^ turn)) =
                        codes_to_bf16<kCode>(reg[i][2 * h], reg[i][2 * h + 1]);
                if constexpr (T::blocks) {
                    // (kUni: the pages' vector is still the one of the loads)
                    float x = 0.f;
                    if constexpr (kUni)
                        x = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(pt_scale), (j + 1) * T::loads + i - pt_first));
                    else x = sreg[i];
                    if (chunk == 0) scale_lds[at * kTile + lrow + i * T::rows] = x * factor;
                }
            }
        }
    };
    auto stage = [&]([[maybe_unused]] int j) {
        if constexpr (!kDma) {
            stage_one(j, j & 1, kreg, ksreg, pt_ks, kScaled ? p.scale_log2 : sp.scale_log2);
            stage_one(j, 2 + (j & 1), vreg, vsreg, pt_vs, 1.f);
        }
    };
    // what went straight to LDS has landed
    auto landed = [] {
        if constexpr (kDma) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    };

    // Operands in LDS: K's piece 2 ks + half of row l32 (and 32 on), V's by transposed reads of rows
    // 4 half + (lane % 16) / 4 (and 8 on), columns 32 db + 16 ((lane % 32) / 16) + 4 (lane % 4) .. +3.
    int k_at[8], v_at[4];
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) k_at[ks] = l32 * kHeadDim + 8 * ((2 * ks + half) ^ (l32 & 15));
#pragma unroll
    for (int db = 0; db < 4; ++db) {
        const int r = 4 * half + ((lane & 15) >> 2), c = 4 * db + 2 * (l32 >> 4) + ((lane & 3) >> 1);
        v_at[db] = r * kHeadDim + 8 * (c ^ (4 * (r & 3))) + 4 * (lane & 1);
    }
    // Block h (0, 1) of K's and of V's tile: operand ks of the scores; columns n % 4 of 16 tokens n / 4
    auto k_operand = [&](int j, int h, int ks) {
        return *reinterpret_cast<const bf16x8_t*>(reinterpret_cast<const __bf16*>(smem + (j & 1) * kTileBytes) + k_at[ks] +
                                                  h * kBlock * kHeadDim);
    };
    auto v_operand = [&](int j, int h, int n) {
        const __bf16* src = reinterpret_cast<const __bf16*>(smem + (2 + (j & 1)) * kTileBytes) + v_at[n & 3] +
                            (h * kBlock + 16 * (n >> 2)) * kHeadDim;
        return __builtin_shufflevector(lds_read_tr16(src), lds_read_tr16(src + 8 * kHeadDim), 0, 1, 2, 3, 4, 5, 6, 7);
    };
    // Of caches with block scales: those of K's or V's tokens 8 q + 4 half + {0..3} of a block.
    auto scales_of = [&](int at, int h, int q) {
        return *reinterpret_cast<const f32x4_t*>(scale_lds + at * kTile + h * kBlock + 8 * q + 4 * half);
    };
    auto mask = [&](int left, f32x16_t& s) {
        left -= 4 * half;
        asm volatile("" : "+v"(left));   // (else the comparands are kept in registers for the whole loop)
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (8 * (i / 4) + i % 4 >= left) s[i] = -INFINITY;
    };
    auto largest = [&](const f32x16_t& s) {
        float x = s[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) x = fmaxf(x, s[i]);
        return x;
    };

    // Block b's tokens, half h of V's tile j: the scores of block b + 1 (half h of K's tile) and P.V of block b, with
    // the softmax of block b and the largest of the next scores spread between the products.  S^T: register i is
    // token 8 (i / 4) + 4 half + i % 4 of its block, of row l32.
    // Written in the order that it is to be issued in: operands three or four products ahead (the first of the
    // tile's second half at the end of its first), nothing that waits for a product right behind it.
    bf16x8_t ring[4], vring[3];
    // kFlat: block h's factor of the scores (above 0: masked scores stay -inf; the least scale times the scores' is no
    // normal number), and of P
    [[maybe_unused]] auto k_factor = [&](int at, int h) { return fmaxf(scale_lds[at * kTile + h * kBlock], __FLT_DENORM_MIN__); };
    auto step = [&](int j, auto half_c, f32x16_t& s, f32x16_t& next, float& top, [[maybe_unused]] float factor,
                    [[maybe_unused]] float& next_factor) {
        constexpr int h = decltype(half_c)::value;
        const int left = t1 - (t0 + j * kTile + h * kBlock);
        if (left < kBlock) {
            mask(left, s);
            top = largest(s);
        }
        if constexpr (h == 0) {
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) ring[ks] = k_operand(j, 0, ks);
        }
        const float c = kFlat ? factor : kScaled ? 1.f : sp.scale_log2;
        [[maybe_unused]] const float by_all = kFlat ? scale_lds[(2 + (j & 1)) * kTile + h * kBlock] : 1.f;
        float sum[2] = {0.f, 0.f}, m_sub = 0.f;
        bf16x8_t pop[2];
        // With block scales P times V's scale is held in two bf16 numbers, its rounding and what that leaves: 16 bits,
        // which the output's 8 do not show, as they do not the 22 of the decode one by one.  (4 prompts of 8000 tokens
        // of e4m3, 16 samples each: 50.2 us, outputs 6e-5 of their norm off the 32-bit form's; one number 47.3 us and 1.6e-3.)
        [[maybe_unused]] bf16x8_t plo[2];
        [[maybe_unused]] f32x4_t by;
        auto softmax = [&](auto ec) {
            constexpr int e = decltype(ec)::value;
            if constexpr (kScaled && e % 4 == 0) by = scales_of(2 + (j & 1), h, e / 4);
            const float w = fast_exp2(kScaled ? s[e] - m_sub : fmaf(s[e], c, -m_sub));
            sum[e & 1] += w;
            const float x = kScaled ? w * by[e & 3] : kFlat ? w * by_all : w;
            pop[e >> 3][e & 7] = (__bf16)x;
            if constexpr (T::blocks) plo[e >> 3][e & 7] = (__bf16)(x - (float)pop[e >> 3][e & 7]);
        };
#pragma unroll
        for (int i = 0; i < 16; ++i) next[i] = 0.f;
        static_for<8>([&](auto ic) {
            constexpr int n = decltype(ic)::value;
            __builtin_amdgcn_sched_barrier(0);
            next = mfma32(ring[n & 3], qop[n], next);
            if constexpr (n < 4) ring[n & 3] = k_operand(j, h, n + 4);
            else if constexpr (n >= 5) vring[n - 5] = v_operand(j, h, n - 5);
            if constexpr (n == 0) {
                const float m_block = half_max(top) * c;
                // What is subtracted is set 8 above a largest score and moves only where one exceeds it: P is
                // at most 1 (P above 1 made sums of values near bf16's largest, and P times a large block's
                // scale, infinite), and 2^-8 at least where it counts, which costs a float no bits.
                if (__any(m_block > m_run)) {
                    const float m_new = m_block > m_run ? m_block + 8.f : m_run;
                    const float alpha = fast_exp2(m_run - (m_new == -INFINITY ? 0.f : m_new));
                    m_run = m_new;
                    l_run *= alpha;
#pragma unroll
                    for (int db = 0; db < 4; ++db) oacc[db] *= alpha;
                }
                m_sub = m_run == -INFINITY ? 0.f : m_run;
            } else if constexpr (n < 6) {
                softmax(std::integral_constant<int, 2 * n - 2>{});
                softmax(std::integral_constant<int, 2 * n - 1>{});
            } else {
                softmax(std::integral_constant<int, n + 4>{});
            }
        });
        // V^T as the A operand: lane holds column 32 db + l32 of the tokens whose P it holds
        float most = 0.f;
        static_for<8>([&](auto ic) {
            constexpr int n = decltype(ic)::value;
            __builtin_amdgcn_sched_barrier(0);
            oacc[n & 3] = mfma32(vring[n % 3], pop[n >> 2], oacc[n & 3]);
            if constexpr (T::blocks) oacc[n & 3] = mfma32(vring[n % 3], plo[n >> 2], oacc[n & 3]);
            if constexpr (n + 3 < 8) vring[n % 3] = v_operand(j, h, n + 3);
            else if constexpr (h == 0) ring[n - 5] = k_operand(j, 1, n - 5);
            if constexpr (n < 2) {
                softmax(std::integral_constant<int, 12 + 2 * n>{});
                softmax(std::integral_constant<int, 13 + 2 * n>{});
            } else if constexpr (n < 6) {   // (4 scores each)
                if constexpr (kScaled) scale4(next, n - 2, scales_of(j & 1, h, n - 2));
                if constexpr (kFlat && n == 2) next_factor = k_factor(j & 1, h);
#pragma unroll
                for (int i = 4 * (n - 2); i < 4 * (n - 1); ++i) most = i == 0 ? next[0] : fmaxf(most, next[i]);
            }
        });
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (h == 0) ring[3] = k_operand(j, 1, 3);
        l_run += sum[0] + sum[1];
        top = most;
    };

    load(-1);
    landed();
    stage(-1);
    load(0);
    landed();
    stage(0);
    if constexpr (!kDma) {
        if (tiles > 1) load(1);
    }
    __syncthreads();
    f32x16_t s0, s1;
    float top = -INFINITY, f0 = 1.f, f1 = 1.f;
    if (active) {   // block 0: the second half of K's tile -1
#pragma unroll
        for (int i = 0; i < 16; ++i) s0[i] = 0.f;
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) s0 = mfma32(k_operand(-1, 1, ks), qop[ks], s0);
        if constexpr (kScaled) {
#pragma unroll
            for (int q = 0; q < 4; ++q) scale4(s0, q, scales_of(1, 1, q));
        }
        if constexpr (kFlat) f0 = k_factor(1, 1);
        top = largest(s0);
    }
    for (int j = 0; j < tiles; ++j) {
        __syncthreads();   // (tile j - 1 has been read, tile j is there)
        if (j + 1 < tiles) {
            stage(j + 1);
            if constexpr (kDma) load(j + 1);
            else if (j + 2 < tiles) load(j + 2);
        }
        if (active) {
            step(j, std::integral_constant<int, 0>{}, s0, s1, top, f0, f1);
            if (t0 + j * kTile + kBlock < t1) step(j, std::integral_constant<int, 1>{}, s1, s0, top, f1, f0);
        }
        landed();
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
    Item it;
    if (p.items == nullptr) {
        __shared__ Item s_item;
        const int count = shared_plan<kThreads>(
            p,
            [&](int first, int n, auto&& item) {
                if (at >= first && at - first < n) s_item = item(at - first);
            },
            [&](int b, const Seq& s) {
                if (blockIdx.x == 0) p.seqs[b] = s;
            });
        if (at >= count) return;
        __syncthreads();
        it = s_item;
    } else {
        it = p.items[at];   // (there is room for every workgroup's)
        if (at >= *p.count) return;
    }
    if (it.rows > 0) {
        shared_item<kKv, kSeg>(p, smem, it, kvh);
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
    if (plan::shared_as_blocks(a, device_cu_count())) {
        const fgqa_decode_blocks_args b = plan::as_decode_blocks(a);
        return fgqa_decode_blocks_workspace_bytes(&b, bytes);
    }
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
    if (plan::shared_as_blocks(a, device_cu_count())) {
        const fgqa_decode_blocks_args b = plan::as_decode_blocks(a);
        return fgqa_decode_blocks(&b, stream);
    }
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
    p.scale_log2 = score_scale(fabsf(d.scale_log2));
    p.q_sign = d.scale_log2 < 0.f ? 0x80008000u : 0u;
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
    if (d.batch <= kThreads && p.num_groups < kThreads && a->max_seqlen > 0) p.items = nullptr;   // (the workgroups plan)
    else hipLaunchKernelGGL(shared_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, p);
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
