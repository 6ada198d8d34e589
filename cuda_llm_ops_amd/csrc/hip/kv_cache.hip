// The paged KV cache's operators (include/fgqa_kv.h): writing tokens, the
// attention weight of each cached token, and eviction.
//
// A block is one page of one KV head: page_size rows of 128 elements.  Blocks
// in 8 bits hold codes c and one scale s, standing for s * c.  The scales that
// are made here are powers of two, so that x / s is exact and a code has one
// rounding, and growing a block's scale rounds its int8 codes once more and its
// e4m3 codes not at all (but where they become subnormal).
#include <algorithm>
#include <math.h>

#include "fgqa_internal.h"
#include "kv_cache_params.h"
#include "kv_codes.h"
#include "../host/kv_plan.h"

namespace fgqa {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kLanesPerRow = 8;                        // 16 elements of a row each
constexpr int kRowsPerSweep = kWave / kLanesPerRow;

typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int m = 1; m < kWave; m *= 2) v = xor_max(v, m);
    return v;
}

// x / s: exact for a power of two, else correctly rounded.
struct Divisor {
    float s, inv;
    bool pow2;
    __device__ explicit Divisor(float scale) : s(scale), inv(1.f / scale) {
        const uint32_t b = __float_as_uint(scale);
        pow2 = (b & 0x7fffffu) == 0 && b >= 0x00800000u && b < 0x7f000000u;
    }
    __device__ f32x4_t operator()(f32x4_t x) const {
        if (pow2) return x * inv;
        return f32x4_t{x[0] / s, x[1] / s, x[2] / s, x[3] / s};
    }
};

// 4 bf16 of two words -> fp32.
__device__ __forceinline__ f32x4_t bf16x4_to_f32(uint32_t w0, uint32_t w1) {
    return f32x4_t{__uint_as_float(w0 << 16), __uint_as_float(w0 & 0xffff0000u), __uint_as_float(w1 << 16),
                   __uint_as_float(w1 & 0xffff0000u)};
}

// How a cache of codes is scaled: not (bf16), as a whole, or block by block.
enum Scaling { kNone, kWhole, kBlocks };

// The waves that write one block and the sweeps (of 8 rows) each holds in
// registers: pages of up to 64 rows take a wave, larger ones a workgroup, which
// goes over pages of more than 256 rows in several rounds, reading them twice.
template <int kSweeps, int kBlockWaves>
struct BlockShape {
    static constexpr int sweeps = kSweeps, waves = kBlockWaves;
    static constexpr int rows = kSweeps * kBlockWaves * kRowsPerSweep;   // of one round
};

// The largest of the block's waves' values.
template <typename Shape>
__device__ __forceinline__ float block_max(float v, float* s_max) {
    v = wave_max(v);
    if constexpr (Shape::waves > 1) {
        const int wave = threadIdx.x / kWave;
        if ((threadIdx.x & (kWave - 1)) == 0) s_max[wave] = v;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < Shape::waves; ++w) v = fmaxf(v, s_max[w]);
    }
    return v;
}

// ---------------------------------------------------------------- append
struct AppendParams {
    CacheParams c;
    const unsigned char* x[2];       // new K, V
    int64_t x_b[2], x_t[2], x_h[2];  // bytes
    const int32_t* block_table;
    int64_t bt_stride;
    const int32_t* seqlens;
    const int32_t* new_lens;
    int max_new, max_tokens;
    int pages;                       // of one sequence that new tokens can touch
    uint32_t items;                  // batch * pages * 2 * hkv, below 2^31
};

// One block per item: item = ((b * pages + j) * 2 + K or V) * hkv + head, heads
// side by side as the new rows lie.  Memory bounds it: the rows stay in registers
// between their maximum and their codes, so each is read once (pages of more than
// 256 rows: twice).  2 x 16384 tokens of 8 heads into e4m3 pages of 64: 155 MB in 35 us,
// 4.4 TB/s where a copy runs at 4.9.  64 single tokens: 4.5 us, a launch.
template <int kCode, Scaling kScaling, typename Shape>
__global__ __launch_bounds__(kThreads) void append_kernel(AppendParams p) {
    __shared__ float s_max[kWaves];
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x / kWave));
    const uint32_t item = blockIdx.x * (uint32_t)(kWaves / Shape::waves) + (uint32_t)(wave / Shape::waves);
    if (item >= p.items) return;
    const int h = (int)(item % (uint32_t)p.c.hkv);
    const uint32_t rest = item / (uint32_t)p.c.hkv;
    const int kv = (int)(rest & 1);
    const int j = (int)((rest >> 1) % (uint32_t)p.pages);
    const int b = (int)((rest >> 1) / (uint32_t)p.pages);

    const int len = max(p.seqlens[b], 0);
    const int want = p.new_lens != nullptr ? min(max(p.new_lens[b], 0), p.max_new) : p.max_new;
    if (len >= p.max_tokens) return;
    const int end = (int)min((int64_t)len + want, (int64_t)p.max_tokens);
    const int page_at = (len >> p.c.page_shift) + j;
    const int64_t t0 = (int64_t)page_at << p.c.page_shift;   // the page's first token
    if (t0 >= end) return;
    const int page_rows = 1 << p.c.page_shift;
    const int slot0 = (int)max((int64_t)len - t0, (int64_t)0);                // new rows: slots [slot0, slot1)
    const int slot1 = (int)min((int64_t)end - t0, (int64_t)page_rows);
    if (slot0 >= slot1) return;
    const int page = p.block_table[(int64_t)b * p.bt_stride + page_at];
    if (page < 0 || page >= p.c.num_pages) return;

    const int row = lane / kLanesPerRow, chunk = lane % kLanesPerRow;
    const int first_row = (wave % Shape::waves) * Shape::sweeps * kRowsPerSweep + row;
    // token of slot 0 in the new rows (below 0 where the sequence's older tokens are)
    const int64_t i0 = t0 - len;
    const unsigned char* src = p.x[kv] + b * p.x_b[kv] + h * p.x_h[kv] + chunk * 32;
    unsigned char* dst = p.c.data[kv] + page * p.c.page[kv] + h * p.c.head[kv] + chunk * (kCode == kCodeBf16 ? 32 : 16);

    u32x4_t raw[Shape::sweeps][2];
    auto load = [&](int base) {
#pragma unroll
        for (int s = 0; s < Shape::sweeps; ++s) {
            const int slot = base + first_row + s * kRowsPerSweep;
            raw[s][0] = raw[s][1] = u32x4_t{0u, 0u, 0u, 0u};
            if (slot >= slot0 && slot < slot1) {
                const u32x4_t* r = reinterpret_cast<const u32x4_t*>(src + (i0 + slot) * p.x_t[kv]);
                raw[s][0] = __builtin_nontemporal_load(r);
                raw[s][1] = __builtin_nontemporal_load(r + 1);
            }
        }
    };
    const int begin = slot0 / Shape::rows * Shape::rows;   // rounds from the first new row's on
    const int last = (slot1 - 1) / Shape::rows * Shape::rows;

    float scale = p.c.scale[kv];
    [[maybe_unused]] bool all_finite = false;
    if constexpr (kScaling == kBlocks) {
        // Without a sign bf16 values order as 16-bit numbers, infinities and NaN
        // above all others; only a block that has such takes the maximum again
        // without them.
        u16x2_t most = {0, 0};
        for (int base = begin; base <= last; base += Shape::rows) {
            load(base);
#pragma unroll
            for (int s = 0; s < Shape::sweeps; ++s)
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2_t, raw[s][i / 4][i % 4] & 0x7fff7fffu));
        }
        const uint32_t top = min((uint32_t)max(most[0], most[1]), 0x7f80u);   // (NaN as inf: a maximum would drop it)
        float amax = block_max<Shape>(__uint_as_float(top << 16), s_max);
        all_finite = amax < INFINITY;
        if (!all_finite) {
            amax = 0.f;
            for (int base = last; base >= begin; base -= Shape::rows) {
                if (base != last) load(base);
#pragma unroll
                for (int s = 0; s < Shape::sweeps; ++s)
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const uint32_t w = raw[s][i / 4][i % 4];
                        amax = fmaxf(amax, fmaxf(finite_abs(__uint_as_float(w << 16)),
                                                 finite_abs(__uint_as_float(w & 0xffff0000u))));
                    }
            }
            if (begin != last) load(last);
            if constexpr (Shape::waves > 1) __syncthreads();   // s_max has been read
            amax = block_max<Shape>(amax, s_max);
        }
        scale = block_scale<kCode>(amax);
        float* at = p.c.scales[kv] + page * p.c.scale_page[kv] + h * p.c.scale_head[kv];
        bool fresh = true;
        if (slot0 > 0) {   // older tokens in the block
            const float old = *at;
            if (!(scale > old)) {
                scale = old;
                fresh = false;
            } else {
                // (codes times old / scale: codes times old can pass fp32's largest
                // number.  old / scale is exact, or 0 to every code.)
                const float ratio = old * (1.f / scale);
                for (int base = 0; base < slot0; base += Shape::rows)
#pragma unroll
                    for (int s = 0; s < Shape::sweeps; ++s) {
                        const int slot = base + first_row + s * kRowsPerSweep;
                        if (slot >= slot0) continue;
                        u32x4_t* r = reinterpret_cast<u32x4_t*>(dst + slot * p.c.slot[kv]);
                        u32x4_t w = *r;
#pragma unroll
                        for (int i = 0; i < 4; ++i) w[i] = to_codes<kCode>(codes_to_f32<kCode>(w[i]) * ratio);
                        *r = w;
                    }
            }
        }
        if constexpr (Shape::waves > 1) __syncthreads();   // every wave has read the old scale
        if (fresh && lane == 0 && wave % Shape::waves == 0) *at = scale;
    }
    const Divisor div(scale);
    for (int base = last; base >= begin; base -= Shape::rows) {
        if (kScaling != kBlocks || base != last) load(base);
#pragma unroll
        for (int s = 0; s < Shape::sweeps; ++s) {
            const int slot = base + first_row + s * kRowsPerSweep;
            if (slot < slot0 || slot >= slot1) continue;
            u32x4_t* r = reinterpret_cast<u32x4_t*>(dst + slot * p.c.slot[kv]);
            if constexpr (kCode == kCodeBf16) {
                r[0] = raw[s][0];
                r[1] = raw[s][1];
            } else {
                if (kScaling == kBlocks && all_finite && div.pow2) {
                    __builtin_nontemporal_store(finite_to_codes<kCode>(raw[s], scale, div.inv), r);
                    continue;
                }
                u32x4_t w;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    w[i] = to_codes<kCode>(div(bf16x4_to_f32(raw[s][i / 2][2 * (i % 2)], raw[s][i / 2][2 * (i % 2) + 1])));
                *r = w;
            }
        }
    }
}

// ---------------------------------------------------------------- weights
struct WeightsParams {
    CacheParams c;
    const __bf16* q;
    const float* lse;
    float* weights;
    int64_t q_b, q_h, w_b, w_h;
    const int32_t* block_table;
    int64_t bt_stride;
    const int32_t* seqlens;
    int max_seqlen, group;
    int waves;        // of one (sequence, head)
    float scale;
    uint32_t items;   // batch * waves * hkv
};

// One wave per 64 tokens of one KV head (plan::weights_waves: or several such
// items), two steps of 32; the waves of a workgroup
// take adjacent heads, so that a token's rows, which lie side by side, are read
// together.  (64 tokens an item are never slower than more, and small calls fill
// the chip; items of 32: 108 us for 92, 64 sequences of up to 16384.)  Memory
// bounds it: those 64 sequences, 64 / 8 heads, e4m3, 499 MB in 89 us, 5.6 TB/s; the
// stores of the weights between the reads of K cost 13 of them.  Rows are
// loaded whole (8 lanes of 16 bytes for codes, 16 for bf16), both steps at once,
// and staged in LDS as they are.
// S[h][t] = Q[h][:] . K[t][:] by v_mfma_f32_16x16x32_bf16 with the 16 query heads
// (zero past the group) as rows: a lane holds one token's scores of 4 heads, and
// the sum over heads takes two exchanges of lane groups.  The order of the head
// dim inside the products is free as long as Q's is the same: lane group g4
// takes the elements of the 16-byte pieces that it reads.
// kSeg (32, 16 or 8): page segments as in the block-scaled decode; 0: any pages.
// kTurns: a wave takes several items (the loop costs calls of an item a wave 1.5 to 3 %).
template <int kCode, Scaling kScaling, int kSeg, bool kTurns>
__global__ __launch_bounds__(kThreads) void weights_kernel(WeightsParams p) {
    constexpr int kStep = 32;
    constexpr int kRowBytes = kCode == kCodeBf16 ? 256 : 128;
    constexpr int kLanes = kRowBytes / 16;          // of a row
    constexpr int kRows = kWave / kLanes;           // of one load instruction
    constexpr int kLoads = kStep / kRows;           // of a step
    constexpr int kStride = kRowBytes + 16;         // LDS bytes of a row: 16 rows spread over all banks
    __shared__ __attribute__((aligned(16))) unsigned char smem[kWaves * kStep * kStride];
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x / kWave));
    const int l16 = lane & 15, g4 = lane >> 4;
    const uint32_t item = blockIdx.x * (uint32_t)kWaves + (uint32_t)wave;
    if (item >= p.items) return;
    const int kvh = (int)(item % (uint32_t)p.c.hkv);
    const uint32_t rest = item / (uint32_t)p.c.hkv;
    const int b = (int)(rest / (uint32_t)p.waves);
    const int first_item = (int)(rest % (uint32_t)p.waves);
    const int len = __builtin_amdgcn_readfirstlane(min(max(p.seqlens[b], 0), p.max_seqlen));
    const int n_items = (len + plan::kWeightsTokens - 1) / plan::kWeightsTokens;
    if (first_item >= n_items) return;

    const int32_t* bt = p.block_table + (int64_t)b * p.bt_stride;
    const int pmask = (1 << p.c.page_shift) - 1;
    const unsigned char* kbase = p.c.data[0] + kvh * p.c.head[0];
    const float* scales = p.c.scales[0] + kvh * p.c.scale_head[0];
    float* wrow = p.weights + b * p.w_b + kvh * p.w_h;
    unsigned char* kl = smem + wave * kStep * kStride;
    const int row = lane / kLanes, piece = lane % kLanes;

    // Segment l of the item (at most 8) has its page and scale in lane l.
    constexpr int kSegs = kSeg > 0 ? kStep / kSeg : 1;
    constexpr int kPer = kLoads / kSegs;
    int t_begin = 0, t_end = 0;
    [[maybe_unused]] int seg_page = 0;
    [[maybe_unused]] float seg_scale = p.scale;
    auto begin = [&](int item) {
        t_begin = item * plan::kWeightsTokens;
        t_end = min(t_begin + plan::kWeightsTokens, len);
        if constexpr (kSeg > 0) {
            seg_page = min(max(bt[min(t_begin + kSeg * lane, t_end - 1) >> p.c.page_shift], 0), p.c.num_pages - 1);
            if constexpr (kScaling == kBlocks) seg_scale = p.scale * scales[(int64_t)seg_page * p.c.scale_page[0]];
        }
    };
    begin(first_item);
    bf16x8_t qop[4];
    {
        const __bf16* qrow = p.q + b * p.q_b + (int64_t)(kvh * p.group + min(l16, p.group - 1)) * p.q_h;
        const u32x4_t zero = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
            const int d = kCode == kCodeBf16 ? 32 * kk + 8 * g4 : 64 * (kk / 2) + 16 * g4 + 8 * (kk % 2);
            const u32x4_t t = *reinterpret_cast<const u32x4_t*>(qrow + d);
            qop[kk] = as_bf16x8(l16 < p.group ? t : zero);
        }
    }
    // Heads past the group: exp(. - inf) = 0.  Their products are 0 * k, NaN where a
    // bf16 key holds an infinity, so bf16 ones are also left out of the sum.  (8-bit
    // keys hold none, and with a NaN the other heads' are NaN too.  Left out there
    // as well, 64 sequences of up to 16384 take 90.7 us for 88.6.)
    // (The difference is formed before log2(e) is multiplied in: its rounding then
    // is relative to the small exponents of the weights that count, not to the
    // LSE's size.)
    float neg_lse[4];
    [[maybe_unused]] bool in_group[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int g = 4 * g4 + i;
        const float l = p.lse[(int64_t)b * p.c.hkv * p.group + kvh * p.group + min(g, p.group - 1)];
        in_group[i] = g < p.group;
        neg_lse[i] = in_group[i] ? -l : -INFINITY;
    }

    struct Step {
        u32x4_t k[kLoads];
        float scale[2];   // kSeg 0: of tokens l16 and 16 + l16
        float w;          // old weight of token lane (below 32)
    };
    const uint32_t kss = (uint32_t)p.c.slot[0];
    [[maybe_unused]] const uint32_t koff = (uint32_t)row * kss + piece * 16;
    auto load = [&](int s, Step& x) {
        const int t0 = t_begin + s * kStep;
        if constexpr (kSeg > 0) {
#pragma unroll
            for (int g = 0; g < kSegs; ++g) {
                const int64_t page = __builtin_amdgcn_readlane(seg_page, s * kSegs + g);
                const int tok = t0 + kSeg * g;
                const int nv = min(kSeg, t_end - tok);   // rows before the item's end; the others read as zeros
                const __amdgpu_buffer_rsrc_t r =
                    make_rsrc(kbase + page * p.c.page[0] + (uint32_t)(tok & pmask) * kss,
                              nv > 0 ? (uint32_t)(nv - 1) * kss + kRowBytes : 0u);
#pragma unroll
                for (int i = 0; i < kPer; ++i) x.k[g * kPer + i] = buf_load16_nt(r, koff + (uint32_t)(kRows * i) * kss);
            }
        } else {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {   // (past the end: its last token, not stored)
                const int tok = min(t0 + kRows * i + row, t_end - 1);
                const int64_t page = min(max(bt[tok >> p.c.page_shift], 0), p.c.num_pages - 1);
                x.k[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(
                    kbase + page * p.c.page[0] + (tok & pmask) * p.c.slot[0] + piece * 16));
            }
#pragma unroll
            for (int tb = 0; tb < 2; ++tb) {
                x.scale[tb] = p.scale;
                if constexpr (kScaling == kBlocks) {
                    const int tok = min(t0 + 16 * tb + l16, t_end - 1);
                    const int64_t page = min(max(bt[tok >> p.c.page_shift], 0), p.c.num_pages - 1);
                    x.scale[tb] *= scales[page * p.c.scale_page[0]];
                }
            }
        }
        x.w = wrow[min(t0 + (lane & 31), t_end - 1)];
    };
    auto compute = [&](int s, const Step& x) {
        const int t0 = t_begin + s * kStep;
#pragma unroll
        for (int i = 0; i < kLoads; ++i)
            *reinterpret_cast<u32x4_t*>(kl + (kRows * i + row) * kStride + piece * 16) = x.k[i];
        const float old = x.w;
        float scale[2];
        if constexpr (kSeg > 0) {
#pragma unroll
            for (int tb = 0; tb < 2; ++tb) {
                auto of = [&](int g) {
                    return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(seg_scale), s * kSegs + g));
                };
                if constexpr (kSegs == 1) scale[tb] = of(0);
                else if constexpr (kSegs == 2) scale[tb] = of(tb);
                else scale[tb] = l16 < 8 ? of(2 * tb) : of(2 * tb + 1);
            }
        } else {
            scale[0] = x.scale[0];
            scale[1] = x.scale[1];
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        float sum[2];
#pragma unroll
        for (int tb = 0; tb < 2; ++tb) {
            f32x4_t c = {0.f, 0.f, 0.f, 0.f};
            const unsigned char* src = kl + (16 * tb + l16) * kStride + 16 * g4;
#pragma unroll
            for (int j = 0; j < kRowBytes / 64; ++j) {
                const u32x4_t w = *reinterpret_cast<const u32x4_t*>(src + 64 * j);
                if constexpr (kCode == kCodeBf16) {
                    c = mfma16(qop[j], as_bf16x8(w), c);
                } else {
                    c = mfma16(qop[2 * j], codes_to_bf16<kCode>(w[0], w[1]), c);
                    c = mfma16(qop[2 * j + 1], codes_to_bf16<kCode>(w[2], w[3]), c);
                }
            }
            sum[tb] = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float e = fast_exp2(fmaf(c[i], scale[tb], neg_lse[i]) * kLog2e);
                sum[tb] += kCode != kCodeBf16 || in_group[i] ? e : 0.f;
            }
        }
        // over the lane groups: groups 0 and 1 get the sums of tokens l16 and 16 + l16
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(sum[0]), __float_as_uint(sum[1]), false, false);
        const float total = half_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
        const int tok = t0 + lane;
        if (lane < kStep && tok < t_end) wrow[tok] = old + total;
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    };
    static_assert(plan::kWeightsTokens == 2 * kStep, "two steps an item");
    for (int item = first_item;;) {
        const bool two = t_begin + kStep < t_end;
        Step first, second;
        load(0, first);
        if (two) load(1, second);
        compute(0, first);
        if (two) compute(1, second);
        if constexpr (!kTurns) break;
        item += p.waves;
        if (item >= n_items) break;
        begin(item);
    }
}

// ---------------------------------------------------------------- evict
struct EvictParams {
    CacheParams c;
    const float* weights;
    float* new_weights;
    int64_t w_b, w_h, nw_b, nw_h;
    const int32_t* block_table;
    const int32_t* new_table;
    int64_t bt_stride, nt_stride;
    const int32_t* seqlens;
    int32_t* new_seqlens;
    int32_t* kept;
    int max_seqlen, weights_len, budget, recent;
    int max_tokens;  // lengths are clamped to it; tokens from max_seqlen on have no weight
    int most;        // tokens of a sequence that are kept: the budget, or what its new pages hold
    int pages;       // new pages of a sequence at most
    int parts;       // workgroups per row of the selection
    uint32_t items;  // batch * pages * 2 * hkv, below 2^31
};

constexpr int kSelectThreads = 1024;
constexpr int kSelectWaves = kSelectThreads / kWave;
constexpr int kBins = 2048;

// Weights in their order as unsigned numbers above 0; NaN above all, -0 as 0.
__device__ __forceinline__ uint32_t weight_key(float w) {
    const uint32_t b = __float_as_uint(w + 0.f);
    const uint32_t k = b ^ (uint32_t)(((int32_t)b >> 31) | (int32_t)0x80000000);
    return w != w ? 0xffffffffu : k;
}

// The weight of a key (of -0 and of a NaN: 0 and a NaN).
__device__ __forceinline__ float weight_of_key(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? (k == 0xffffffffu ? 0x7fc00000u : k ^ 0x80000000u) : ~k);
}

// Lanes of m before this one.
__device__ __forceinline__ uint32_t lanes_below(uint64_t m) {
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
}

// dst[from, to) = value by `threads` threads, 16 bytes at a time where they are aligned.
template <typename T>
__device__ __forceinline__ void fill_row(T* dst, int from, int to, T value, int thread, int threads) {
    static_assert(sizeof(T) == 4, "");
    typedef T vec __attribute__((ext_vector_type(4)));
    const int head = min(from + (int)((0 - (reinterpret_cast<uintptr_t>(dst + from) >> 2)) & 3), to);
    const int vecs = (to - head) / 4;
    if (thread < head - from) dst[from + thread] = value;
    for (int i = thread; i < vecs; i += threads) reinterpret_cast<vec*>(dst + head)[i] = vec{value, value, value, value};
    if (thread < to - head - 4 * vecs) dst[head + 4 * vecs + thread] = value;
}

// One workgroup per (sequence, head): the `need` largest keys of the candidates
// (tokens before the recent ones) by their digits from the top, 11, 11 and 10
// bits: the histogram of the keys that share the digits found so far says which
// digit the last kept key has.  Then every wave walks its part of the candidates
// in order and writes what is kept.  Integer sums only: no order matters.
// kHeld: candidates whose keys are held in LDS, read once, all loads in
// flight together; 0 for longer rows, which every pass reads again.  (In 32
// registers of a thread instead, whose passes cannot be loops, 23.3 us where LDS
// took 22.1.)
// The vector units of a row's one CU bound it: an operation on each of 32K keys
// takes 0.2 us, the first histogram 3.5.  Shared out over workgroups, the
// histograms would take further launches (that form was not built or timed);
// where there are fewer rows than CUs, `parts` workgroups find the same
// threshold, and each writes its part of every wave's steps.  8 rows of 32K: 17.2
// us (22.1 in one part), 256 of 8K 13.2, 4 of 600 6.9: the latency of loads, three
// histograms and their scans, and stores (the passes in a loop of one body: 0.8 us
// more).
template <int kHeld>
__global__ __launch_bounds__(kSelectThreads) void select_kernel(EvictParams p) {
    __shared__ __attribute__((aligned(16))) uint32_t s_keys[kHeld > 0 ? kHeld : 4];
    __shared__ __attribute__((aligned(16))) int s_hist[kBins];
    __shared__ __attribute__((aligned(16))) int s_wave[3][kSelectWaves];
    __shared__ int s_found[2];
    const int tid = threadIdx.x, lane = tid & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int part = (int)(blockIdx.x % (unsigned)p.parts);
    const unsigned row = blockIdx.x / (unsigned)p.parts;
    const int h = (int)(row % (unsigned)p.c.hkv), b = (int)(row / (unsigned)p.c.hkv);
    const int len = min(max(p.seqlens[b], 0), p.max_tokens);
    const int count = min(len, p.most);
    // (tokens without a weight count as recent: the candidates all have one)
    const int recent = len > p.most ? min(max(p.recent, len - p.max_seqlen), p.most) : len;
    const int cand = len - recent;
    const int need = count - recent;
    const float* w = p.weights + b * p.w_b + h * p.w_h;
    float* nw = p.new_weights + b * p.nw_b + h * p.nw_h;
    int32_t* kept = p.kept + ((int64_t)b * p.c.hkv + h) * p.budget;

    // each wave's run of the candidates: steps of 4 in a row per lane, the key 0,
    // which no weight has, past the end
    const int steps = (int)(((unsigned)cand + kSelectThreads * 4 - 1) / (kSelectThreads * 4));
    const int lo = wave * steps * (kWave * 4) + lane * 4;
    // 4 weights from i on; past the row's end the last 4, which to_keys puts in place
    // (no load in a branch, where each would be waited for)
    auto read = [&](int i) -> f32x4_t {
        typedef f32x4_t loose __attribute__((aligned(4)));
        if (cand >= 4) return *reinterpret_cast<const loose*>(w + min(i, cand - 4));
        return f32x4_t{w[0], w[min(1, cand - 1)], w[cand - 1], 0.f};
    };
    auto to_keys = [&](int i, f32x4_t v) {
        const int over = cand >= 4 ? i - (cand - 4) : i;   // of 4, how many lie past the end
        if (over > 0) v = f32x4_t{over == 1 ? v[1] : over == 2 ? v[2] : v[3], over == 1 ? v[2] : v[3], v[3], 0.f};
        u32x4_t k;
#pragma unroll
        for (int e = 0; e < 4; ++e) k[e] = i + e < cand ? weight_key(v[e]) : 0u;
        return k;
    };
    // f(index of the first, keys) for each of these steps of the wave's, in order
    auto each = [&](int from, int end, auto&& f) {
        if constexpr (kHeld > 0) {
            for (int s = from; s < end; ++s) {
                const int i = lo + s * (kWave * 4);
                f(i, *reinterpret_cast<const u32x4_t*>(s_keys + i));
            }
        } else {
            constexpr int kBatch = 4;
            for (int s = from; s < end; s += kBatch) {
                f32x4_t v[kBatch];
#pragma unroll
                for (int e = 0; e < kBatch; ++e) v[e] = s + e < end ? read(lo + (s + e) * (kWave * 4)) : f32x4_t{};
#pragma unroll
                for (int e = 0; e < kBatch; ++e)
                    if (s + e < end) {
                        const int i = lo + (s + e) * (kWave * 4);
                        f(i, to_keys(i, v[e]));
                    }
            }
        }
    };
    auto waves_before = [&](const int* of_waves) {   // their sum over the waves before this one
        int x = 0;
#pragma unroll
        for (int v = 0; v < kSelectWaves; v += 4) {
            const int4 q = *reinterpret_cast<const int4*>(of_waves + v);
            x += (v < wave ? q.x : 0) + (v + 1 < wave ? q.y : 0) + (v + 2 < wave ? q.z : 0) + (v + 3 < wave ? q.w : 0);
        }
        return x;
    };
    constexpr int kMost = kHeld / (kSelectThreads * 4);   // steps of a held row
    f32x4_t raw[kMost > 0 ? kMost : 1];
    if (kHeld > 0 && need > 0) {
#pragma unroll
        for (int s = 0; s < kMost; ++s)
            if (s < steps) raw[s] = read(lo + s * (kWave * 4));
    }

    // what needs no choice: the recent tokens, and what lies behind the kept ones
    const int at_thread = part * kSelectThreads + tid, threads = p.parts * kSelectThreads;
    if (h == 0 && at_thread == 0) p.new_seqlens[b] = count;
    for (int i = at_thread; i < recent; i += threads) {
        kept[need + i] = cand + i;
        if (need + i < p.weights_len) nw[need + i] = cand + i < p.max_seqlen ? w[cand + i] : 0.f;
    }
    auto fill = [&] {
        fill_row(kept, count, p.budget, (int32_t)-1, at_thread, threads);
        fill_row(nw, count, p.weights_len, 0.f, at_thread, threads);
    };
    if (need <= 0) return fill();

    for (int i = tid; i < kBins / 4; i += kSelectThreads) reinterpret_cast<int4*>(s_hist)[i] = int4{0, 0, 0, 0};
    if constexpr (kHeld > 0) {
#pragma unroll
        for (int s = 0; s < kMost; ++s) {
            const int i = lo + s * (kWave * 4);
            if (s < steps) *reinterpret_cast<u32x4_t*>(s_keys + i) = to_keys(i, raw[s]);
        }
    }
    fill();   // (after the loads: a wait for those would wait for its stores too)
    __syncthreads();

    // keys above `prefix` are kept, and the first `left` of those equal to it
    uint32_t prefix = 0;
    int left = need;
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
        const uint32_t digits = pass == 2 ? 1023u : 2047u;
        const uint32_t mask = pass == 0 ? 0u : pass == 1 ? 0xffe00000u : 0xfffffc00u;
        each(0, steps, [&](int, u32x4_t k) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (pass == 0 ? k[e] != 0u : (k[e] & mask) == prefix)   // (no weight's key has the top digit 0)
                    atomicAdd(&s_hist[(k[e] >> shift) & digits], 1);
        });
        __syncthreads();
        // thread t: bins kBins - 2 - 2t and the one above, from the top down, left
        // zero for the next pass
        int2* pair = reinterpret_cast<int2*>(s_hist) + (kBins / 2 - 1 - tid);
        const int top = pair->y, next = pair->x;
        *pair = int2{0, 0};
        const int incl = wave_fold(top + next, [](int x, int y) { return x + y; });
        if (lane == kWave - 1) s_wave[0][wave] = incl;
        __syncthreads();
        const int before = incl - top - next + waves_before(s_wave[0]);
        if (before < left && before + top >= left) {
            s_found[0] = kBins - 1 - 2 * tid;
            s_found[1] = left - before;
        } else if (before + top < left && before + top + next >= left) {
            s_found[0] = kBins - 2 - 2 * tid;
            s_found[1] = left - before - top;
        }
        __syncthreads();
        prefix |= (uint32_t)s_found[0] << shift;
        left = s_found[1];
    }

    // of this wave, and before its steps of this part
    const int first = p.parts == 1 ? 0 : (int)((unsigned)(part * steps) / (unsigned)p.parts);
    const int end = p.parts == 1 ? steps : (int)((unsigned)((part + 1) * steps) / (unsigned)p.parts);
    int n_above = 0, n_same = 0;
    int above_before = 0, same_before = 0;
    each(0, steps, [&](int i, u32x4_t k) {
        const bool here = i - lo >= first * (kWave * 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            n_above += __popcll(__ballot(k[e] > prefix));
            n_same += __popcll(__ballot(k[e] == prefix));
        }
        above_before = here ? above_before : n_above;
        same_before = here ? same_before : n_same;
    });
    if (lane == 0) {
        s_wave[1][wave] = n_above;
        s_wave[2][wave] = n_same;
    }
    __syncthreads();
    int seen = __builtin_amdgcn_readfirstlane(waves_before(s_wave[2])) + same_before;
    int at = __builtin_amdgcn_readfirstlane(waves_before(s_wave[1])) + above_before + min(seen, left);
    each(first, end, [&](int i, u32x4_t k) {
        // ties: the first of them in the lanes before, then in this lane's order
        bool keep[4];
        uint64_t same[4];
        bool any = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            keep[e] = k[e] > prefix;
            same[e] = __ballot(k[e] == prefix);
            any |= same[e] != 0;
        }
        if (any) {
            int tie = seen;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                tie += (int)lanes_below(same[e]);
                seen += __popcll(same[e]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                keep[e] = keep[e] || (k[e] == prefix && tie < left);
                tie += k[e] == prefix ? 1 : 0;
            }
        }
        int to = at;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint64_t m = __ballot(keep[e]);
            to += (int)lanes_below(m);
            at += __popcll(m);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (keep[e]) {
                kept[to] = i + e;
                nw[to] = weight_of_key(k[e]);
                ++to;
            }
    });
}

// Moves the kept tokens: one block of the new pages per item, as append_kernel,
// its rows gathered through `kept` and the block table.  Memory bounds it: 32
// sequences cut to 4000 tokens, 8 heads, e4m3 pages of 64: 530 MB in 110 us, 4.8 TB/s,
// the rate of a copy.
template <int kCode, Scaling kScaling, typename Shape>
__global__ __launch_bounds__(kThreads) void move_kernel(EvictParams p) {
    __shared__ float s_max[kWaves];
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x / kWave));
    const uint32_t item = blockIdx.x * (uint32_t)(kWaves / Shape::waves) + (uint32_t)(wave / Shape::waves);
    if (item >= p.items) return;
    const int h = (int)(item % (uint32_t)p.c.hkv);
    const uint32_t rest = item / (uint32_t)p.c.hkv;
    const int kv = (int)(rest & 1);
    const int j = (int)((rest >> 1) % (uint32_t)p.pages);
    const int b = (int)((rest >> 1) / (uint32_t)p.pages);
    const int len = min(max(p.seqlens[b], 0), p.max_tokens);
    const int rows = min(min(len, p.most) - (j << p.c.page_shift), 1 << p.c.page_shift);
    if (rows <= 0) return;
    const int page = p.new_table[(int64_t)b * p.nt_stride + j];
    if (page < 0 || page >= p.c.num_pages) return;

    constexpr int kPieces = kCode == kCodeBf16 ? 2 : 1;   // 16-byte pieces of a row that a lane holds
    const int row = lane / kLanesPerRow, chunk = lane % kLanesPerRow;
    const int first_row = (wave % Shape::waves) * Shape::sweeps * kRowsPerSweep + row;
    const int32_t* kept = p.kept + ((int64_t)b * p.c.hkv + h) * p.budget + (j << p.c.page_shift);
    const int32_t* bt = p.block_table + (int64_t)b * p.bt_stride;
    const unsigned char* src = p.c.data[kv] + h * p.c.head[kv] + chunk * 16 * kPieces;
    unsigned char* dst = p.c.data[kv] + page * p.c.page[kv] + h * p.c.head[kv] + chunk * 16 * kPieces;
    const int pmask = (1 << p.c.page_shift) - 1;

    // A wave's rows of a round: lane l looks up row l (its place and scale), and
    // the lanes of a row get them from there, so that all rows load together.
    static_assert(Shape::sweeps * kRowsPerSweep <= kWave, "a lane for each of the wave's rows");
    u32x4_t raw[Shape::sweeps][kPieces];
    float from[Shape::sweeps];
    auto load = [&](int base) {
        const int slot_l = min(base + (wave % Shape::waves) * Shape::sweeps * kRowsPerSweep + lane, rows - 1);
        const int t = kept[slot_l];
        const int64_t old = min(max(bt[t >> p.c.page_shift], 0), p.c.num_pages - 1);
        const int64_t place = old * p.c.page[kv] + (t & pmask) * p.c.slot[kv];
        float scale_l = 0.f;
        if constexpr (kScaling == kBlocks) scale_l = p.c.scales[kv][old * p.c.scale_page[kv] + h * p.c.scale_head[kv]];
#pragma unroll
        for (int s = 0; s < Shape::sweeps; ++s) {
            const int from_lane = s * kRowsPerSweep + row;
            const uint32_t lo = __shfl((int)place, from_lane, kWave), hi = __shfl((int)(place >> 32), from_lane, kWave);
            const u32x4_t* r =
                reinterpret_cast<const u32x4_t*>(src + (int64_t)(((uint64_t)hi << 32) | lo));
#pragma unroll
            for (int i = 0; i < kPieces; ++i) raw[s][i] = __builtin_nontemporal_load(r + i);   // (past the end: the last row)
            if constexpr (kScaling == kBlocks) from[s] = __shfl(scale_l, from_lane, kWave);
        }
    };
    const int last = (rows - 1) / Shape::rows * Shape::rows;
    float scale = 1.f;
    if constexpr (kScaling == kBlocks) {
        float amax = 0.f;
        for (int base = 0; base <= last; base += Shape::rows) {
            load(base);
#pragma unroll
            for (int s = 0; s < Shape::sweeps; ++s)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const f32x4_t x = codes_to_f32<kCode>(raw[s][0][i]) * from[s];
#pragma unroll
                    for (int e = 0; e < 4; ++e) amax = fmaxf(amax, capped_abs(x[e]));
                }
        }
        scale = block_scale<kCode>(block_max<Shape>(amax, s_max));
        if (lane == 0 && wave % Shape::waves == 0)
            p.c.scales[kv][page * p.c.scale_page[kv] + h * p.c.scale_head[kv]] = scale;
    }
    // (codes times from / scale, as the append's older ones; past fp32's largest number
    // only for rows whose codes are all 0)
    const float inv = 1.f / scale;
    for (int base = last; base >= 0; base -= Shape::rows) {
        if (kScaling != kBlocks || base != last) load(base);
#pragma unroll
        for (int s = 0; s < Shape::sweeps; ++s) {
            const int slot = base + first_row + s * kRowsPerSweep;
            if (slot >= rows) continue;
            u32x4_t* r = reinterpret_cast<u32x4_t*>(dst + slot * p.c.slot[kv]);
            if constexpr (kScaling == kBlocks) {
                const float ratio = fminf(from[s] * inv, kLargest);
                u32x4_t w;
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = to_codes<kCode>(codes_to_f32<kCode>(raw[s][0][i]) * ratio);
                *r = w;
            } else {
#pragma unroll
                for (int i = 0; i < kPieces; ++i) r[i] = raw[s][i];
            }
        }
    }
}

// ---------------------------------------------------------------- launches
// Calls f with the block shape for pages of page_size rows.
template <typename F>
void with_shape(int page_size, F&& f) {
    static_assert(plan::kWavePageRows == 64, "larger pages take a workgroup");
    if (page_size <= 8) f(BlockShape<1, 1>{});
    else if (page_size <= 16) f(BlockShape<2, 1>{});
    else if (page_size <= 32) f(BlockShape<4, 1>{});
    else if (page_size <= 64) f(BlockShape<8, 1>{});
    else if (page_size <= 128) f(BlockShape<4, 4>{});
    else f(BlockShape<8, 4>{});
}

template <typename Shape>
unsigned block_grid(int64_t items) {
    return (unsigned)ceil_div(items, kWaves / Shape::waves);
}

template <int kCode, Scaling kScaling>
void launch_append(const AppendParams& p, int page_size, hipStream_t s) {
    with_shape(page_size, [&](auto shape) {
        using Shape = decltype(shape);
        hipLaunchKernelGGL((append_kernel<kCode, kScaling, Shape>), dim3(block_grid<Shape>(p.items)), dim3(kThreads), 0,
                           s, p);
    });
}

template <int kCode, Scaling kScaling, bool kTurns>
void launch_weights_pages(const WeightsParams& p, int page_size, hipStream_t s) {
    const dim3 grid((unsigned)ceil_div(p.items, kWaves)), block(kThreads);
    if (page_size >= 32) hipLaunchKernelGGL((weights_kernel<kCode, kScaling, 32, kTurns>), grid, block, 0, s, p);
    else if (page_size == 16) hipLaunchKernelGGL((weights_kernel<kCode, kScaling, 16, kTurns>), grid, block, 0, s, p);
    else if (page_size == 8) hipLaunchKernelGGL((weights_kernel<kCode, kScaling, 8, kTurns>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((weights_kernel<kCode, kScaling, 0, kTurns>), grid, block, 0, s, p);
}

template <int kCode, Scaling kScaling>
void launch_weights(const WeightsParams& p, int page_size, hipStream_t s) {
    if ((int64_t)p.waves * plan::kWeightsTokens < p.max_seqlen) launch_weights_pages<kCode, kScaling, true>(p, page_size, s);
    else launch_weights_pages<kCode, kScaling, false>(p, page_size, s);
}

template <int kCode, Scaling kScaling>
void launch_move(const EvictParams& p, int page_size, hipStream_t s) {
    with_shape(page_size, [&](auto shape) {
        using Shape = decltype(shape);
        hipLaunchKernelGGL((move_kernel<kCode, kScaling, Shape>), dim3(block_grid<Shape>(p.items)), dim3(kThreads), 0, s,
                           p);
    });
}

}  // namespace
}  // namespace fgqa

using namespace fgqa;

extern "C" int fgqa_kv_append(const fgqa_kv_append_args* a, void* stream) {
    const int st = plan::validate_kv_append(a);
    if (st != FGQA_OK) return st;
    if (a->batch == 0 || a->max_new == 0 || a->max_pages == 0) return FGQA_OK;
    AppendParams p;
    p.c = cache_params(a->cache);
    const void* x[2] = {a->k_new, a->v_new};
    const int64_t* xs[2] = {a->k_new_stride, a->v_new_stride};
    for (int i = 0; i < 2; ++i) {
        p.x[i] = static_cast<const unsigned char*>(x[i]);
        p.x_b[i] = xs[i][0] * 2;
        p.x_t[i] = xs[i][1] * 2;
        p.x_h[i] = xs[i][2] * 2;
    }
    p.block_table = a->block_table;
    p.bt_stride = a->block_table_stride;
    p.seqlens = a->seqlens;
    p.new_lens = a->new_lens;
    p.max_new = a->max_new;
    p.max_tokens = a->max_pages * a->cache.page_size;
    p.pages = (int)plan::append_pages(a->max_new, a->cache.page_size);
    p.items = (uint32_t)((int64_t)a->batch * p.pages * 2 * p.c.hkv);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const int page = a->cache.page_size;
    const bool blocks = a->cache.k_scales != nullptr;
    if (a->cache.kv_dtype == FGQA_KV_BF16) launch_append<kCodeBf16, kNone>(p, page, s);
    else if (a->cache.kv_dtype == FGQA_KV_INT8) launch_append<kCodeInt8, kBlocks>(p, page, s);
    else if (blocks) launch_append<kCodeFp8, kBlocks>(p, page, s);
    else launch_append<kCodeFp8, kWhole>(p, page, s);
    return hipGetLastError() == hipSuccess ? FGQA_OK : FGQA_ERR_HIP;
}

extern "C" int fgqa_kv_weights(const fgqa_kv_weights_args* a, void* stream) {
    const int st = plan::validate_kv_weights(a);
    if (st != FGQA_OK) return st;
    if (a->batch == 0 || a->max_seqlen == 0) return FGQA_OK;
    WeightsParams p;
    p.c = cache_params(a->cache);
    p.q = static_cast<const __bf16*>(a->q);
    p.lse = a->lse;
    p.weights = a->weights;
    p.q_b = a->q_stride[0];
    p.q_h = a->q_stride[1];
    p.w_b = a->weights_stride[0];
    p.w_h = a->weights_stride[1];
    p.block_table = a->block_table;
    p.bt_stride = a->block_table_stride;
    p.seqlens = a->seqlens;
    p.max_seqlen = a->max_seqlen;
    p.group = a->num_q_heads / p.c.hkv;
    p.waves = plan::weights_waves(a->batch, p.c.hkv, a->max_seqlen);
    p.items = (uint32_t)((int64_t)a->batch * p.waves * p.c.hkv);
    const bool blocks = a->cache.k_scales != nullptr;
    const bool whole = a->cache.kv_dtype == FGQA_KV_FP8_E4M3 && !blocks;
    p.scale = a->scale * (whole ? a->cache.k_scale : 1.f);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    // Page segments of at least 8 rows, where a page's bytes stay below 2^31.
    const int page = (int64_t)a->cache.page_size * p.c.slot[0] < ((int64_t)1 << 31) ? a->cache.page_size : 1;
    if (a->cache.kv_dtype == FGQA_KV_BF16) launch_weights<kCodeBf16, kNone>(p, page, s);
    else if (a->cache.kv_dtype == FGQA_KV_INT8) launch_weights<kCodeInt8, kBlocks>(p, page, s);
    else if (blocks) launch_weights<kCodeFp8, kBlocks>(p, page, s);
    else launch_weights<kCodeFp8, kWhole>(p, page, s);
    return hipGetLastError() == hipSuccess ? FGQA_OK : FGQA_ERR_HIP;
}

extern "C" int fgqa_kv_evict(const fgqa_kv_evict_args* a, void* stream) {
    const int st = plan::validate_kv_evict(a);
    if (st != FGQA_OK) return st;
    if (a->batch == 0) return FGQA_OK;
    EvictParams p;
    p.c = cache_params(a->cache);
    p.weights = a->weights;
    p.new_weights = a->new_weights;
    p.w_b = a->weights_stride[0];
    p.w_h = a->weights_stride[1];
    p.nw_b = a->new_weights_stride[0];
    p.nw_h = a->new_weights_stride[1];
    p.block_table = a->block_table;
    p.new_table = a->new_block_table;
    p.bt_stride = a->block_table_stride;
    p.nt_stride = a->new_block_table_stride;
    p.seqlens = a->seqlens;
    p.new_seqlens = a->new_seqlens;
    p.kept = a->kept;
    p.max_seqlen = a->max_seqlen;
    p.weights_len = a->weights_len;
    p.budget = a->budget;
    p.recent = a->recent;
    p.max_tokens = plan::evict_tokens(*a);
    p.most = plan::evict_most(*a);
    p.pages = (int)ceil_div(std::min(p.most, p.max_tokens), a->cache.page_size);
    p.items = (uint32_t)((int64_t)a->batch * p.pages * 2 * p.c.hkv);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const int64_t rows = (int64_t)a->batch * p.c.hkv;
    const int cus = device_cu_count();
    if (cus <= 0) return FGQA_ERR_HIP;
    p.parts = (int)std::max<int64_t>(1, std::min(cus / rows, ceil_div(a->max_seqlen, 4 * kSelectThreads)));
    const dim3 grid((unsigned)(rows * p.parts)), block(kSelectThreads);
    if (a->max_seqlen <= 8 * kSelectThreads) hipLaunchKernelGGL(select_kernel<8 * kSelectThreads>, grid, block, 0, s, p);
    else if (a->max_seqlen <= 32 * kSelectThreads) hipLaunchKernelGGL(select_kernel<32 * kSelectThreads>, grid, block, 0, s, p);
    else hipLaunchKernelGGL(select_kernel<0>, grid, block, 0, s, p);
    if (p.items > 0) {
        const int page = a->cache.page_size;
        if (a->cache.kv_dtype == FGQA_KV_BF16) launch_move<kCodeBf16, kNone>(p, page, s);
        else if (a->cache.kv_dtype == FGQA_KV_INT8) launch_move<kCodeInt8, kBlocks>(p, page, s);
        else if (a->cache.k_scales != nullptr) launch_move<kCodeFp8, kBlocks>(p, page, s);
        else launch_move<kCodeFp8, kWhole>(p, page, s);
    }
    return hipGetLastError() == hipSuccess ? FGQA_OK : FGQA_ERR_HIP;
}
