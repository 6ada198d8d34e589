// One decode item, tokens of one sequence and KV head run by a few waves, over
// contiguous and paged caches (the math and layout are decode_flash_gqa.hip's, whose
// kernels and decode_shared.hip's share the work out and merge the items).
#pragma once

#include <math.h>
#include <stdint.h>

#include "fgqa_device.h"
#include "../host/kv_plan.h"

namespace fgqa {

struct DecodeParams {
    const __bf16* q;
    const __bf16* k;
    const __bf16* v;
    __bf16* o;
    float* lse;
    const int32_t* seqlens;
    float* part_o;   // [B, Hkv, nsplit, G, 128]
    float* part_ml;  // [B, Hkv, nsplit, G, 2]  (max in log2 units, sum)
    int64_t q_sb, q_sh;
    int64_t k_sb, k_ss, k_sh;
    int64_t v_sb, v_ss, v_sh;
    int64_t o_sb, o_sh;
    const int32_t* work;   // ragged work list: [0] = entries, then (b << 16 | split) per entry; or null
    int64_t* prefix;       // teams: [B + 1] 128-token blocks before each sequence, then their total
    int teams;             // > 0: the ragged batch's blocks are shared out evenly over this many teams
    int batch, max_seqlen, hq, hkv, group;
    int nsplit, chunk;
    float scale_log2;
    // paged KV: k/v are the page caches, strides {page, slot, head} in elements
    // of the cache type; page of token t = block_table[b * bt_stride + (t >> page_shift)]
    const int32_t* block_table;
    int64_t bt_stride;
    int page_shift;
    int num_pages;      // page indices are clamped to [0, num_pages)
    float v_scale;      // multiplies O (the fp8 V scale; 1 otherwise)
    // block scales of an 8-bit cache, strides {page, head}
    const float* k_scales;
    const float* v_scales;
    int64_t ks_sp, ks_sh, vs_sp, vs_sh;
};

// Cache layouts the decode items read (the last two: codes with block scales).
enum DecKv { kKvContig = 0, kKvPagedBf16 = 1, kKvPagedFp8 = 2, kKvBlocksFp8 = 3, kKvBlocksInt8 = 4 };

// 16 OCP fp8 e4m3 values -> 16 bf16 (exact: every e4m3 value is a bf16 value).
__device__ __forceinline__ void fp8x16_to_bf16(u32x4_t in, u32x4_t* lo, u32x4_t* hi) {
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        w[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(in[i], 1.0f, false));
        w[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(in[i], 1.0f, true));
    }
    *lo = u32x4_t{w[0], w[1], w[2], w[3]};
    *hi = u32x4_t{w[4], w[5], w[6], w[7]};
}

constexpr int kDecThreads = 256;
constexpr int kDecWaves = kDecThreads / kWave;
constexpr int kDecStep = 32;        // tokens per wave step (two 16-token MFMA blocks)
constexpr int kDecRowStride = 136;  // LDS row stride (elements) of a staged K or V row: 272 B
                                    // spreads 16 rows over all 64 banks for b128 reads
constexpr int kDecTileElems = kDecStep * kDecRowStride;
constexpr int kDecSmemBytes = kDecWaves * 2 * kDecTileElems * 2;  // per wave: K tile + V tile
static_assert(kDecWaves * 16 * kHeadDim * 4 + kDecWaves * 16 * 2 * 4 <= kDecSmemBytes,
              "wave merge buffers must fit in the staging area");

__device__ __forceinline__ int clamp_len(const DecodeParams& p, int b) {
    int len = p.seqlens ? p.seqlens[b] : p.max_seqlen;
    return min(max(len, 0), p.max_seqlen);
}

// One item of pass 1: tokens [t_begin, t_end) (not empty) of one sequence and
// kv head, run by 4 waves (tid: the thread's index among them, smem: their
// kDecSmemBytes of LDS).  whole: the item is the sequence's only one and
// writes O and the LSE; otherwise its fp32 partial goes to rows slot0 + head
// of the workspace.  kSeg (paged
// caches, 0 or a power of two from one load instruction's rows up to 32): the
// rows of a 32-token step fall into page segments of kSeg rows
// (kSeg = min(page, 32)), each read through one buffer resource; 0 is the
// general form, with a page lookup and a 64-bit address per row.
// The only workgroup barriers are the two of the wave merge, so two items of
// the same tokens can share a workgroup.
// kInf: a step's scores may all be -inf (infinite bf16 keys).
template <int kKv, int kSeg = 0, bool kInf = false>
__device__ __forceinline__ void dec_item(const DecodeParams& p, unsigned char* smem, int t_begin, int t_end, int kvh,
                                         int b, int tid, bool whole, int64_t slot0) {
    const int lane = tid & (kWave - 1);
    constexpr bool kUni = kSeg > 0;
    const int wave = kUni ? __builtin_amdgcn_readfirstlane(tid / kWave) : tid / kWave;
    const int l16 = lane & 15;
    const int g4 = lane >> 4;

    __bf16* kl = reinterpret_cast<__bf16*>(smem) + wave * 2 * kDecTileElems;
    __bf16* vl = kl + kDecTileElems;

    // Q^T as the B operand: lane holds Q[h = l16][32*kk + 8*g4 .. +7]; heads >= G are zero.
    bf16x8_t qop[4];
    {
        const bool hv = l16 < p.group;
        const __bf16* qrow = p.q + b * p.q_sb + (int64_t)(kvh * p.group + (hv ? l16 : 0)) * p.q_sh;
        const u32x4_t zero = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
            u32x4_t t = *reinterpret_cast<const u32x4_t*>(qrow + kk * 32 + g4 * 8);
            qop[kk] = as_bf16x8(hv ? t : zero);
        }
    }

    float m_run = -INFINITY;
    float l_run = 0.f;  // this lane's share of the rowsum of head l16
    f32x4_t oacc[8];
#pragma unroll
    for (int db = 0; db < 8; ++db) oacc[db] = f32x4_t{0.f, 0.f, 0.f, 0.f};

    const int n_steps = (t_end - t_begin + kDecStep - 1) / kDecStep;
    // One step = 32 token rows of K and of V.  bf16: load r (0..7) of a lane
    // covers row 4*r + g4, 16-byte chunk l16, so each quarter-wave reads one
    // whole 256-byte row (the coalesced pattern).  fp8: rows are 128 bytes;
    // load r (0..3) covers row 8*r + lane/8, chunk lane%8.
    constexpr int kRows = (kKv == kKvPagedFp8) ? 4 : 8;
    const int fp8_row = lane >> 3;
    const int fp8_chunk = lane & 7;
    auto row_of = [&](int r) { return (kKv == kKvPagedFp8) ? 8 * r + fp8_row : 4 * r + g4; };
    u32x4_t kreg[kRows];
    u32x4_t vreg[kRows];

    // Contiguous cache: buffer resources end at the split's last valid token,
    // so later tokens read as zero.
    const uint32_t kss = (uint32_t)(p.k_ss * 2);
    const uint32_t vss = (uint32_t)(p.v_ss * 2);
    __amdgpu_buffer_rsrc_t krs, vrs;
    if constexpr (kKv == kKvContig) {
        krs = make_rsrc(p.k + b * p.k_sb + kvh * p.k_sh, (uint32_t)(t_end - 1) * kss + kHeadDim * 2);
        vrs = make_rsrc(p.v + b * p.v_sb + kvh * p.v_sh, (uint32_t)(t_end - 1) * vss + kHeadDim * 2);
    }
    // Paged cache: each row's page comes from the block table one step ahead
    // of its load.  Tokens past the split's end reuse its last token (their
    // scores are masked; the row only has to be finite).
    constexpr int kElemBytes = (kKv == kKvPagedFp8) ? 1 : 2;
    const unsigned char* kbase = reinterpret_cast<const unsigned char*>(p.k) + kvh * p.k_sh * kElemBytes;
    const unsigned char* vbase = reinterpret_cast<const unsigned char*>(p.v) + kvh * p.v_sh * kElemBytes;
    const int32_t* bt = p.block_table + (int64_t)b * p.bt_stride;
    const int pmask = (1 << p.page_shift) - 1;
    int pg[kRows];
    // kSeg > 0: segment g of a step (rows kSeg*g .. +kSeg-1, one page) is
    // read through one buffer resource per cache, starting at the segment's
    // first row and ending at the split's last token (rows past it read as
    // zeros).  The wave's segment pages come 64 at a time from one vector
    // load of the block table (lane l: the wave's segment pt_first + l, its
    // segments numbered n * kSegs + g for its n-th step) and are taken out
    // with v_readlane (a scalar load would share its wait counter with the
    // LDS traffic).  Load instruction i
    // of a segment reads its rows kR*i .. kR*i + kR - 1 at a per-lane offset
    // that is the same in every segment and step.  The host picks kSeg only
    // when a page's bytes stay below 2^31.
    constexpr int kR = (kKv == kKvPagedFp8) ? 8 : 4;           // rows per load instruction
    constexpr int kSegs = kUni ? kDecStep / kSeg : 1;          // segments per step
    constexpr int kPerSeg = kRows / kSegs;                     // load instructions per segment
    static_assert(!kUni || (kSeg >= kR && kSeg <= kDecStep && kPerSeg * kSegs == kRows), "page segment");
    constexpr uint32_t kRowBytes = kHeadDim * kElemBytes;
    const uint32_t kss_e = (uint32_t)(p.k_ss * kElemBytes);
    const uint32_t vss_e = (uint32_t)(p.v_ss * kElemBytes);
    const int64_t ksb_e = p.k_sb * kElemBytes;
    const int64_t vsb_e = p.v_sb * kElemBytes;
    const int t_end_u = kUni ? __builtin_amdgcn_readfirstlane(t_end) : t_end;
    [[maybe_unused]] uint32_t kvoff[kPerSeg], vvoff[kPerSeg];
    if constexpr (kUni) {
        const int lr = (kKv == kKvPagedFp8) ? fp8_row : g4;             // the lane's row in an instruction
        const int cb = (kKv == kKvPagedFp8) ? fp8_chunk * 16 : l16 * 16;
#pragma unroll
        for (int i = 0; i < kPerSeg; ++i) {
            kvoff[i] = (uint32_t)(kR * i + lr) * kss_e + cb;
            vvoff[i] = (uint32_t)(kR * i + lr) * vss_e + cb;
        }
    }
    [[maybe_unused]] int pt_lane = 0;       // block table entry of segment pt_first + lane
    [[maybe_unused]] int pt_first = -kWave;
    [[maybe_unused]] auto pt_load = [&](int first) {
        const int n = first + lane;
        const int tok = min(t_begin + (wave + kDecWaves * (n / kSegs)) * kDecStep + kSeg * (n % kSegs), t_end_u - 1);
        pt_lane = bt[tok >> p.page_shift];
        pt_first = first;
    };
    if constexpr (kUni) pt_load(0);
    auto fetch_pages = [&](int s) {
        if constexpr (kUni) {
            (void)s;   // the pages are taken out in load_step
        } else if constexpr (kKv != kKvContig) {
            // Raw entries: they are clamped where load_step uses them.  A
            // clamp here would make the wave wait for the table loads at once,
            // and vector loads complete in order, so that wait would also take
            // the K/V loads issued just before, leaving none in flight while
            // the step computes.
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
                const int tok = min(t_begin + s * kDecStep + row_of(r), t_end - 1);
                pg[r] = bt[tok >> p.page_shift];
            }
        }
    };
    auto load_step = [&](int s) {
        const int t0 = t_begin + s * kDecStep;
        if constexpr (kUni) {
            const int n0 = ((s - wave) / kDecWaves) * kSegs;   // the wave's first segment of step s
            if (n0 + kSegs > pt_first + kWave) pt_load(n0);
#pragma unroll
            for (int g = 0; g < kSegs; ++g) {
                pg[g] = min(max(__builtin_amdgcn_readlane(pt_lane, n0 - pt_first + g), 0), p.num_pages - 1);
            }
#pragma unroll
            for (int g = 0; g < kSegs; ++g) {
                const int tok = t0 + kSeg * g;
                const int nv = min(kSeg, t_end_u - tok);   // rows before the split's end
                const uint32_t slot = (uint32_t)(tok & pmask);
                const __amdgpu_buffer_rsrc_t kr = make_rsrc(kbase + pg[g] * ksb_e + slot * kss_e,
                                                            nv > 0 ? (uint32_t)(nv - 1) * kss_e + kRowBytes : 0u);
                const __amdgpu_buffer_rsrc_t vr = make_rsrc(vbase + pg[g] * vsb_e + slot * vss_e,
                                                            nv > 0 ? (uint32_t)(nv - 1) * vss_e + kRowBytes : 0u);
#pragma unroll
                for (int i = 0; i < kPerSeg; ++i) {
                    kreg[g * kPerSeg + i] = buf_load16_nt(kr, kvoff[i]);
                    vreg[g * kPerSeg + i] = buf_load16_nt(vr, vvoff[i]);
                }
            }
        } else if constexpr (kKv == kKvContig) {
#pragma unroll
            for (int r = 0; r < 8; ++r) kreg[r] = buf_load16_nt(krs, (uint32_t)(t0 + r * 4 + g4) * kss + l16 * 16);
#pragma unroll
            for (int r = 0; r < 8; ++r) vreg[r] = buf_load16_nt(vrs, (uint32_t)(t0 + r * 4 + g4) * vss + l16 * 16);
        } else {
            const int cb = (kKv == kKvPagedFp8) ? fp8_chunk * 16 : l16 * 16;
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
                const int slot = min(t0 + row_of(r), t_end - 1) & pmask;
                const int page = min(max(pg[r], 0), p.num_pages - 1);
                const int64_t ko = ((int64_t)page * p.k_sb + (int64_t)slot * p.k_ss) * kElemBytes + cb;
                const int64_t vo = ((int64_t)page * p.v_sb + (int64_t)slot * p.v_ss) * kElemBytes + cb;
                kreg[r] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(kbase + ko));
                vreg[r] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(vbase + vo));
            }
        }
    };

    int st = wave;
    if (st < n_steps) {
        fetch_pages(st);
        load_step(st);
    }
    if (st + kDecWaves < n_steps) fetch_pages(st + kDecWaves);
    for (; st < n_steps; st += kDecWaves) {
        // Stage this step's rows (fp8 widened to bf16), then put the next
        // step's loads and the page lookups of the step after in flight.
        if constexpr (kKv == kKvPagedFp8) {
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
                u32x4_t lo, hi;
                __bf16* kd = kl + row_of(r) * kDecRowStride + fp8_chunk * 16;
                __bf16* vd = vl + row_of(r) * kDecRowStride + fp8_chunk * 16;
                fp8x16_to_bf16(kreg[r], &lo, &hi);
                *reinterpret_cast<u32x4_t*>(kd) = lo;
                *reinterpret_cast<u32x4_t*>(kd + 8) = hi;
                fp8x16_to_bf16(vreg[r], &lo, &hi);
                *reinterpret_cast<u32x4_t*>(vd) = lo;
                *reinterpret_cast<u32x4_t*>(vd + 8) = hi;
            }
        } else {
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                *reinterpret_cast<u32x4_t*>(kl + (r * 4 + g4) * kDecRowStride + l16 * 8) = kreg[r];
                *reinterpret_cast<u32x4_t*>(vl + (r * 4 + g4) * kDecRowStride + l16 * 8) = vreg[r];
            }
        }
        if (st + kDecWaves < n_steps) load_step(st + kDecWaves);
        if (st + 2 * kDecWaves < n_steps) fetch_pages(st + 2 * kDecWaves);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");

        // S^T = K Q^T; K as the A operand: lane holds K[16*tb + l16][32*kk + 8*g4 .. +7].
        const int t0 = t_begin + st * kDecStep;
        f32x4_t s[2];
#pragma unroll
        for (int tb = 0; tb < 2; ++tb) {
            s[tb] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
                const bf16x8_t ka =
                    *reinterpret_cast<const bf16x8_t*>(kl + (tb * 16 + l16) * kDecRowStride + kk * 32 + g4 * 8);
                s[tb] = mfma16(ka, qop[kk], s[tb]);
            }
        }

        // Online softmax for head l16 over tokens t0 + 16*tb + 4*g4 + i.
        float x[8];
        float tmax = -INFINITY;
#pragma unroll
        for (int tb = 0; tb < 2; ++tb)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int tok = t0 + tb * 16 + g4 * 4 + i;
                const float val = (tok < t_end) ? s[tb][i] * p.scale_log2 : -INFINITY;
                x[tb * 4 + i] = val;
                tmax = fmaxf(tmax, val);
            }
        tmax = xor_max(xor_max(tmax, 16), 32);
        const float m_new = fmaxf(m_run, tmax);  // finite (but for kInf): every step holds a valid token
        const float m_sub = kInf && m_new == -INFINITY ? 0.f : m_new;
        const float alpha = fast_exp2(m_run - m_sub);
        float psum = 0.f;
        bf16x8_t pop;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float pv = fast_exp2(x[j] - m_sub);
            psum += pv;
            pop[j] = (__bf16)pv;
        }
        l_run = l_run * alpha + psum;
        m_run = m_new;
#pragma unroll
        for (int db = 0; db < 8; ++db) oacc[db] *= alpha;

        // V^T as the A operand: lane holds V[token(slot)][16*db + l16] for the
        // 8 slots of group g4: tokens 4*g4 + {0..3} and 16 + 4*g4 + {0..3},
        // the same tokens whose P this lane already holds.  Two transposed
        // reads (ds_read_b64_tr_b16) per column block: source lane l16 of the
        // group points at row 4*g4 + l16/4 (+16), columns 16*db + 4*(l16%4) .. +3.
        const __bf16* vsrc = vl + (4 * g4 + (l16 >> 2)) * kDecRowStride + 4 * (l16 & 3);
#pragma unroll
        for (int db = 0; db < 8; ++db) {
            const bf16x4_t lo = lds_read_tr16(vsrc + db * 16);
            const bf16x4_t hi = lds_read_tr16(vsrc + 16 * kDecRowStride + db * 16);
            oacc[db] = mfma16(__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7), pop, oacc[db]);
        }

        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }

    l_run = xor_sum(xor_sum(l_run, 16), 32);

    // Merge the 4 waves in LDS (reusing the staging area).
    __syncthreads();
    float* ow = reinterpret_cast<float*>(smem);        // [wave][16][128]
    float* mlw = ow + kDecWaves * 16 * kHeadDim;       // [wave][16][2]
#pragma unroll
    for (int db = 0; db < 8; ++db)
#pragma unroll
        for (int i = 0; i < 4; ++i) ow[(wave * 16 + l16) * kHeadDim + db * 16 + g4 * 4 + i] = oacc[db][i];
    if (g4 == 0) {
        mlw[(wave * 16 + l16) * 2 + 0] = m_run;
        mlw[(wave * 16 + l16) * 2 + 1] = l_run;
    }
    __syncthreads();

    const int h = tid >> 4;
    const int d0 = (tid & 15) * 8;
    if (h >= p.group) return;
    float mw[kDecWaves];
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < kDecWaves; ++w) {
        mw[w] = mlw[(w * 16 + h) * 2];
        M = fmaxf(M, mw[w]);
    }
    float L = 0.f;
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kDecWaves; ++w) {
        const float c = (mw[w] == -INFINITY) ? 0.f : fast_exp2(mw[w] - M);
        L += c * mlw[(w * 16 + h) * 2 + 1];
        const float* src = ow + (w * 16 + h) * kHeadDim + d0;
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] += c * src[j];
    }
    const int qh = kvh * p.group + h;
    if (whole) {
        const float inv = p.v_scale / L;
        bf16x8_t out;
#pragma unroll
        for (int j = 0; j < 8; ++j) out[j] = (__bf16)(acc[j] * inv);
        *reinterpret_cast<bf16x8_t*>(p.o + b * p.o_sb + qh * p.o_sh + d0) = out;
        if (p.lse != nullptr && (tid & 15) == 0) p.lse[(int64_t)b * p.hq + qh] = M * kLn2 + logf(L);
    } else {
        const int64_t slot = slot0 + h;
        float* po = p.part_o + slot * kHeadDim + d0;
        const float vs = p.v_scale;
        *reinterpret_cast<f32x4_t*>(po) = f32x4_t{acc[0] * vs, acc[1] * vs, acc[2] * vs, acc[3] * vs};
        *reinterpret_cast<f32x4_t*>(po + 4) = f32x4_t{acc[4] * vs, acc[5] * vs, acc[6] * vs, acc[7] * vs};
        if ((tid & 15) == 0) {
            p.part_ml[slot * 2 + 0] = M;
            p.part_ml[slot * 2 + 1] = L;
        }
    }
}

}  // namespace fgqa

#include "decode_block8.h"

namespace fgqa {

// The item of each layout, and its LDS, for kNw waves.
template <int kKv, int kNw>
constexpr int kDecItemSmem = kKv >= kKvBlocksFp8 ? dec8_smem_bytes(kNw) : kDecSmemBytes;

template <int kKv, int kSeg, int kNw, bool kInf = false>
__device__ __forceinline__ void dec_item_of(const DecodeParams& p, unsigned char* smem, int t_begin, int t_end, int kvh,
                                            int b, int tid, bool whole, int64_t slot0) {
    if constexpr (kKv >= kKvBlocksFp8)
        dec_item8<kKv == kKvBlocksFp8 ? kCodeFp8 : kCodeInt8, kSeg, kNw>(p, smem, t_begin, t_end, kvh, b, tid, whole,
                                                                         slot0);
    else
        dec_item<kKv, kSeg, kInf>(p, smem, t_begin, t_end, kvh, b, tid, whole, slot0);
}

}  // namespace fgqa
