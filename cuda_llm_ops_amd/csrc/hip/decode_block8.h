// One decode item over a paged cache of 8-bit codes with block scales (included
// by decode_flash_gqa.hip, whose kernels share the work out and merge the items).
//
// The mathematics is that of dec_item, on codes: with K = sK c_K and V = sV c_V
// (one scale per page and KV head),
//     s_t = scale sK(t) (q . c_K[t]),   o = sum_t softmax(s)_t sV(t) c_V[t].
// Codes are widened exactly (to bf16 for K, fp16 for V).  sK multiplies the
// scores in fp32.  sV is folded into P in fp32, and P sV, at 2^14 times its ratio to
// the head's largest so far (vref), is held in two fp16 numbers, its rounding and
// what that leaves: 22 bits, and down to 2^-39 of the largest.  (Relative to the
// largest sV instead, a block of a far larger scale took the bits of the tokens that
// get the attention, whatever it got itself.  One fp16 number alone moves 7.5 % of the
// bf16 outputs to a neighbour of the 32-bit form's, two 0.07 %.)
//
// K and V rows are loaded whole, 8 lanes of 16 bytes a row, and staged in LDS
// as codes, half the bytes of bf16 rows.  (Reading K's MFMA operand straight
// from memory touches each 128-byte row twice, 64 bytes at a time: 381 us instead
// of 357 for the loads alone of 1M tokens of 8 heads.)  V comes back transposed
// (ds_read_b64_tr_b8: 8 tokens of one column per lane).  The K operand's
// contraction index is reordered so that a lane's 16-byte pieces 16 g4 and
// 64 + 16 g4 of a row are two operands each (Q is loaded in the same order).
//
// Four heads a workgroup of 8 waves where they divide by 4: the rows of a token
// lie side by side over its heads, and what limits the stream is how much of
// them is read together (loads alone, 64-token pages in random order: 5.95,
// 6.59 and 7.00 TB/s with 1, 2 and 4 heads a workgroup; one step or three in
// flight per wave change nothing).  The read stream bounds it: 64 sequences of up to
// 32768 tokens, 64 / 8 heads, e4m3 pages of 64: 2155 MB in 328 us, 6.6 TB/s, and 4 to 7
// for the combine.
#pragma once

#include "fgqa_device.h"
#include "kv_codes.h"

namespace fgqa {

constexpr int kDec8RowStride = 144;   // LDS bytes of a row: 16 rows spread over all 64 banks
constexpr int kDec8TileBytes = kDecStep * kDec8RowStride;
constexpr int kDec8WaveBytes = 2 * kDec8TileBytes + kDecStep * 2 * 4;   // K, V, their scales
constexpr int kDec8MergeStride = kHeadDim + 4;   // floats of a merged row: 16 rows spread over all 64 banks
constexpr int dec8_smem_bytes(int waves) {
    const int merge = waves * 16 * kDec8MergeStride * 4 + waves * 16 * 2 * 4;
    return waves * kDec8WaveBytes > merge ? waves * kDec8WaveBytes : merge;
}
constexpr float kDec8PScale = 16384.f;   // P's scale in fp16

__device__ __forceinline__ f32x4_t mfma16_f16(f16x8_t a, f16x8_t b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// Transposed LDS read of bytes: within 16 lanes, lane i gets bytes 0 .. 7 of
// column i of the 8 x 16 bytes whose row j lies at the addresses of lanes 2j
// (columns 0 .. 7) and 2j + 1 (8 .. 15).
__device__ __forceinline__ u32x2_t lds_read_tr8(const unsigned char* p) {
    typedef int s32x2_t __attribute__((ext_vector_type(2)));
    const s32x2_t v = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
        (__attribute__((address_space(3))) s32x2_t*)(__attribute__((address_space(3))) void*)(p));
    return __builtin_bit_cast(u32x2_t, v);
}

// The loads of one 32-token step, row 8 r + lane / 8 and piece lane % 8 each, and
// the scales of its tokens' blocks: of the step's kSegs segments, or (kSeg 0) of
// this lane's rows.
struct Step8 {
    u32x4_t k[4], v[4];
    float ks[4], vs[4];
};

// As dec_item: tokens [t_begin, t_end) (not empty, t_begin a multiple of 128)
// of one sequence and kv head, by kNw waves.  Two steps' loads are in flight per
// wave.
// kSeg (32, 16 or 8, for pages of at least that many rows whose bytes stay below
// 2^31): a step is 1, 2 or 4 page segments, read through buffer resources that
// end at the item's last token (rows past it are zeros), their pages and scales
// taken 64 segments at a time from one vector load each.  0: any pages, a lookup
// and a 64-bit address per row.
template <int kCode, int kSeg, int kNw>
__device__ __forceinline__ void dec_item8(const DecodeParams& p, unsigned char* smem, int t_begin, int t_end, int kvh,
                                          int b, int tid, bool whole, int64_t slot0) {
    const int lane = tid & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int l16 = lane & 15;
    const int g4 = lane >> 4;
    unsigned char* kl = smem + wave * kDec8WaveBytes;
    unsigned char* vl = kl + kDec8TileBytes;
    float* sl = reinterpret_cast<float*>(vl + kDec8TileBytes);   // kSeg 0: [32] K scales, [32] V scales

    // Q^T as the B operand: lane holds Q[h = l16] at the elements that its
    // pieces of K hold; heads >= G are zero.
    bf16x8_t qop[4];
    {
        const bool hv = l16 < p.group;
        const __bf16* qrow = p.q + b * p.q_sb + (int64_t)(kvh * p.group + (hv ? l16 : 0)) * p.q_sh;
        const u32x4_t zero = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
            const u32x4_t t = *reinterpret_cast<const u32x4_t*>(qrow + 64 * (kk / 2) + 16 * g4 + 8 * (kk % 2));
            qop[kk] = as_bf16x8(hv ? t : zero);
        }
    }

    float m_run = -INFINITY;
    float l_run = 0.f;   // this lane's share of the rowsum of head l16
    // head l16's largest |P sV| so far, P relative to m_run, and 2^-112 at least: 2^14 /
    // vref is a number (blocks of zeros have the scale 2^-126)
    constexpr uint32_t kLeastRef = 0x07800000u;
    float vref = __uint_as_float(kLeastRef);
    f32x4_t oacc[8];
#pragma unroll
    for (int db = 0; db < 8; ++db) oacc[db] = f32x4_t{0.f, 0.f, 0.f, 0.f};

    const unsigned char* kbase = reinterpret_cast<const unsigned char*>(p.k) + kvh * p.k_sh;
    const unsigned char* vbase = reinterpret_cast<const unsigned char*>(p.v) + kvh * p.v_sh;
    const float* kscales = p.k_scales + kvh * p.ks_sh;
    const float* vscales = p.v_scales + kvh * p.vs_sh;
    const int32_t* bt = p.block_table + (int64_t)b * p.bt_stride;
    const int pmask = (1 << p.page_shift) - 1;
    const int row8 = lane >> 3, piece = lane & 7;
    const int t_end_u = __builtin_amdgcn_readfirstlane(t_end);
    const int n_steps = (t_end - t_begin + kDecStep - 1) / kDecStep;

    // kSeg > 0
    constexpr int kSegs = kSeg > 0 ? kDecStep / kSeg : 1;
    const uint32_t kss = (uint32_t)p.k_ss, vss = (uint32_t)p.v_ss;
    [[maybe_unused]] const uint32_t koff = (uint32_t)row8 * kss + piece * 16;
    [[maybe_unused]] const uint32_t voff = (uint32_t)row8 * vss + piece * 16;
    [[maybe_unused]] int pt_page = 0, pt_first = -kWave;   // lane l: the wave's segment pt_first + l
    [[maybe_unused]] float pt_ks = 0.f, pt_vs = 0.f;
    [[maybe_unused]] auto pt_load = [&](int first) {
        const int n = first + lane;
        const int tok = min(t_begin + (wave + kNw * (n / kSegs)) * kDecStep + kSeg * (n % kSegs), t_end_u - 1);
        pt_page = min(max(bt[tok >> p.page_shift], 0), p.num_pages - 1);
        pt_ks = kscales[(int64_t)pt_page * p.ks_sp];
        pt_vs = vscales[(int64_t)pt_page * p.vs_sp];
        pt_first = first;
    };
    // kSeg 0: the table's entries are loaded two steps before they are used, and
    // before the rows of the step between: vector loads complete in order, so
    // waiting for them then waits for no row that is not needed yet.
    [[maybe_unused]] int pg[2][4];   // of the lane's rows
    [[maybe_unused]] auto fetch_pages = [&](int s, int (&to)[4]) {
        const int t0 = t_begin + s * kDecStep;
#pragma unroll
        for (int r = 0; r < 4; ++r) to[r] = bt[min(t0 + 8 * r + row8, t_end - 1) >> p.page_shift];
    };
    auto load_step = [&](int s, Step8& x, [[maybe_unused]] const int (&pages)[4]) {
        const int t0 = t_begin + s * kDecStep;
        if constexpr (kSeg > 0) {
            const int n0 = ((s - wave) / kNw) * kSegs;   // the wave's first segment of step s
            if (n0 + kSegs > pt_first + kWave) pt_load(n0);
#pragma unroll
            for (int g = 0; g < kSegs; ++g) {
                const int at = n0 - pt_first + g;
                const int64_t page = __builtin_amdgcn_readlane(pt_page, at);
                x.ks[g] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(pt_ks), at));
                x.vs[g] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(pt_vs), at));
                const int tok = t0 + kSeg * g;
                const int nv = min(kSeg, t_end_u - tok);   // rows before the item's end
                const uint32_t slot = (uint32_t)(tok & pmask);
                const __amdgpu_buffer_rsrc_t kr =
                    make_rsrc(kbase + page * p.k_sb + slot * kss, nv > 0 ? (uint32_t)(nv - 1) * kss + kHeadDim : 0u);
                const __amdgpu_buffer_rsrc_t vr =
                    make_rsrc(vbase + page * p.v_sb + slot * vss, nv > 0 ? (uint32_t)(nv - 1) * vss + kHeadDim : 0u);
#pragma unroll
                for (int i = 0; i < 4 / kSegs; ++i)
                    x.k[g * (4 / kSegs) + i] = buf_load16_nt(kr, koff + (uint32_t)(8 * i) * kss);
#pragma unroll
                for (int i = 0; i < 4 / kSegs; ++i)
                    x.v[g * (4 / kSegs) + i] = buf_load16_nt(vr, voff + (uint32_t)(8 * i) * vss);
            }
        } else {
#pragma unroll
            for (int r = 0; r < 4; ++r) {   // (past the item's end: its last token)
                const int64_t slot = min(t0 + 8 * r + row8, t_end - 1) & pmask;
                const int64_t page = min(max(pages[r], 0), p.num_pages - 1);
                x.k[r] = __builtin_nontemporal_load(
                    reinterpret_cast<const u32x4_t*>(kbase + page * p.k_sb + slot * p.k_ss + piece * 16));
                x.v[r] = __builtin_nontemporal_load(
                    reinterpret_cast<const u32x4_t*>(vbase + page * p.v_sb + slot * p.v_ss + piece * 16));
                x.ks[r] = kscales[page * p.ks_sp];
                x.vs[r] = vscales[page * p.vs_sp];
            }
        }
    };

    // One step; its registers are free for the next loads once `reload` is called.
    auto compute = [&](int st, Step8& x, auto&& reload) {
        const int t0 = t_begin + st * kDecStep;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            *reinterpret_cast<u32x4_t*>(kl + (8 * r + row8) * kDec8RowStride + piece * 16) = x.k[r];
            *reinterpret_cast<u32x4_t*>(vl + (8 * r + row8) * kDec8RowStride + piece * 16) = x.v[r];
        }
        if constexpr (kSeg == 0) {
            if (piece == 0) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    sl[8 * r + row8] = x.ks[r];
                    sl[kDecStep + 8 * r + row8] = x.vs[r];
                }
            }
        }
        float ks_seg[4], vs_seg[4];
#pragma unroll
        for (int g = 0; g < kSegs; ++g) {
            ks_seg[g] = x.ks[g];
            vs_seg[g] = x.vs[g];
        }
        reload();
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");

        // S^T = K Q^T (codes), K as the A operand
        f32x4_t s[2];
#pragma unroll
        for (int tb = 0; tb < 2; ++tb) {
            s[tb] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const u32x4_t c =
                    *reinterpret_cast<const u32x4_t*>(kl + (16 * tb + l16) * kDec8RowStride + 64 * j + 16 * g4);
                s[tb] = mfma16(codes_to_bf16<kCode>(c[0], c[1]), qop[2 * j], s[tb]);
                s[tb] = mfma16(codes_to_bf16<kCode>(c[2], c[3]), qop[2 * j + 1], s[tb]);
            }
        }
        // scales of tokens t0 + 16*tb + 4*g4 + i
        float ks[8], vs[8];
        if constexpr (kSeg > 0) {
#pragma unroll
            for (int tb = 0; tb < 2; ++tb) {
                const int g = kSegs == 1 ? 0 : kSegs == 2 ? tb : 2 * tb;
                const bool second = kSegs == 4 && g4 >= 2;
                const float k1 = second ? ks_seg[kSegs == 4 ? g + 1 : g] : ks_seg[g];
                const float v1 = second ? vs_seg[kSegs == 4 ? g + 1 : g] : vs_seg[g];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    ks[4 * tb + i] = k1 * p.scale_log2;
                    vs[4 * tb + i] = v1;
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int at = 16 * (j / 4) + 4 * g4 + j % 4;
                ks[j] = sl[at] * p.scale_log2;
                vs[j] = sl[kDecStep + at];
            }
        }

        // Online softmax for head l16 over tokens t0 + 16*tb + 4*g4 + i.
        float y[8];
        float tmax = -INFINITY;
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = s[j >> 2][j & 3] * ks[j];
        if (t0 + kDecStep > t_end_u) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (t0 + (j >> 2) * 16 + g4 * 4 + (j & 3) >= t_end) y[j] = -INFINITY;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) tmax = fmaxf(tmax, y[j]);
        tmax = groups_max(tmax);
        const float m_new = fmaxf(m_run, tmax);
        // (-inf, no score above it yet: what is subtracted has to be a number)
        const float m_sub = m_new == -INFINITY ? 0.f : m_new;
        const float alpha = fast_exp2(m_run - m_sub);
        float psum = 0.f;
        float pv[8], pmax = __uint_as_float(kLeastRef);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float e = fast_exp2(y[j] - m_sub);
            psum += e;
            pv[j] = e * vs[j];
            pmax = fmaxf(pmax, fabsf(pv[j]));
        }
        pmax = groups_max(pmax);
        // The sums so far are relative to vref, which a larger m_run lowers with them:
        // only a larger P sV rescales them (or vref at its least).
        const float vold = vref * alpha;
        vref = fmaxf(vold, pmax);
        const float vinv = __builtin_amdgcn_rcpf(vref);
        // (exactly 1 where nothing changed: vref * (1 / vref) need not be)
        const float oalpha = vref > vold ? vold * vinv : 1.f;
        f16x8_t pop, plo;   // P sV: rounded, and the rest
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float x = pv[j] * (vinv * kDec8PScale);
            pop[j] = (_Float16)x;
            plo[j] = (_Float16)(x - (float)pop[j]);
        }
        l_run = l_run * alpha + psum;
        m_run = m_new;
        // (most steps raise no head's largest)
        if (__any(oalpha != 1.f)) {
#pragma unroll
            for (int db = 0; db < 8; ++db) oacc[db] *= oalpha;
        }

        // V^T as the A operand: tokens 4*g4 + {0..3} and 16 + 4*g4 + {0..3}
        // of column 16*db + l16, those whose P this lane holds.  Row j of the
        // group's 8 is addressed by lanes 2j and 2j + 1.
        const int row = l16 >> 1;
        const unsigned char* vsrc =
            vl + (4 * g4 + (row & 3) + 16 * (row >> 2)) * kDec8RowStride + 8 * (l16 & 1);
        // (4 columns at a time: a column's second product waits for its first)
#pragma unroll
        for (int d4 = 0; d4 < 8; d4 += 4) {
            f16x8_t v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const u32x2_t c = lds_read_tr8(vsrc + 16 * (d4 + i));
                v[i] = codes_to_f16<kCode>(c[0], c[1]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) oacc[d4 + i] = mfma16_f16(v[i], pop, oacc[d4 + i]);
#pragma unroll
            for (int i = 0; i < 4; ++i) oacc[d4 + i] = mfma16_f16(v[i], plo, oacc[d4 + i]);
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    };

    Step8 step_a, step_b;
    auto load_if = [&](int s, Step8& x, int (&pages)[4], int (&next)[4]) {
        if (kSeg == 0 && s + kNw < n_steps) fetch_pages(s + kNw, next);
        if (s < n_steps) load_step(s, x, pages);
    };
    int st = wave;
    if (kSeg == 0 && st < n_steps) fetch_pages(st, pg[0]);
    load_if(st, step_a, pg[0], pg[1]);
    load_if(st + kNw, step_b, pg[1], pg[0]);
    for (; st < n_steps; st += 2 * kNw) {
        compute(st, step_a, [&] { load_if(st + 2 * kNw, step_a, pg[0], pg[1]); });
        if (st + kNw < n_steps) compute(st + kNw, step_b, [&] { load_if(st + 3 * kNw, step_b, pg[1], pg[0]); });
    }

    l_run = groups_sum(l_run);

    // Merge the waves in LDS (reusing the staging area).
    __syncthreads();
    float* ow = reinterpret_cast<float*>(smem);       // [wave][16][kDec8MergeStride]
    float* mlw = ow + kNw * 16 * kDec8MergeStride;    // [wave][16][2]
    const float oscale = vref * (1.f / kDec8PScale);
#pragma unroll
    for (int db = 0; db < 8; ++db)
        *reinterpret_cast<f32x4_t*>(ow + (wave * 16 + l16) * kDec8MergeStride + db * 16 + g4 * 4) = oacc[db] * oscale;
    if (g4 == 0) {
        mlw[(wave * 16 + l16) * 2 + 0] = m_run;
        mlw[(wave * 16 + l16) * 2 + 1] = l_run;
    }
    __syncthreads();

    const int d0 = (tid & 15) * 8;
    for (int h = tid >> 4; h < p.group; h += kNw * 4) {
        float mw[kNw];
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < kNw; ++w) {
            mw[w] = mlw[(w * 16 + h) * 2];
            M = fmaxf(M, mw[w]);
        }
        float L = 0.f;
        float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kNw; ++w) {
            const float c = (mw[w] == -INFINITY) ? 0.f : fast_exp2(mw[w] - M);
            L += c * mlw[(w * 16 + h) * 2 + 1];
            const float* src = ow + (w * 16 + h) * kDec8MergeStride + d0;
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[j] += c * src[j];
        }
        const int qh = kvh * p.group + h;
        if (whole) {
            const float inv = 1.f / L;
            bf16x8_t out;
#pragma unroll
            for (int j = 0; j < 8; ++j) out[j] = (__bf16)(acc[j] * inv);
            *reinterpret_cast<bf16x8_t*>(p.o + b * p.o_sb + qh * p.o_sh + d0) = out;
            if (p.lse != nullptr && (tid & 15) == 0) p.lse[(int64_t)b * p.hq + qh] = M * kLn2 + logf(L);
        } else {
            const int64_t slot = slot0 + h;
            float* po = p.part_o + slot * kHeadDim + d0;
            *reinterpret_cast<f32x4_t*>(po) = f32x4_t{acc[0], acc[1], acc[2], acc[3]};
            *reinterpret_cast<f32x4_t*>(po + 4) = f32x4_t{acc[4], acc[5], acc[6], acc[7]};
            if ((tid & 15) == 0) {
                p.part_ml[slot * 2 + 0] = M;
                p.part_ml[slot * 2 + 1] = L;
            }
        }
    }
}

}  // namespace fgqa
