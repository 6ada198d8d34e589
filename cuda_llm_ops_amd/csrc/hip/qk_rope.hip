// Queries and keys normalised for each head and rotated to their positions, in one
// pass, and the gradients of that (include/fgqa_rope.h).
//
// A row is one token's query or key of one head, D elements of bf16.  A group of
// 4, 8 or 16 lanes (D up to 64, 128, 256) holds a row, two 16-byte pieces a lane
// with the elements that a rotation pairs, so nothing but the norm's sums goes
// between lanes.  A lane group takes up to 4 rows of one token, with one set of
// angles (8 pairs a lane; the backward's up to 8 rows).
//
// Both directions are bound by the bytes of the rows.  Forward, [4, 6001] tokens of 28
// and 4 heads of 128: 72 us for 393 MB, 5.4 TB/s; one token of 64 conversations, 64 and
// 8 heads: 3.7 us, of a launch.  Backward, [3, 5003] tokens of 32 and 8 heads: 103 us
// for 461 MB with its second launch, 4.5 TB/s.  A large copy reaches 4.96 TB/s.
#include <algorithm>
#include <math.h>

#include <type_traits>

#include "fgqa_device.h"
#include "fgqa_internal.h"
#include "../host/rope_plan.h"

namespace fgqa {
namespace {

constexpr int kThreads = plan::kRopeThreads;

// Rows of one tensor [B, S, H, D], strides in elements.
struct Rows {
    const __bf16* in;
    const __bf16* grad;   // backward: of the outputs
    __bf16* out;
    const void* weight;
    int64_t in_s[3], grad_s[3], out_s[3];
    int heads;
    int per, slices;       // heads an item takes, items of a token
    FastDiv div_slices;
    uint32_t items;
};

struct RopeParams {
    Rows x[2];             // Q, K
    unsigned first_k;      // workgroups from here on take K
    const void* positions;
    const float* inv_freq;
    const int32_t* axes;
    int64_t pos_a, pos_b, pos_s;
    int pos64, weights_bf16, num_axes;
    int seqlen, head_dim, rotary_dim, interleaved;
    FastDiv div_seqlen;
    float eps, inv_dim, sin_sign;
    float* partial;        // backward: [workgroups, D], the workgroups' sums of the weights' gradients
};

// Sum over the lanes of a row, in each of them: neighbours, pairs, then mirrored
// halves of 8 and 16 lanes (DPP, without LDS).
template <int kLanes>
__device__ __forceinline__ float row_sum(float v) {
    auto add = [](float x, auto ctrl) {
        const int o = __builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), decltype(ctrl)::value, 0xF, 0xF, true);
        return x + __uint_as_float((uint32_t)o);
    };
    v = add(v, std::integral_constant<int, 0xB1>{});
    v = add(v, std::integral_constant<int, 0x4E>{});
    if constexpr (kLanes >= 8) v = add(v, std::integral_constant<int, 0x141>{});
    if constexpr (kLanes >= 16) v = add(v, std::integral_constant<int, 0x140>{});
    return v;
}

// cos and sin of t turns, |t| <= 1/2, by the chip's instructions, which take turns: over
// every float of 2^-29 to 1/2 they were off by at most 2^-22.9 (sin 2^-20 relative).
__device__ __forceinline__ void cos_sin_turns(float t, float* c, float* s) {
    *c = __builtin_amdgcn_cosf(t);
    *s = __builtin_amdgcn_sinf(t);
}

typedef float f32x4u_t __attribute__((ext_vector_type(4), aligned(4)));
typedef int i32x4u_t __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x4u_t __attribute__((ext_vector_type(4), aligned(2)));

// 16 bytes of a row; kStream: past the caches, which more rows than they hold would only churn.
template <bool kStream>
__device__ __forceinline__ u32x4_t load16(const __bf16* at) {
    const u32x4_t* p = reinterpret_cast<const u32x4_t*>(at);
    if constexpr (kStream) return __builtin_nontemporal_load(p);
    else return *p;
}
template <bool kStream>
__device__ __forceinline__ void store16(__bf16* at, u32x4_t v) {
    u32x4_t* p = reinterpret_cast<u32x4_t*>(at);
    if constexpr (kStream) __builtin_nontemporal_store(v, p);
    else *p = v;
}

// What a lane holds of each row: 16 elements, those of pieces off[0] and off[1].
struct LaneShape {
    int off[2];
    int pair[2];    // its first pair and its fifth
    bool rotated;
    bool active;    // (lanes past the row's end hold nothing)
};

__device__ __forceinline__ LaneShape lane_shape(const RopeParams& p, int l) {
    LaneShape s;
    s.rotated = 16 * l < p.rotary_dim;
    s.active = 16 * l < p.head_dim;
    // A piece of each half of what is rotated, or of what is not, side by side with the next lanes' (where
    // neighbours are pairs any two would do: the backward of [3, 5003] tokens took 11 to 18 us more with two that
    // follow each other).
    const int base = s.rotated ? 0 : p.rotary_dim, span = s.rotated ? p.rotary_dim : p.head_dim - p.rotary_dim;
    s.off[0] = base + 8 * (l - base / 16);
    s.off[1] = s.off[0] + span / 2;
    s.pair[0] = p.interleaved ? 4 * l : 8 * l;
    s.pair[1] = p.interleaved ? p.rotary_dim / 4 + 4 * l : 8 * l + 4;
    return s;
}

// The lane's 8 angles: positions times inverse frequencies in turns, in 64 bits as
// far as the fraction (a position of 2^20 would leave 32-bit angles 2^-4 off).
__device__ __forceinline__ void lane_angles(const RopeParams& p, const LaneShape& ls, int b, int s, float (&cs)[8],
                                            float (&sn)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        cs[j] = 1.f;
        sn[j] = 0.f;
    }
    if (!ls.rotated) return;
    const int64_t at = b * p.pos_b + s * p.pos_s;
    auto position = [&](int axis) {
        const int64_t i = at + axis * p.pos_a;
        return p.pos64 ? (double)static_cast<const int64_t*>(p.positions)[i]
                       : (double)static_cast<const int32_t*>(p.positions)[i];
    };
    double pos[8];
    if (p.axes != nullptr) {
        const i32x4u_t a0 = *reinterpret_cast<const i32x4u_t*>(p.axes + ls.pair[0]);
        const i32x4u_t a1 = *reinterpret_cast<const i32x4u_t*>(p.axes + ls.pair[1]);
#pragma unroll
        for (int j = 0; j < 8; ++j) pos[j] = position(min(max(j < 4 ? a0[j & 3] : a1[j & 3], 0), p.num_axes - 1));
    } else {
        const double one = position(0);
#pragma unroll
        for (int j = 0; j < 8; ++j) pos[j] = one;
    }
    const f32x4u_t f0 = *reinterpret_cast<const f32x4u_t*>(p.inv_freq + ls.pair[0]);
    const f32x4u_t f1 = *reinterpret_cast<const f32x4u_t*>(p.inv_freq + ls.pair[1]);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const double turns = pos[j] * ((double)(j < 4 ? f0[j & 3] : f1[j & 3]) * 0.15915494309189533577);
        cos_sin_turns((float)(turns - __builtin_rint(turns)), &cs[j], &sn[j]);
        sn[j] *= p.sin_sign;
    }
}

// Two 16-byte pieces <-> 16 fp32: v[0..7] the first's, v[8..15] the second's.
__device__ __forceinline__ void widen(const u32x4_t (&raw)[2], float (&v)[16]) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[8 * i + 2 * j] = __uint_as_float(raw[i][j] << 16);
            v[8 * i + 2 * j + 1] = __uint_as_float(raw[i][j] & 0xffff0000u);
        }
}

__device__ __forceinline__ u32x4_t narrow8(const float* v) {
    bf16x8_t r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = (__bf16)v[i];
    return __builtin_bit_cast(u32x4_t, r);
}

__device__ __forceinline__ void lane_weights(const RopeParams& p, const Rows& x, const LaneShape& ls, float (&w)[16]) {
    if (p.weights_bf16) {
        u32x4_t raw[2];
#pragma unroll
        for (int i = 0; i < 2; ++i)
            raw[i] = *reinterpret_cast<const u32x4u_t*>(static_cast<const __bf16*>(x.weight) + ls.off[i]);
        widen(raw, w);
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const f32x4u_t f = *reinterpret_cast<const f32x4u_t*>(static_cast<const float*>(x.weight) + ls.off[i] + 4 * j);
#pragma unroll
                for (int e = 0; e < 4; ++e) w[8 * i + 4 * j + e] = f[e];
            }
    }
}

// Pairs (a, b) turned by the lane's angles: elements (v[j], v[8 + j]), or, interleaved,
// (v[2j], v[2j + 1]).  Elements that are not rotated stay as they are (an infinity
// times sin 0 would not).
template <bool kInterleaved, bool kBack>
__device__ __forceinline__ void rotate(float (&v)[16], const float (&cs)[8], const float (&sn)[8], bool rotated) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        float& a = v[kInterleaved ? 2 * j : j];
        float& b = v[kInterleaved ? 2 * j + 1 : 8 + j];
        const float s = kBack ? -sn[j] : sn[j];
        const float ra = a * cs[j] - b * s, rb = b * cs[j] + a * s;
        a = rotated ? ra : a;
        b = rotated ? rb : b;
    }
}

struct Item {
    int b, s, h0, rows;
};

__device__ __forceinline__ Item item_of(const RopeParams& p, const Rows& x, uint32_t item) {
    Item r;
    const int token = fast_div((int)item, x.div_slices);
    r.h0 = ((int)item - token * x.slices) * x.per;
    r.rows = min(x.per, x.heads - r.h0);
    r.b = fast_div(token, p.div_seqlen);
    r.s = token - r.b * p.seqlen;
    return r;
}

// Forward; without a norm and with sin negated, also the gradients of a rotation alone.
template <int kLanes, int kHeads, bool kInterleaved, bool kNorm, bool kStream>
__global__ __launch_bounds__(kThreads) void rope_kernel(RopeParams p) {
    const int which = blockIdx.x >= p.first_k ? 1 : 0;
    const Rows& x = p.x[which];
    const unsigned block = blockIdx.x - (which ? p.first_k : 0u);
    const uint32_t item = block * (uint32_t)(kThreads / kLanes) + threadIdx.x / kLanes;
    const LaneShape ls = lane_shape(p, threadIdx.x % kLanes);
    const bool mine = item < x.items && ls.active;   // (all lanes of a row stay for its sum)
    const Item it = item_of(p, x, item < x.items ? item : 0u);

    u32x4_t raw[kHeads][2];
    const __bf16* src = x.in + it.b * x.in_s[0] + it.s * x.in_s[1] + it.h0 * x.in_s[2];
#pragma unroll
    for (int r = 0; r < kHeads; ++r)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            raw[r][i] = u32x4_t{0u, 0u, 0u, 0u};
            if (mine && r < it.rows) raw[r][i] = load16<kStream>(src + r * x.in_s[2] + ls.off[i]);
        }
    float w[16];
    if constexpr (kNorm) {
#pragma unroll
        for (int i = 0; i < 16; ++i) w[i] = 0.f;
        if (ls.active) lane_weights(p, x, ls, w);
    }
    float cs[8], sn[8];
    lane_angles(p, ls, it.b, it.s, cs, sn);

    __bf16* dst = x.out + it.b * x.out_s[0] + it.s * x.out_s[1] + it.h0 * x.out_s[2];
#pragma unroll
    for (int r = 0; r < kHeads; ++r) {
        float v[16];
        widen(raw[r], v);
        if constexpr (kNorm) {
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) sum = fmaf(v[i], v[i], sum);
            const float inv = rsqrtf(row_sum<kLanes>(sum) * p.inv_dim + p.eps);
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = v[i] * inv * w[i];
        }
        rotate<kInterleaved, false>(v, cs, sn, ls.rotated);
        if (mine && r < it.rows) {
#pragma unroll
            for (int i = 0; i < 2; ++i) store16<kStream>(dst + r * x.out_s[2] + ls.off[i], narrow8(v + 8 * i));
        }
    }
}

// Backward with a norm.  With g = R^T dy, u = x / sqrt(mean(x^2) + eps) = x r:
//   dw = sum over rows of g u,   dx = r (w g - u mean(w g u)).
// A workgroup walks items of one tensor and keeps its sums of dw in registers, each
// lane those of its 16 elements, so that no gradient goes through an atomic.  A lane
// group goes through its item's rows one by one with one set of angles, and has the
// next row's loads in flight.
template <int kLanes, bool kInterleaved, bool kStream>
__global__ __launch_bounds__(kThreads) void rope_backward_kernel(RopeParams p) {
    __shared__ float s_dw[kThreads / kWave][plan::kRopeMaxHeadDim];
    const int which = blockIdx.x >= p.first_k ? 1 : 0;
    const Rows& x = p.x[which];
    const unsigned block = blockIdx.x - (which ? p.first_k : 0u);
    const uint32_t blocks = which ? gridDim.x - p.first_k : p.first_k;
    constexpr uint32_t kGroups = kThreads / kLanes;
    const LaneShape ls = lane_shape(p, threadIdx.x % kLanes);
    float w[16], dw[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i] = dw[i] = 0.f;
    if (ls.active) lane_weights(p, x, ls, w);

    struct Place {
        const __bf16 *src, *grad;
        __bf16* dst;
        int b, s, rows;   // (no rows: past the items or the row's end)
    };
    auto place = [&](uint32_t first) {   // (items + a round stay below 2^32)
        const uint32_t item = first + threadIdx.x / kLanes;
        const Item it = item_of(p, x, item < x.items ? item : 0u);
        Place at;
        at.src = x.in + it.b * x.in_s[0] + it.s * x.in_s[1] + it.h0 * x.in_s[2];
        at.grad = x.grad + it.b * x.grad_s[0] + it.s * x.grad_s[1] + it.h0 * x.grad_s[2];
        at.dst = x.out + it.b * x.out_s[0] + it.s * x.out_s[1] + it.h0 * x.out_s[2];
        at.b = it.b;
        at.s = it.s;
        at.rows = item < x.items && ls.active ? it.rows : 0;
        return at;
    };
    u32x4_t raw[2], graw[2];
    auto load = [&](const Place& at, int r) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            raw[i] = graw[i] = u32x4_t{0u, 0u, 0u, 0u};
            if (r < at.rows) {
                raw[i] = load16<kStream>(at.src + r * x.in_s[2] + ls.off[i]);
                graw[i] = load16<kStream>(at.grad + r * x.grad_s[2] + ls.off[i]);
            }
        }
    };
    uint32_t first = block * kGroups;
    Place at = place(first);
    load(at, 0);
    while (first < x.items) {
        const uint32_t next = first + blocks * kGroups;
        float cs[8], sn[8];
        lane_angles(p, ls, at.b, at.s, cs, sn);
        const Place after = place(next);
        for (int r = 0; r < x.per; ++r) {
            float v[16], g[16];
            widen(raw, v);
            widen(graw, g);
            if (r + 1 < x.per) load(at, r + 1);
            else load(after, 0);
            rotate<kInterleaved, true>(g, cs, sn, ls.rotated);
            float sum = 0.f, dot = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) sum = fmaf(v[i], v[i], sum);
            const float inv_row = rsqrtf(row_sum<kLanes>(sum) * p.inv_dim + p.eps);
            const float inv = r < at.rows ? inv_row : 0.f;   // (of rows that are not there eps 0 would make it infinite)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                v[i] *= inv;
                dw[i] = fmaf(g[i], v[i], dw[i]);
                g[i] *= w[i];
                dot = fmaf(g[i], v[i], dot);
            }
            const float mean = row_sum<kLanes>(dot) * p.inv_dim;
#pragma unroll
            for (int i = 0; i < 16; ++i) g[i] = inv * (g[i] - v[i] * mean);
            if (r < at.rows) {
#pragma unroll
                for (int i = 0; i < 2; ++i) store16<kStream>(at.dst + r * x.out_s[2] + ls.off[i], narrow8(g + 8 * i));
            }
        }
        at = after;
        first = next;
    }

    // the wave's lane groups, then the waves in order
#pragma unroll
    for (int i = 0; i < 16; ++i) {
#pragma unroll
        for (int m = kLanes; m < kWave; m *= 2) dw[i] = xor_sum(dw[i], m);
    }
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    if (lane < kLanes && ls.active) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s_dw[wave][ls.off[i / 8] + i % 8] = dw[i];
    }
    __syncthreads();
    for (int d = threadIdx.x; d < p.head_dim; d += kThreads) {
        float sum = 0.f;
#pragma unroll
        for (int v = 0; v < kThreads / kWave; ++v) sum += s_dw[v][d];
        p.partial[(int64_t)blockIdx.x * p.head_dim + d] = sum;
    }
}

// The workgroups' sums to the weights' gradients, 16 elements of one tensor a workgroup.
constexpr int kSumThreads = 1024;
__global__ __launch_bounds__(kSumThreads) void rope_weights_kernel(const float* partial, int head_dim, int blocks_q, int blocks_k,
                                                                   float* dq, float* dk) {
    __shared__ float s_sum[kSumThreads / 16][17];
    const int slices = head_dim / 16;
    const bool k = (int)blockIdx.x >= slices;
    const int d0 = 16 * ((int)blockIdx.x - (k ? slices : 0));
    const int col = threadIdx.x % 16, row = threadIdx.x / 16;
    const int n = k ? blocks_k : blocks_q;
    const float* src = partial + (int64_t)(k ? blocks_q : 0) * head_dim + d0 + col;
    float sum = 0.f;
#pragma unroll 4
    for (int i = row; i < n; i += kSumThreads / 16) sum += src[(int64_t)i * head_dim];
    s_sum[row][col] = sum;
    __syncthreads();
    for (int m = kSumThreads / 32; m > 0; m /= 2) {
        if (row < m) s_sum[row][col] += s_sum[row + m][col];
        __syncthreads();
    }
    if (row == 0) (k ? dk : dq)[d0 + col] = s_sum[0][col];
}

// Calls f with the compile-time lanes of a row and pairing.
template <typename F>
void with_shape(const fgqa_rope_args& a, F&& f) {
    auto pairing = [&](auto lanes) {
        if (a.interleaved) f(lanes, std::true_type{});
        else f(lanes, std::false_type{});
    };
    const int lanes = plan::rope_row_lanes(a.head_dim);
    if (lanes == 4) pairing(std::integral_constant<int, 4>{});
    else if (lanes == 8) pairing(std::integral_constant<int, 8>{});
    else pairing(std::integral_constant<int, 16>{});
}

RopeParams rope_params(const fgqa_rope_args& a, const plan::RopeSlices (&slices)[2]) {
    RopeParams p = {};
    const int64_t tokens = (int64_t)a.batch * a.seqlen;
    const int heads[2] = {a.num_q_heads, a.num_kv_heads};
    const void* weights[2] = {a.q_weight, a.k_weight};
    for (int i = 0; i < 2; ++i) {
        Rows& x = p.x[i];
        x.weight = weights[i];
        x.heads = heads[i];
        x.per = slices[i].per;
        x.slices = slices[i].count;
        x.div_slices = make_fast_div(x.slices);
        x.items = (uint32_t)(tokens * x.slices);
    }
    p.positions = a.positions;
    p.inv_freq = a.inv_freq;
    p.axes = a.axes;
    p.pos_a = a.positions_stride[0];
    p.pos_b = a.positions_stride[1];
    p.pos_s = a.positions_stride[2];
    p.pos64 = a.positions_int64;
    p.weights_bf16 = a.weights_bf16;
    p.num_axes = a.num_axes;
    p.seqlen = a.seqlen;
    p.head_dim = a.head_dim;
    p.rotary_dim = a.rotary_dim;
    p.interleaved = a.interleaved;
    p.div_seqlen = make_fast_div(a.seqlen);
    p.eps = a.eps;
    p.inv_dim = 1.f / (float)a.head_dim;
    p.sin_sign = 1.f;
    return p;
}

void set_rows(Rows* x, const void* in, const int64_t (&is)[3], void* out, const int64_t (&os)[3]) {
    x->in = static_cast<const __bf16*>(in);
    x->out = static_cast<__bf16*>(out);
    for (int i = 0; i < 3; ++i) {
        x->in_s[i] = is[i];
        x->out_s[i] = os[i];
    }
}

template <bool kNorm>
void launch_rope(const fgqa_rope_args& a, RopeParams p, int heads_per, hipStream_t s) {
    with_shape(a, [&](auto lanes, auto inter) {
        constexpr int kLanes = decltype(lanes)::value;
        constexpr bool kInter = decltype(inter)::value;
        const int64_t groups = kThreads / kLanes;
        p.first_k = (unsigned)ceil_div(p.x[0].items, groups);
        const unsigned grid = p.first_k + (unsigned)ceil_div(p.x[1].items, groups);
        auto launch = [&](auto h, auto stream) {
            hipLaunchKernelGGL((rope_kernel<kLanes, decltype(h)::value, kInter, kNorm, decltype(stream)::value>), dim3(grid),
                               dim3(kThreads), 0, s, p);
        };
        if (heads_per != 4) launch(std::integral_constant<int, 1>{}, std::false_type{});
        else if (plan::rope_streams(a, 2)) launch(std::integral_constant<int, 4>{}, std::true_type{});
        else launch(std::integral_constant<int, 4>{}, std::false_type{});
    });
}

// The forward's items.
RopeParams forward_params(const fgqa_rope_args& a, int heads_per) {
    const plan::RopeSlices slices[2] = {plan::rope_slices(a.num_q_heads, heads_per), plan::rope_slices(a.num_kv_heads, heads_per)};
    return rope_params(a, slices);
}

}  // namespace
}  // namespace fgqa

using namespace fgqa;

extern "C" int fgqa_qk_norm_rope(const fgqa_rope_args* a, void* stream) {
    const int st = plan::validate_rope(a);
    if (st != FGQA_OK) return st;
    if (a->batch == 0 || a->seqlen == 0) return FGQA_OK;
    const int heads_per = plan::rope_heads_per(*a);
    RopeParams p = forward_params(*a, heads_per);
    set_rows(&p.x[0], a->q, a->q_stride, a->q_out, a->q_out_stride);
    set_rows(&p.x[1], a->k, a->k_stride, a->k_out, a->k_out_stride);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (a->q_weight != nullptr) launch_rope<true>(*a, p, heads_per, s);
    else launch_rope<false>(*a, p, heads_per, s);
    return hipGetLastError() == hipSuccess ? FGQA_OK : FGQA_ERR_HIP;
}

extern "C" int fgqa_qk_norm_rope_backward_workspace_bytes(const fgqa_rope_backward_args* a, size_t* bytes) {
    if (a == nullptr || bytes == nullptr) return FGQA_ERR_INVALID_ARGUMENT;
    const int st = plan::validate_rope_sizes(a->fwd);
    if (st != FGQA_OK) return st;
    *bytes = a->fwd.q_weight != nullptr ? plan::rope_grad_plan(a->fwd).ws_bytes : 0;
    return FGQA_OK;
}

extern "C" int fgqa_qk_norm_rope_backward(const fgqa_rope_backward_args* a, void* stream) {
    const int st = plan::validate_rope_backward(a);
    if (st != FGQA_OK) return st;
    const fgqa_rope_args& f = a->fwd;
    const bool norm = f.q_weight != nullptr, empty = f.batch == 0 || f.seqlen == 0;
    if (empty && !norm) return FGQA_OK;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (!norm) {
        const int heads_per = plan::rope_heads_per(f);
        RopeParams p = forward_params(f, heads_per);
        set_rows(&p.x[0], a->grad_q_out, a->grad_q_out_stride, a->grad_q, a->grad_q_stride);
        set_rows(&p.x[1], a->grad_k_out, a->grad_k_out_stride, a->grad_k, a->grad_k_stride);
        p.sin_sign = -1.f;
        launch_rope<false>(f, p, heads_per, s);
        return hipGetLastError() == hipSuccess ? FGQA_OK : FGQA_ERR_HIP;
    }
    const plan::RopeGradPlan pl = plan::rope_grad_plan(f);
    std::unique_lock<std::mutex> lock;
    void* ws = a->workspace;
    if (pl.ws_bytes > 0) {
        if (ws == nullptr && a->workspace_bytes == 0) {
            lock = workspace_lock();
            int got = FGQA_OK;
            ws = internal_workspace(pl.ws_bytes, &got);
            if (got != FGQA_OK) return got;
        } else if (ws == nullptr || a->workspace_bytes < pl.ws_bytes) {
            return FGQA_ERR_WORKSPACE;
        } else if ((reinterpret_cast<uintptr_t>(ws) & 255u) != 0) {
            return FGQA_ERR_UNSUPPORTED;
        }
    }
    if (!empty) {
        RopeParams p = rope_params(f, pl.slices);
        set_rows(&p.x[0], f.q, f.q_stride, a->grad_q, a->grad_q_stride);
        set_rows(&p.x[1], f.k, f.k_stride, a->grad_k, a->grad_k_stride);
        p.x[0].grad = static_cast<const __bf16*>(a->grad_q_out);
        p.x[1].grad = static_cast<const __bf16*>(a->grad_k_out);
        for (int i = 0; i < 3; ++i) {
            p.x[0].grad_s[i] = a->grad_q_out_stride[i];
            p.x[1].grad_s[i] = a->grad_k_out_stride[i];
        }
        p.partial = static_cast<float*>(ws);
        p.first_k = (unsigned)pl.blocks[0];
        with_shape(f, [&](auto lanes, auto inter) {
            auto launch = [&](auto stream) {
                hipLaunchKernelGGL((rope_backward_kernel<decltype(lanes)::value, decltype(inter)::value, decltype(stream)::value>),
                                   dim3((unsigned)(pl.blocks[0] + pl.blocks[1])), dim3(kThreads), 0, s, p);
            };
            if (plan::rope_streams(f, 3)) launch(std::true_type{});
            else launch(std::false_type{});
        });
    }
    hipLaunchKernelGGL(rope_weights_kernel, dim3((unsigned)(2 * (f.head_dim / 16))), dim3(kSumThreads), 0, s,
                       static_cast<const float*>(ws), f.head_dim, pl.blocks[0], pl.blocks[1], a->grad_q_weight,
                       a->grad_k_weight);
    return hipGetLastError() == hipSuccess ? FGQA_OK : FGQA_ERR_HIP;
}
