// Host-only argument validation of include/fgqa_rope.h (see rope_plan.h).
// Products of caller-supplied sizes are formed in 128 bits.
#include "rope_plan.h"

#include <math.h>

namespace fgqa {
namespace plan {

namespace {
typedef __int128 i128;

constexpr int64_t kLim31 = (int64_t)1 << 31;

bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

// Strides of a [B, S, H, D] tensor: not negative, in 16-byte pieces, the last row within 2^60 elements.
int check_strides(const fgqa_rope_args& a, int heads, const int64_t (&s)[3]) {
    const int64_t n[3] = {a.batch, a.seqlen, heads};
    i128 off = 0;
    for (int i = 0; i < 3; ++i) {
        if (s[i] < 0) return FGQA_ERR_INVALID_ARGUMENT;
        off += (i128)(n[i] > 0 ? n[i] - 1 : 0) * s[i];
    }
    if (off >= ((i128)1 << 60)) return FGQA_ERR_UNSUPPORTED;
    for (int i = 0; i < 3; ++i)
        if (s[i] & 7) return FGQA_ERR_UNSUPPORTED;
    return FGQA_OK;
}

int check_rows(const void* p) {
    if (p == nullptr) return FGQA_ERR_INVALID_ARGUMENT;
    return aligned16(p) ? FGQA_OK : FGQA_ERR_UNSUPPORTED;
}

bool same_strides(const int64_t (&x)[3], const int64_t (&y)[3]) {
    return x[0] == y[0] && x[1] == y[1] && x[2] == y[2];
}

// An output at an input's address is that input, element for element.
bool in_place_or_apart(const void* out, const int64_t (&os)[3], const void* in, const int64_t (&is)[3]) {
    return out != in || same_strides(os, is);
}

// Sizes of the forward's arguments that both directions use.
int validate_sizes(const fgqa_rope_args& a) {
    if (a.batch < 0 || a.seqlen < 0 || a.num_q_heads <= 0 || a.num_kv_heads <= 0 || a.num_axes <= 0 || a.head_dim <= 0 ||
        a.rotary_dim < 0 || a.rotary_dim > a.head_dim)
        return FGQA_ERR_INVALID_ARGUMENT;
    if (!isfinite(a.eps) || a.eps < 0.f) return FGQA_ERR_INVALID_ARGUMENT;
    if ((a.q_weight == nullptr) != (a.k_weight == nullptr)) return FGQA_ERR_INVALID_ARGUMENT;
    if (a.head_dim % 16 != 0 || a.head_dim > kRopeMaxHeadDim || a.rotary_dim % 16 != 0) return FGQA_ERR_UNSUPPORTED;
    const int64_t n[3] = {a.num_axes, a.batch, a.seqlen};
    i128 off = 0;
    for (int i = 0; i < 3; ++i) {
        if (a.positions_stride[i] < 0) return FGQA_ERR_INVALID_ARGUMENT;
        off += (i128)(n[i] > 0 ? n[i] - 1 : 0) * a.positions_stride[i];
    }
    if (off >= ((i128)1 << 60)) return FGQA_ERR_UNSUPPORTED;
    // one row an item: its items, and its threads of a launch
    const i128 rows = (i128)a.batch * a.seqlen * ((i128)a.num_q_heads + a.num_kv_heads);
    if (rows >= kLim31 || rows * rope_row_lanes(a.head_dim) + 2 * kRopeThreads >= ((i128)1 << 32)) return FGQA_ERR_UNSUPPORTED;
    return FGQA_OK;
}

// What the angles and the norm read.
int validate_shared_pointers(const fgqa_rope_args& a) {
    if (a.rotary_dim > 0) {
        if (a.positions == nullptr || a.inv_freq == nullptr) return FGQA_ERR_INVALID_ARGUMENT;
        const uintptr_t mask = a.positions_int64 ? 7 : 3;
        if ((reinterpret_cast<uintptr_t>(a.positions) & mask) != 0 || !aligned4(a.inv_freq) || !aligned4(a.axes))
            return FGQA_ERR_UNSUPPORTED;
    }
    const uintptr_t mask = a.weights_bf16 ? 1 : 3;
    if (((reinterpret_cast<uintptr_t>(a.q_weight) | reinterpret_cast<uintptr_t>(a.k_weight)) & mask) != 0)
        return FGQA_ERR_UNSUPPORTED;
    return FGQA_OK;
}

int first_error(int a, int b) { return a != FGQA_OK ? a : b; }
}  // namespace

int validate_rope_sizes(const fgqa_rope_args& a) { return validate_sizes(a); }

// Waves of the items of both tensors, up to `most` heads an item.
static int64_t waves(const fgqa_rope_args& a, int most) {
    const int64_t items =
        (int64_t)a.batch * a.seqlen * (rope_slices(a.num_q_heads, most).count + rope_slices(a.num_kv_heads, most).count);
    return items * rope_row_lanes(a.head_dim) / 64;
}

int rope_heads_per(const fgqa_rope_args& a) {
    // 4 rows share a lane group's angles and have their loads in flight together, as far as there is a wave
    // of them for each SIMD: 1 and 4 rows took 10.2 and 9.3 us on 81,920 rows of 128 (2,560 waves of 4), 6.5 and 6.3
    // on 40,960, but 4.8 and 5.4 on 10,240 (320 waves).
    constexpr int64_t kRopeWaves = 1024;
    return waves(a, 4) >= kRopeWaves ? 4 : 1;
}

bool rope_streams(const fgqa_rope_args& a, int passes) {
    // The last cache holds 2^28 bytes.  Loads and stores of the forward through the caches and past them took 28.8
    // and 30.7 us for 168 MB, 43.8 and 44.8 for 256, 51.9 and 50.7 for 287, 92.3 and 86.1 for 492; those of the
    // backward 47.6 and 54.0 for 252, 70.0 and 69.0 for 307, 98 and 83.5 for 430, 148 and 136 for 737.  (Its loads alone
    // past them took 80 for 430, but 113 for 461 between other calls' data, where both took 103 and neither 110.)
    // A prefill behind the forward, which reads what was written, takes the difference back: [4, 6001] tokens of 28 and 4
    // heads 71 and 81 us, with the prefill 1020 and 1022 (window 512: 362 and 353), [2, 8192] of 32 and 8 heads 62 and 71,
    // 967 and 964 (252 and 251).
    constexpr int64_t kRopeCache = (int64_t)1 << 28;
    const int64_t rows = (int64_t)a.batch * a.seqlen * ((int64_t)a.num_q_heads + a.num_kv_heads);   // (below 2^31)
    return rows * a.head_dim * 2 * passes > kRopeCache;
}

RopeGradPlan rope_grad_plan(const fgqa_rope_args& a) {
    // As many workgroups as the kernel's registers let on the chip at once (3 waves a SIMD);
    // 1024, of which the last wait for a place, took 120 against 108 us on 600,360 rows.
    // Up to 8 rows an item as far as two thirds of those waves have one: 1, 2, 4 and 8 rows
    // took 141, 117, 108 and 108 us there, and 19.0, 18.1, 17.3 and 17.5 us on 73,728 rows.
    constexpr int64_t kRopeGradBlocks = 768, kRopeGradWaves = 2048;
    RopeGradPlan p = {};
    const int64_t tokens = (int64_t)a.batch * a.seqlen;
    const int64_t groups = kRopeThreads / rope_row_lanes(a.head_dim);   // items of a workgroup at a time
    int most = 8;
    while (most > 1 && waves(a, most) < kRopeGradWaves) most /= 2;
    const int heads[2] = {a.num_q_heads, a.num_kv_heads};
    int64_t left = kRopeGradBlocks;
    for (int i = 0; i < 2; ++i) {
        p.slices[i] = rope_slices(heads[i], most);
        const int64_t all = ceil_div(tokens * p.slices[i].count, groups);
        const int64_t part = kRopeGradBlocks * heads[0] / ((int64_t)heads[0] + heads[1]);
        const int64_t share = i == 0 ? (part > 1 ? part : 1) : left;
        p.blocks[i] = (int)(all < share ? all : share);
        left -= share;
    }
    p.ws_bytes = (size_t)(p.blocks[0] + p.blocks[1]) * a.head_dim * sizeof(float);
    return p;
}

int validate_rope(const fgqa_rope_args* a) {
    if (a == nullptr) return FGQA_ERR_INVALID_ARGUMENT;
    int st = validate_sizes(*a);
    if (st == FGQA_OK) st = check_strides(*a, a->num_q_heads, a->q_stride);
    if (st == FGQA_OK) st = check_strides(*a, a->num_kv_heads, a->k_stride);
    if (st == FGQA_OK) st = check_strides(*a, a->num_q_heads, a->q_out_stride);
    if (st == FGQA_OK) st = check_strides(*a, a->num_kv_heads, a->k_out_stride);
    if (st != FGQA_OK || a->batch == 0 || a->seqlen == 0) return st;
    st = first_error(check_rows(a->q), check_rows(a->k));
    st = first_error(st, first_error(check_rows(a->q_out), check_rows(a->k_out)));
    st = first_error(st, validate_shared_pointers(*a));
    if (st != FGQA_OK) return st;
    if (a->q_out == a->k_out || a->q_out == a->k || a->k_out == a->q ||
        !in_place_or_apart(a->q_out, a->q_out_stride, a->q, a->q_stride) ||
        !in_place_or_apart(a->k_out, a->k_out_stride, a->k, a->k_stride))
        return FGQA_ERR_INVALID_ARGUMENT;
    return FGQA_OK;
}

int validate_rope_backward(const fgqa_rope_backward_args* a) {
    if (a == nullptr) return FGQA_ERR_INVALID_ARGUMENT;
    const fgqa_rope_args& f = a->fwd;
    int st = validate_sizes(f);
    if (st == FGQA_OK) st = check_strides(f, f.num_q_heads, a->grad_q_out_stride);
    if (st == FGQA_OK) st = check_strides(f, f.num_kv_heads, a->grad_k_out_stride);
    if (st == FGQA_OK) st = check_strides(f, f.num_q_heads, a->grad_q_stride);
    if (st == FGQA_OK) st = check_strides(f, f.num_kv_heads, a->grad_k_stride);
    const bool norm = f.q_weight != nullptr;
    if (norm) {
        if (st == FGQA_OK) st = check_strides(f, f.num_q_heads, f.q_stride);
        if (st == FGQA_OK) st = check_strides(f, f.num_kv_heads, f.k_stride);
    }
    if (st != FGQA_OK) return st;
    if (norm) {
        if (a->grad_q_weight == nullptr || a->grad_k_weight == nullptr || a->grad_q_weight == a->grad_k_weight)
            return FGQA_ERR_INVALID_ARGUMENT;
        if (!aligned4(a->grad_q_weight) || !aligned4(a->grad_k_weight)) return FGQA_ERR_UNSUPPORTED;
    }
    if (f.batch == 0 || f.seqlen == 0) return FGQA_OK;
    st = first_error(check_rows(a->grad_q_out), check_rows(a->grad_k_out));
    st = first_error(st, first_error(check_rows(a->grad_q), check_rows(a->grad_k)));
    if (norm) st = first_error(st, first_error(check_rows(f.q), check_rows(f.k)));
    st = first_error(st, validate_shared_pointers(f));
    if (st != FGQA_OK) return st;
    if (a->grad_q == a->grad_k || a->grad_q == a->grad_k_out || a->grad_k == a->grad_q_out ||
        !in_place_or_apart(a->grad_q, a->grad_q_stride, a->grad_q_out, a->grad_q_out_stride) ||
        !in_place_or_apart(a->grad_k, a->grad_k_stride, a->grad_k_out, a->grad_k_out_stride))
        return FGQA_ERR_INVALID_ARGUMENT;
    if (norm && (a->grad_q == f.q || a->grad_q == f.k || a->grad_k == f.q || a->grad_k == f.k)) return FGQA_ERR_INVALID_ARGUMENT;
    return FGQA_OK;
}

}  // namespace plan
}  // namespace fgqa
