// Host-only argument validation of the paged KV cache's C ABI (see kv_plan.h).
// Products of caller-supplied sizes are formed in 128 bits.
#include "kv_plan.h"

#include <math.h>

namespace fgqa {
namespace plan {

namespace {
typedef __int128 i128;

constexpr int64_t kLim31 = (int64_t)1 << 31;

// The element offset of the last row stays below 2^60 (strides are not negative).
template <int K>
bool extent_ok(const int64_t (&n)[K], const int64_t* s) {
    i128 off = 0;
    for (int i = 0; i < K; ++i) off += (i128)(n[i] > 0 ? n[i] - 1 : 0) * s[i];
    return off < ((i128)1 << 60);
}

template <int K>
bool non_negative(const int64_t (&s)[K]) {
    for (int i = 0; i < K; ++i)
        if (s[i] < 0) return false;
    return true;
}

bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

bool finite_positive(float x) { return isfinite(x) && x > 0.f; }

// The cache's sizes, type, strides and which scales there are.
// writes: codes are written, so a scale for the whole cache divides.
int validate_cache(const fgqa_kv_cache& c, bool with_v, bool writes) {
    if (c.num_kv_heads <= 0 || c.head_dim <= 0 || c.page_size <= 0 || c.num_pages < 0) return FGQA_ERR_INVALID_ARGUMENT;
    if (c.kv_dtype != FGQA_KV_BF16 && c.kv_dtype != FGQA_KV_FP8_E4M3 && c.kv_dtype != FGQA_KV_INT8)
        return FGQA_ERR_INVALID_ARGUMENT;
    const bool scaled = c.k_scales != nullptr;
    if (with_v && scaled != (c.v_scales != nullptr)) return FGQA_ERR_INVALID_ARGUMENT;
    if (scaled && c.kv_dtype == FGQA_KV_BF16) return FGQA_ERR_INVALID_ARGUMENT;
    if (!scaled && c.kv_dtype == FGQA_KV_INT8) return FGQA_ERR_INVALID_ARGUMENT;
    if (!scaled && c.kv_dtype == FGQA_KV_FP8_E4M3) {
        if (!isfinite(c.k_scale) || (writes && !finite_positive(c.k_scale))) return FGQA_ERR_INVALID_ARGUMENT;
        if (with_v && (!isfinite(c.v_scale) || (writes && !finite_positive(c.v_scale)))) return FGQA_ERR_INVALID_ARGUMENT;
    }
    if (!non_negative(c.k_stride) || (with_v && !non_negative(c.v_stride))) return FGQA_ERR_INVALID_ARGUMENT;
    if (scaled && (!non_negative(c.k_scales_stride) || (with_v && !non_negative(c.v_scales_stride))))
        return FGQA_ERR_INVALID_ARGUMENT;
    if ((c.page_size & (c.page_size - 1)) != 0 || c.page_size > (1 << 20)) return FGQA_ERR_UNSUPPORTED;
    if (c.head_dim != kHeadDim) return FGQA_ERR_UNSUPPORTED;
    const int64_t n[3] = {c.num_pages, c.page_size, c.num_kv_heads};
    const int64_t sn[2] = {c.num_pages, c.num_kv_heads};
    if (!extent_ok(n, c.k_stride) || (with_v && !extent_ok(n, c.v_stride))) return FGQA_ERR_UNSUPPORTED;
    if (scaled && (!extent_ok(sn, c.k_scales_stride) || (with_v && !extent_ok(sn, c.v_scales_stride))))
        return FGQA_ERR_UNSUPPORTED;
    const int64_t m = c.kv_dtype == FGQA_KV_BF16 ? 7 : 15;   // strides in 16-byte pieces
    for (int i = 0; i < 3; ++i)
        if ((c.k_stride[i] & m) || (with_v && (c.v_stride[i] & m))) return FGQA_ERR_UNSUPPORTED;
    return FGQA_OK;
}

int validate_cache_pointers(const fgqa_kv_cache& c, bool with_v) {
    if (c.num_pages == 0 || c.k == nullptr || (with_v && c.v == nullptr)) return FGQA_ERR_INVALID_ARGUMENT;
    if (!aligned16(c.k) || (with_v && !aligned16(c.v))) return FGQA_ERR_UNSUPPORTED;
    if (!aligned4(c.k_scales) || (with_v && !aligned4(c.v_scales))) return FGQA_ERR_UNSUPPORTED;
    return FGQA_OK;
}

// K's and V's data and block scales, which the call writes, are not the same memory.
bool written_apart(const fgqa_kv_cache& c) {
    return c.k != c.v && (c.k_scales == nullptr || c.k_scales != c.v_scales);
}

// A launch has fewer than 2^31 workgroups and 2^32 threads.
bool grid_ok(i128 workgroups, int threads) {
    return workgroups < kLim31 && workgroups * threads < ((i128)1 << 32);
}

// Blocks of the append's and the eviction's pages.
bool blocks_ok(i128 blocks, int page_size) {
    return blocks < kLim31 && grid_ok(page_size <= kWavePageRows ? (blocks + 3) / 4 : blocks, 256);
}
}  // namespace

int validate_kv_append(const fgqa_kv_append_args* a) {
    if (a == nullptr) return FGQA_ERR_INVALID_ARGUMENT;
    const int st = validate_cache(a->cache, true, true);
    if (st != FGQA_OK) return st;
    if (a->batch < 0 || a->max_new < 0 || a->max_pages < 0 || a->block_table_stride < 0) return FGQA_ERR_INVALID_ARGUMENT;
    if (!non_negative(a->k_new_stride) || !non_negative(a->v_new_stride)) return FGQA_ERR_INVALID_ARGUMENT;
    if (a->max_new > kMaxTokens || (i128)a->max_pages * a->cache.page_size > kMaxTokens) return FGQA_ERR_UNSUPPORTED;
    const int64_t n[3] = {a->batch, a->max_new, a->cache.num_kv_heads};
    const int64_t bn[1] = {a->batch};
    if (!extent_ok(n, a->k_new_stride) || !extent_ok(n, a->v_new_stride) || !extent_ok(bn, &a->block_table_stride))
        return FGQA_ERR_UNSUPPORTED;
    if (!blocks_ok((i128)a->batch * append_pages(a->max_new, a->cache.page_size) * 2 * a->cache.num_kv_heads,
                   a->cache.page_size))
        return FGQA_ERR_UNSUPPORTED;
    if (a->batch == 0 || a->max_new == 0 || a->max_pages == 0) return FGQA_OK;
    if (a->k_new == nullptr || a->v_new == nullptr || a->block_table == nullptr || a->seqlens == nullptr)
        return FGQA_ERR_INVALID_ARGUMENT;
    if (!aligned16(a->k_new) || !aligned16(a->v_new) || !aligned4(a->block_table) || !aligned4(a->seqlens) ||
        !aligned4(a->new_lens))
        return FGQA_ERR_UNSUPPORTED;
    for (int i = 0; i < 3; ++i)
        if ((a->k_new_stride[i] & 7) || (a->v_new_stride[i] & 7)) return FGQA_ERR_UNSUPPORTED;
    const int pointers = validate_cache_pointers(a->cache, true);
    if (pointers != FGQA_OK) return pointers;
    return written_apart(a->cache) ? FGQA_OK : FGQA_ERR_INVALID_ARGUMENT;
}

int validate_kv_weights(const fgqa_kv_weights_args* a) {
    if (a == nullptr) return FGQA_ERR_INVALID_ARGUMENT;
    const int st = validate_cache(a->cache, false, false);
    if (st != FGQA_OK) return st;
    if (a->batch < 0 || a->max_seqlen < 0 || a->num_q_heads <= 0 || a->block_table_stride < 0)
        return FGQA_ERR_INVALID_ARGUMENT;
    if (a->num_q_heads % a->cache.num_kv_heads != 0 || !isfinite(a->scale)) return FGQA_ERR_INVALID_ARGUMENT;
    if (!non_negative(a->q_stride) || !non_negative(a->weights_stride)) return FGQA_ERR_INVALID_ARGUMENT;
    // the block table row covers max_seqlen tokens
    if ((i128)a->max_seqlen > (i128)a->block_table_stride * a->cache.page_size)
        return FGQA_ERR_INVALID_ARGUMENT;
    if (a->num_q_heads / a->cache.num_kv_heads > 16) return FGQA_ERR_UNSUPPORTED;
    if (a->max_seqlen > kMaxTokens) return FGQA_ERR_UNSUPPORTED;
    const int64_t qn[2] = {a->batch, a->num_q_heads};
    const int64_t wn[3] = {a->batch, a->cache.num_kv_heads, a->max_seqlen};
    const int64_t ws[3] = {a->weights_stride[0], a->weights_stride[1], 1};
    const int64_t bn[1] = {a->batch};
    if (!extent_ok(qn, a->q_stride) || !extent_ok(wn, ws) || !extent_ok(bn, &a->block_table_stride))
        return FGQA_ERR_UNSUPPORTED;
    if (a->batch == 0 || a->max_seqlen == 0) return FGQA_OK;
    if (!grid_ok(((i128)a->batch * a->cache.num_kv_heads * weights_waves(a->batch, a->cache.num_kv_heads, a->max_seqlen) + 3) / 4,
                 256))
        return FGQA_ERR_UNSUPPORTED;
    if (a->q == nullptr || a->lse == nullptr || a->weights == nullptr || a->block_table == nullptr ||
        a->seqlens == nullptr)
        return FGQA_ERR_INVALID_ARGUMENT;
    if (!aligned16(a->q) || (a->q_stride[0] & 7) || (a->q_stride[1] & 7)) return FGQA_ERR_UNSUPPORTED;
    if (!aligned4(a->lse) || !aligned4(a->weights) || !aligned4(a->block_table) || !aligned4(a->seqlens))
        return FGQA_ERR_UNSUPPORTED;
    return validate_cache_pointers(a->cache, false);
}

int validate_kv_evict(const fgqa_kv_evict_args* a) {
    if (a == nullptr) return FGQA_ERR_INVALID_ARGUMENT;
    const int st = validate_cache(a->cache, true, false);
    if (st != FGQA_OK) return st;
    if (a->batch < 0 || a->max_seqlen < 0 || a->weights_len < a->max_seqlen || a->budget <= 0 || a->recent < 0 ||
        a->max_tokens < 0 || a->new_tokens < 0)
        return FGQA_ERR_INVALID_ARGUMENT;
    if (a->block_table_stride < 0 || a->new_block_table_stride < 0 || !non_negative(a->weights_stride) ||
        !non_negative(a->new_weights_stride))
        return FGQA_ERR_INVALID_ARGUMENT;
    const int64_t longest = evict_tokens(*a);
    const int64_t most = evict_most(*a) < longest ? evict_most(*a) : longest;
    // the block tables' rows cover the tokens
    if ((i128)longest > (i128)a->block_table_stride * a->cache.page_size ||
        (i128)most > (i128)a->new_block_table_stride * a->cache.page_size)
        return FGQA_ERR_INVALID_ARGUMENT;
    if (a->weights_len > kMaxTokens || a->budget > kMaxTokens || longest > kMaxTokens) return FGQA_ERR_UNSUPPORTED;
    const int64_t wn[3] = {a->batch, a->cache.num_kv_heads, a->weights_len};
    const int64_t ws[3] = {a->weights_stride[0], a->weights_stride[1], 1};
    const int64_t ns[3] = {a->new_weights_stride[0], a->new_weights_stride[1], 1};
    const int64_t bn[1] = {a->batch};
    if (!extent_ok(wn, ws) || !extent_ok(wn, ns) || !extent_ok(bn, &a->block_table_stride) ||
        !extent_ok(bn, &a->new_block_table_stride) ||
        (i128)a->batch * a->cache.num_kv_heads * a->budget >= ((i128)1 << 60))
        return FGQA_ERR_UNSUPPORTED;
    const i128 rows = (i128)a->batch * a->cache.num_kv_heads;
    if (!grid_ok(rows, 1024) || !blocks_ok(rows * 2 * ceil_div(most, a->cache.page_size), a->cache.page_size))
        return FGQA_ERR_UNSUPPORTED;
    if (a->batch == 0) return FGQA_OK;
    if (a->seqlens == nullptr || a->new_seqlens == nullptr || a->kept == nullptr) return FGQA_ERR_INVALID_ARGUMENT;
    if (!aligned4(a->seqlens) || !aligned4(a->new_seqlens) || !aligned4(a->kept)) return FGQA_ERR_UNSUPPORTED;
    // (workgroups write outputs while others still read these)
    if (a->new_seqlens == a->seqlens || a->new_seqlens == a->kept) return FGQA_ERR_INVALID_ARGUMENT;
    if (a->weights_len > 0) {
        if (a->new_weights == nullptr) return FGQA_ERR_INVALID_ARGUMENT;
        if (!aligned4(a->new_weights)) return FGQA_ERR_UNSUPPORTED;
    }
    if (longest == 0) return FGQA_OK;
    if (a->block_table == nullptr || a->new_block_table == nullptr) return FGQA_ERR_INVALID_ARGUMENT;
    if (a->max_seqlen > 0 && (a->weights == nullptr || a->weights == a->new_weights)) return FGQA_ERR_INVALID_ARGUMENT;
    if (!aligned4(a->weights) || !aligned4(a->block_table) || !aligned4(a->new_block_table)) return FGQA_ERR_UNSUPPORTED;
    const int pointers = validate_cache_pointers(a->cache, true);
    if (pointers != FGQA_OK) return pointers;
    return written_apart(a->cache) ? FGQA_OK : FGQA_ERR_INVALID_ARGUMENT;
}

fgqa_decode_paged_args as_decode_paged(const fgqa_decode_blocks_args* a) {
    fgqa_decode_paged_args p = {};
    p.q = a->q;
    p.k_cache = a->cache.k;
    p.v_cache = a->cache.v;
    p.o = a->o;
    p.lse = a->lse;
    p.block_table = a->block_table;
    p.seqlens = a->seqlens;
    p.batch = a->batch;
    p.max_seqlen = a->max_seqlen;
    p.num_q_heads = a->num_q_heads;
    p.num_kv_heads = a->cache.num_kv_heads;
    p.head_dim = a->cache.head_dim;
    p.page_size = a->cache.page_size;
    p.num_pages = a->cache.num_pages;
    p.kv_dtype = FGQA_KV_FP8_E4M3;
    p.scale = a->scale;
    p.k_scale = p.v_scale = 1.f;
    for (int i = 0; i < 2; ++i) {
        p.q_stride[i] = a->q_stride[i];
        p.o_stride[i] = a->o_stride[i];
    }
    for (int i = 0; i < 3; ++i) {
        p.k_stride[i] = a->cache.k_stride[i];
        p.v_stride[i] = a->cache.v_stride[i];
    }
    p.block_table_stride = a->block_table_stride;
    p.split_tokens = a->split_tokens;
    p.workspace = a->workspace;
    p.workspace_bytes = a->workspace_bytes;
    return p;
}

// Splits of the tokens that a CU gets of a full batch, so that one round of
// workgroups runs, down to a step of 8 waves; no splits where the sequences are
// at most kSplitSlack longer (the combine's launch costs what those take).  Hq / Hkv,
// 16-token pages, lengths up to S, us teams / splits: 16 / 1, 1 x 512 11.1 / 6.0; 32 / 8,
// 4 x 1024 16.0 / 9.4, 16 x 4096 30.7 / 28.1, 1 x 32768 25.0 / 21.6 (but 17.7 / 18.6
// where the one sequence has 8806 tokens of them).  Teams share out uneven lengths,
// and 4 heads of theirs read side by side: they are taken for more than kSplitMost
// tokens a CU (16 x 8192 40.3 / 46.2, 128 x 2048 63.2 / 75.5) or two workgroups a CU
// (32 / 8, 128 x 512 26.1 / 30.4).  The lines are those of 8 KV heads; 28 / 4, 64 x
// 4096 is the other way, 41.3 / 36.5, which they do not tell apart.
int blocks_split(int64_t batch, int64_t num_kv_heads, int64_t max_seqlen, int cus) {
    constexpr int64_t kSplitMost = 2048, kSplitSlack = 512;
    const i128 heads = (i128)batch * num_kv_heads;
    const i128 tokens = heads * max_seqlen;
    if (max_seqlen <= 0 || tokens > (i128)kSplitMost * cus || heads > 2 * (i128)cus) return 0;
    const int64_t step = kDecodeStepRound;   // what 4 waves take at a time
    const int64_t chunk = ceil_div(ceil_div((int64_t)tokens, cus), step) * step;
    return (int)(max_seqlen <= chunk + kSplitSlack ? ceil_div(max_seqlen, step) * step : chunk);
}

int plan_blocks(const fgqa_decode_paged_args* a, int cus, DecodePlan* plan) {
    fgqa_decode_paged_args split = *a;
    if (a->split_tokens == 0)
        split.split_tokens = blocks_split(a->batch, a->num_kv_heads, a->max_seqlen, cus > 0 ? cus : 256);
    const int st = split.split_tokens > 0 ? plan_paged(&split, plan) : plan_paged(a, plan, block_item_slots(a->num_kv_heads));
    if (st != FGQA_OK) return st;
    const bool splits = grid_ok((i128)a->batch * plan->nsplit * a->num_kv_heads, 512);
    if (plan->teams > 0) {
        if (!splits) plan->least_bytes = plan->ws_bytes;   // teams or nothing
        return FGQA_OK;
    }
    plan->list = false;
    plan->ws_bytes = plan->least_bytes = plan->part_o_bytes + plan->part_ml_bytes;
    return splits ? FGQA_OK : FGQA_ERR_UNSUPPORTED;
}

int validate_decode_blocks(const fgqa_decode_blocks_args* a) {
    if (a == nullptr) return FGQA_ERR_INVALID_ARGUMENT;
    if (a->cache.kv_dtype != FGQA_KV_FP8_E4M3 && a->cache.kv_dtype != FGQA_KV_INT8) return FGQA_ERR_INVALID_ARGUMENT;
    const fgqa_decode_paged_args p = as_decode_paged(a);
    return validate_paged(&p);
}

int validate_decode_blocks_pointers(const fgqa_decode_blocks_args* a) {
    const fgqa_decode_paged_args p = as_decode_paged(a);
    int st = validate_paged_pointers(&p);
    if (st != FGQA_OK || a->batch == 0 || a->max_seqlen == 0) return st;
    if (a->cache.k_scales == nullptr || a->cache.v_scales == nullptr) return FGQA_ERR_INVALID_ARGUMENT;
    st = validate_cache(a->cache, true, false);
    return st != FGQA_OK ? st : validate_cache_pointers(a->cache, true);
}

}  // namespace plan
}  // namespace fgqa
