/*
 * fgqa_kv.h -- C ABI of the paged KV cache's operators of libfgqa.so: writing
 * tokens to it, single-token attention over a cache in 8 bits with a scale for
 * each block, the attention weight each cached token gets, and the eviction of
 * the tokens that got least.  Conventions, status codes and the bf16 / fp8
 * caches' layout are fgqa.h's.
 *
 * No counterpart in the reference: it has no paged cache and none in 8 bits.
 */
#ifndef FGQA_KV_H
#define FGQA_KV_H

#include "fgqa.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Continues fgqa_kv_dtype: two's complement bytes, -127 .. 127, in blocks with scales. */
#define FGQA_KV_INT8 2

/*
 * A paged KV cache.
 *   k, v      [num_pages, page_size, num_kv_heads, head_dim] of kv_dtype, strides
 *             {page, slot, head} in elements; 16-byte aligned, strides multiples
 *             of 16 bytes; head_dim 128; page_size a power of two.
 *   k_scales, v_scales   fp32 [num_pages, num_kv_heads], strides {page, head} in
 *             elements: the scale of each block, one page of one KV head, whose
 *             codes c stand for c * scale.  Both or neither (NULL); required
 *             with FGQA_KV_INT8, NULL with FGQA_KV_BF16.  Scales are positive
 *             and at most 2^126 (the append and the eviction write powers of two).
 *             K's and V's data and scales lie apart where a call writes them (one
 *             address for both is refused there); the decode takes shared ones.
 *   k_scale, v_scale     one scale for a whole FGQA_KV_FP8_E4M3 cache without
 *             block scales (finite, and above 0 where tokens are written);
 *             ignored otherwise.
 * Token t of sequence b is slot t % page_size of page block_table[b][t / page_size].
 */
typedef struct fgqa_kv_cache {
    void* k;
    void* v;
    float* k_scales;
    float* v_scales;
    int32_t kv_dtype;
    int32_t num_kv_heads;
    int32_t head_dim;
    int32_t page_size;
    int32_t num_pages;
    float k_scale;
    float v_scale;
    int64_t k_stride[3];
    int64_t v_stride[3];
    int64_t k_scales_stride[2];
    int64_t v_scales_stride[2];
} fgqa_kv_cache;

/*
 * Writes new tokens to the cache: tokens i = 0 .. n-1 of k_new / v_new's row b
 * become tokens seqlens[b] + i of sequence b (seqlens itself is not changed).
 *
 *   k_new, v_new  bf16 [B, max_new, Hkv, D], strides {b, token, head}
 *   block_table   device int32 [B, max_pages], rows block_table_stride apart
 *   seqlens       device int32 [B], tokens the sequences hold (below 0: as 0)
 *   new_lens      device int32 [B], new tokens, each clamped to [0, max_new]
 *                 (nullable: max_new each)
 *
 * Block scales: a block whose first slot gets a new token gets the smallest
 * power of two s (at least 2^-126) with max|x| <= s * 448 (e4m3) or s * 127
 * (int8) over its new tokens' finite values.  A block that holds older tokens
 * keeps its scale or, where its new tokens need a larger one, gets theirs, and
 * its older codes are rounded again to it (exact for e4m3 codes of scales that
 * are powers of two, but for those that become subnormal).  Codes are x / s
 * rounded to nearest even; +-inf becomes the largest code of its sign; NaN
 * stays NaN in e4m3 and becomes 0 in int8.
 *
 * Tokens at or past max_pages * page_size, and those whose page is not in
 * [0, num_pages), are not written.  Slots without a new token keep their
 * bytes (but for older codes rounded again).  The pages that a call writes
 * must not be shared between its sequences.
 */
typedef struct fgqa_kv_append_args {
    fgqa_kv_cache cache;
    const void* k_new;
    const void* v_new;
    int64_t k_new_stride[3];
    int64_t v_new_stride[3];
    const int32_t* block_table;
    int64_t block_table_stride;
    const int32_t* seqlens;
    const int32_t* new_lens;
    int32_t batch;
    int32_t max_new;
    int32_t max_pages;
} fgqa_kv_append_args;

int fgqa_kv_append(const fgqa_kv_append_args* args, void* stream);

/*
 * fgqa_decode_paged over a cache with block scales (e4m3 or int8): scores use
 * q.c * k_scales[page][head] * scale, and O sums p * c * v_scales[page][head].
 * q, o, lse, block_table, seqlens, scale, split_tokens, workspace: as there.
 * Codes are widened exactly; P times the V scale is held in two fp16 numbers (22
 * bits) for P.V, sums are fp32.  Sequences are cut into splits of split_tokens or, where that is 0, as
 * the batch's size asks: outputs may differ in rounding between batches, not
 * between runs of one.  A call whose sequences run whole needs no workspace
 * (fgqa_decode_blocks_workspace_bytes gives 0).
 */
typedef struct fgqa_decode_blocks_args {
    fgqa_kv_cache cache;
    const void* q;
    void* o;
    float* lse;
    const int32_t* block_table;
    const int32_t* seqlens;
    int32_t batch;
    int32_t max_seqlen;
    int32_t num_q_heads;
    float scale;
    int64_t q_stride[2];
    int64_t o_stride[2];
    int64_t block_table_stride;
    int32_t split_tokens;
    void* workspace;
    size_t workspace_bytes;
} fgqa_decode_blocks_args;

int fgqa_decode_blocks_workspace_bytes(const fgqa_decode_blocks_args* args, size_t* bytes);

int fgqa_decode_blocks(const fgqa_decode_blocks_args* args, void* stream);

/*
 * Adds to each cached token's weight what a single-token attention gave it:
 *   weights[b][h][t] += sum over the query heads g of KV head h of
 *                       exp(scale * q[b][g] . k[b][t][h] - lse[b][g]),  t < seqlens[b].
 * Any cache (bf16, e4m3 with one scale or block scales, int8); only K is read.
 *
 *   q        bf16 [B, Hq, D], strides {b, h}
 *   lse      fp32 [B, Hq], contiguous, natural log, as the decode entries write it
 *   weights  fp32 [B, Hkv, at least max_seqlen], strides {b, h}; those at or past
 *            a sequence's length are left as they are.  Rows do not overlap.
 *   block_table, seqlens, max_seqlen, scale: as fgqa_decode_paged.
 * Each weight is added once, without atomics: the same bits from run to run.
 */
typedef struct fgqa_kv_weights_args {
    fgqa_kv_cache cache; /* v, v_scales, v_scale and v_stride are not used */
    const void* q;
    const float* lse;
    float* weights;
    int64_t q_stride[2];
    int64_t weights_stride[2];
    const int32_t* block_table;
    int64_t block_table_stride;
    const int32_t* seqlens;
    int32_t batch;
    int32_t max_seqlen;
    int32_t num_q_heads;
    float scale;
} fgqa_kv_weights_args;

int fgqa_kv_weights(const fgqa_kv_weights_args* args, void* stream);

/*
 * Cuts each sequence to at most `budget` tokens, chosen for each KV head by its
 * weights, and moves those to new pages.
 *
 * A sequence of n <= budget tokens keeps all.  A longer one keeps its last
 * `recent` tokens (at most budget; tokens at or past max_seqlen, which have no
 * weight, all count as recent) and, of those before, the budget - recent of
 * largest weight; of equal weights the one of lower index, NaN counting as
 * larger than any number.  Kept tokens stay in order: token kept[b][h][i] becomes token i,
 * in page new_block_table[b][i / page_size].
 *
 *   weights      fp32 [B, Hkv, at least max_seqlen], strides {b, h}
 *   new_weights  fp32 [B, Hkv, weights_len], strides {b, h}: the kept tokens'
 *                weights, then zeros to weights_len (>= max_seqlen)
 *                (of older tokens, -0 as 0 and a NaN as some NaN,
 *                and 0 of tokens without one; tokens past weights_len have none)
 *   kept         int32 [B, Hkv, budget], contiguous; -1 past the kept tokens
 *   new_seqlens  int32 [B]: min(n, budget)
 *   block_table, seqlens: as fgqa_decode_paged.
 *   max_seqlen   tokens that have weights.  Lengths are clamped to it, or to
 *                max_tokens where that is more: max_tokens is what a row of the block
 *                table holds (0: max_seqlen).
 *   new_block_table  int32 [B, at least min(budget, longest sequence) / page_size
 *                rounded up].  Pages outside [0, num_pages) are not written.
 *                new_tokens: tokens its rows have pages for, where that can be less
 *                (0: enough); sequences are cut to them as if they were the budget.
 *
 * Blocks with scales are scaled anew, as fgqa_kv_append scales new tokens (from
 * the values that the kept codes stand for); other caches' bytes are copied.
 * Slots behind the last kept token keep their bytes.
 *
 * The new pages must be apart from all pages that the call reads, and not
 * shared between its sequences; new_seqlens, new_weights and kept apart from each
 * other and from all that the call reads (weights or seqlens in place are refused).
 * The old pages are left as they are, so pages shared with other sequences stay valid.
 */
typedef struct fgqa_kv_evict_args {
    fgqa_kv_cache cache;
    const float* weights;
    float* new_weights;
    int64_t weights_stride[2];
    int64_t new_weights_stride[2];
    const int32_t* block_table;
    const int32_t* new_block_table;
    int64_t block_table_stride;
    int64_t new_block_table_stride;
    const int32_t* seqlens;
    int32_t* new_seqlens;
    int32_t* kept;
    int32_t batch;
    int32_t max_seqlen;
    int32_t weights_len;
    int32_t budget;
    int32_t recent;
    int32_t max_tokens;
    int32_t new_tokens;
} fgqa_kv_evict_args;

int fgqa_kv_evict(const fgqa_kv_evict_args* args, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* FGQA_KV_H */
