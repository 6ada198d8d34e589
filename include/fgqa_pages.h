/*
 * fgqa_pages.h -- C ABI of sequences that share pages of a paged KV cache in
 * libfgqa.so: forking and freeing sequences, moving the pages in use together, and
 * the decode of sequences that begin alike.  The cache, conventions and status codes
 * are fgqa_kv.h's.
 *
 * No counterpart in the reference: it has no paged cache.
 */
#ifndef FGQA_PAGES_H
#define FGQA_PAGES_H

#include "fgqa_kv.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * New rows of a block table that go on from old ones, with room for new tokens.
 *
 * New row i goes on from old row p = parents[i] (outside [0, batch): from an empty
 * sequence) with n = seqlens[p] tokens (clamped to what the two tables' rows hold) and room
 * for new_lens[i] more.  Its cells, of page_size tokens each:
 *   full pages of the n tokens   the old row's pages, shared
 *   a partly filled last page    the old row's page for the first new row that goes on
 *                                from p (unless held), which may go on filling it; every other
 *                                row gets a page of its own with a copy of the filled slots
 *                                (and, of caches with block scales, of the scales)
 *   further cells up to n + new_lens[i] tokens   pages of its own
 *   the rest                     -1
 * Pages of its own are free ones: pages that are not held and that no new row has from an
 * old one, in ascending order, given to the rows in order and to their cells in order.  So
 * pages that only rows without a successor had are free at once, and so are pages of an old row past its tokens.
 * Where the free pages do not suffice the last cells get -1; a row whose copy got no
 * page is cut to its full pages.
 * An old row's entries outside [0, num_pages) stay as they are (and are nobody's pages).  The
 * page of a partly filled last cell must be in no other place of the old table.
 *
 *   block_table   device int32 [batch, max_pages], rows block_table_stride apart
 *   seqlens       device int32 [batch]
 *   parents       device int32 [new_batch] (nullable: row i goes on from row i)
 *   new_lens      device int32 [new_batch], below 0 as 0 (nullable: 0)
 *   held          device uint8 [num_pages], pages with a value other than 0 are in use
 *                 elsewhere: never given out, and not gone on filling (nullable: none)
 *   new_block_table  device int32 [new_batch, new_max_pages]
 *   new_seqlens   device int32 [new_batch]
 *   num_free      device int32 [1]: free pages that are left, or, below 0, how many were missing
 *   workspace     16-byte aligned, fgqa_kv_fork_workspace_bytes; NULL and 0: the library's buffer
 * What is written lies apart from all that is read, and from each other (one address for two is refused).
 */
typedef struct fgqa_kv_fork_args {
    fgqa_kv_cache cache;
    const int32_t* block_table;
    const int32_t* seqlens;
    const int32_t* parents;
    const int32_t* new_lens;
    const uint8_t* held;
    int32_t* new_block_table;
    int32_t* new_seqlens;
    int32_t* num_free;
    int64_t block_table_stride;
    int64_t new_block_table_stride;
    int32_t batch;
    int32_t max_pages;
    int32_t new_batch;
    int32_t new_max_pages;
    void* workspace;
    size_t workspace_bytes;
} fgqa_kv_fork_args;

int fgqa_kv_fork_workspace_bytes(const fgqa_kv_fork_args* args, size_t* bytes);

int fgqa_kv_fork(const fgqa_kv_fork_args* args, void* stream);

/*
 * Moves the pages in use to the lowest page numbers and renumbers the block table.
 *
 * In use are the pages of the cells that hold seqlens' tokens.  With L of them that are not
 * held, they end up in the first L pages that are not held: those already there stay, the
 * others move, in ascending order, into the pages free there, in ascending order (K and V,
 * every slot, and the scales).  Held pages stay.  The pages that were left keep their bytes.
 *
 *   block_table, seqlens, held, workspace   as fgqa_kv_fork
 *   new_block_table  device int32 [batch, max_pages]: the new numbers; -1 in cells
 *                    past a sequence's tokens; entries outside [0, num_pages) as they are
 *   num_used         device int32 [1]: all pages from there on are free
 * What is written lies apart from all that is read, and from each other (as above).
 */
typedef struct fgqa_kv_compact_args {
    fgqa_kv_cache cache;
    const int32_t* block_table;
    const int32_t* seqlens;
    const uint8_t* held;
    int32_t* new_block_table;
    int32_t* num_used;
    int64_t block_table_stride;
    int64_t new_block_table_stride;
    int32_t batch;
    int32_t max_pages;
    void* workspace;
    size_t workspace_bytes;
} fgqa_kv_compact_args;

int fgqa_kv_compact_workspace_bytes(const fgqa_kv_compact_args* args, size_t* bytes);

int fgqa_kv_compact(const fgqa_kv_compact_args* args, void* stream);

/*
 * Single-token attention over a paged cache, as fgqa_decode_paged and
 * fgqa_decode_blocks, for sequences that begin alike: what group n's sequences,
 * group_starts[n] .. group_starts[n + 1] - 1, share is read once for all of them.
 *
 *   group_starts  device int32 [num_groups + 1], ascending (each taken as at least the
 *                 one before it, and as at most the batch); sequences outside have nothing in common
 *   shared_lens   device int32 [num_groups]: the group's sequences of at least one token have the
 *                 same pages for their first shared_lens[n] tokens: those of the
 *                 first of them are read for all.  What is taken of it is whole pages, at most the shortest such
 *                 sequence; a value of 0 or less is nothing.
 *   cache         any of fgqa_kv.h's (v is read only, as K is)
 *   q, o, lse, block_table, seqlens, max_seqlen, scale   as fgqa_decode_paged
 *   workspace     256-byte aligned, fgqa_decode_shared_workspace_bytes (it depends on the
 *                 sizes and the device, not on lengths); NULL and 0: the library's buffer
 * Sums and statistics are fp32.  For P.V over shared tokens P is rounded to bf16 or, with block
 * scales, held times V's scale in two bf16 numbers (16 bits, products below 2^-126 as 0).  The work is cut as the lengths of all sequences ask: outputs may differ in
 * rounding between batches, not between runs of one.  num_groups is at most 4096, batch below 32768.
 * Over a cache with block scales a call of few tokens (batch * KV heads * max_seqlen at most
 * 1152 a CU) is fgqa_decode_blocks, which then takes less time.
 */
typedef struct fgqa_decode_shared_args {
    fgqa_kv_cache cache;
    const void* q;
    void* o;
    float* lse;
    const int32_t* block_table;
    const int32_t* seqlens;
    const int32_t* group_starts;
    const int32_t* shared_lens;
    int32_t batch;
    int32_t max_seqlen;
    int32_t num_q_heads;
    int32_t num_groups;
    float scale;
    int64_t q_stride[2];
    int64_t o_stride[2];
    int64_t block_table_stride;
    void* workspace;
    size_t workspace_bytes;
} fgqa_decode_shared_args;

int fgqa_decode_shared_workspace_bytes(const fgqa_decode_shared_args* args, size_t* bytes);

int fgqa_decode_shared(const fgqa_decode_shared_args* args, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* FGQA_PAGES_H */
