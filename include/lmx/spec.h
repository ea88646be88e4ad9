/*
 * lmx/spec.h -- one step with drafted tokens (speculative decoding) over the
 * paged KV cache of lmx/paged.h: its pages and row maps, its trees, its
 * prologue, its attention, the verification of the drafts and the keeping of
 * the accepted rows.  The conventions are lmx/attn.h's: plain C types,
 * caller-owned device memory, work enqueued on `stream`, nothing allocated or
 * synchronized, arguments validated on the host before anything is enqueued,
 * lmx_status results.  The reference decodes one token at a time for one
 * sequence (docs/limitations.md:21); nothing here has a counterpart there
 * beyond what lmxs_prologue and lmxs_attn name.
 *
 * A step.  Request b has lens[b] positions in the cache and brings some rows:
 * row 0 its last accepted token, whose K and V the cache lacks, and behind it
 * drafted tokens.  parent[i] is the row (within the request's) that row i
 * continues: parents come before their children; -1, or anything else that is
 * not an earlier row, makes a row a root.  Row i is stored in slot lens[b] + i
 * and stands at position lens[b] + its depth.
 *     lmxs_plan      pages, offsets, lengths, slots        once a step
 *     lmxs_tree      positions, and who sees whom          once a step
 *     lmxs_prologue  norm, rotate at the positions, store  each layer
 *     lmxs_attn      attention                             each layer
 *     lmxs_verify    accepted rows, next token             once a step
 *     lmxs_keep      accepted rows to consecutive slots    once a step, all layers
 * Lengths, tables, trees and paths are read on the device, so that one captured
 * graph serves every step within its bounds.  Device contents that break the
 * rules below give unspecified results for the requests that they belong to,
 * but no access outside the buffers.
 */
#ifndef LMX_SPEC_H
#define LMX_SPEC_H

#include "lmx/paged.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Most rows of a request in lmxs_tree, lmxs_attn, lmxs_verify and lmxs_keep. */
#define LMXS_MAX_ROWS 1024

/* ------------------------------------------------------------------------
 * The step's pages and row maps from the requests' lengths.  Request b, with
 * lens[b] positions cached and new_rows[b] rows to come, needs
 * ceil((lens[b] + new_rows[b]) / page_size) table entries and has held[b].
 *  - trim: entries beyond what is needed are given back (the last request's
 *    first, its last entry first) and become -1; those that are no page are
 *    only dropped.  A request that left has length 0 and no rows.
 *  - Then requests take the entries that they lack, in order, each from the top
 *    of the list of free pages.  Where the list ends, what is still lacking is
 *    left out: held[b] says how many entries there are, later positions are in
 *    no page, and the next call tries again.
 * A call that takes pages and one with the lengths before it that trims them
 * leave table and list as they were.  A page goes back for every entry that names
 * it: one that requests share has to be in no more than one of the tables by then.
 *   lens, new_rows  device int32 [n_seq]
 *   page_table      int32 [n_seq, table_stride]; what lies from held[b] on is not
 *                   read, and written where the request needs it
 *   held            int32 [n_seq], updated
 *   free_pages      int32 [n_pages]; n_free[0] of them are free.  What lies
 *                   behind them is not read and stays.
 *   n_free          int32 [2], updated: pages that are free, entries lacking
 *   cu, ctx_lens    int32 [n_seq + 1] and [n_seq], written: lmxp_batch's.
 *                   ctx_lens[b] is lens[b] + new_rows[b], also where the table ends
 *                   before that: the rows behind its end are in no page, and what
 *                   is cached stays as it is
 *   slots           int64 [n_tokens] or NULL, written: page * page_size + slot
 *                   of each row, -1 for a row in no page or of no request
 *   pos             int32 [n_tokens] or NULL, written: lens[b] + its place among
 *                   its request's rows; -1 for a row of no request
 * Negative lengths count as 0.  A request of more rows than its table has positions
 * cannot be served: its ctx_lens is the table's positions, and the calls below put
 * none of its rows in a page.  None of these may overlap. */
typedef struct {
    uint32_t n_seq;
    uint32_t n_tokens;    /* rows of slots and pos: at least the new rows     */
    uint32_t page_size;   /* 16, 32, 64, 128 or 256                           */
    uint32_t table_stride;
    uint32_t n_pages;     /* pages of the pool, and entries of free_pages     */
    uint32_t trim;        /* 1: give back what is not needed                  */
} lmxs_plan_desc;

lmx_status lmxs_plan(const lmxs_plan_desc *d, const int32_t *lens, const int32_t *new_rows,
                     int32_t *page_table, int32_t *held, int32_t *free_pages, int32_t *n_free,
                     int32_t *cu, int32_t *ctx_lens, int64_t *slots, int32_t *pos,
                     lmx_stream stream);

/* ------------------------------------------------------------------------
 * Positions and sight of a step's rows from their parents.
 *   parent  int32 [n_tokens]
 *   words   64-bit words a row of seen, at least max_new / 64; 1 to 16
 *   window  0, or rows see only ancestors less than `window` behind them
 *   pos     int32 [n_tokens] or NULL, written: ctx_lens[b] less its rows, plus
 *           the row's depth
 *   seen    uint64 [n_tokens, words] or NULL, written: bit j of row i: it sees
 *           row j of its request (itself and its ancestors)
 * Of the batch n_seq, n_tokens, max_new, cu and ctx_lens count.  Rows of no
 * request are left as they are. */
lmx_status lmxs_tree(const lmxp_batch *b, const int32_t *parent, uint32_t words, uint32_t window,
                     int32_t *pos, uint64_t *seen, lmx_stream stream);

/* ------------------------------------------------------------------------
 * lmxp_prologue with positions apart from slots, either order of pairs, and
 * turns that are scaled.  The row's K and V go to its slot; q and k turn by
 *   pos[i] * rope_base^(-2j/n_rot) / rope_factors[j]
 * in pair j, (j, j + n_rot/2) or, interleaved, (2j, 2j + 1), times turn_scale.
 * Factors and turn_scale express linear, per-band and YaRN scaling for long
 * contexts.  Everything else is lmxp_prologue's.
 *   pos     device int32 [n_tokens]; NULL: the rows' slots' positions */
typedef struct {
    uint32_t interleaved; /* 0: pairs are half a rotation apart, 1: neighbours */
    float turn_scale;     /* factor of sine and cosine (1: a rotation)         */
} lmxs_rope;

lmx_status lmxs_prologue(const lmxp_pool *p, const lmxp_batch *b, const lmxp_prologue_desc *d,
                         const lmxs_rope *r, const int32_t *pos, const float *q,
                         const float *k_new, const float *v_new, const float *q_gain,
                         const float *k_gain, const float *rope_factors, void *q_out,
                         lmx_dtype q_out_dt, lmx_stream stream);

/* ------------------------------------------------------------------------
 * lmxp_attn for rows that see each other by a mask: row i of a request sees
 *  - the positions before the request's rows, [0, ctx - rows), in a window those
 *    above pos[i] - window, and
 *  - row j of the request where bit j of its seen is set,
 * as far as they are in a page.  The window says nothing of the rows (lmxs_tree
 * leaves those behind it out of seen); pos[i] is taken as at least ctx - rows
 * and below ctx.  A row that sees nothing, or whose every score is -infinity,
 * gets zeros, and what a row does not see has no part in its result.
 *   seen   uint64 [n_tokens, words], 8-byte aligned; words 1 to 16, 64 * words
 *          at least max_new
 *   pos    int32 [n_tokens]; may be NULL without a window
 * Types, layouts and precision are lmxp_attn's, but that f16 q and out always have
 * weights of 22 bits, as f32 q and out have.  The workspace is used as lmxp_attn's:
 * lmxs_attn_workspace_bytes gives what serves this batch and every one whose n_seq,
 * n_tokens, max_new and max_ctx are at most its own, for either dt and any window (0 for a description that is
 * refused). */
size_t lmxs_attn_workspace_bytes(const lmxp_pool *p, const lmxp_batch *b,
                                 const lmxp_attn_desc *d);

lmx_status lmxs_attn(const lmxp_pool *p, const lmxp_batch *b, const lmxp_attn_desc *d,
                     const uint64_t *seen, uint32_t words, const int32_t *pos, const void *q,
                     lmx_dtype dt, void *out, void *ws, size_t ws_bytes, lmx_stream stream);

/* ------------------------------------------------------------------------
 * Which drafted rows the target model accepts, and the token behind them, from
 * given random numbers, so that what comes out is distributed as the target's
 * own samples.  Rows are gone through in order; a row is tested if its parent is
 * the last accepted row (row 0 at first), and the first that passes is the next
 * accepted row.  p is the target's distribution behind each row, W = 1 at first:
 *   q given   the distribution that each row's children were drawn from, each
 *             by itself.  w = (p - a q)+, a = 0 at first; child c passes if
 *             u W q(c) < w(c); after one that does not, a += W and
 *             W = sum of (p - a q)+.
 *   q NULL    the children were chosen (the draft's best): c passes if
 *             u W < w(c), w = p; after one that does not, W -= w(c), w(c) = 0.
 * In the end the token is the least t with w(0) + .. + w(t) > r * sum of w, of
 * the last accepted row's w.  All of this is in 64 bits.  Where nothing of w is left
 * the token comes from p; where p has nothing either it is -1.
 *   greedy    a child passes if it is the largest p's index (the lowest of
 *             equals, NaN none of them); so the token.  p may be logits; q, u
 *             and r are not read.  -1 where every p is NaN.
 *   cu        device int32 [n_seq + 1], as lmxp_batch's
 *   tokens    int32 [n_tokens]; one outside [0, vocab) never passes and changes
 *             nothing
 *   parent    int32 [n_tokens], or NULL: each row continues the one before it
 *   p, q      [n_tokens, vocab] of dt (LMX_F32 or LMX_F16), rows p_stride,
 *             q_stride elements apart; entries that are not above 0 and finite
 *             count as 0.  Rows are taken to sum to 1.
 *   u         f32 [n_tokens] in [0, 1): the test of each row
 *   r         f32 [n_seq] in [0, 1)
 *   path      int32 [n_seq, max_new], written: the accepted rows (0 first)
 *             within the request, then -1
 *   accepted  int32 [n_seq], written: their number, 0 for a request of no rows
 *   token     int32 [n_seq], written; -1 for a request of no rows
 *   lens      int32 [n_seq] or NULL: accepted is added to it
 * The workspace (16-byte aligned) is needed for large vocabularies unless greedy, where
 * lmxs_verify_workspace_bytes is not 0; every byte read from it was written by the same
 * call.  Outputs overlap nothing. */
typedef struct {
    uint32_t n_seq;
    uint32_t n_tokens;
    uint32_t max_new;     /* most rows of a request, at most LMXS_MAX_ROWS     */
    uint32_t vocab;       /* at most 2^24                                      */
    uint32_t p_stride;    /* 0: vocab                                          */
    uint32_t q_stride;    /* 0: vocab                                          */
    uint32_t greedy;
} lmxs_verify_desc;

size_t lmxs_verify_workspace_bytes(const lmxs_verify_desc *d);

lmx_status lmxs_verify(const lmxs_verify_desc *d, const int32_t *cu, const int32_t *tokens,
                       const int32_t *parent, const void *p, const void *q, lmx_dtype dt,
                       const float *u, const float *r, int32_t *path, int32_t *accepted,
                       int32_t *token, int32_t *lens, void *ws, size_t ws_bytes,
                       lmx_stream stream);

/* ------------------------------------------------------------------------
 * Moves the accepted rows' K and V to the slots behind the cached positions:
 * row path[b][j] of request b to where its row j is, for 0 < j < accepted[b].
 * path rises and path[b][j] >= j, as lmxs_verify writes it; an entry that does
 * not, and one that is no row of the request, is not moved, nor one from or to a
 * position in no page.
 *   pools     host array of n_pools (1 to 1024) pointers to pools (a layer each) of
 *             one geometry and store, whose pages the batch's table names; their K,
 *             V and scales do not overlap
 *   b         the step's batch, its lengths with all of its rows
 *   path      int32 [n_seq, path_stride], path_stride at least max_new
 *   accepted  int32 [n_seq] */
lmx_status lmxs_keep(const lmxp_pool *const *pools, uint32_t n_pools, const lmxp_batch *b,
                     const int32_t *path, uint32_t path_stride, const int32_t *accepted,
                     lmx_stream stream);

#ifdef __cplusplus
}
#endif

#endif /* LMX_SPEC_H */
