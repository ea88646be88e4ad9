/*
 * lmx/paged.h -- the paged KV cache of libllmoxide_amd.so: its write (f16 or
 * 8-bit), its read-back, the attention prologue in front of it and the
 * attention over it.  The conventions are lmx/attn.h's: plain C types,
 * caller-owned device memory, work enqueued on `stream`, nothing allocated or
 * synchronized, arguments validated on the host before anything is enqueued,
 * lmx_status results.  The reference keeps one contiguous cache per session
 * (cache.rs:65-154) and serves one sequence (docs/limitations.md:21); these
 * entry points have no counterpart there beyond what each one names.
 *
 * Pool.  A page holds page_size consecutive positions of one sequence, for
 * every kv head:
 *     k [n_pages, n_kv_heads, page_size, head_dim]
 *     v [n_pages, n_kv_heads, head_dim, page_size]      (V is kept transposed)
 * f16, or int8 with one f32 scale per position and head,
 *     k_scale, v_scale [n_pages, n_kv_heads, page_size];  value = int * scale.
 * head_dim: 64, 128, 256 or 512.  page_size: 16, 32, 64, 128 or 256.
 *
 * Batch.  Sequence b of n_seq brings rows cu[b] .. cu[b+1]-1 of the batch's
 * n_tokens rows: its last cu[b+1]-cu[b] positions of ctx_lens[b] (the lengths
 * count the new rows).  Position p of it lives in page
 * page_table[b*table_stride + p / page_size], slot p % page_size.
 *   cu          int32 [n_seq+1], rising from >= 0; rows outside [cu[0],
 *               cu[n_seq]) belong to no sequence: nothing is read or written
 *               for them.  Two equal entries: a sequence without new rows.
 *   ctx_lens    int32 [n_seq], each at most max_ctx and at least its new rows
 *   max_new     at least the largest number of new rows of a sequence
 *   max_ctx     at most table_stride * page_size
 * A call whose work would take 2^24 workgroups or more (some 10^8 row heads) is
 * refused with LMX_E_SHAPE.
 * cu, ctx_lens and page_table are read on the device, so a captured graph
 * replays with the lengths that they hold then.  A position whose table entry
 * is not in [0, n_pages) is in no page: it is not stored, reads back as 0 and
 * no query sees it (which is how pages behind a window are let go).  Lengths
 * and tables that break the rules above give unspecified results for the
 * sequences that they belong to, but no access outside the buffers.  Several
 * sequences may share pages; a position that one call writes must be in one
 * sequence's pages only.  A call's other tensors do not overlap the pool.
 *
 * An 8-bit row head x is stored as scale = amax(|x|) / 127, rounded to f32,
 * and int = x / scale rounded to the nearest, ties to even, from the exact
 * quotient.  amax below 2^-100 stores scale 0 and zeros.  A head that holds an
 * infinity or a NaN stores scale NaN (all of it reads back as NaN).
 */
#ifndef LMX_PAGED_H
#define LMX_PAGED_H

#include "lmx/attn.h"

#ifdef __cplusplus
extern "C" {
#endif

/* What a pool holds. */
typedef enum { LMXP_F16 = 1, LMXP_I8 = 2 } lmxp_store;

typedef struct {
    uint32_t n_pages;
    uint32_t page_size;   /* positions a page: 16, 32, 64, 128 or 256         */
    uint32_t n_kv_heads;
    uint32_t head_dim;    /* 64, 128, 256 or 512                              */
    uint32_t store;       /* lmxp_store                                       */
    void *k;              /* 16-byte aligned, as all pool buffers             */
    void *v;
    float *k_scale;       /* LMXP_I8; NULL for LMXP_F16                       */
    float *v_scale;
} lmxp_pool;

typedef struct {
    uint32_t n_seq;
    uint32_t n_tokens;    /* rows of the batch's tensors                      */
    uint32_t max_new;     /* most new rows of one sequence                    */
    uint32_t max_ctx;     /* longest sequence, its new rows included          */
    uint32_t table_stride;/* page-table entries per sequence                  */
    const int32_t *cu;         /* device [n_seq + 1]                          */
    const int32_t *ctx_lens;   /* device [n_seq]                              */
    const int32_t *page_table; /* device [n_seq, table_stride]                */
} lmxp_batch;

/* ------------------------------------------------------------------------
 * Write the batch's K and V rows into the pages (the paged, ragged form of
 * lmx_kv_append; f16 rounds to nearest even).  Row i, head h starts at
 * k_new + i*row_stride + h*head_dim (likewise v_new).
 *   src_dt      LMX_F32 or LMX_F16
 *   row_stride  elements between rows (0: n_kv_heads*head_dim); a multiple of
 *               4, so rows can be columns of a fused projection.  The rows are
 *               16-byte (f32) or 8-byte (f16) aligned.
 * Either of k_new / v_new may be NULL to write only the other. */
lmx_status lmxp_append(const lmxp_pool *p, const lmxp_batch *b, const void *k_new,
                       const void *v_new, lmx_dtype src_dt, uint32_t row_stride,
                       lmx_stream stream);

/* ------------------------------------------------------------------------
 * Read the batch's rows back from the pages: the inverse of lmxp_append for
 * the same batch.  (To read positions [a, e) of a sequence, give it e - a rows
 * and length e.)  k_out, v_out [n_tokens, row_stride] of out_dt (LMX_F32 or
 * LMX_F16; an 8-bit value is int * scale rounded to f32, and for LMX_F16 that to
 * f16, which is one place off the nearest f16 once in some 17000); row_stride and
 * alignment as for lmxp_append.  Rows of positions in no page are written as
 * zeros.  Either output may be NULL. */
lmx_status lmxp_read(const lmxp_pool *p, const lmxp_batch *b, void *k_out, void *v_out,
                     lmx_dtype out_dt, uint32_t row_stride, lmx_stream stream);

/* ------------------------------------------------------------------------
 * Attention prologue over pages: lmx_attn_prologue's steps for a ragged batch
 * (per-head RMS norm with gain, NeoX rotation of the first n_rot dims at the
 * row's position, optional V norm), K and V stored as lmxp_append stores them.
 *   q        f32, head h of row i at q + i*q_row_stride + h*q_head_stride
 *   q_out    [n_tokens, n_heads, head_dim] of q_out_dt (LMX_F32 or LMX_F16),
 *            contiguous.  It may be q itself where q is contiguous and
 *            q_out_dt is LMX_F32; any other overlap is refused.
 *   k_new, v_new   f32, kv_row_stride floats between rows
 *   q_gain, k_gain, rope_factors   as lmx_attn_prologue's; each may be NULL
 * Strides are in elements and multiples of 4, buffers 16-byte aligned.
 * n_rot even, <= head_dim. */
typedef struct {
    uint32_t n_heads;
    uint32_t n_rot;
    uint32_t v_norm;         /* 1: RMS-normalize V per head                    */
    uint32_t q_head_stride;  /* 0: head_dim                                   */
    uint32_t q_row_stride;   /* 0: n_heads * q_head_stride                    */
    uint32_t kv_row_stride;  /* 0: n_kv_heads * head_dim                      */
    float rms_eps;
    float rope_base;
} lmxp_prologue_desc;

lmx_status lmxp_prologue(const lmxp_pool *p, const lmxp_batch *b, const lmxp_prologue_desc *d,
                         const float *q, const float *k_new, const float *v_new,
                         const float *q_gain, const float *k_gain, const float *rope_factors,
                         void *q_out, lmx_dtype q_out_dt, lmx_stream stream);

/* ------------------------------------------------------------------------
 * Attention of the batch's rows over the pages (lmx_attn_fwd's formula, causal,
 * for a ragged batch of chunks and single tokens):
 *   out[i,h,:] = sum_p softmax_p(scale * q[i,h,:] . K[p, h/G, :]) V[p, h/G, :]
 * over the positions p of row i's sequence with
 *   (window ? max(0, pos-window+1) : 0) <= p <= pos
 * that are in a page, pos being the row's position.  The batch's own rows are
 * read from the pages: append them first.  A row that sees no position, or
 * whose every score is -infinity, gets zeros.  What a row does not see has no
 * part in its result, infinities and NaN included.  An 8-bit V scale below
 * 2^-90 (values below 1e-25) is taken as 2^-90; beside one above 2^100 (values
 * above 1e32) keys of far smaller scales may lose their part of the softmax.
 *   dt   LMX_F16: q and out are f16, the sums fp32.  The weights p are rounded
 *        to f16 (11 bits) before they meet V in sequences that bring many rows
 *        (n_heads / n_kv_heads times its new rows above 32 to 128, by head_dim
 *        and store; any number, where n_seq is 1 and max_new allows that many)
 *        and carried as two f16 parts (22 bits) in the others.
 *        A result is off by some 2.8e-4 of itself in the former and 2.1e-4 in
 *        the latter (root mean square), its own rounding to f16 included.
 *        LMX_F32: q and out are f32; q and p are carried as two f16 parts each
 *        (22 bits; an element of q below 2^-39 of its row's largest counts as
 *        0) whatever the lengths.
 *   q    head h of row i at q + i*q_row_stride + h*q_head_stride (elements,
 *        multiples of 8; 0: contiguous); 16-byte aligned
 *   out  [n_tokens, n_heads, head_dim] contiguous, 16-byte aligned, not
 *        overlapping q (LMX_E_SHAPE)
 * n_heads: a multiple of n_kv_heads.  The workspace (16-byte aligned) holds
 * partial results where a key range is split; every byte read from it was
 * written by the same call.  A call that needs more than ws_bytes is refused
 * with LMX_E_WORKSPACE; what one needs does not rise with its batch (only batches
 * that leave compute units idle are split, so a long prompt needs less than a
 * short chunk), which is why lmxp_attn_workspace_bytes answers for smaller ones
 * too.  Calls that overlap in time (two streams, two replayed graphs) need one
 * each. */
typedef struct {
    uint32_t n_heads;
    uint32_t window;         /* 0: every earlier position                     */
    uint32_t q_head_stride;  /* 0: head_dim                                   */
    uint32_t q_row_stride;   /* 0: n_heads * q_head_stride                    */
    float scale;
} lmxp_attn_desc;

/* Bytes that serve lmxp_attn with this pool and these n_heads on this batch and
 * on every one whose n_seq, n_tokens, max_new and max_ctx are at most its own,
 * for either dt and any window (0 for a description that lmxp_attn refuses). */
size_t lmxp_attn_workspace_bytes(const lmxp_pool *p, const lmxp_batch *b, const lmxp_attn_desc *d);

lmx_status lmxp_attn(const lmxp_pool *p, const lmxp_batch *b, const lmxp_attn_desc *d,
                     const void *q, lmx_dtype dt, void *out, void *ws, size_t ws_bytes,
                     lmx_stream stream);

#ifdef __cplusplus
}
#endif

#endif /* LMX_PAGED_H */
