// Host-side validation that the paged entry points share.
#pragma once

#include <cmath>

#include "paged.hpp"

namespace lmx {

inline bool at16(const void* p) { return ((uintptr_t)p & 15) == 0; }
inline bool overlap(const void* a, uint64_t na, const void* b, uint64_t nb) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return x < y + nb && y < x + na;
}
// Bytes from a tensor's first element to behind its last: `rows` rows a
// row_stride apart, `heads` heads a head_stride apart, hd elements.
inline uint64_t extent(uint64_t rows, uint64_t row_stride, uint64_t heads, uint64_t head_stride, uint64_t hd,
                       uint64_t es) {
    return ((rows - 1) * row_stride + (heads - 1) * head_stride + hd) * es;
}

inline lmx_status check_pool(const lmxp_pool* p) {
    if (!p) return LMX_E_NULL;
    if (p->store != LMXP_F16 && p->store != LMXP_I8) return LMX_E_UNSUPPORTED;
    if (p->head_dim != 64 && p->head_dim != 128 && p->head_dim != 256 && p->head_dim != 512) return LMX_E_UNSUPPORTED;
    const uint32_t ps = p->page_size;
    if (ps != 16 && ps != 32 && ps != 64 && ps != 128 && ps != 256) return LMX_E_UNSUPPORTED;
    if (p->n_kv_heads == 0 || p->n_kv_heads > 4096 || p->n_pages == 0 || p->n_pages > (1u << 30)) return LMX_E_SHAPE;
    if (!p->k || !p->v) return LMX_E_NULL;
    if (!at16(p->k) || !at16(p->v)) return LMX_E_ALIGN;
    if (p->store == LMXP_I8) {
        if (!p->k_scale || !p->v_scale) return LMX_E_NULL;
        if (!at16(p->k_scale) || !at16(p->v_scale)) return LMX_E_ALIGN;
    }
    return LMX_OK;
}

inline lmx_status check_batch(const lmxp_pool* p, const lmxp_batch* b) {
    if (!b) return LMX_E_NULL;
    if (!b->cu || !b->ctx_lens || !b->page_table) return LMX_E_NULL;
    for (const void* x : {(const void*)b->cu, (const void*)b->ctx_lens, (const void*)b->page_table})
        if ((uintptr_t)x & 3) return LMX_E_ALIGN;
    if (b->n_seq == 0 || b->n_seq > (1u << 20) || b->n_tokens == 0 || b->n_tokens > (1u << 28)) return LMX_E_SHAPE;
    if (b->max_new == 0 || b->max_new > b->n_tokens || b->max_ctx == 0 || b->table_stride == 0) return LMX_E_SHAPE;
    if (b->max_ctx >= (1u << 30) || b->table_stride >= (1u << 30)) return LMX_E_CONTEXT;
    if ((uint64_t)b->max_ctx > (uint64_t)b->table_stride * p->page_size) return LMX_E_CONTEXT;
    return LMX_OK;
}

// row_stride of rows of n_kv_heads heads: 0 or at least a row, a multiple of 4.
inline lmx_status check_kv_rows(const lmxp_pool* p, uint32_t row_stride) {
    if (row_stride && (row_stride < p->n_kv_heads * p->head_dim || row_stride % 4)) return LMX_E_SHAPE;
    return LMX_OK;
}

struct QLayout {
    uint64_t head, row;
};
inline lmx_status check_q(uint32_t n_heads, uint32_t hd, uint32_t head_stride, uint32_t row_stride, uint32_t mult,
                          QLayout* l) {
    if (n_heads == 0 || n_heads > 65536) return LMX_E_SHAPE;
    l->head = head_stride ? head_stride : hd;
    l->row = row_stride ? row_stride : l->head * n_heads;
    if (l->head < hd || l->head % mult || l->row % mult) return LMX_E_SHAPE;
    if (l->row < (n_heads - 1) * l->head + hd) return LMX_E_SHAPE;
    return LMX_OK;
}

inline lmx_status check_attn(const lmxp_pool* p, const lmxp_batch* b, const lmxp_attn_desc* d, QLayout* l) {
    lmx_status s = check_pool(p);
    if (s != LMX_OK) return s;
    s = check_batch(p, b);
    if (s != LMX_OK) return s;
    if (!d) return LMX_E_NULL;
    s = check_q(d->n_heads, p->head_dim, d->q_head_stride, d->q_row_stride, 8, l);
    if (s != LMX_OK) return s;
    if (d->n_heads % p->n_kv_heads) return LMX_E_SHAPE;
    if (!std::isfinite(d->scale)) return LMX_E_SHAPE;
    if (d->window >= (1u << 30)) return LMX_E_SHAPE;
    // query rows of a sequence, and work items, are counted in 32 bits
    if ((uint64_t)b->n_tokens * d->n_heads >= (1ull << 30)) return LMX_E_SHAPE;
    if ((uint64_t)b->max_new * d->n_heads * b->n_seq >= (1ull << 31)) return LMX_E_SHAPE;
    return LMX_OK;
}

// A prologue's arguments.
inline lmx_status check_prologue(const lmxp_pool* p, const lmxp_batch* b, const lmxp_prologue_desc* d, const float* q,
                                 const float* k_new, const float* v_new, const float* q_gain, const float* k_gain,
                                 const float* rope_factors, const void* q_out, lmx_dtype q_out_dt) {
    lmx_status s = check_pool(p);
    if (s != LMX_OK) return s;
    if ((s = check_batch(p, b)) != LMX_OK) return s;
    if (!d || !q || !k_new || !v_new || !q_out) return LMX_E_NULL;
    if (q_out_dt != LMX_F32 && q_out_dt != LMX_F16) return LMX_E_UNSUPPORTED;
    QLayout l;
    if ((s = check_q(d->n_heads, p->head_dim, d->q_head_stride, d->q_row_stride, 4, &l)) != LMX_OK) return s;
    if ((s = check_kv_rows(p, d->kv_row_stride)) != LMX_OK) return s;
    if (d->n_rot > p->head_dim || d->n_rot % 2 || d->v_norm > 1) return LMX_E_SHAPE;
    if (!std::isfinite(d->rms_eps) || d->rms_eps < 0.f) return LMX_E_SHAPE;
    if (d->n_rot && !(d->rope_base > 0.f && std::isfinite(d->rope_base))) return LMX_E_SHAPE;
    for (const void* x : {(const void*)q, (const void*)k_new, (const void*)v_new, (const void*)q_gain,
                          (const void*)k_gain, (const void*)q_out})
        if (!at16(x)) return LMX_E_ALIGN;
    if ((uintptr_t)rope_factors & 3) return LMX_E_ALIGN;
    // q_out beside q, or exactly q: a row that is written is read by the same lanes first
    const uint64_t es = q_out_dt == LMX_F32 ? 4 : 2, dense = (uint64_t)d->n_heads * p->head_dim;
    const bool in_place = q_out == (const void*)q && es == 4 && l.head == p->head_dim && l.row == dense;
    if (!in_place && overlap(q, extent(b->n_tokens, l.row, d->n_heads, l.head, p->head_dim, 4), q_out,
                             b->n_tokens * dense * es))
        return LMX_E_SHAPE;
    // k_new and v_new are read while q_out is written
    const uint64_t kv_row = d->kv_row_stride ? d->kv_row_stride : (uint64_t)p->n_kv_heads * p->head_dim;
    const uint64_t kv_bytes = extent(b->n_tokens, kv_row, p->n_kv_heads, p->head_dim, p->head_dim, 4);
    for (const void* x : {(const void*)k_new, (const void*)v_new})
        if (overlap(x, kv_bytes, q_out, b->n_tokens * dense * es)) return LMX_E_SHAPE;
    return LMX_OK;
}

// An attention call's arguments but for the workspace.
inline lmx_status check_attn_call(const lmxp_pool* p, const lmxp_batch* b, const lmxp_attn_desc* d, const void* q,
                                  lmx_dtype dt, const void* out) {
    QLayout l;
    lmx_status s = check_attn(p, b, d, &l);
    if (s != LMX_OK) return s;
    if (!q || !out) return LMX_E_NULL;
    if (dt != LMX_F32 && dt != LMX_F16) return LMX_E_UNSUPPORTED;
    if (!at16(q) || !at16(out)) return LMX_E_ALIGN;
    const uint64_t es = dt == LMX_F32 ? 4 : 2;
    if (overlap(q, extent(b->n_tokens, l.row, d->n_heads, l.head, p->head_dim, es), out,
                (uint64_t)b->n_tokens * d->n_heads * p->head_dim * es))
        return LMX_E_SHAPE;
    return LMX_OK;
}

}  // namespace lmx
