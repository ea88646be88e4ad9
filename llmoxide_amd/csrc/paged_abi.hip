// extern "C" entry points of the paged KV cache (declared in lmx/paged.h):
// host-side validation, as in abi.hip.
#include "paged_check.hpp"

namespace lmx {

lmx_status paged_append(const lmxp_pool* p, const lmxp_batch* b, const void* k_new, const void* v_new,
                        lmx_dtype src_dt, uint32_t row_stride, hipStream_t st);
lmx_status paged_read(const lmxp_pool* p, const lmxp_batch* b, void* k_out, void* v_out, lmx_dtype out_dt,
                      uint32_t row_stride, hipStream_t st);
lmx_status paged_prologue(const lmxp_pool* p, const lmxp_batch* b, const lmxp_prologue_desc* d, const float* q,
                          const float* k_new, const float* v_new, const float* q_gain, const float* k_gain,
                          const float* factors, void* q_out, lmx_dtype q_out_dt, hipStream_t st);
size_t paged_attn_workspace(const lmxp_pool* p, const lmxp_batch* b, const lmxp_attn_desc* d, bool seen);
bool paged_attn_need(const lmxp_pool* p, const lmxp_batch* b, const lmxp_attn_desc* d, bool f32, bool seen, size_t* bytes);
lmx_status paged_attn(const lmxp_pool* p, const lmxp_batch* b, const lmxp_attn_desc* d, const void* q, lmx_dtype dt,
                      void* out, void* ws, hipStream_t st);

static int log2_of(uint32_t x) {
    int l = 0;
    while ((1u << l) < x) ++l;
    return l;
}

PagedArgs paged_args(const lmxp_pool* p, const lmxp_batch* b) {
    PagedArgs a{};
    a.g.n_seq = (int)b->n_seq;
    a.g.n_tokens = (int)b->n_tokens;
    a.g.max_new = (int)b->max_new;
    a.g.max_ctx = (int)b->max_ctx;
    a.g.table_stride = (int)b->table_stride;
    a.g.n_pages = (int)p->n_pages;
    a.g.ps_log2 = log2_of(p->page_size);
    a.g.Hkv = (int)p->n_kv_heads;
    a.g.G = 1;
    a.hd = (int)p->head_dim;
    a.k = static_cast<char*>(p->k);
    a.v = static_cast<char*>(p->v);
    a.k_scale = p->k_scale;
    a.v_scale = p->v_scale;
    a.cu = b->cu;
    a.ctx = b->ctx_lens;
    a.table = b->page_table;
    return a;
}

}  // namespace lmx

using namespace lmx;

extern "C" {

lmx_status lmxp_append(const lmxp_pool* p, const lmxp_batch* b, const void* k_new, const void* v_new,
                       lmx_dtype src_dt, uint32_t row_stride, lmx_stream stream) {
    lmx_status s = check_pool(p);
    if (s != LMX_OK) return s;
    if ((s = check_batch(p, b)) != LMX_OK) return s;
    if (!k_new && !v_new) return LMX_E_NULL;
    if (src_dt != LMX_F32 && src_dt != LMX_F16) return LMX_E_UNSUPPORTED;
    if ((s = check_kv_rows(p, row_stride)) != LMX_OK) return s;
    const uintptr_t mask = src_dt == LMX_F32 ? 15 : 7;
    if (((uintptr_t)k_new & mask) || ((uintptr_t)v_new & mask)) return LMX_E_ALIGN;
    return paged_append(p, b, k_new, v_new, src_dt, row_stride, (hipStream_t)stream);
}

lmx_status lmxp_read(const lmxp_pool* p, const lmxp_batch* b, void* k_out, void* v_out, lmx_dtype out_dt,
                     uint32_t row_stride, lmx_stream stream) {
    lmx_status s = check_pool(p);
    if (s != LMX_OK) return s;
    if ((s = check_batch(p, b)) != LMX_OK) return s;
    if (!k_out && !v_out) return LMX_E_NULL;
    if (out_dt != LMX_F32 && out_dt != LMX_F16) return LMX_E_UNSUPPORTED;
    if ((s = check_kv_rows(p, row_stride)) != LMX_OK) return s;
    const uintptr_t mask = out_dt == LMX_F32 ? 15 : 7;
    if (((uintptr_t)k_out & mask) || ((uintptr_t)v_out & mask)) return LMX_E_ALIGN;
    return paged_read(p, b, k_out, v_out, out_dt, row_stride, (hipStream_t)stream);
}

lmx_status lmxp_prologue(const lmxp_pool* p, const lmxp_batch* b, const lmxp_prologue_desc* d, const float* q,
                         const float* k_new, const float* v_new, const float* q_gain, const float* k_gain,
                         const float* rope_factors, void* q_out, lmx_dtype q_out_dt, lmx_stream stream) {
    const lmx_status s = check_prologue(p, b, d, q, k_new, v_new, q_gain, k_gain, rope_factors, q_out, q_out_dt);
    if (s != LMX_OK) return s;
    return paged_prologue(p, b, d, q, k_new, v_new, q_gain, k_gain, rope_factors, q_out, q_out_dt,
                          (hipStream_t)stream);
}

size_t lmxp_attn_workspace_bytes(const lmxp_pool* p, const lmxp_batch* b, const lmxp_attn_desc* d) {
    QLayout l;
    return check_attn(p, b, d, &l) == LMX_OK ? paged_attn_workspace(p, b, d, false) : 0;
}

lmx_status lmxp_attn(const lmxp_pool* p, const lmxp_batch* b, const lmxp_attn_desc* d, const void* q, lmx_dtype dt,
                     void* out, void* ws, size_t ws_bytes, lmx_stream stream) {
    lmx_status s = check_attn_call(p, b, d, q, dt, out);
    if (s != LMX_OK) return s;
    size_t need;
    if (!paged_attn_need(p, b, d, dt == LMX_F32, false, &need)) return LMX_E_SHAPE;
    if (need && (!ws || ws_bytes < need)) return LMX_E_WORKSPACE;
    if (need && !at16(ws)) return LMX_E_ALIGN;
    return paged_attn(p, b, d, q, dt, out, ws, (hipStream_t)stream);
}

}  // extern "C"
