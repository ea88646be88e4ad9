// extern "C" entry points of steps with drafted tokens (declared in lmx/spec.h):
// host-side validation, as in abi.hip.
#include <algorithm>

#include "paged_check.hpp"
#include "spec.hpp"

namespace lmx {

lmx_status spec_plan(const lmxs_plan_desc* d, const int32_t* lens, const int32_t* new_rows, int32_t* table, int32_t* held,
                     int32_t* free_pages, int32_t* n_free, int32_t* cu, int32_t* ctx, int64_t* slots, int32_t* pos,
                     hipStream_t st);
lmx_status spec_tree(const lmxp_batch* b, const int32_t* parent, uint32_t words, uint32_t window, int32_t* pos,
                     uint64_t* seen, hipStream_t st);
lmx_status paged_prologue_at(const lmxp_pool* p, const lmxp_batch* b, const lmxp_prologue_desc* d, const lmxs_rope* r,
                             const int32_t* pos, const float* q, const float* k_new, const float* v_new,
                             const float* q_gain, const float* k_gain, const float* factors, void* q_out,
                             lmx_dtype q_out_dt, hipStream_t st);
bool paged_attn_need(const lmxp_pool* p, const lmxp_batch* b, const lmxp_attn_desc* d, bool f32, bool seen, size_t* bytes);
size_t paged_attn_workspace(const lmxp_pool* p, const lmxp_batch* b, const lmxp_attn_desc* d, bool seen);
lmx_status paged_attn_seen(const lmxp_pool* p, const lmxp_batch* b, const lmxp_attn_desc* d, const uint64_t* seen,
                           uint32_t words, const int32_t* pos, const void* q, lmx_dtype dt, void* out, void* ws,
                           hipStream_t st);
size_t spec_verify_workspace(const lmxs_verify_desc* d);
bool spec_verify_fits(const lmxs_verify_desc* d);
lmx_status spec_verify(const lmxs_verify_desc* d, const int32_t* cu, const int32_t* tokens, const int32_t* parent,
                       const void* p, const void* q, lmx_dtype dt, const float* u, const float* r, int32_t* path,
                       int32_t* accepted, int32_t* token, int32_t* lens, void* ws, hipStream_t st);
lmx_status spec_keep(const lmxp_pool* const* pools, uint32_t n_pools, const lmxp_batch* b, const int32_t* path,
                     uint32_t path_stride, const int32_t* accepted, hipStream_t st);

constexpr uint32_t kMostPools = 1024;  // a call to lmxs_keep

// A call's arrays: one that is written may overlap none of the others.
struct Span {
    const void* at;
    uint64_t bytes;
    bool written;
};
template <int N>
static bool apart(const Span (&s)[N]) {
    for (int i = 0; i < N; ++i)
        for (int j = 0; j < i; ++j)
            if ((s[i].written || s[j].written) && s[i].at && s[j].at && s[i].bytes && s[j].bytes &&
                overlap(s[i].at, s[i].bytes, s[j].at, s[j].bytes))
                return false;
    return true;
}
static bool aligned(const void* p, uintptr_t to) { return ((uintptr_t)p & (to - 1)) == 0; }

// What a batch's rows need where no pool is at hand.
static lmx_status check_rows(const lmxp_batch* b) {
    if (!b) return LMX_E_NULL;
    if (!b->cu || !b->ctx_lens) return LMX_E_NULL;
    if (!aligned(b->cu, 4) || !aligned(b->ctx_lens, 4)) return LMX_E_ALIGN;
    if (b->n_seq == 0 || b->n_seq > (1u << 20) || b->n_tokens == 0 || b->n_tokens > (1u << 28)) return LMX_E_SHAPE;
    if (b->max_new == 0 || b->max_new > b->n_tokens) return LMX_E_SHAPE;
    return LMX_OK;
}
// Words of sight that rows of max_new need.
static lmx_status check_words(uint32_t max_new, uint32_t words) {
    return words == 0 || words > LMXS_MAX_ROWS / 64 || max_new > 64 * words ? LMX_E_SHAPE : LMX_OK;
}

static lmx_status check_verify(const lmxs_verify_desc* d) {
    if (!d) return LMX_E_NULL;
    if (d->n_seq == 0 || d->n_seq > (1u << 20) || d->n_tokens == 0 || d->n_tokens > (1u << 28)) return LMX_E_SHAPE;
    if (d->max_new == 0 || d->max_new > LMXS_MAX_ROWS || d->max_new > d->n_tokens) return LMX_E_SHAPE;
    if (d->vocab == 0 || d->vocab > (1u << 24) || d->greedy > 1) return LMX_E_SHAPE;
    if ((d->p_stride && d->p_stride < d->vocab) || (d->q_stride && d->q_stride < d->vocab)) return LMX_E_SHAPE;
    return spec_verify_fits(d) ? LMX_OK : LMX_E_SHAPE;
}

// Whether arrays of pools of one geometry share memory: an array's moves are made in
// order by the threads that own it, so none may reach into another.  Sorted by their
// addresses, some neighbours overlap if any two do.  (36 layers of four arrays 0.6 us;
// each with each, without the scales, 4.)
enum Shared { NONE, WITHIN_A_POOL, BETWEEN_POOLS };
static Shared shared_memory(const lmxp_pool* const* pools, uint32_t n_pools) {
    struct Array {
        uintptr_t at;
        uint32_t pool, scale;
    };
    Array all[4 * kMostPools];
    const lmxp_pool& p = *pools[0];
    const bool i8 = p.store == LMXP_I8;
    const uint64_t slots = (uint64_t)p.n_pages * p.n_kv_heads * p.page_size, bytes = slots * p.head_dim * (i8 ? 1 : 2);
    uint32_t n = 0;
    for (uint32_t i = 0; i < n_pools; ++i) {
        const lmxp_pool& x = *pools[i];
        for (const void* at : {x.k, x.v}) all[n++] = Array{(uintptr_t)at, i, 0};
        if (i8)
            for (const void* at : {x.k_scale, x.v_scale}) all[n++] = Array{(uintptr_t)at, i, 1};
    }
    std::sort(all, all + n, [](const Array& x, const Array& y) { return x.at < y.at; });
    Shared found = NONE;
    for (uint32_t i = 1; i < n; ++i)
        if (all[i].at - all[i - 1].at < (all[i - 1].scale ? 4 * slots : bytes)) {
            if (all[i].pool != all[i - 1].pool) return BETWEEN_POOLS;
            found = WITHIN_A_POOL;
        }
    return found;
}

}  // namespace lmx

using namespace lmx;

extern "C" {

lmx_status lmxs_plan(const lmxs_plan_desc* d, const int32_t* lens, const int32_t* new_rows, int32_t* page_table,
                     int32_t* held, int32_t* free_pages, int32_t* n_free, int32_t* cu, int32_t* ctx_lens,
                     int64_t* slots, int32_t* pos, lmx_stream stream) {
    if (!d || !lens || !new_rows || !page_table || !held || !free_pages || !n_free || !cu || !ctx_lens) return LMX_E_NULL;
    const uint32_t ps = d->page_size;
    if (ps != 16 && ps != 32 && ps != 64 && ps != 128 && ps != 256) return LMX_E_UNSUPPORTED;
    if (d->n_seq == 0 || d->n_seq > (1u << 20) || d->n_tokens == 0 || d->n_tokens > (1u << 28)) return LMX_E_SHAPE;
    if (d->table_stride == 0 || d->n_pages == 0 || d->n_pages >= (1u << 30) || d->trim > 1) return LMX_E_SHAPE;
    // entries are gone through by one workgroup
    if ((uint64_t)d->n_seq * d->table_stride > (1u << 28)) return LMX_E_SHAPE;
    for (const void* x : {(const void*)lens, (const void*)new_rows, (const void*)page_table, (const void*)held,
                          (const void*)free_pages, (const void*)n_free, (const void*)cu, (const void*)ctx_lens, (const void*)pos})
        if (!aligned(x, 4)) return LMX_E_ALIGN;
    if (!aligned(slots, 8)) return LMX_E_ALIGN;
    const uint64_t n = 4ull * d->n_seq, t = d->n_tokens;
    const Span all[] = {{lens, n, false}, {new_rows, n, false}, {page_table, n * d->table_stride, true}, {held, n, true},
                        {free_pages, 4ull * d->n_pages, true}, {n_free, 8, true}, {cu, n + 4, true}, {ctx_lens, n, true},
                        {slots, 8 * t, true}, {pos, 4 * t, true}};
    if (!apart(all)) return LMX_E_SHAPE;
    return spec_plan(d, lens, new_rows, page_table, held, free_pages, n_free, cu, ctx_lens, slots, pos,
                     (hipStream_t)stream);
}

lmx_status lmxs_tree(const lmxp_batch* b, const int32_t* parent, uint32_t words, uint32_t window, int32_t* pos,
                     uint64_t* seen, lmx_stream stream) {
    lmx_status s = check_rows(b);
    if (s != LMX_OK) return s;
    if (!parent || (!pos && !seen)) return LMX_E_NULL;
    if ((s = check_words(b->max_new, words)) != LMX_OK) return s;
    if (window >= (1u << 30)) return LMX_E_SHAPE;
    if (!aligned(parent, 4) || !aligned(pos, 4) || !aligned(seen, 8)) return LMX_E_ALIGN;
    const uint64_t t = b->n_tokens, n = 4ull * b->n_seq;
    const Span all[] = {{b->cu, n + 4, false}, {b->ctx_lens, n, false}, {parent, 4 * t, false}, {pos, 4 * t, true},
                        {seen, 8 * t * words, true}};
    if (!apart(all)) return LMX_E_SHAPE;
    return spec_tree(b, parent, words, window, pos, seen, (hipStream_t)stream);
}

lmx_status lmxs_prologue(const lmxp_pool* p, const lmxp_batch* b, const lmxp_prologue_desc* d, const lmxs_rope* r,
                         const int32_t* pos, const float* q, const float* k_new, const float* v_new, const float* q_gain,
                         const float* k_gain, const float* rope_factors, void* q_out, lmx_dtype q_out_dt,
                         lmx_stream stream) {
    const lmx_status s = check_prologue(p, b, d, q, k_new, v_new, q_gain, k_gain, rope_factors, q_out, q_out_dt);
    if (s != LMX_OK) return s;
    if (!r) return LMX_E_NULL;
    if (r->interleaved > 1 || !std::isfinite(r->turn_scale)) return LMX_E_SHAPE;
    if (!aligned(pos, 4)) return LMX_E_ALIGN;
    const uint64_t out = (uint64_t)b->n_tokens * d->n_heads * p->head_dim * (q_out_dt == LMX_F32 ? 4 : 2);
    if (pos && overlap(pos, 4ull * b->n_tokens, q_out, out)) return LMX_E_SHAPE;
    return paged_prologue_at(p, b, d, r, pos, q, k_new, v_new, q_gain, k_gain, rope_factors, q_out, q_out_dt,
                             (hipStream_t)stream);
}

size_t lmxs_attn_workspace_bytes(const lmxp_pool* p, const lmxp_batch* b, const lmxp_attn_desc* d) {
    QLayout l;
    return check_attn(p, b, d, &l) == LMX_OK && b->max_new <= LMXS_MAX_ROWS ? paged_attn_workspace(p, b, d, true) : 0;
}

lmx_status lmxs_attn(const lmxp_pool* p, const lmxp_batch* b, const lmxp_attn_desc* d, const uint64_t* seen,
                     uint32_t words, const int32_t* pos, const void* q, lmx_dtype dt, void* out, void* ws,
                     size_t ws_bytes, lmx_stream stream) {
    lmx_status s = check_attn_call(p, b, d, q, dt, out);
    if (s != LMX_OK) return s;
    if (!seen || (d->window && !pos)) return LMX_E_NULL;
    if ((s = check_words(b->max_new, words)) != LMX_OK) return s;
    if (!aligned(seen, 8) || !aligned(pos, 4)) return LMX_E_ALIGN;
    const uint64_t bytes = (uint64_t)b->n_tokens * d->n_heads * p->head_dim * (dt == LMX_F32 ? 4 : 2);
    if (overlap(seen, 8ull * b->n_tokens * words, out, bytes)) return LMX_E_SHAPE;
    if (pos && overlap(pos, 4ull * b->n_tokens, out, bytes)) return LMX_E_SHAPE;
    size_t need;
    if (!paged_attn_need(p, b, d, dt == LMX_F32, true, &need)) return LMX_E_SHAPE;
    if (need && (!ws || ws_bytes < need)) return LMX_E_WORKSPACE;
    if (need && !at16(ws)) return LMX_E_ALIGN;
    return paged_attn_seen(p, b, d, seen, words, pos, q, dt, out, ws, (hipStream_t)stream);
}

size_t lmxs_verify_workspace_bytes(const lmxs_verify_desc* d) {
    return check_verify(d) == LMX_OK ? spec_verify_workspace(d) : 0;
}

lmx_status lmxs_verify(const lmxs_verify_desc* d, const int32_t* cu, const int32_t* tokens, const int32_t* parent,
                       const void* p, const void* q, lmx_dtype dt, const float* u, const float* r, int32_t* path,
                       int32_t* accepted, int32_t* token, int32_t* lens, void* ws, size_t ws_bytes, lmx_stream stream) {
    const lmx_status s = check_verify(d);
    if (s != LMX_OK) return s;
    if (!cu || !tokens || !p || !path || !accepted || !token) return LMX_E_NULL;
    if (!d->greedy && (!u || !r)) return LMX_E_NULL;
    if (dt != LMX_F32 && dt != LMX_F16) return LMX_E_UNSUPPORTED;
    const uintptr_t es = dt == LMX_F32 ? 4 : 2;
    if (!aligned(p, es) || !aligned(q, es)) return LMX_E_ALIGN;
    for (const void* x : {(const void*)cu, (const void*)tokens, (const void*)parent, (const void*)u, (const void*)r,
                          (const void*)path, (const void*)accepted, (const void*)token, (const void*)lens})
        if (!aligned(x, 4)) return LMX_E_ALIGN;
    const size_t need = spec_verify_workspace(d);
    if (need && (!ws || ws_bytes < need)) return LMX_E_WORKSPACE;
    if (need && !at16(ws)) return LMX_E_ALIGN;
    const uint64_t n = 4ull * d->n_seq, t = 4ull * d->n_tokens;
    auto rows = [&](uint32_t stride) { return ((uint64_t)(d->n_tokens - 1) * (stride ? stride : d->vocab) + d->vocab) * es; };
    const Span all[] = {{cu, n + 4, false}, {tokens, t, false}, {parent, t, false}, {p, rows(d->p_stride), false},
                        {d->greedy ? nullptr : q, rows(d->q_stride), false}, {d->greedy ? nullptr : u, t, false},
                        {d->greedy ? nullptr : r, n, false}, {path, n * d->max_new, true}, {accepted, n, true},
                        {token, n, true}, {lens, n, true}, {need ? ws : nullptr, need, true}};
    if (!apart(all)) return LMX_E_SHAPE;
    return spec_verify(d, cu, tokens, parent, p, d->greedy ? nullptr : q, dt, u, r, path, accepted, token, lens, ws,
                       (hipStream_t)stream);
}

lmx_status lmxs_keep(const lmxp_pool* const* pools, uint32_t n_pools, const lmxp_batch* b, const int32_t* path,
                     uint32_t path_stride, const int32_t* accepted, lmx_stream stream) {
    if (!pools) return LMX_E_NULL;
    if (n_pools == 0 || n_pools > kMostPools) return LMX_E_SHAPE;
    for (uint32_t i = 0; i < n_pools; ++i) {
        const lmx_status s = check_pool(pools[i]);
        if (s != LMX_OK) return s;
        const lmxp_pool &x = *pools[i], &y = *pools[0];
        if (x.n_pages != y.n_pages || x.page_size != y.page_size || x.store != y.store || x.n_kv_heads != y.n_kv_heads ||
            x.head_dim != y.head_dim)
            return LMX_E_SHAPE;
    }
    const lmxp_pool* const p = pools[0];
    const lmx_status s = check_batch(p, b);
    if (s != LMX_OK) return s;
    const Shared shared = shared_memory(pools, n_pools);
    if (shared == BETWEEN_POOLS) return LMX_E_SHAPE;
    if (!path || !accepted) return LMX_E_NULL;
    if (b->max_new > LMXS_MAX_ROWS || path_stride < b->max_new || path_stride >= (1u << 30)) return LMX_E_SHAPE;
    if (!aligned(path, 4) || !aligned(accepted, 4)) return LMX_E_ALIGN;
    if (shared != NONE) return LMX_E_SHAPE;
    // pieces of 16 bytes of K and elements of V, 256 a workgroup, and 64 layers a launch at most
    const uint64_t pieces = (uint64_t)p->n_kv_heads * (p->head_dim + p->head_dim / 8 + 2);
    if ((uint64_t)b->n_seq * ((pieces + 255) / 256) * 64 >= (1u << 24)) return LMX_E_SHAPE;
    return spec_keep(pools, n_pools, b, path, path_stride, accepted, (hipStream_t)stream);
}

}  // extern "C"
