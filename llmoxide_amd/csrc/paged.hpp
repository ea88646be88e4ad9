// Device-side view of a paged pool and batch, and the lookups the kernels share.
#pragma once

#include "common.hpp"
#include "lmx/paged.h"
#include "paged_index.hpp"

namespace lmx {

struct PagedArgs {
    PagedGeom g;
    int hd;
    char* k;
    char* v;
    float* k_scale;
    float* v_scale;
    const int32_t* cu;
    const int32_t* ctx;
    const int32_t* table;
};

// Host: the kernels' view of a validated pool and batch (paged_abi.hip).
PagedArgs paged_args(const lmxp_pool* p, const lmxp_batch* b);

// Where one row of the batch lives.
struct RowPlace {
    int page;  // -1: in no page, or the row belongs to no sequence
    int slot;
    int pos;
    bool owned;  // belongs to a sequence
};

// The place of row `row` (a value of the lane's own; rows first .. last are
// the wave's).  All lanes take part.  A sequence's index is the number of
// ends cu[b+1] at or below the row: 64 ends at a time sit one in a lane, ends
// at or below `first` count for every lane, and the others are searched by
// halves among the lanes.
__device__ __forceinline__ RowPlace locate_row(const PagedArgs& a, int row, int first, int last) {
    const int lane = __lane_id();
    int seq = 0;
    for (int c0 = 0; c0 < a.g.n_seq; c0 += 64) {
        const int b = c0 + lane;
        const int end = b < a.g.n_seq ? a.cu[b + 1] : 0x7fffffff;
        const uint64_t below = __ballot(end <= first), upto = __ballot(end <= last);
        if (below == upto) {
            seq += __popcll(below);
        } else {
            int at = 0;
#pragma unroll
            for (int step = 32; step > 0; step >>= 1)
                at += __shfl(end, at + step - 1, 64) <= row ? step : 0;
            at += __shfl(end, at, 64) <= row ? 1 : 0;
            seq += at;
        }
        if (upto != ~0ull) break;
    }
    RowPlace p{-1, 0, 0, false};
    if (seq >= a.g.n_seq || row >= a.g.n_tokens) return p;
    const int cu0 = a.cu[seq], cu1 = a.cu[seq + 1];
    const PagedSeq s = paged_seq(a.g, cu0, cu1, a.ctx[seq]);
    if (row < s.row0 || row >= s.row0 + s.n) return p;
    p.owned = true;
    p.pos = s.ctx - s.n + (row - s.row0);
    const int e = p.pos < s.ctx ? paged_entry(a.g, p.pos) : -1;
    if (e < 0) return p;
    p.page = paged_page(a.g, a.table[(size_t)seq * a.g.table_stride + e]);
    p.slot = p.pos & ((1 << a.g.ps_log2) - 1);
    return p;
}

// Offset in elements of (page, head, slot)'s K row, of its V column's first
// element, and of its scale.
__device__ __forceinline__ size_t k_offset(const PagedArgs& a, int page, int head, int slot) {
    return ((((size_t)page * a.g.Hkv + head) << a.g.ps_log2) + slot) * a.hd;
}
__device__ __forceinline__ size_t v_offset(const PagedArgs& a, int page, int head, int slot) {
    return (((size_t)page * a.g.Hkv + head) * a.hd << a.g.ps_log2) + slot;
}
__device__ __forceinline__ size_t scale_offset(const PagedArgs& a, int page, int head, int slot) {
    return (((size_t)page * a.g.Hkv + head) << a.g.ps_log2) + slot;
}

}  // namespace lmx
