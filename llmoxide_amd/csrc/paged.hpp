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
    int seq;   // -1: none
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
    RowPlace p{-1, 0, 0, -1};
    if (seq >= a.g.n_seq || row >= a.g.n_tokens) return p;
    const int cu0 = a.cu[seq], cu1 = a.cu[seq + 1];
    const PagedSeq s = paged_seq(a.g, cu0, cu1, a.ctx[seq]);
    if (row < s.row0 || row >= s.row0 + s.n) return p;
    p.seq = seq;
    p.pos = s.ctx - s.n + (row - s.row0);
    const int e = p.pos < s.ctx ? paged_entry(a.g, p.pos) : -1;
    if (e < 0) return p;
    p.page = paged_page(a.g, a.table[(size_t)seq * a.g.table_stride + e]);
    p.slot = p.pos & ((1 << a.g.ps_log2) - 1);
    return p;
}

// Inclusive sum over the wave's lanes.
__device__ __forceinline__ int wave_scan(int x) {
    const int lane = __lane_id();
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int y = __shfl_up(x, d, 64);
        x += lane >= d ? y : 0;
    }
    return x;
}

// Row block `id` of the batch (every wave for itself): its first row r0 and row
// count, and in lane l the place of row r0 + l % R.  False: no such block.
template <int LOG2_R>
__device__ __forceinline__ bool find_block(const PagedArgs& a, int id, int& r0, int& n_rows, RowPlace& at) {
    const int lane = __lane_id();
    int base = 0;
    for (int c0 = 0; c0 < a.g.n_seq; c0 += 64) {
        const int b = c0 + lane;
        PagedSeq s{0, 0, 0};
        if (b < a.g.n_seq) s = paged_seq(a.g, a.cu[b], a.cu[b + 1], a.ctx[b]);
        const int n = row_blocks(s, LOG2_R), upto = a.g.n_seq == 1 ? n : wave_scan(n);
        const uint64_t has = __ballot(base + upto > id);
        if (has) {
            const int l = __builtin_ctzll(has);
            auto get = [&](int x) { return __builtin_amdgcn_readlane(x, l); };
            const PagedSeq q{get(s.row0), get(s.n), get(s.ctx)};
            const RowBlock blk = row_block(q, id - base - (get(upto) - get(n)), LOG2_R);
            r0 = q.row0 + blk.first;
            n_rows = blk.count;
            at = RowPlace{-1, 0, 0, -1};
            const int row = lane & ((1 << LOG2_R) - 1);
            if (row < n_rows) {
                at.seq = c0 + l;
                at.pos = q.ctx - q.n + blk.first + row;
                const int e = paged_entry(a.g, at.pos);
                if (e >= 0) {
                    at.page = paged_page(a.g, a.table[(size_t)at.seq * a.g.table_stride + e]);
                    at.slot = at.pos & ((1 << a.g.ps_log2) - 1);
                }
            }
            return n_rows > 0;
        }
        base += __builtin_amdgcn_readlane(upto, 63);
    }
    return false;
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
