// Index arithmetic of the paged cache: which rows, positions, pages and work
// items a batch has.  Plain C++ with no HIP in it, so that a host program can
// walk the same functions over lengths and tables of any content: whatever
// cu, ctx_lens and page_table hold, nothing here names a row outside
// [0, n_tokens), a table entry outside the table or a page outside the pool.
#pragma once

#include <stdint.h>

#if defined(__HIP__) || defined(__HIPCC__)
#define LMX_FN __host__ __device__ __forceinline__
#else
#define LMX_FN inline
#endif

namespace lmx {

// The geometry of a batch that index arithmetic needs.
struct PagedGeom {
    int n_seq, n_tokens, max_new, max_ctx, table_stride;
    int n_pages, ps_log2;
    int Hkv, G;       // kv heads; query heads a kv head (attention only)
    int window;       // 0: none
};

LMX_FN int imin(int a, int b) { return a < b ? a : b; }
LMX_FN int imax(int a, int b) { return a > b ? a : b; }

// One sequence's rows [row0, row0 + n) and length, forced into range.
struct PagedSeq {
    int row0, n, ctx;
};
LMX_FN PagedSeq paged_seq(const PagedGeom& g, int cu0, int cu1, int ctx) {
    PagedSeq s;
    s.row0 = imin(imax(cu0, 0), g.n_tokens);
    s.n = imin(imax(cu1, s.row0), g.n_tokens) - s.row0;
    s.ctx = imin(imax(ctx, 0), g.max_ctx);
    return s;
}

// Index of position pos's entry within a sequence's table row, or -1 where
// the row has none.
LMX_FN int paged_entry(const PagedGeom& g, int pos) {
    if (pos < 0) return -1;
    const int e = pos >> g.ps_log2;
    return e < g.table_stride ? e : -1;
}

// A table entry as a page, or -1.
LMX_FN int paged_page(const PagedGeom& g, int entry) {
    return (uint32_t)entry < (uint32_t)g.n_pages ? entry : -1;
}

// ---- row blocks: a sequence's new rows, cut where its positions are multiples
// of R (a power of two), so that a block's rows meet whole granules of a page
// except at the sequence's own ends.  A first position below 0 (a length
// shorter than its new rows) is cut the same way.
LMX_FN int row_blocks(const PagedSeq& s, int log2_r) {
    return s.n ? ((s.ctx - 1) >> log2_r) - ((s.ctx - s.n) >> log2_r) + 1 : 0;
}
// Block i's rows: [first, first + count) of the sequence's.
struct RowBlock {
    int first, count;
};
LMX_FN RowBlock row_block(const PagedSeq& s, int i, int log2_r) {
    const int p0 = s.ctx - s.n, lo = ((p0 >> log2_r) + i) * (1 << log2_r);
    RowBlock b;
    b.first = imax(lo - p0, 0);
    b.count = imin(lo + (1 << log2_r) - p0, s.n) - b.first;
    return b;
}
// Blocks of all sequences together: a sequence of n rows has at most n / R + 2,
// and no more than n.
LMX_FN int64_t row_blocks_bound(const PagedGeom& g, int log2_r) {
    const int64_t a = ((int64_t)g.n_tokens >> log2_r) + 2 * (int64_t)g.n_seq;
    return a < g.n_tokens ? a : g.n_tokens;
}

// ---- attention's work items.
//
// A sequence's rows meet a kv head as n * G query rows (row r: token r / G,
// query head kvh * G + r % G), cut into row tiles of `bm`.  Its visible keys
// are [lo, ctx), lo the first position that its first row sees, rounded down
// to a 64-key unit; they are cut into splits of `per` units.
constexpr int kUnit = 64;

struct SeqWork {
    int rt;      // row tiles
    int lo;      // first key, a multiple of kUnit
    int units;   // 64-key units from lo to ctx
};
LMX_FN SeqWork seq_work(const PagedGeom& g, const PagedSeq& s, int bm) {
    SeqWork w;
    w.rt = (int)(((int64_t)s.n * g.G + bm - 1) / bm);
    const int first = s.ctx - s.n;  // position of the first row
    int lo = g.window && first + 1 > g.window ? first + 1 - g.window : 0;
    lo = imin(lo, s.ctx) & ~(kUnit - 1);
    w.lo = lo;
    w.units = (s.ctx - lo + kUnit - 1) / kUnit;
    return w;
}
// Splits of a sequence whose splits are `per` units long (at least one, so
// that every row is written).
LMX_FN int seq_splits(const SeqWork& w, int per) { return w.units > per ? (w.units + per - 1) / per : 1; }

// Row tiles of all sequences together: an upper bound from the shapes alone,
// and the least where every row of the batch is some sequence's.
LMX_FN int64_t row_tiles_least(const PagedGeom& g, int bm) { return ((int64_t)g.n_tokens * g.G + bm - 1) / bm; }
LMX_FN int64_t row_tiles_bound(const PagedGeom& g, int bm) {
    const int64_t a = ((int64_t)g.n_tokens * g.G + (int64_t)g.n_seq * (bm - 1)) / bm;
    const int64_t b = (int64_t)g.n_tokens * ((g.G + bm - 1) / bm);
    return a < b ? a : b;
}

// Units a split, for a total of `work` (units x row tiles x kv heads) cut for
// about `target` items.  The items of all sequences together are then at most
// target + Hkv * row tiles: a sequence with u units in rt tiles has
// rt * Hkv * ceil(u / per) < rt * Hkv * (u / per + 1), and the factor above
// 1 covers the float sum's rounding.
LMX_FN int units_per_split(float work, int target, int least) {
    const float per = work * 1.0001f / (float)target;
    return per <= (float)least ? least : (per < 1e9f ? (int)per + 1 : 1000000000);
}

}  // namespace lmx
