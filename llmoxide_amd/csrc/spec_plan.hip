// Pages and row maps of a step from its requests' lengths, and positions and
// sight of its rows from their parents.
//
// The list of free pages is a stack: given-back pages go on top, then requests
// take from the top in order, so a request's first page lies at a place that
// sums over the requests before it name.  One workgroup makes these sums (1024
// requests at a time) and moves the pages, a thread an entry, whatever request
// it is of; the order of everything is that of the sums, none of arrivals.
//
// Bound by latency: a step's entries and rows are a few KB, read once through
// four dependent steps (lengths, sums, free list, table).  Sixteen requests of 32
// rows 6.6 us, 64 requests with 42000 rows 6.6 and 2.7 for the map.
#include "spec.hpp"

namespace lmx {

struct PlanArgs {
    int n_seq, n_tokens, ps_log2, stride, n_pages, trim;
    int rows_here;  // 1: the plan's workgroup maps the rows too
    const int32_t* lens;
    const int32_t* fresh;
    int32_t* table;
    int32_t* held;
    int32_t* free_pages;
    int32_t* n_free;
    int32_t* cu;
    int32_t* ctx;
    int64_t* slots;
    int32_t* pos;
};

constexpr int kPlan = 1024;  // threads, and requests at a time

struct Request {
    int len, rows, need, held;
};
__device__ __forceinline__ int room_of(const PlanArgs& a) {
    const int64_t table = (int64_t)a.stride << a.ps_log2;
    return (int)(table < kMost ? table : kMost);
}
__device__ __forceinline__ Request load_request(const PlanArgs& a, int b) {
    Request r;
    r.len = imax(a.lens[b], 0);
    r.rows = imin(imax(a.fresh[b], 0), a.n_tokens);
    r.held = imin(imax(a.held[b], 0), a.stride);
    const int64_t total = (int64_t)r.len + r.rows, room = room_of(a);
    r.need = (int)(((total < room ? total : room) + (1 << a.ps_log2) - 1) >> a.ps_log2);
    return r;
}
// Length with n rows, from which their positions count back: not cut where the table
// ends, which would move them onto cached ones.  (More rows than the table has positions
// are a length below the rows, which have no positions.)
__device__ __forceinline__ int length_with(const PlanArgs& a, int len, int n) {
    const int64_t total = (int64_t)len + n;
    return n > room_of(a) ? room_of(a) : (int)(total < 0x7fffffff ? total : 0x7fffffff);
}

// Inclusive scans over the workgroup of three counts that only its first `waves`
// waves have (the others get the totals, so that places behind the last request hold
// no less than its: last_at needs rising numbers); `sums` (48 words of LDS) may be used
// again afterwards.
struct Three {
    int x[3];
};
__device__ __forceinline__ Three block_scan(Three v, int waves, int* sums, Three& total) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    if (w < waves) {
#pragma unroll
        for (int d = 1; d < 64; d <<= 1)
#pragma unroll
            for (int i = 0; i < 3; ++i) {
                const int y = __shfl_up(v.x[i], d, 64);
                v.x[i] = lane >= d ? add_sat(v.x[i], y) : v.x[i];
            }
        if (lane == 63)
#pragma unroll
            for (int i = 0; i < 3; ++i) sums[3 * w + i] = v.x[i];
    }
    __syncthreads();
    Three before{{0, 0, 0}};
    total = before;
    for (int k = 0; k < waves; ++k) {
        if (k == w) before = total;
#pragma unroll
        for (int i = 0; i < 3; ++i) total.x[i] = add_sat(total.x[i], sums[3 * k + i]);
    }
    if (w >= waves) before = total;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 3; ++i) v.x[i] = add_sat(v.x[i], before.x[i]);
    return v;
}
// Of `n` rising numbers (n a power of two), the last at or below i (the first one is).
__device__ __forceinline__ int last_at(const int* start, int n, int i) {
    int at = 0;
    for (int step = n >> 1; step > 0; step >>= 1) at += start[at + step] <= i ? step : 0;
    return at;
}

// Row j of request b, whose rows begin behind `len` positions.
__device__ __forceinline__ void map_row(const PlanArgs& a, int row, int b, int len, int j) {
    const int64_t p = (int64_t)len + j, e = p >> a.ps_log2;
    int page = -1;
    if (e < a.stride && p < kMost) page = a.table[(size_t)b * a.stride + e];
    if (a.slots)
        a.slots[row] = (uint32_t)page < (uint32_t)a.n_pages ? ((int64_t)page << a.ps_log2) + (p & ((1 << a.ps_log2) - 1)) : -1;
    if (a.pos) a.pos[row] = (int32_t)(p < 0x7fffffff ? p : 0x7fffffff);
}
__device__ __forceinline__ void map_none(const PlanArgs& a, int row) {
    if (a.slots) a.slots[row] = -1;
    if (a.pos) a.pos[row] = -1;
}

// Up to kPlan requests, a thread each, and the sums over them.
enum { kBack, kWant, kRows };
struct Chunk {
    Request r;
    int had, want, back;
    Three upto, all;
};
__device__ __forceinline__ Chunk load_chunk(const PlanArgs& a, int c0, int waves, int* sums) {
    Chunk c;
    c.r = Request{0, 0, 0, 0};
    if (c0 + (int)threadIdx.x < a.n_seq) c.r = load_request(a, c0 + threadIdx.x);
    c.back = a.trim ? imax(c.r.held - c.r.need, 0) : 0;
    c.had = c.r.held - c.back;
    c.want = imax(c.r.need - c.had, 0);
    c.upto = block_scan(Three{{c.back, c.want, c.r.rows}}, waves, sums, c.all);
    return c;
}

__global__ __launch_bounds__(kPlan) void spec_plan_kernel(PlanArgs a) {
    __shared__ int sums[3 * kPlan / 64];
    __shared__ int start[kPlan], from[kPlan];        // of entries: a request's first, and its place in the table
    __shared__ int row_start[kPlan], row_len[kPlan];  // of rows
    const int tid = threadIdx.x;
    int top = imin(imax(a.n_free[0], 0), a.n_pages);  // free pages
    const int waves = imin((a.n_seq + 63) / 64, kPlan / 64);
    int size = 1;  // of `start` and `row_start`: places of requests, rounded up
    while (size < a.n_seq && size < kPlan) size <<= 1;

    Chunk c = load_chunk(a, 0, waves, sums);
    if (a.trim)
        for (int c0 = (a.n_seq - 1) / kPlan * kPlan; c0 >= 0; c0 -= kPlan) {  // the last requests first
            if (a.n_seq > kPlan) c = load_chunk(a, c0, waves, sums);
            const int total = c.all.x[kBack];
            if (total == 0) continue;  // uniform
            // place k of start: the request k from behind
            if (tid < size) {
                start[size - 1 - tid] = total - c.upto.x[kBack];
                from[size - 1 - tid] = c.r.held - 1;
            }
            __syncthreads();
            for (int i0 = 0; i0 < total; i0 += kPlan) {
                const int i = i0 + tid;
                int id = -1;
                if (i < total) {
                    const int t = last_at(start, size, i);
                    int32_t* at = a.table + (size_t)(c0 + size - 1 - t) * a.stride + (from[t] - (i - start[t]));
                    id = *at;
                    *at = -1;
                }
                const bool page = (uint32_t)id < (uint32_t)a.n_pages;
                Three back;
                const Three rank = block_scan(Three{{page, 0, 0}}, kPlan / 64, sums, back);
                const int to = top + rank.x[0] - 1;
                if (page && to < a.n_pages) a.free_pages[to] = id;
                top = imin(top + back.x[0], a.n_pages);
            }
        }
    __syncthreads();

    int rows = 0, taken = 0;  // of the requests before
    for (int c0 = 0; c0 < a.n_seq; c0 += kPlan) {
        if (c0) c = load_chunk(a, c0, waves, sums);  // (the first chunk is at hand)
        const int b = c0 + tid, all_rows = c.all.x[kRows], all_want = c.all.x[kWant];
        if (b < a.n_seq) {
            const int upto = imin(add_sat(rows, c.upto.x[kRows]), a.n_tokens);
            a.cu[b + 1] = upto;
            a.ctx[b] = length_with(a, c.r.len, upto - imin(add_sat(rows, c.upto.x[kRows] - c.r.rows), a.n_tokens));
            a.held[b] = c.had + imin(imax(top - add_sat(taken, c.upto.x[kWant] - c.want), 0), c.want);
        }
        if (tid < size) {
            start[tid] = c.upto.x[kWant] - c.want;
            from[tid] = c.had;
            row_start[tid] = c.upto.x[kRows] - c.r.rows;
            row_len[tid] = c.r.len;
        }
        __syncthreads();
        for (int i = tid; i < all_want; i += kPlan) {
            const int t = last_at(start, size, i), at = top - 1 - add_sat(taken, i);
            a.table[(size_t)(c0 + t) * a.stride + from[t] + (i - start[t])] = at >= 0 ? a.free_pages[at] : -1;
        }
        if (a.rows_here) {
            __syncthreads();
            for (int i = tid; i < all_rows && rows + i < a.n_tokens; i += kPlan) {
                const int t = last_at(row_start, size, i);
                map_row(a, rows + i, c0 + t, row_len[t], i - row_start[t]);
            }
        }
        rows = add_sat(rows, all_rows);
        taken = add_sat(taken, all_want);
        __syncthreads();
    }
    if (a.rows_here)
        for (int row = rows + tid; row < a.n_tokens; row += kPlan) map_none(a, row);
    if (tid == 0) {
        a.cu[0] = 0;
        a.n_free[0] = imax(top - taken, 0);
        a.n_free[1] = imax(taken - top, 0);
    }
}

// The map of many rows: a thread a row.
__global__ __launch_bounds__(256) void spec_rows_kernel(PlanArgs a) {
    const int row = blockIdx.x * 256 + threadIdx.x;
    if (row >= a.n_tokens) return;
    if (row >= a.cu[a.n_seq]) return map_none(a, row);
    int lo = 0, hi = a.n_seq;  // the last request that begins at or below the row
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.cu[mid] <= row) lo = mid;
        else hi = mid;
    }
    map_row(a, row, lo, imax(a.lens[lo], 0), row - a.cu[lo]);
}

// Rows that the plan's workgroup maps itself.  Here and in a kernel of their own, us a
// plan: 4096 rows 6.5 and 8.9, 8192 rows 8.4 and 9.2, 16384 rows 10.1 and 9.1.
constexpr int kRowsHere = 8192;

lmx_status spec_plan(const lmxs_plan_desc* d, const int32_t* lens, const int32_t* new_rows, int32_t* table, int32_t* held,
                     int32_t* free_pages, int32_t* n_free, int32_t* cu, int32_t* ctx, int64_t* slots, int32_t* pos,
                     hipStream_t st) {
    PlanArgs a{};
    a.n_seq = (int)d->n_seq;
    a.n_tokens = (int)d->n_tokens;
    while ((1u << a.ps_log2) < d->page_size) ++a.ps_log2;
    a.stride = (int)d->table_stride;
    a.n_pages = (int)d->n_pages;
    a.trim = (int)d->trim;
    a.lens = lens;
    a.fresh = new_rows;
    a.table = table;
    a.held = held;
    a.free_pages = free_pages;
    a.n_free = n_free;
    a.cu = cu;
    a.ctx = ctx;
    a.slots = slots;
    a.pos = pos;
    const bool map = slots || pos;
    a.rows_here = map && a.n_tokens <= kRowsHere;
    (void)hipGetLastError();
    hipLaunchKernelGGL(spec_plan_kernel, dim3(1), dim3(kPlan), 0, st, a);
    LMX_CHECK_LAUNCH();
    if (map && !a.rows_here) {
        hipLaunchKernelGGL(spec_rows_kernel, dim3((unsigned)((a.n_tokens + 255) / 256)), dim3(256), 0, st, a);
        LMX_CHECK_LAUNCH();
    }
    return LMX_OK;
}

// ------------------------------------------------------------------- trees --
// A workgroup takes a request.  A row's ancestors among the 64 rows of its own word
// come from a walk up the parents, which lie in LDS: at most 63 steps, some ten in a
// tree of 64 drafts.  The words before are those of its first ancestor there, and so
// on: at most 15 more steps, whatever the depth (1024 rows in a chain 26 us,
// eight trees of 1024 13; with a walk up to the root for each word 2940 and 444).
//
// Bound by latency: sixteen trees of 32 rows 3.4 us, 8 KB.
struct Above {
    int next, n;    // the row's first ancestor in an earlier word (-1: none); bits set
    uint64_t bits;  // the row and its ancestors in its own word
};
__global__ __launch_bounds__(256) void spec_tree_kernel(int n_tokens, int words, int window, const int32_t* cu,
                                                        const int32_t* ctx, const int32_t* parent, int32_t* pos,
                                                        uint64_t* seen) {
    __shared__ int up[LMXS_MAX_ROWS];
    __shared__ Above above[LMXS_MAX_ROWS];
    const SpecRows s = spec_rows(cu, blockIdx.x, n_tokens, 64 * words);
    for (int i = threadIdx.x; i < s.n; i += 256) {
        const int p = parent[s.row0 + i];
        up[i] = p >= 0 && p < i ? p : -1;
    }
    const int first = imax(ctx[blockIdx.x] - s.n, 0);
    __syncthreads();
    for (int i = threadIdx.x; i < s.n; i += 256) {
        Above x{up[i], 1, 1ull << (i & 63)};
        while (x.next >= 0 && x.next >> 6 == i >> 6) {
            x.bits |= 1ull << (x.next & 63);
            ++x.n;
            x.next = up[x.next];
        }
        above[i] = x;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < s.n; i += 256) {
        int depth = -1;  // of the row, less those still to come
        int p = i;
        for (int w = words - 1; w >= 0; --w) {
            uint64_t bits = 0;
            if (p >= 0 && p >> 6 == w) {
                const Above x = above[p];
                bits = x.bits;
                // ancestors come before: those behind the window are the lowest bits
                if (window)
                    for (int drop = imin(depth + 1 + x.n - window, x.n); drop > 0; --drop) bits &= bits - 1;
                depth += x.n;
                p = x.next;
            }
            if (seen) seen[(size_t)(s.row0 + i) * words + w] = bits;
        }
        if (pos) pos[s.row0 + i] = first + depth;
    }
}

lmx_status spec_tree(const lmxp_batch* b, const int32_t* parent, uint32_t words, uint32_t window, int32_t* pos,
                     uint64_t* seen, hipStream_t st) {
    (void)hipGetLastError();
    hipLaunchKernelGGL(spec_tree_kernel, dim3(b->n_seq), dim3(256), 0, st, (int)b->n_tokens, (int)words, (int)window,
                       b->cu, b->ctx_lens, parent, pos, seen);
    LMX_CHECK_LAUNCH();
    return LMX_OK;
}

}  // namespace lmx
