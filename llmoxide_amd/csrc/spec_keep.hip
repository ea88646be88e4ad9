// Moves the accepted rows of a step to consecutive slots, in all layers at once.
//
// A thread owns one 16-byte piece of K's rows, or one dim of V's columns, of one
// head in one layer, and moves it for every accepted row in order.  A row moves
// to a slot at or before its own, and rows rise, so a slot that is written has
// been read before if it had to be: by the same thread, four moves at once.  No
// barrier, no second buffer.  Every wave looks the moves up for itself, one a
// lane; they then come from the lanes' registers as scalars.
//
// Bound by latency (four dependent loads: lengths, path, table, rows) and, in many
// layers, by V's sectors: it lies transposed, so that a position's dims are 2 bytes
// each in a page's 32 to 512 bytes a dim.  Sixteen requests' paths through trees of 32
// rows, 36 layers of 8 heads of 128 dims, f16 (24 MB read and written): 12 us, 2 TB/s;
// one request, 8 layers: 3.7 us, 7 with the launch and the host.
#include "spec.hpp"

namespace lmx {

constexpr int kPools = 64;  // layers a launch

struct KeepArgs {
    PagedArgs p;  // its pool pointers are not used
    const int32_t* path;
    const int32_t* accepted;
    int path_stride;
    int pieces;   // threads' pieces of one layer and request
    char* k[kPools];
    char* v[kPools];
    float* k_scale[kPools];
    float* v_scale[kPools];
};

// A lane's position as (page, slot); page -1: none.  (Position 0's entry is read
// where the position has none: no branch, so that two lookups go out together.)
struct Place {
    int page, slot;
};
__device__ __forceinline__ Place place_of(const PagedArgs& a, int b, int pos) {
    const int e = paged_entry(a.g, pos);
    const int page = paged_page(a.g, a.table[(size_t)b * a.g.table_stride + imax(e, 0)]);
    return Place{e < 0 ? -1 : page, pos & ((1 << a.g.ps_log2) - 1)};
}

// N moves of one element, all read before the first is written: from and to are
// the same for the whole wave.
template <int N, typename T>
__device__ __forceinline__ void move_some(char* base, const int64_t* from, const int64_t* to) {
    T x[N];
#pragma unroll
    for (int u = 0; u < N; ++u) x[u] = *reinterpret_cast<const T*>(base + from[u]);
#pragma unroll
    for (int u = 0; u < N; ++u) *reinterpret_cast<T*>(base + to[u]) = x[u];
}

template <bool I8>
__global__ __launch_bounds__(256) void spec_keep_kernel(KeepArgs a) {
    using E = std::conditional_t<I8, uint8_t, uint16_t>;
    constexpr int ES = sizeof(E);
    const PagedGeom& g = a.p.g;
    const int b = blockIdx.x, layer = blockIdx.z, lane = threadIdx.x & 63;
    const int x = blockIdx.y * 256 + threadIdx.x;  // the thread's piece
    const int cu0 = a.p.cu[b], cu1 = a.p.cu[b + 1], ctx = a.p.ctx[b], accepted = a.accepted[b];
    args_in_sgprs(cu0, cu1, ctx, accepted);  // one round of loads
    const PagedSeq s = paged_seq(g, cu0, cu1, ctx);
    const int n = imin(imin(imax(accepted, 0), s.n), a.path_stride), first = s.first;
    const int ps = 1 << g.ps_log2, hd = a.p.hd;
    const int chunks = hd * ES / 16;  // 16-byte pieces of a K row
    const int kp = g.Hkv * chunks, vp = g.Hkv * hd;
    const bool is_k = x < kp, is_v = !is_k && x < kp + vp;
    // The thread's place in a page; bytes from page to page and from slot to slot.
    char* base;
    int64_t page_bytes;
    int slot_bytes;
    if (is_k) {
        const int h = (int)((uint32_t)x / (uint32_t)chunks), c = x - h * chunks;
        base = a.k[layer] + ((size_t)h << g.ps_log2) * (hd * ES) + 16 * c;
        page_bytes = ((int64_t)g.Hkv << g.ps_log2) * (hd * ES);
        slot_bytes = hd * ES;
    } else if (is_v) {
        base = a.v[layer] + ((size_t)(x - kp) << g.ps_log2) * ES;
        page_bytes = ((int64_t)vp << g.ps_log2) * ES;
        slot_bytes = ES;
    } else {  // 8 bits: scales
        const int y = x - kp - vp;
        base = reinterpret_cast<char*>(y < g.Hkv ? a.k_scale[layer] : a.v_scale[layer]) + (((size_t)(y < g.Hkv ? y : y - g.Hkv) << g.ps_log2) * 4);
        page_bytes = ((int64_t)g.Hkv << g.ps_log2) * 4;
        slot_bytes = 4;
    }
    for (int j0 = 1; j0 < n; j0 += 64) {
        const int j = imin(j0 + lane, n - 1);
        const int p = a.path[(size_t)b * a.path_stride + j], before = a.path[(size_t)b * a.path_stride + j - 1];
        const bool row = j0 + lane < n && p > j && p < s.n && p > before;
        const Place from = place_of(a.p, b, first + (row ? p : j)), to = place_of(a.p, b, first + j);
        uint64_t left = __ballot(row && from.page >= 0 && to.page >= 0);
        while (left) {  // (all lanes: what is read from a lane has to be made there)
            int64_t f[4], t[4];
            int m = 0;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int l = left ? (int)__builtin_ctzll(left) : 0;
                m += left != 0;
                left &= left - 1;
                f[u] = __builtin_amdgcn_readlane(from.page, l) * page_bytes + __builtin_amdgcn_readlane(from.slot, l) * slot_bytes;
                t[u] = __builtin_amdgcn_readlane(to.page, l) * page_bytes + __builtin_amdgcn_readlane(to.slot, l) * slot_bytes;
            }
            auto go = [&](auto tag) {
                using T = decltype(tag);
                if (m == 1) move_some<1, T>(base, f, t);
                else if (m == 2) move_some<2, T>(base, f, t);
                else if (m == 3) move_some<3, T>(base, f, t);
                else move_some<4, T>(base, f, t);
            };
            if (is_k) go(f32x4{});
            else if (is_v) go(E{});
            else if (x < a.pieces) go(0.f);
        }
    }
}

lmx_status spec_keep(const lmxp_pool* const* pools, uint32_t n_pools, const lmxp_batch* b, const int32_t* path,
                     uint32_t path_stride, const int32_t* accepted, hipStream_t st) {
    KeepArgs a{};
    const lmxp_pool& p = *pools[0];
    a.p = paged_args(&p, b);
    a.path = path;
    a.accepted = accepted;
    a.path_stride = (int)path_stride;
    const bool i8 = p.store == LMXP_I8;
    const int es = i8 ? 1 : 2, hd = (int)p.head_dim, kv = (int)p.n_kv_heads;
    a.pieces = kv * (hd * es / 16) + kv * hd + (i8 ? 2 * kv : 0);
    (void)hipGetLastError();
    for (uint32_t at = 0; at < n_pools; at += kPools) {
        const uint32_t n = n_pools - at < kPools ? n_pools - at : kPools;
        for (uint32_t i = 0; i < n; ++i) {
            a.k[i] = static_cast<char*>(pools[at + i]->k);
            a.v[i] = static_cast<char*>(pools[at + i]->v);
            a.k_scale[i] = pools[at + i]->k_scale;
            a.v_scale[i] = pools[at + i]->v_scale;
        }
        const dim3 grid(b->n_seq, (unsigned)((a.pieces + 255) / 256), n);
        if (i8) hipLaunchKernelGGL(spec_keep_kernel<true>, grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL(spec_keep_kernel<false>, grid, dim3(256), 0, st, a);
        LMX_CHECK_LAUNCH();
    }
    return LMX_OK;
}

}  // namespace lmx
