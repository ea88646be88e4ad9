// Moves the accepted rows of a step to consecutive slots, in all layers at once.
//
// A thread owns one 16-byte piece of K's rows, or one dim of V's columns, of one
// head in one layer, and moves it for every accepted row in order.  A row moves
// to a slot at or before its own, and rows rise, so a slot that is written has
// been read before if it had to be: by the same thread, up to eight moves at
// once.  No barrier, no second buffer.
//
// Bound by the cache lines of V: the lanes of a wave take the dims of one
// position, each in a line of its own (V lies transposed), and a dim's moves
// mostly share that line.
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

// Slots (page * page_size + slot) of one move; -1: none.
struct Move {
    int64_t src, dst;
};
__device__ __forceinline__ int64_t slot_of(const PagedArgs& a, int b, int pos) {
    const int e = paged_entry(a.g, pos);
    if (e < 0) return -1;
    const int page = paged_page(a.g, a.table[(size_t)b * a.g.table_stride + e]);
    return page < 0 ? -1 : ((int64_t)page << a.g.ps_log2) + (pos & ((1 << a.g.ps_log2) - 1));
}

// Moves of one element that lies at[slot-dependent offset]: up to eight are read
// before the first is written.
template <typename T, typename F>
__device__ __forceinline__ void move_all(T* base, const Move* moves, int n, const F& offset) {
    constexpr int U = 8;
    for (int j0 = 0; j0 < n; j0 += U) {
        T x[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (j0 + u < n && moves[j0 + u].src >= 0) x[u] = base[offset(moves[j0 + u].src)];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (j0 + u < n && moves[j0 + u].src >= 0) base[offset(moves[j0 + u].dst)] = x[u];
    }
}

template <bool I8>
__global__ __launch_bounds__(256) void spec_keep_kernel(KeepArgs a) {
    using E = std::conditional_t<I8, uint8_t, uint16_t>;
    __shared__ Move moves[64];
    const PagedGeom& g = a.p.g;
    const int b = blockIdx.x, layer = blockIdx.z, tid = threadIdx.x;
    const PagedSeq s = paged_seq(g, a.p.cu[b], a.p.cu[b + 1], a.p.ctx[b]);
    const int n = imin(imin(imax(a.accepted[b], 0), s.n), a.path_stride), first = s.ctx - s.n;
    const int psm = (1 << g.ps_log2) - 1, hd = a.p.hd;
    const int x = blockIdx.y * 256 + tid;                 // the thread's piece
    const int chunks = hd * (int)sizeof(E) / 16;          // 16-byte pieces of a K row
    const int kp = g.Hkv * chunks, vp = g.Hkv * hd;
    for (int j0 = 1; j0 < n; j0 += 64) {
        const int m = imin(64, n - j0);
        if (tid < m) {
            const int j = j0 + tid, p = a.path[(size_t)b * a.path_stride + j];
            const int before = a.path[(size_t)b * a.path_stride + j - 1];
            Move v{-1, -1};
            if (p > j && p < s.n && p > before) v = Move{slot_of(a.p, b, first + p), slot_of(a.p, b, first + j)};
            if (v.dst < 0) v.src = -1;
            moves[tid] = v;
        }
        __syncthreads();
        if (x < kp) {
            const int h = x / chunks, c = x % chunks;
            move_all(reinterpret_cast<uint4*>(a.k[layer]), moves, m, [&](int64_t at) {
                return ((((at >> g.ps_log2) * g.Hkv + h) << g.ps_log2) + (at & psm)) * chunks + c;
            });
        } else if (x < kp + vp) {
            const int h = (x - kp) / hd, d = (x - kp) % hd;
            move_all(reinterpret_cast<E*>(a.v[layer]), moves, m, [&](int64_t at) {
                return ((((at >> g.ps_log2) * g.Hkv + h) * hd + d) << g.ps_log2) + (at & psm);
            });
        } else if (I8 && x < kp + vp + 2 * g.Hkv) {
            const int y = x - kp - vp, h = y % g.Hkv;
            move_all(y < g.Hkv ? a.k_scale[layer] : a.v_scale[layer], moves, m, [&](int64_t at) {
                return (((at >> g.ps_log2) * g.Hkv + h) << g.ps_log2) + (at & psm);
            });
        }
        __syncthreads();
    }
}

lmx_status spec_keep(const lmxp_pool* pools, uint32_t n_pools, const lmxp_batch* b, const int32_t* path,
                     uint32_t path_stride, const int32_t* accepted, hipStream_t st) {
    KeepArgs a{};
    a.p = paged_args(pools, b);
    a.path = path;
    a.accepted = accepted;
    a.path_stride = (int)path_stride;
    const bool i8 = pools->store == LMXP_I8;
    const int es = i8 ? 1 : 2, hd = (int)pools->head_dim, kv = (int)pools->n_kv_heads;
    a.pieces = kv * (hd * es / 16) + kv * hd + (i8 ? 2 * kv : 0);
    (void)hipGetLastError();
    for (uint32_t at = 0; at < n_pools; at += kPools) {
        const uint32_t n = n_pools - at < kPools ? n_pools - at : kPools;
        for (uint32_t i = 0; i < n; ++i) {
            a.k[i] = static_cast<char*>(pools[at + i].k);
            a.v[i] = static_cast<char*>(pools[at + i].v);
            a.k_scale[i] = pools[at + i].k_scale;
            a.v_scale[i] = pools[at + i].v_scale;
        }
        const dim3 grid(b->n_seq, (unsigned)((a.pieces + 255) / 256), n);
        if (i8) hipLaunchKernelGGL(spec_keep_kernel<true>, grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL(spec_keep_kernel<false>, grid, dim3(256), 0, st, a);
        LMX_CHECK_LAUNCH();
    }
    return LMX_OK;
}

}  // namespace lmx
