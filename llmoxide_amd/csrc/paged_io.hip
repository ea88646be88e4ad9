// Writes into and reads from the paged KV cache on gfx950: append, prologue
// (norm, rotate, store) and read-back.
//
// All three move rows [token, head, dim] to or from pages where K keeps its
// rows and V lies transposed, [dim, slot].  A workgroup takes R consecutive
// rows of the batch and one kind of head.  A row's lane holds dims 4i .. 4i+3
// of its first half and the same of its second, so that the rotation of a
// whole head stays in the lane.  K goes straight between memory and registers.
// V turns in LDS: 16 rows of one sequence that fill a 16-slot granule move as
// 4 x 4 (8 bits) or 2 x 2 (f16) blocks turned by byte permutes, 16 bytes a
// transfer; rows at a chunk's ragged ends, and single tokens, element by
// element.  Attention reads V's operand fragments straight from such columns,
// which is what the transposed layout is for; the price is paid here, once a
// row.
//
// Bound by HBM: the rows in, the pages out (8 bits: 1 + 4 / head_dim bytes a
// value), nothing else.  Measured (8 kv heads; a copy reaches 5.13 TB/s):
//   eight prompts to 8 bits and back, 228 MB, 128 dims   59 us, 3.87 TB/s (store
//   22.9 us, read 20.1 us a kernel, the rest lies between the two)
//   a read of 32768 8-bit positions to f16, 203 MB       46 us, 4.38 TB/s
//   the prologue of six 8-bit chunks, 256 dims, 310 MB   87 us, 3.6 TB/s: two
//   thirds of the LDS cycles are conflicts of the angle table's stores (13% of
//   the CU cycles); the next head's loads ahead of the stores, or four
//   workgroups a CU, are not faster
//   one decode step of 32 sequences (append) 4.0 us, of 16 (prologue) 4.6 us a
//   kernel; a call 9.5 and 14.1 us, the host's
// Counters: profiles/paged_cache.md.
#include <cmath>

#include "lds_dma.hpp"
#include "paged.hpp"

namespace lmx {

template <int HD>
struct RowLanes {
    static constexpr int LPR = HD / 8;                   // lanes a row: 4 dims of each half a lane
    static constexpr int RPI = 64 / LPR;                 // rows a wave at once
    static constexpr int LOG2_R = HD <= 128 ? 6 : HD == 256 ? 5 : 4;
    static constexpr int R = 1 << LOG2_R;                // rows a workgroup
    static constexpr int NI = R / 4 / RPI;               // a wave's turns over its rows
};

template <int LPR>
__device__ __forceinline__ float sum_row(float x) {
    if constexpr (LPR == 64) return wave_sum64(x);
    if constexpr (LPR == 8) {
        x += dpp<0xB1>(x);   // quad_perm [1,0,3,2]
        x += dpp<0x4E>(x);   // quad_perm [2,3,0,1]
        return x + dpp<0x141>(x);  // row_half_mirror
    }
    x = row_sum16(x);
    if constexpr (LPR == 32) x += shfl_xor(x, 16);
    return x;
}
template <int CTRL>
__device__ __forceinline__ uint32_t max_dpp(uint32_t x) {
    const uint32_t y = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xF, 0xF, false);
    return x > y ? x : y;
}
template <int LPR>
__device__ __forceinline__ uint32_t max_row(uint32_t x) {
    x = max_dpp<0xB1>(x);
    x = max_dpp<0x4E>(x);
    x = max_dpp<0x141>(x);
    if constexpr (LPR >= 16) x = max_dpp<0x140>(x);
#pragma unroll
    for (int m = 16; m < LPR; m <<= 1) {
        const uint32_t y = (uint32_t)__shfl_xor((int)x, m, 64);
        x = x > y ? x : y;
    }
    return x;
}

// 4 x 4 bytes turned: out[d] holds byte d of in[0..3].
__device__ __forceinline__ void turn4(const uint32_t (&in)[4], uint32_t (&out)[4]) {
    const uint32_t a = __builtin_amdgcn_perm(in[1], in[0], 0x05010400u);  // 0.0 1.0 0.1 1.1
    const uint32_t b = __builtin_amdgcn_perm(in[3], in[2], 0x05010400u);
    const uint32_t c = __builtin_amdgcn_perm(in[1], in[0], 0x07030602u);  // 0.2 1.2 0.3 1.3
    const uint32_t d = __builtin_amdgcn_perm(in[3], in[2], 0x07030602u);
    out[0] = __builtin_amdgcn_perm(b, a, 0x05040100u);
    out[1] = __builtin_amdgcn_perm(b, a, 0x07060302u);
    out[2] = __builtin_amdgcn_perm(d, c, 0x05040100u);
    out[3] = __builtin_amdgcn_perm(d, c, 0x07060302u);
}

// A workgroup's V rows in LDS, one word (4 int8 or 2 f16 dims) beside the
// next, rows an odd number of words apart.
template <int HD, bool I8>
struct VTile {
    static constexpr int DW = I8 ? 4 : 2;        // dims a word
    static constexpr int W = HD / DW;            // words a row
    static constexpr int P = W + 1;
    static constexpr int BYTES = RowLanes<HD>::R * P * 4;
};

// Which of the workgroup's rows move as whole granules: row t has position
// pos0 + t, granule i starts at row first + 16 i (first < 0 where a sequence's
// rows begin inside one).
struct Granules {
    int first, count;
    __device__ __forceinline__ void of(const RowPlace& at, int n_rows) {
        first = -(__builtin_amdgcn_readfirstlane(at.pos) & 15);
        count = (n_rows - first + 15) >> 4;
    }
    __device__ __forceinline__ bool full(int i, int n_rows) const {
        return first + 16 * i >= 0 && first + 16 * i + 16 <= n_rows;
    }
    __device__ __forceinline__ bool full_row(int t, int n_rows) const { return full((t - first) >> 4, n_rows); }
};

// The 8-bit scale of a row from the largest |x|'s bits (which order as the
// magnitudes do, NaN above infinity above all numbers): amax / 127, correctly
// rounded; 0 below 2^-100, so that 1 / scale below is finite; NaN for a row
// that holds an infinity or a NaN.
__device__ __forceinline__ float scale_of(uint32_t amax_bits) {
    if (amax_bits >= 0x7f800000u) return __builtin_nanf("");
    const float amax = __builtin_bit_cast(float, amax_bits);
    return amax < 0x1p-100f ? 0.f : amax / 127.f;
}
// Eight x / s rounded to the nearest integers, ties to even, from the exact
// quotients, as bytes.  t = x * inv is off by 2^-23 of itself at most, so its
// rounding (the low byte of t + 1.5 2^23) is the quotient's unless t lies
// within 2^-15 of a half.  Such a k is settled by x - k s, which is exact in
// f32 (near s / 2, and a multiple of the smaller of x's and s's last places).
// inv = 0 (scale 0 or NaN) gives zeros, whatever x holds.
__device__ __forceinline__ void quantize8(const f32x4 (&x)[2], float s, float inv, uint32_t (&out)[2]) {
    constexpr float kMagic = 12582912.f;
    const uint32_t on = inv == 0.f ? 0u : ~0u;
    float k[2][4], off = 0.f;
#pragma unroll
    for (int v = 0; v < 2; ++v)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float y = x[v][j] * inv;  // NaN where inv is 0 and x is not finite
            const float t = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, y) & on);
            k[v][j] = t + kMagic;
            off = fmaxf(off, fabsf(t - (k[v][j] - kMagic)));
        }
    if (__ballot(off > 0.5f - 0x1p-15f)) {
#pragma unroll
        for (int v = 0; v < 2; ++v)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float n = k[v][j] - kMagic;
                const float r = fmaf(-n, s, x[v][j]), h = 0.5f * s;
                const bool odd = ((int)n) & 1;
                if (on && (r > h || (r == h && odd))) k[v][j] += 1.f;
                if (on && (r < -h || (r == -h && odd))) k[v][j] -= 1.f;
            }
    }
#pragma unroll
    for (int v = 0; v < 2; ++v) {
        uint32_t u[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) u[j] = __builtin_bit_cast(uint32_t, k[v][j]);
        out[v] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(u[3], u[2], 0x0c0c0400u),
                                       __builtin_amdgcn_perm(u[1], u[0], 0x0c0c0400u), 0x05040100u);
    }
}

template <typename T>
__device__ __forceinline__ f32x4 load4(const T* p) {
    if constexpr (sizeof(T) == 4) {
        return *reinterpret_cast<const f32x4*>(p);
    } else {
        const f16x4 h = *reinterpret_cast<const f16x4*>(p);
        return f32x4{(float)h[0], (float)h[1], (float)h[2], (float)h[3]};
    }
}
template <typename T>
__device__ __forceinline__ void store4(T* p, f32x4 x) {
    if constexpr (sizeof(T) == 4)
        *reinterpret_cast<f32x4*>(p) = x;
    else
        *reinterpret_cast<f16x4*>(p) = f16x4{(f16)x[0], (f16)x[1], (f16)x[2], (f16)x[3]};
}

// V element (page, head, dim, slot).  The address is opaque: what follows from
// it stays where it is used, and is not held in registers across a loop.
template <typename T>
__device__ __forceinline__ T* column(T* v, const PagedArgs& a, int page, int head, int slot, int dim) {
    uint64_t x = reinterpret_cast<uint64_t>(v + v_offset(a, page, head, slot) + ((size_t)dim << a.g.ps_log2));
    opaque(x);
    return reinterpret_cast<T*>(x);
}

struct StoreArgs {
    PagedArgs p;
    const void* k_new;
    const void* v_new;
    size_t row_stride;  // elements
    int n_k, n_v, n_q;  // heads to take: K heads, V heads, query heads
    int g_k, g_v, g_q;  // groups of hpw heads, a workgroup each
    int hpw;
    // prologue only
    const float* q;
    void* q_out;
    size_t q_row_stride, q_head_stride;
    const float* q_gain;
    const float* k_gain;
    const float* factors;
    int n_rot, v_norm, q_out_f16;
    float eps;
    double scale_pow[8];  // s^(2^k), s = base^(-2/n_rot): pair i turns by pos * s^i
};

// sin and cos of theta (double): the multiple of pi/2 is taken off in double,
// what is left (|r| <= pi/4) goes through its Taylor series in f32: the terms
// left out are below 2e-9, the rounding 6e-8.  Angles of far positions keep
// their 53 bits up to there.
__device__ __forceinline__ void turn_of(double theta, float& c, float& s) {
    const double n = rint(theta * 0.63661977236758134308);
    double r = fma(-n, 1.57079632679489655800, theta);
    r = fma(-n, 6.12323399573676603587e-17, r);
    const float x = (float)r, x2 = x * x;
    const float sn = fmaf(x * x2, fmaf(x2, fmaf(x2, fmaf(x2, 1.f / 362880, -1.f / 5040), 1.f / 120), -1.f / 6), x);
    const float cs = fmaf(x2, fmaf(x2, fmaf(x2, fmaf(x2, fmaf(x2, -1.f / 3628800, 1.f / 40320), -1.f / 720), 1.f / 24), -0.5f), 1.f);
    const int q = (int)((long long)n & 3);
    c = (q & 1) ? sn : cs;
    s = (q & 1) ? cs : sn;
    if (q == 1 || q == 2) c = -c;
    if (q >= 2) s = -s;
}

// Where a lane's turn of a whole head comes from, and the norm before it.
template <int LPR, int HD>
__device__ __forceinline__ void norm_row(f32x4 (&e)[2], const float* gain, float eps, int li) {
    float ss = 0.f;
#pragma unroll
    for (int v = 0; v < 2; ++v)
#pragma unroll
        for (int j = 0; j < 4; ++j) ss = fmaf(e[v][j], e[v][j], ss);
    const float sc = __builtin_amdgcn_rsqf(sum_row<LPR>(ss) / (float)HD + eps);
#pragma unroll
    for (int v = 0; v < 2; ++v) {
        const f32x4 g = gain ? load4(gain + 4 * li + HD / 2 * v) : f32x4{1.f, 1.f, 1.f, 1.f};
#pragma unroll
        for (int j = 0; j < 4; ++j) e[v][j] = e[v][j] * sc * g[j];
    }
}
// The whole head turns: dim d's partner d + HD/2 is the lane's own.
__device__ __forceinline__ void turn_row(f32x4 (&e)[2], const float (&c)[4], const float (&s)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float p = e[0][j], q = e[1][j];
        e[0][j] = p * c[j] - q * s[j];
        e[1][j] = q * c[j] + p * s[j];
    }
}
// The first 2 * half dims turn: partners lie in other lanes as a rule, so the
// row goes through LDS (rs: the row's floats).  turn_at(i): (cos, sin) of pair i.
template <int HD, typename F>
__device__ __forceinline__ void turn_part(f32x4 (&e)[2], float* rs, int li, int half, const F& turn_at) {
#pragma unroll
    for (int v = 0; v < 2; ++v) store4(rs + 4 * li + HD / 2 * v, e[v]);
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
    for (int v = 0; v < 2; ++v)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int d = 4 * li + HD / 2 * v + j;
            if (d < 2 * half) {
                const bool lo = d < half;
                const float2 t = turn_at(lo ? d : d - half);
                const float o = rs[lo ? d + half : d - half];
                e[v][j] = e[v][j] * t.x + (lo ? -o : o) * t.y;
            }
        }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
// The largest |x| of a row, as bits.
template <int LPR>
__device__ __forceinline__ uint32_t row_amax(const f32x4 (&e)[2]) {
    uint32_t m = 0;
#pragma unroll
    for (int v = 0; v < 2; ++v)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float f = e[v][j];
            const uint32_t u = __builtin_bit_cast(uint32_t, f) & 0x7fffffffu;
            m = m > u ? m : u;
        }
    return max_row<LPR>(m);
}
__device__ __forceinline__ double freq_of(const StoreArgs& a, int i) {
    double f = 1.0;  // s^i by the bits of i (i < 256)
#pragma unroll
    for (int k = 0; k < 8; ++k) f *= (i >> k) & 1 ? a.scale_pow[k] : 1.0;
    return a.factors ? f / (double)a.factors[i] : f;
}

// Rows of prompts.  PRO: norm and rotate on the way, and take the query heads
// too.
template <typename SRC, bool I8, int HD, bool PRO>
__global__ __launch_bounds__(256) void paged_store_kernel(StoreArgs a) {
    using L = RowLanes<HD>;
    using VT = VTile<HD, I8>;
    using DT = std::conditional_t<I8, int8_t, f16>;
    constexpr int R = L::R, NI = L::NI, LPR = L::LPR, H2 = HD / 2;
    // a workgroup holds V's rows, or the angles (cos, sin) of its rows
    constexpr int kTurn = PRO ? R * H2 * 8 : 0, kBytes = VT::BYTES > kTurn ? VT::BYTES : kTurn;
    __shared__ __align__(16) char smem[kBytes];
    __shared__ __align__(16) float rows_s[PRO ? 4 : 1][PRO ? 512 : 4];
    __shared__ double freq_s[PRO ? H2 : 1];
    uint32_t* const vt = reinterpret_cast<uint32_t*>(smem);
    float2* const turn = reinterpret_cast<float2*>(smem);  // [row][pair]

    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int sub = lane / LPR, li = lane % LPR;
    const int y = blockIdx.y;
    const bool is_k = y < a.g_k, is_v = !is_k && y < a.g_k + a.g_v, is_q = PRO && !is_k && !is_v;
    const int h_lo = (is_k ? y : is_v ? y - a.g_k : y - a.g_k - a.g_v) * a.hpw;
    const int h_hi = imin(h_lo + a.hpw, is_k ? a.n_k : is_v ? a.n_v : a.n_q);
    const int half = a.n_rot / 2;
    int r0, n_rows;
    RowPlace at;
    if (!find_block<L::LOG2_R>(a.p, blockIdx.x, r0, n_rows, at)) return;

    f32x4 x[NI][2];
    auto load = [&](int h) {
#pragma unroll
        for (int it = 0; it < NI; ++it) {
            const int row = r0 + imin(w * (R / 4) + it * L::RPI + sub, n_rows - 1);
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                const int d = 4 * li + H2 * v;
                if (is_q)
                    x[it][v] = load4(a.q + row * a.q_row_stride + h * a.q_head_stride + d);
                else
                    x[it][v] = load4(static_cast<const SRC*>(is_k ? a.k_new : a.v_new) + row * a.row_stride + h * HD + d);
            }
        }
    };
    load(h_lo);
    if (PRO && !is_v) {
        for (int i = tid; i < half; i += 256) freq_s[i] = freq_of(a, i);
        __syncthreads();
        // a thread keeps to one row: the rows that exist, rounded up to a power of two, side by side
        int rl2 = 0;
        while ((1 << rl2) < n_rows) ++rl2;
        const int row = tid & ((1 << rl2) - 1);
        const double pos = (double)__shfl(at.pos, row, 64);
        for (int i = tid >> rl2; i < half; i += 256 >> rl2) {
            float c, s;
            turn_of(pos * freq_s[i], c, s);
            turn[row * H2 + i] = make_float2(c, s);
        }
        __syncthreads();
    }
    Granules gr;
    gr.of(at, n_rows);

    for (int h = h_lo; h < h_hi; ++h) {
        if (h > h_lo) load(h);
#pragma unroll
        for (int it = 0; it < NI; ++it) {
            const int rl = w * (R / 4) + it * L::RPI + sub;  // row within the workgroup
            if (w * (R / 4) + it * L::RPI >= n_rows) break;  // uniform: none of these rows exists
            f32x4(&e)[2] = x[it];
            if constexpr (PRO) {
                const float* gain = is_v ? nullptr : is_k ? a.k_gain : a.q_gain;
                if (is_v ? a.v_norm != 0 : gain != nullptr) norm_row<LPR, HD>(e, gain, a.eps, li);
                if (!is_v && half == H2) {
                    const f32x4* t = reinterpret_cast<const f32x4*>(&turn[rl * H2 + 4 * li]);
                    const f32x4 t0 = t[0], t1 = t[1];
                    turn_row(e, {t0[0], t0[2], t1[0], t1[2]}, {t0[1], t0[3], t1[1], t1[3]});
                } else if (!is_v && half) {
                    turn_part<HD>(e, rows_s[w] + sub * HD, li, half, [&](int i) { return turn[rl * H2 + i]; });
                }
                if (is_q) {
                    if (rl < n_rows) {
                        const size_t o = ((size_t)(r0 + rl) * a.n_q + h) * HD + 4 * li;
#pragma unroll
                        for (int v = 0; v < 2; ++v) {
                            if (a.q_out_f16)
                                store4(static_cast<f16*>(a.q_out) + o + H2 * v, e[v]);
                            else
                                store4(static_cast<float*>(a.q_out) + o + H2 * v, e[v]);
                        }
                    }
                    continue;
                }
            }
            const int page = __shfl(at.page, rl, 64), slot = __shfl(at.slot, rl, 64);
            const bool live = rl < n_rows && page >= 0;
            uint32_t bytes[2];
            if constexpr (I8) {
                const float s = scale_of(row_amax<LPR>(e));
                if (live && li == 0) (is_k ? a.p.k_scale : a.p.v_scale)[scale_offset(a.p, page, h, slot)] = s;
                quantize8(e, s, s > 0.f ? 1.f / s : 0.f, bytes);  // NaN compares false
            }
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                const int d = 4 * li + H2 * v;
                if constexpr (I8) {
                    if (is_v)
                        vt[rl * VT::P + d / 4] = bytes[v];
                    else if (live)
                        *reinterpret_cast<uint32_t*>(a.p.k + k_offset(a.p, page, h, slot) + d) = bytes[v];
                } else if (is_v) {
                    vt[rl * VT::P + d / 2] = __builtin_bit_cast(uint32_t, f16x2{(f16)e[v][0], (f16)e[v][1]});
                    vt[rl * VT::P + d / 2 + 1] = __builtin_bit_cast(uint32_t, f16x2{(f16)e[v][2], (f16)e[v][3]});
                } else if (live) {
                    store4(reinterpret_cast<f16*>(a.p.k) + k_offset(a.p, page, h, slot) + d, e[v]);
                }
            }
        }
        if (!is_v) continue;  // uniform
        __syncthreads();
        for (int i0 = 0; i0 < VT::W * gr.count; i0 += 256) {
            const int i = i0 + tid, word = i % VT::W, g = i / VT::W, t0 = gr.first + 16 * g;
            const int row = imin(imax(t0, 0), R - 1);
            const int page = __shfl(at.page, row, 64), slot = __shfl(at.slot, row, 64);
            if (g >= gr.count || !gr.full(g, n_rows) || page < 0) continue;
            char* col = a.p.v + (v_offset(a.p, page, h, slot) + ((size_t)(word * VT::DW) << a.p.g.ps_log2)) * sizeof(DT);
            const uint32_t* src = vt + t0 * VT::P + word;
            const size_t step = sizeof(DT) << a.p.g.ps_log2;  // bytes from a dim to the next
            if constexpr (I8) {
                uint32_t o[4][4];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const uint32_t in[4] = {src[(4 * q) * VT::P], src[(4 * q + 1) * VT::P], src[(4 * q + 2) * VT::P], src[(4 * q + 3) * VT::P]};
                    uint32_t t[4];
                    turn4(in, t);
#pragma unroll
                    for (int d = 0; d < 4; ++d) o[d][q] = t[d];
                }
#pragma unroll
                for (int d = 0; d < 4; ++d)
                    *reinterpret_cast<uint4*>(col + d * step) = uint4{o[d][0], o[d][1], o[d][2], o[d][3]};
            } else {
                uint32_t o[2][8];
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    const uint32_t b0 = src[(2 * q) * VT::P], b1 = src[(2 * q + 1) * VT::P];
                    o[0][q] = __builtin_amdgcn_perm(b1, b0, 0x05040100u);
                    o[1][q] = __builtin_amdgcn_perm(b1, b0, 0x07060302u);
                }
#pragma unroll
                for (int d = 0; d < 2; ++d) {
                    *reinterpret_cast<uint4*>(col + d * step) = uint4{o[d][0], o[d][1], o[d][2], o[d][3]};
                    *reinterpret_cast<uint4*>(col + d * step + 16) = uint4{o[d][4], o[d][5], o[d][6], o[d][7]};
                }
            }
        }
        const int tok = lane & (R - 1);
        const bool single = tok < n_rows && at.page >= 0 && !gr.full_row(tok, n_rows);
        if (__ballot(single)) {
            constexpr int DPI = 64 / R;  // dims a wave at once
            DT* col = column(reinterpret_cast<DT*>(a.p.v), a.p, imax(at.page, 0), h, at.slot, w * DPI + lane / R);
            const size_t step = (size_t)(4 * DPI) << a.p.g.ps_log2;
            if (single)
#pragma unroll 8
                for (int i = 0; i < HD / 4 / DPI; ++i, col += step)
                    *col = reinterpret_cast<const DT*>(vt + tok * VT::P)[(i * 4 + w) * DPI + lane / R];
        }
        __syncthreads();  // the next head's rows go where these are
    }
}

// Single tokens: a row head is LPR lanes of a wave, from load to store; no LDS
// but for a partial turn, V's column element by element.
template <typename SRC, bool I8, int HD, bool PRO>
__global__ __launch_bounds__(256) void paged_store_tokens_kernel(StoreArgs a) {
    using L = RowLanes<HD>;
    using DT = std::conditional_t<I8, int8_t, f16>;
    constexpr int LPR = L::LPR, RPI = L::RPI, H2 = HD / 2;
    __shared__ __align__(16) float rows_s[PRO ? 4 : 1][PRO ? 512 : 4];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int sub = lane / LPR, li = lane % LPR;
    const int heads = a.n_k + a.n_v + a.n_q;
    const int64_t units = (int64_t)a.p.g.n_tokens * heads, u0 = ((int64_t)blockIdx.x * 4 + w) * RPI;
    if (u0 >= units) return;  // uniform; no barrier below
    const int64_t u = u0 + sub < units ? u0 + sub : units - 1;
    const bool have = u0 + sub < units;
    const int row = (int)(u / heads), head = (int)(u % heads);
    const bool is_k = head < a.n_k, is_v = !is_k && head < a.n_k + a.n_v, is_q = !is_k && !is_v;
    const int h = is_k ? head : is_v ? head - a.n_k : head - a.n_k - a.n_v;
    f32x4 e[2];
#pragma unroll
    for (int v = 0; v < 2; ++v) {
        const int d = 4 * li + H2 * v;
        if (PRO && is_q)
            e[v] = load4(a.q + row * a.q_row_stride + h * a.q_head_stride + d);
        else
            e[v] = load4(static_cast<const SRC*>(is_k ? a.k_new : a.v_new) + row * a.row_stride + h * HD + d);
    }
    const int64_t u1 = u0 + RPI - 1 < units ? u0 + RPI - 1 : units - 1;
    const RowPlace at = locate_row(a.p, row, (int)(u0 / heads), (int)(u1 / heads));
    if constexpr (PRO) {
        const int half = a.n_rot / 2;
        const float* gain = is_k ? a.k_gain : is_q ? a.q_gain : nullptr;
        // the lanes of a row agree; all lanes of the wave take part in the sums
        f32x4 n[2] = {e[0], e[1]};
        norm_row<LPR, HD>(n, gain, a.eps, li);
        if (is_v ? a.v_norm != 0 : gain != nullptr) {
            e[0] = n[0];
            e[1] = n[1];
        }
        if (half == H2) {
            float c[4], s[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) turn_of((double)at.pos * freq_of(a, 4 * li + j), c[j], s[j]);
            if (!is_v) turn_row(e, c, s);
        } else if (half) {
            n[0] = e[0];
            n[1] = e[1];
            turn_part<HD>(n, rows_s[w] + sub * HD, li, half, [&](int i) {
                float2 t;
                turn_of((double)at.pos * freq_of(a, i), t.x, t.y);
                return t;
            });
            if (!is_v) {
                e[0] = n[0];
                e[1] = n[1];
            }
        }
    }
    if (PRO && is_q) {
        if (have && at.seq >= 0) {
            const size_t o = ((size_t)row * a.n_q + h) * HD + 4 * li;
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                if (a.q_out_f16)
                    store4(static_cast<f16*>(a.q_out) + o + H2 * v, e[v]);
                else
                    store4(static_cast<float*>(a.q_out) + o + H2 * v, e[v]);
            }
        }
    }
    uint32_t bytes[2];
    float s = 0.f;
    if constexpr (I8) {
        s = scale_of(row_amax<LPR>(e));
        quantize8(e, s, s > 0.f ? 1.f / s : 0.f, bytes);  // NaN compares false
    }
    if (!have || at.page < 0 || is_q) return;
    if (I8 && li == 0) (is_k ? a.p.k_scale : a.p.v_scale)[scale_offset(a.p, at.page, h, at.slot)] = s;
#pragma unroll
    for (int v = 0; v < 2; ++v) {
        const int d = 4 * li + H2 * v;
        if (is_k) {
            DT* dst = reinterpret_cast<DT*>(a.p.k) + k_offset(a.p, at.page, h, at.slot) + d;
            if constexpr (I8) *reinterpret_cast<uint32_t*>(dst) = bytes[v];
            else store4(dst, e[v]);
        } else {
            DT* dst = reinterpret_cast<DT*>(a.p.v) + v_offset(a.p, at.page, h, at.slot) + ((size_t)d << a.p.g.ps_log2);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (I8) dst[(size_t)j << a.p.g.ps_log2] = (int8_t)(bytes[v] >> (8 * j));
                else dst[(size_t)j << a.p.g.ps_log2] = (f16)e[v][j];
            }
        }
    }
}

struct ReadArgs {
    PagedArgs p;
    void* k_out;
    void* v_out;
    size_t row_stride;
    int n_k, n_v, g_k, g_v, hpw;  // heads, groups of hpw heads (a workgroup each)
};

template <typename OUT, bool I8, int HD>
__global__ __launch_bounds__(256) void paged_read_kernel(ReadArgs a) {
    using L = RowLanes<HD>;
    using VT = VTile<HD, I8>;
    using DT = std::conditional_t<I8, int8_t, f16>;
    using KW = std::conditional_t<I8, uint32_t, uint2>;  // four dims
    constexpr int R = L::R, NI = L::NI, LPR = L::LPR, H2 = HD / 2;
    // granules a thread takes: the rows touch R / 16 + 1 of them at most
    constexpr int NG = (VT::W * (R / 16 + 1) + 255) / 256, GD = VT::DW, GQ = I8 ? 1 : 2;
    __shared__ __align__(16) uint32_t vt[VT::BYTES / 4];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int sub = lane / LPR, li = lane % LPR;
    const int y = blockIdx.y;
    const bool is_k = y < a.g_k;
    const int h_lo = (is_k ? y : y - a.g_k) * a.hpw, h_hi = imin(h_lo + a.hpw, is_k ? a.n_k : a.n_v);
    int r0, n_rows;
    RowPlace at;
    if (!find_block<L::LOG2_R>(a.p, blockIdx.x, r0, n_rows, at)) return;
    Granules gr;
    gr.of(at, n_rows);

    int pages[NI], slots[NI];
    bool own[NI];
#pragma unroll
    for (int it = 0; it < NI; ++it) {
        const int rl = w * (R / 4) + it * L::RPI + sub;
        pages[it] = __shfl(at.page, rl, 64);
        slots[it] = __shfl(at.slot, rl, 64);
        own[it] = rl < n_rows;
    }
    // Of the thread's granules, -1: none.  One at a ragged end is read whole
    // too, and the rows that are not the batch's left out.
    int g_page[NG], g_slot[NG];
#pragma unroll
    for (int n = 0; n < NG; ++n) {
        const int g = (tid + 256 * n) / VT::W, row = imin(imax(gr.first + 16 * g, 0), R - 1);
        g_page[n] = __shfl(at.page, row, 64);
        g_slot[n] = __shfl(at.slot, row, 64) & ~15;
        if (g >= gr.count) g_page[n] = -1;
    }
    KW rk[NI][2];
    uint4 rv[NG][GD][GQ];
    float rs[NI];
    auto load = [&](int h) {  // pages that are none read page 0; their rows are written as zeros
        if (I8)
#pragma unroll
            for (int it = 0; it < NI; ++it)
                rs[it] = (is_k ? a.p.k_scale : a.p.v_scale)[scale_offset(a.p, imax(pages[it], 0), h, slots[it])];
        if (is_k) {
#pragma unroll
            for (int it = 0; it < NI; ++it)
#pragma unroll
                for (int v = 0; v < 2; ++v)
                    rk[it][v] = *reinterpret_cast<const KW*>(
                        a.p.k + (k_offset(a.p, imax(pages[it], 0), h, slots[it]) + 4 * li + H2 * v) * sizeof(DT));
        } else {
#pragma unroll
            for (int n = 0; n < NG; ++n)
                if (g_page[n] >= 0) {
                    const char* col = a.p.v + (v_offset(a.p, g_page[n], h, g_slot[n]) +
                                               ((size_t)((tid + 256 * n) % VT::W * GD) << a.p.g.ps_log2)) * sizeof(DT);
#pragma unroll
                    for (int d = 0; d < GD; ++d)
#pragma unroll
                        for (int k = 0; k < GQ; ++k)
                            rv[n][d][k] = *reinterpret_cast<const uint4*>(col + d * (sizeof(DT) << a.p.g.ps_log2) + 16 * k);
                }
        }
    };
    load(h_lo);
    OUT* out = static_cast<OUT*>(is_k ? a.k_out : a.v_out);
    for (int h = h_lo; h < h_hi; ++h) {
        if (!is_k) {
#pragma unroll
            for (int n = 0; n < NG; ++n)
                if (g_page[n] >= 0) {
                    const int i = tid + 256 * n;
                    const int t0 = gr.first + 16 * (i / VT::W);
                    uint32_t* dst = vt + t0 * VT::P + i % VT::W;
                    const bool full = t0 >= 0 && t0 + 16 <= R;
                    auto put = [&](int t, uint32_t x) {
                        if (full || (t0 + t >= 0 && t0 + t < R)) dst[t * VT::P] = x;
                    };
                    if constexpr (I8) {
                        const uint32_t x[4][4] = {{rv[n][0][0].x, rv[n][0][0].y, rv[n][0][0].z, rv[n][0][0].w},
                                                  {rv[n][1][0].x, rv[n][1][0].y, rv[n][1][0].z, rv[n][1][0].w},
                                                  {rv[n][2][0].x, rv[n][2][0].y, rv[n][2][0].z, rv[n][2][0].w},
                                                  {rv[n][3][0].x, rv[n][3][0].y, rv[n][3][0].z, rv[n][3][0].w}};
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const uint32_t in[4] = {x[0][q], x[1][q], x[2][q], x[3][q]};
                            uint32_t t[4];
                            turn4(in, t);
#pragma unroll
                            for (int j = 0; j < 4; ++j) put(4 * q + j, t[j]);
                        }
                    } else {
#pragma unroll
                        for (int k = 0; k < GQ; ++k) {
                            const uint32_t x[2][4] = {{rv[n][0][k].x, rv[n][0][k].y, rv[n][0][k].z, rv[n][0][k].w},
                                                      {rv[n][1][k].x, rv[n][1][k].y, rv[n][1][k].z, rv[n][1][k].w}};
#pragma unroll
                            for (int q = 0; q < 4; ++q) {
                                put(8 * k + 2 * q, __builtin_amdgcn_perm(x[1][q], x[0][q], 0x05040100u));
                                put(8 * k + 2 * q + 1, __builtin_amdgcn_perm(x[1][q], x[0][q], 0x07060302u));
                            }
                        }
                    }
                }
            __syncthreads();
        }
        KW zk[NI][2];
        float zs[NI];
#pragma unroll
        for (int it = 0; it < NI; ++it) {
            zk[it][0] = rk[it][0];
            zk[it][1] = rk[it][1];
            zs[it] = rs[it];
        }
        if (h + 1 < h_hi) load(h + 1);
#pragma unroll
        for (int it = 0; it < NI; ++it) {
            const int rl = w * (R / 4) + it * L::RPI + sub;
            if (!own[it]) continue;
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                const int d = 4 * li + H2 * v;
                KW b;
                if (is_k) {
                    b = zk[it][v];
                } else {
                    const uint32_t* src = &vt[rl * VT::P + d / VT::DW];
                    if constexpr (I8) b = src[0];
                    else b = uint2{src[0], src[1]};
                }
                f32x4 y = {0.f, 0.f, 0.f, 0.f};
                if (pages[it] >= 0) {
                    if constexpr (I8) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) y[j] = zs[it] * (float)(int8_t)(b >> (8 * j));
                    } else {
                        const f16x2 lo = __builtin_bit_cast(f16x2, b.x), hi = __builtin_bit_cast(f16x2, b.y);
                        y = f32x4{(float)lo[0], (float)lo[1], (float)hi[0], (float)hi[1]};
                    }
                }
                store4(out + (size_t)(r0 + rl) * a.row_stride + h * HD + d, y);
            }
        }
        if (!is_k) __syncthreads();
    }
}

// Heads a workgroup that makes its rows' angles once for them; short batches
// take a head each, so that the heads run side by side.  5407 rows of 32 heads:
// 1, 2, 4, 8 heads 98, 82, 79, 82 us; 1024 rows one head 17.8, four 20.5; 2048
// rows one head 25.6, four 23.9.
static int heads_a_group(uint32_t n_tokens) { return n_tokens <= 1024 ? 1 : 4; }
// A grid that the launch can name: 256 threads a workgroup in 32 bits, and 16 bits across.
static bool grid_fits(int64_t x, int64_t y) { return x < (1 << 24) && y < (1 << 16); }
// Batches of few rows a sequence: whole granules are rare, and a block of rows
// would be a row or two.  One row: append 4.0 us a kernel against 6.2, prologue
// 4.4 against 12.6; four rows: 15.4 us a prologue call on either.
static bool few_rows(const PagedGeom& g) { return g.max_new <= 4; }

template <bool PRO, typename SRC, bool I8>
static lmx_status launch_store_hd(const StoreArgs& a, int hd, hipStream_t st) {
    auto go = [&](auto tag) {
        constexpr int HD = decltype(tag)::value;
        using L = RowLanes<HD>;
        if (few_rows(a.p.g)) {
            const int64_t units = (int64_t)a.p.g.n_tokens * (a.n_k + a.n_v + a.n_q);
            const int64_t x = (units + 4 * L::RPI - 1) / (4 * L::RPI);
            if (!grid_fits(x, 1)) return LMX_E_SHAPE;
            hipLaunchKernelGGL((paged_store_tokens_kernel<SRC, I8, HD, PRO>), dim3((unsigned)x), dim3(256), 0, st, a);
        } else {
            const int64_t x = row_blocks_bound(a.p.g, L::LOG2_R), y = a.g_k + a.g_v + a.g_q;
            if (!grid_fits(x, y)) return LMX_E_SHAPE;
            hipLaunchKernelGGL((paged_store_kernel<SRC, I8, HD, PRO>), dim3((unsigned)x, (unsigned)y), dim3(256), 0, st, a);
        }
        LMX_CHECK_LAUNCH();
        return LMX_OK;
    };
    switch (hd) {
        case 64: return go(std::integral_constant<int, 64>{});
        case 128: return go(std::integral_constant<int, 128>{});
        case 256: return go(std::integral_constant<int, 256>{});
        default: return go(std::integral_constant<int, 512>{});
    }
}

lmx_status paged_append(const lmxp_pool* p, const lmxp_batch* b, const void* k_new, const void* v_new,
                        lmx_dtype src_dt, uint32_t row_stride, hipStream_t st) {
    StoreArgs a{};
    a.p = paged_args(p, b);
    a.k_new = k_new;
    a.v_new = v_new;
    a.row_stride = row_stride ? row_stride : (size_t)p->n_kv_heads * p->head_dim;
    a.n_k = k_new ? (int)p->n_kv_heads : 0;
    a.n_v = v_new ? (int)p->n_kv_heads : 0;
    a.hpw = 1;
    a.g_k = a.n_k;
    a.g_v = a.n_v;
    (void)hipGetLastError();
    const bool i8 = p->store == LMXP_I8;
    const int hd = (int)p->head_dim;
    if (src_dt == LMX_F32)
        return i8 ? launch_store_hd<false, float, true>(a, hd, st) : launch_store_hd<false, float, false>(a, hd, st);
    return i8 ? launch_store_hd<false, f16, true>(a, hd, st) : launch_store_hd<false, f16, false>(a, hd, st);
}

lmx_status paged_prologue(const lmxp_pool* p, const lmxp_batch* b, const lmxp_prologue_desc* d, const float* q,
                          const float* k_new, const float* v_new, const float* q_gain, const float* k_gain,
                          const float* factors, void* q_out, lmx_dtype q_out_dt, hipStream_t st) {
    StoreArgs a{};
    a.p = paged_args(p, b);
    a.k_new = k_new;
    a.v_new = v_new;
    a.row_stride = d->kv_row_stride ? d->kv_row_stride : (size_t)p->n_kv_heads * p->head_dim;
    a.n_k = a.n_v = (int)p->n_kv_heads;
    a.n_q = (int)d->n_heads;
    a.q = q;
    a.q_out = q_out;
    a.q_head_stride = d->q_head_stride ? d->q_head_stride : p->head_dim;
    a.q_row_stride = d->q_row_stride ? d->q_row_stride : a.q_head_stride * d->n_heads;
    a.q_gain = q_gain;
    a.k_gain = k_gain;
    a.factors = factors;
    a.n_rot = (int)d->n_rot;
    a.v_norm = (int)d->v_norm;
    a.q_out_f16 = q_out_dt == LMX_F16;
    a.eps = d->rms_eps;
    double s = d->n_rot ? std::pow((double)d->rope_base, -2.0 / (double)d->n_rot) : 1.0;
    for (int k = 0; k < 8; ++k, s *= s) a.scale_pow[k] = s;
    a.hpw = heads_a_group(b->n_tokens);
    a.g_k = (a.n_k + a.hpw - 1) / a.hpw;
    a.g_v = (a.n_v + a.hpw - 1) / a.hpw;
    a.g_q = (a.n_q + a.hpw - 1) / a.hpw;
    (void)hipGetLastError();
    const int hd = (int)p->head_dim;
    return p->store == LMXP_I8 ? launch_store_hd<true, float, true>(a, hd, st)
                               : launch_store_hd<true, float, false>(a, hd, st);
}

template <typename OUT, bool I8>
static lmx_status launch_read(const ReadArgs& a, int hd, hipStream_t st) {
    auto go = [&](auto tag) {
        constexpr int HD = decltype(tag)::value;
        const int64_t x = row_blocks_bound(a.p.g, RowLanes<HD>::LOG2_R), y = a.g_k + a.g_v;
        if (!grid_fits(x, y)) return LMX_E_SHAPE;
        hipLaunchKernelGGL((paged_read_kernel<OUT, I8, HD>), dim3((unsigned)x, (unsigned)y), dim3(256), 0, st, a);
        LMX_CHECK_LAUNCH();
        return LMX_OK;
    };
    switch (hd) {
        case 64: return go(std::integral_constant<int, 64>{});
        case 128: return go(std::integral_constant<int, 128>{});
        case 256: return go(std::integral_constant<int, 256>{});
        default: return go(std::integral_constant<int, 512>{});
    }
}

lmx_status paged_read(const lmxp_pool* p, const lmxp_batch* b, void* k_out, void* v_out, lmx_dtype out_dt,
                      uint32_t row_stride, hipStream_t st) {
    ReadArgs a{};
    a.p = paged_args(p, b);
    a.k_out = k_out;
    a.v_out = v_out;
    a.row_stride = row_stride ? row_stride : (size_t)p->n_kv_heads * p->head_dim;
    a.n_k = k_out ? (int)p->n_kv_heads : 0;
    a.n_v = v_out ? (int)p->n_kv_heads : 0;
    // the second head's loads go out beside the first's stores (to 2048 rows no difference)
    a.hpw = b->n_tokens <= 1024 ? 1 : 2;
    a.g_k = (a.n_k + a.hpw - 1) / a.hpw;
    a.g_v = (a.n_v + a.hpw - 1) / a.hpw;
    (void)hipGetLastError();
    const bool i8 = p->store == LMXP_I8;
    const int hd = (int)p->head_dim;
    if (out_dt == LMX_F32) return i8 ? launch_read<float, true>(a, hd, st) : launch_read<float, false>(a, hd, st);
    return i8 ? launch_read<f16, true>(a, hd, st) : launch_read<f16, false>(a, hd, st);
}

}  // namespace lmx
