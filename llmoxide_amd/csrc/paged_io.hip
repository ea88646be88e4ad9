// Writes into and reads from the paged KV cache on gfx950: append, prologue
// (norm, rotate, store) and read-back.
//
// All three move rows [token, head, dim] to or from pages where K keeps its
// rows and V lies transposed, [dim, slot].  A workgroup takes R consecutive
// rows of the batch and one head at a time.  K goes straight between memory
// and registers, a row across 16-64 lanes, 16 bytes of f32 a lane.  V turns
// in LDS: rows go in, columns come out with lane = row, so that the lanes of
// a store are neighbouring slots of one dim (R * 2 bytes together in f16).
// Attention reads V's operand fragments straight from such columns, which is
// what the transposed layout is for; the price is paid here once a row.
#include <cmath>

#include "paged.hpp"

namespace lmx {

template <int HD>
struct RowLanes {
    static constexpr int LPR = HD >= 256 ? 64 : HD / 4;  // lanes a row
    static constexpr int VPL = HD / 4 / LPR;             // float4s a lane
    static constexpr int RPI = 64 / LPR;                 // rows a wave at once
    static constexpr int R = HD <= 128 ? 64 : HD == 256 ? 32 : 16;  // rows a workgroup
    static constexpr int NI = R / 4 / RPI;               // a wave's turns over its rows
};

template <int LPR>
__device__ __forceinline__ float sum_row(float x) {
    if constexpr (LPR == 64) return wave_sum64(x);
    x = row_sum16(x);
    if constexpr (LPR == 32) x += shfl_xor(x, 16);
    return x;
}
template <int LPR>
__device__ __forceinline__ uint32_t max_row(uint32_t x) {
#pragma unroll
    for (int m = 1; m < LPR; m <<= 1) {
        const uint32_t y = (uint32_t)__shfl_xor((int)x, m, 64);
        x = x > y ? x : y;
    }
    return x;
}

// The 8-bit scale of a row from the largest |x|'s bits (which order as the
// magnitudes do, NaN above infinity above all numbers): amax / 127, correctly
// rounded; 0 below 2^-100, so that 1 / scale below is finite; NaN for a row
// that holds an infinity or a NaN.
__device__ __forceinline__ float scale_of(uint32_t amax_bits) {
    if (amax_bits >= 0x7f800000u) return __builtin_nanf("");
    const float amax = __builtin_bit_cast(float, amax_bits);
    return amax < 0x1p-100f ? 0.f : amax / 127.f;
}
// x / s rounded to the nearest integer, ties to even, from the exact quotient.
// k = rint(x * inv) is off by one at most, and where the product rounds across
// a half.  x - k s is exact in f32 (|x - k s| is near s / 2 and a multiple of
// the smaller of x's and s's last places), so comparing it with s / 2 settles
// the border.  inv = 0 (scale 0 or NaN) gives 0.
__device__ __forceinline__ int quantize(float x, float s, float inv) {
    if (inv == 0.f) return 0;
    float k = rintf(x * inv);
    const float r = fmaf(-k, s, x), h = 0.5f * s;
    const bool odd = ((int)k) & 1;
    if (r > h || (r == h && odd)) k += 1.f;
    if (r < -h || (r == -h && odd)) k -= 1.f;
    return (int)fminf(fmaxf(k, -127.f), 127.f);
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

struct StoreArgs {
    PagedArgs p;
    const void* k_new;
    const void* v_new;
    size_t row_stride;  // elements
    int n_k, n_v, n_q;  // heads to take: K heads, V heads, then query heads
    int hpw;            // heads a workgroup
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

// PRO: norm and rotate on the way, and take the query heads too.
template <typename SRC, bool I8, int HD, bool PRO>
__global__ __launch_bounds__(256) void paged_store_kernel(StoreArgs a) {
    using L = RowLanes<HD>;
    using DT = std::conditional_t<I8, int8_t, f16>;
    constexpr int R = L::R, VPL = L::VPL, NI = L::NI, LPR = L::LPR;
    constexpr int VP = HD + (I8 ? 4 : 2);  // an odd number of words a row: columns spread over the banks
    __shared__ __align__(16) DT vt[R][VP];
    __shared__ float2 turn[PRO ? R : 1][PRO ? HD / 2 : 1];
    __shared__ __align__(16) float rows_s[PRO ? 4 : 1][PRO ? 256 * VPL : 1];
    __shared__ double freq_s[PRO ? HD / 2 : 1];

    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int sub = lane / LPR, li = lane % LPR;
    const int r0 = blockIdx.x * R, last = imin(r0 + R, a.p.g.n_tokens) - 1;
    const int first_head = blockIdx.y * a.hpw, heads = a.n_k + a.n_v + a.n_q;
    const int end_head = imin(first_head + a.hpw, heads);
    const int half = a.n_rot / 2;

    if constexpr (PRO) {
        for (int i = tid; i < half; i += 256) {
            double f = 1.0;  // s^i by the bits of i (i < 256)
#pragma unroll
            for (int k = 0; k < 8; ++k) f *= (i >> k) & 1 ? a.scale_pow[k] : 1.0;
            freq_s[i] = a.factors ? f / (double)a.factors[i] : f;
        }
    }
    const RowPlace at = locate_row(a.p, r0 + (lane & (R - 1)), r0, last);
    if constexpr (PRO) {
        __syncthreads();
        // lane & (R-1) = row: each thread fills its own row's angles
        for (int i = tid / R; i < half; i += 256 / R) {
            float c, s;
            turn_of((double)at.pos * freq_s[i], c, s);
            turn[lane & (R - 1)][i] = make_float2(c, s);
        }
        __syncthreads();
    }

    for (int head = first_head; head < end_head; ++head) {
        const bool is_k = head < a.n_k, is_v = !is_k && head < a.n_k + a.n_v;
        const int h = is_k ? head : is_v ? head - a.n_k : head - a.n_k - a.n_v;
        f32x4 x[NI][VPL];
#pragma unroll
        for (int it = 0; it < NI; ++it) {
            const int row = imin(r0 + w * (R / 4) + it * L::RPI + sub, last);
#pragma unroll
            for (int v = 0; v < VPL; ++v) {
                const int d = 4 * li + 256 * v;
                if (PRO && !is_k && !is_v)
                    x[it][v] = load4(a.q + row * a.q_row_stride + h * a.q_head_stride + d);
                else
                    x[it][v] = load4(static_cast<const SRC*>(is_k ? a.k_new : a.v_new) + row * a.row_stride + h * HD + d);
            }
        }
#pragma unroll
        for (int it = 0; it < NI; ++it) {
            const int rl = w * (R / 4) + it * L::RPI + sub;  // row within the workgroup
            if (r0 + w * (R / 4) + it * L::RPI > last) break;  // uniform: none of these rows exists
            f32x4* y = x[it];
            if constexpr (PRO) {
                const float* gain = is_v ? nullptr : is_k ? a.k_gain : a.q_gain;
                if (is_v ? a.v_norm != 0 : gain != nullptr) {
                    float ss = 0.f;
#pragma unroll
                    for (int v = 0; v < VPL; ++v)
#pragma unroll
                        for (int j = 0; j < 4; ++j) ss = fmaf(y[v][j], y[v][j], ss);
                    const float sc = __builtin_amdgcn_rsqf(sum_row<LPR>(ss) / (float)HD + a.eps);
#pragma unroll
                    for (int v = 0; v < VPL; ++v) {
                        const f32x4 g = gain ? load4(gain + 4 * li + 256 * v) : f32x4{1.f, 1.f, 1.f, 1.f};
#pragma unroll
                        for (int j = 0; j < 4; ++j) y[v][j] = y[v][j] * sc * g[j];
                    }
                }
                if (!is_v && half) {
                    // the partner of dim d is d +- half, in another lane as a rule: through LDS
                    float* rs = rows_s[w] + sub * HD;
#pragma unroll
                    for (int v = 0; v < VPL; ++v) store4(rs + 4 * li + 256 * v, y[v]);
                    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
                    __builtin_amdgcn_wave_barrier();
                    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
                    for (int v = 0; v < VPL; ++v)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int d = 4 * li + 256 * v + j;
                            if (d < a.n_rot) {
                                const bool lo = d < half;
                                const float2 t = turn[rl][lo ? d : d - half];
                                const float o = rs[lo ? d + half : d - half];
                                y[v][j] = y[v][j] * t.x + (lo ? -o : o) * t.y;
                            }
                        }
                    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
                    __builtin_amdgcn_wave_barrier();
                    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
                }
                if (!is_k && !is_v) {
                    const int owned = __shfl((int)at.owned, rl & (R - 1), 64);
                    if (r0 + rl <= last && owned) {
                        const size_t o = ((size_t)(r0 + rl) * a.n_q + h) * HD + 4 * li;
#pragma unroll
                        for (int v = 0; v < VPL; ++v) {
                            if (a.q_out_f16)
                                store4(static_cast<f16*>(a.q_out) + o + 256 * v, y[v]);
                            else
                                store4(static_cast<float*>(a.q_out) + o + 256 * v, y[v]);
                        }
                    }
                    continue;
                }
            }
            const int page = __shfl(at.page, rl, 64), slot = __shfl(at.slot, rl, 64);
            const bool live = r0 + rl <= last && page >= 0;
            float s = 0.f, inv = 0.f;
            if constexpr (I8) {
                uint32_t m = 0;
#pragma unroll
                for (int v = 0; v < VPL; ++v)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float e = y[v][j];
                        const uint32_t u = __builtin_bit_cast(uint32_t, e) & 0x7fffffffu;
                        m = m > u ? m : u;
                    }
                s = scale_of(max_row<LPR>(m));
                inv = s > 0.f ? 1.f / s : 0.f;  // NaN compares false
                if (live && li == 0) (is_k ? a.p.k_scale : a.p.v_scale)[scale_offset(a.p, page, h, slot)] = s;
            }
#pragma unroll
            for (int v = 0; v < VPL; ++v) {
                const int d = 4 * li + 256 * v;
                if constexpr (I8) {
                    uint32_t b = 0;
#pragma unroll
                    for (int j = 0; j < 4; ++j) b |= (uint32_t)(quantize(y[v][j], s, inv) & 255) << (8 * j);
                    if (is_v)
                        *reinterpret_cast<uint32_t*>(&vt[rl][d]) = b;
                    else if (live)
                        *reinterpret_cast<uint32_t*>(a.p.k + k_offset(a.p, page, h, slot) + d) = b;
                } else if (is_v) {  // rows of an odd number of words: two 4-byte stores
                    *reinterpret_cast<f16x2*>(&vt[rl][d]) = f16x2{(f16)y[v][0], (f16)y[v][1]};
                    *reinterpret_cast<f16x2*>(&vt[rl][d + 2]) = f16x2{(f16)y[v][2], (f16)y[v][3]};
                } else if (live) {
                    store4(reinterpret_cast<f16*>(a.p.k) + k_offset(a.p, page, h, slot) + d, y[v]);
                }
            }
        }
        if (!is_v) continue;  // uniform
        __syncthreads();
        const int tok = lane & (R - 1);
        if (r0 + tok <= last && at.page >= 0) {
            DT* col = reinterpret_cast<DT*>(a.p.v) + v_offset(a.p, at.page, h, at.slot);
            constexpr int DPI = 64 / R;  // dims a wave at once
#pragma unroll 8
            for (int i = 0; i < HD / 4 / DPI; ++i) {
                const int d = (i * 4 + w) * DPI + lane / R;
                col[(size_t)d << a.p.g.ps_log2] = vt[tok][d];
            }
        }
        __syncthreads();
    }
}

struct ReadArgs {
    PagedArgs p;
    void* k_out;
    void* v_out;
    size_t row_stride;
    int n_k, n_v;
};

template <typename OUT, bool I8, int HD>
__global__ __launch_bounds__(256) void paged_read_kernel(ReadArgs a) {
    using L = RowLanes<HD>;
    using DT = std::conditional_t<I8, int8_t, f16>;
    constexpr int R = L::R, VPL = L::VPL, NI = L::NI, LPR = L::LPR;
    constexpr int VP = HD + (I8 ? 4 : 2);
    __shared__ __align__(16) DT vt[R][VP];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int sub = lane / LPR, li = lane % LPR;
    const int r0 = blockIdx.x * R, last = imin(r0 + R, a.p.g.n_tokens) - 1;
    const int head = blockIdx.y;
    const bool is_k = head < a.n_k;
    const int h = is_k ? head : head - a.n_k;
    const RowPlace at = locate_row(a.p, r0 + (lane & (R - 1)), r0, last);

    if (!is_k) {
        const int tok = lane & (R - 1);
        constexpr int DPI = 64 / R;
        if (at.page >= 0) {
            const DT* col = reinterpret_cast<const DT*>(a.p.v) + v_offset(a.p, at.page, h, at.slot);
#pragma unroll 16
            for (int i = 0; i < HD / 4 / DPI; ++i) {
                const int d = (i * 4 + w) * DPI + lane / R;
                vt[tok][d] = col[(size_t)d << a.p.g.ps_log2];
            }
        }
        __syncthreads();
    }
    OUT* out = static_cast<OUT*>(is_k ? a.k_out : a.v_out);
#pragma unroll
    for (int it = 0; it < NI; ++it) {
        const int rl = w * (R / 4) + it * L::RPI + sub;
        const int page = __shfl(at.page, rl, 64), slot = __shfl(at.slot, rl, 64);
        const int owned = __shfl((int)at.owned, rl, 64);
        if (r0 + rl > last || !owned) continue;
        const float s = I8 && page >= 0 ? (is_k ? a.p.k_scale : a.p.v_scale)[scale_offset(a.p, page, h, slot)] : 1.f;
#pragma unroll
        for (int v = 0; v < VPL; ++v) {
            const int d = 4 * li + 256 * v;
            f32x4 y = {0.f, 0.f, 0.f, 0.f};
            if (page >= 0) {
                if constexpr (I8) {
                    uint32_t b;
                    if (is_k)
                        b = *reinterpret_cast<const uint32_t*>(a.p.k + k_offset(a.p, page, h, slot) + d);
                    else
                        b = *reinterpret_cast<const uint32_t*>(&vt[rl][d]);
#pragma unroll
                    for (int j = 0; j < 4; ++j) y[j] = s * (float)(int8_t)(b >> (8 * j));
                } else if (is_k) {
                    y = load4(reinterpret_cast<const f16*>(a.p.k) + k_offset(a.p, page, h, slot) + d);
                } else {
                    const f16x2 lo = *reinterpret_cast<const f16x2*>(&vt[rl][d]);
                    const f16x2 hi = *reinterpret_cast<const f16x2*>(&vt[rl][d + 2]);
                    y = f32x4{(float)lo[0], (float)lo[1], (float)hi[0], (float)hi[1]};
                }
            }
            store4(out + (size_t)(r0 + rl) * a.row_stride + h * HD + d, y);
        }
    }
}

template <bool PRO, typename SRC, bool I8>
static lmx_status launch_store_hd(const StoreArgs& a, int hd, hipStream_t st) {
    const int heads = a.n_k + a.n_v + a.n_q;
    auto go = [&](auto tag) {
        constexpr int HD = decltype(tag)::value;
        const dim3 grid((a.p.g.n_tokens + RowLanes<HD>::R - 1) / RowLanes<HD>::R, (heads + a.hpw - 1) / a.hpw);
        hipLaunchKernelGGL((paged_store_kernel<SRC, I8, HD, PRO>), grid, dim3(256), 0, st, a);
    };
    switch (hd) {
        case 64: go(std::integral_constant<int, 64>{}); break;
        case 128: go(std::integral_constant<int, 128>{}); break;
        case 256: go(std::integral_constant<int, 256>{}); break;
        default: go(std::integral_constant<int, 512>{}); break;
    }
    LMX_CHECK_LAUNCH();
    return LMX_OK;
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
    a.hpw = b->n_tokens <= 512 ? 1 : 8;
    (void)hipGetLastError();
    const int hd = (int)p->head_dim;
    return p->store == LMXP_I8 ? launch_store_hd<true, float, true>(a, hd, st)
                               : launch_store_hd<true, float, false>(a, hd, st);
}

template <typename OUT, bool I8>
static lmx_status launch_read(const ReadArgs& a, int hd, hipStream_t st) {
    auto go = [&](auto tag) {
        constexpr int HD = decltype(tag)::value;
        const dim3 grid((a.p.g.n_tokens + RowLanes<HD>::R - 1) / RowLanes<HD>::R, a.n_k + a.n_v);
        hipLaunchKernelGGL((paged_read_kernel<OUT, I8, HD>), grid, dim3(256), 0, st, a);
    };
    switch (hd) {
        case 64: go(std::integral_constant<int, 64>{}); break;
        case 128: go(std::integral_constant<int, 128>{}); break;
        case 256: go(std::integral_constant<int, 256>{}); break;
        default: go(std::integral_constant<int, 512>{}); break;
    }
    LMX_CHECK_LAUNCH();
    return LMX_OK;
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
    (void)hipGetLastError();
    const bool i8 = p->store == LMXP_I8;
    const int hd = (int)p->head_dim;
    if (out_dt == LMX_F32) return i8 ? launch_read<float, true>(a, hd, st) : launch_read<float, false>(a, hd, st);
    return i8 ? launch_read<f16, true>(a, hd, st) : launch_read<f16, false>(a, hd, st);
}

}  // namespace lmx
