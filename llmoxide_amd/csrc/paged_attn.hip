// Attention of few query rows (decode) over pages on gfx950, and the merge of
// key splits.
//
// A work item is 16 query rows of one kv head (row r: token r / G, head r % G)
// over one split of the visible keys; a workgroup's four waves take a quarter
// of the split each and join in LDS.  Everything goes from memory to MFMA
// operands without LDS: both products are computed transposed,
//   S^T[key, row] = K Q^T      A = K  (lane: one key, 8 dims)
//   O^T[dim, row] += V^T P^T   A = V^T (lane: one dim, 8 keys), B = P^T
// and v_mfma_f32_16x16x32_f16 leaves S^T with a lane holding one row's scores
// for keys 4g..4g+3 of each 16-key block (g = lane / 16).  Which keys a block
// takes is free, so block j takes keys 8g + 4j + (0..3) of each group g: the
// two blocks of a 32-key tile give a lane 8 consecutive keys, exactly what the
// B operand of the second product and a 16-byte load of a V column want.  8-bit
// tiles are 64 keys in four blocks, 16 consecutive keys a lane.
//
// Softmax: one running reference m per row (log2 units), taken from the first
// tile and moved only when a score passes it by 2^4; weights are
// exp2(s - m + 10) <= 2^14, so f16 holds them, with a residual in a second f16
// (22 bits together); sums are fp32.  An 8-bit V's scale joins the exponent as
// its logarithm, so that what f16 holds are the weights that V's integers meet,
// row by row; the sum takes an exponential without it (log_v_scale).
//
// Bound by HBM: every visible K and V byte once, 4 * G * hd operations for 4 * hd
// bytes of f16 a position and kv head.  The waves share nothing and the
// transposed V makes every load a whole operand, so nothing is staged in LDS.
// Loads run one tile ahead in the registers that the
// tile before leaves; with K's and V's waits counted apart and the four waves'
// tiles side by side (V's 128-byte lines then meet in the caches) an 8-bit step
// of 32 sequences fell from 145 to 110 us and one f16 token over 32k keys from
// 38.9 to 33.9 us.  Measured (128-dim heads, 8 of them for 32 query heads):
//   one token over 32768 f16 keys     34.4 us a call, 3.9 TB/s (25 us + merge 4)
//   32 tokens, 8 bits, 527 MB         112 us, 4.7 TB/s (a copy reaches 5.1)
//   one token over 512 keys           9.6 us a call, the launch and the host
// Counters: profiles/paged_cache.md.
#include <algorithm>

#include "paged_attn.hpp"

namespace lmx {

constexpr int kBM = 16;       // query rows an item
// Weights are exp2(s - m + kLift), and a score may pass m by kSlack before m
// moves: at most 2^14, with the smallest f16 step 2^-34 of a weight at m.
constexpr float kLift = 10.f;
constexpr float kSlack = 4.f;

__device__ __forceinline__ f32x4 mfma16(f16x8 a, f16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
// Maximum over the four lanes (g) that share a row.
__device__ __forceinline__ float max_groups(float x) {
    x = fmaxf(x, shfl_xor(x, 16));
    return fmaxf(x, shfl_xor(x, 32));
}
__device__ __forceinline__ float sum_groups(float x) {
    x += shfl_xor(x, 16);
    return x + shfl_xor(x, 32);
}

// LDS traffic among the lanes of one wave, in program order.
__device__ __forceinline__ void wave_lds_order() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

template <int HD, bool I8>
struct Tile {
    static constexpr int KEYS = I8 ? 64 : 32;
    static constexpr int NB = KEYS / 16;          // 16-key blocks
    static constexpr int GR = KEYS / 16;          // 16-key granules, each in one page
    static constexpr int KL = I8 ? HD / 64 : HD / 32;  // 16-byte K loads a block
    static constexpr int VL = HD / 16;            // 16-byte V loads
    uint4 k[NB][KL];
    uint4 v[VL];
    float ks, vs;                                 // 8-bit: the scales of key t0 + lane
};

// Positions of the pool before the (page, head) block of granule i of a tile;
// a missing page reads page 0, and is masked.
template <int HD, bool I8>
__device__ __forceinline__ size_t granule_base(const AttnPagedArgs& a, const int (&pages)[Tile<HD, I8>::GR], int h, int i) {
    constexpr int GR = Tile<HD, I8>::GR;
    // (Values first, then the choice: a choice among elements makes the array
    // one in memory, which the compiler then keeps in LDS.)
    const int p0 = pages[0], p1 = pages[1];
    int p = i & 1 ? p1 : p0;
    if constexpr (GR == 4) {
        const int p2 = pages[2], p3 = pages[3], q = i & 1 ? p3 : p2;
        p = i & 2 ? q : p;
    }
    return ((size_t)imax(p, 0) * a.p.g.Hkv + h) << a.p.g.ps_log2;
}

// The tile's K operands (and 8-bit scales): the lane's key in block j is
// KEYS/4 * (c/4) + 4j + c%4; those of a lane do not leave a granule.
template <int HD, bool I8>
__device__ __forceinline__ void load_k(const AttnPagedArgs& a, const int (&pages)[Tile<HD, I8>::GR], int h, int t0, Tile<HD, I8>& t) {
    using T = Tile<HD, I8>;
    constexpr int ES = I8 ? 1 : 2, QUART = T::KEYS / 4;
    const int lane = __lane_id(), c = lane & 15, g = lane >> 4, psm = (1 << a.p.g.ps_log2) - 1;
    const size_t kb = granule_base<HD, I8>(a, pages, h, QUART * (c >> 2) / 16);
    const char* kr = a.p.k + (kb + ((t0 + QUART * (c >> 2)) & psm) + (c & 3)) * (HD * ES) + 16 * g;
#pragma unroll
    for (int j = 0; j < T::NB; ++j)
#pragma unroll
        for (int l = 0; l < T::KL; ++l) t.k[j][l] = *reinterpret_cast<const uint4*>(kr + 4 * j * HD * ES + 64 * l);
    if constexpr (I8) {
        const size_t at = granule_base<HD, I8>(a, pages, h, g) + ((t0 + lane) & psm);
        t.ks = a.p.k_scale[at];
        t.vs = a.p.v_scale[at];
    }
}
// Its V operands: the lane's KEYS/4 consecutive keys of dims c, c + 16, ...
template <int HD, bool I8>
__device__ __forceinline__ void load_v(const AttnPagedArgs& a, const int (&pages)[Tile<HD, I8>::GR], int h, int t0, Tile<HD, I8>& t) {
    using T = Tile<HD, I8>;
    constexpr int ES = I8 ? 1 : 2, QUART = T::KEYS / 4;
    const int lane = __lane_id(), c = lane & 15, g = lane >> 4, psm = (1 << a.p.g.ps_log2) - 1;
    const size_t vb = granule_base<HD, I8>(a, pages, h, QUART * g / 16);
    const char* vc = a.p.v + (vb * HD + ((size_t)c << a.p.g.ps_log2) + ((t0 + QUART * g) & psm)) * ES;
    const uint32_t vstep = (16u * ES) << a.p.g.ps_log2;
#pragma unroll
    for (int l = 0; l < T::VL; ++l) t.v[l] = *reinterpret_cast<const uint4*>(vc + l * vstep);
}

// F32: q and out are f32 and q has a residual part.  SEEN: rows see each other by
// a mask, and all of them what lies before them (in their windows).
template <int HD, bool I8, bool F32, bool SEEN>
__global__ __launch_bounds__(256, HD <= 128 ? 2 : 1) void paged_rows_kernel(AttnPagedArgs a) {
    using T = Tile<HD, I8>;
    using QT = std::conditional_t<F32, float, f16>;
    constexpr int KS = HD / 32;   // k-steps of QK
    constexpr int DT = HD / 16;   // 16-dim blocks of the output
    constexpr bool QLDS = HD == 512;
    constexpr int OP = HD + 4;  // floats a row of the exchange (16-byte rows, rows 4 banks apart)
    constexpr size_t kEx = 512 + 4 * 16 * OP * 4, kQ = QLDS ? (F32 ? 2 : 1) * KS * 64 * 16 : 0;
    __shared__ __align__(16) char smem[kEx > kQ ? kEx : kQ];
    // By masks, 8 bits: one exponential a key, exp2(score - m), is the sum's, and times
    // V's scale the weight.  Scales of 2^-90 to 2^100 keep both in range as above.  Eight
    // sequences of 16 rows, us with one and with two exponentials: 128 dims 42.3 and 43.2,
    // 256 dims 80.4 and 82.2; 512 dims, where it spills more registers, f32 queries 191 and
    // 162 (f16 queries 160 and 158).
    constexpr bool LEAN = I8 && SEEN && HD <= 256;
    __shared__ __align__(16) float scales[I8 ? 4 : 1][LEAN ? 3 : 2][64];  // a wave's: K's, log2 of V's, LEAN: V's
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 15, g = lane >> 4;

    Item it;
    if (!find_item(a, blockIdx.x, kBM, true, false, it)) return;
    const PagedGeom& pg = a.p.g;
    if (it.split == 0 && tid == 0 && it.tile < a.rt_max)
        a.rows[((size_t)it.b * pg.Hkv + it.h) * a.rt_max + it.tile] = make_int4(it.first, it.stride, it.splits, 0);

    // The split's tiles go round the four waves: what shares a 128-byte line of V
    // (a column's neighbouring tiles) is asked for at one time, not once and
    // again when the caches have lost it.
    const int split_lo = it.w.lo + it.split * it.per * kUnit;
    const int split_hi = it.splits > 1 ? imin(it.s.ctx, split_lo + it.per * kUnit) : it.s.ctx;
    constexpr int STEP = 4 * T::KEYS;
    const int key_lo = split_lo + w * T::KEYS, key_hi = split_hi;

    // The lane's query row.
    const int row = it.tile * kBM + c;
    const bool have = row < it.s.n * pg.G;
    const int tok = have ? row / pg.G : 0, head = it.h * pg.G + (have ? row % pg.G : 0);
    const int pos = have ? it.s.first + tok : -1;
    const int seen_lo = pg.window ? imax(pos - pg.window + 1, 0) : 0, seen_hi = imin(pos, it.s.ctx - 1);
    Sight sight;
    if constexpr (SEEN) sight = sight_of(a, it.s, have, tok);
    // Keys that every row of the tile sees need no mask.
    const int r_last = imin(it.tile * kBM + kBM, it.s.n * pg.G) - 1;
    const int p_first = it.s.first + (SEEN ? 0 : (it.tile * kBM) / pg.G);      // the first row's position, or the least
    const int p_last = it.s.first + (SEEN ? it.s.n - 1 : r_last / pg.G);       // the last row's, or the largest
    const int all_hi = imin(SEEN ? p_first - 1 : p_first, it.s.ctx - 1);
    const int all_lo = pg.window ? imax(p_last - pg.window + 1, 0) : 0;
    // Keys that some row sees: up to the last row's position, from the first row's window.
    const int any_hi = imin(p_last, it.s.ctx - 1);
    const int any_lo = pg.window ? imax(p_first - pg.window + 1, 0) : 0;

    // Q: k-step s holds dims 32s + 8g (f16 tiles); an 8-bit tile's 16-byte load
    // spans two k-steps, so there k-step 2l + e holds dims 64l + 16g + 8e.
    f16x8 qh[QLDS ? 1 : KS], ql[F32 && !QLDS ? KS : 1];
    float qscale = a.c;
    auto q_dim = [&](int s) { return I8 ? 64 * (s >> 1) + 16 * g + 8 * (s & 1) : 32 * s + 8 * g; };
    f16x8* const q_lds = reinterpret_cast<f16x8*>(smem);  // QLDS: [part][KS][64]
    {
        const QT* qr = static_cast<const QT*>(a.q) + (size_t)(it.s.row0 + tok) * a.q_row_stride + head * a.q_head_stride;
        if constexpr (F32) {
            // The row times a power of two that brings its largest element to
            // [2^14, 2^15): both f16 parts then keep their bits.
            float m = 0.f;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                float x[8];
                load_f32<8>(qr + q_dim(s), x);
#pragma unroll
                for (int j = 0; j < 8; ++j) m = fmaxf(m, finite_or_0(fabsf(x[j])));
            }
            m = max_groups(m);
            int e = 0;
            if (m > 0.f) e = 15 - (__builtin_amdgcn_frexp_expf(m));
            e = imin(imax(e, -120), 120);
            const float up = ldexpf(1.f, e);
            qscale = ldexpf(a.c, -e);
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                float x[8];
                load_f32<8>(qr + q_dim(s), x);
                f16x8 hi, lo;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float y = have ? x[j] * up : 0.f;
                    hi[j] = (f16)y;
                    lo[j] = (f16)finite_or_0(y - (float)hi[j]);
                }
                if constexpr (QLDS) {
                    if (w == 0) {
                        q_lds[s * 64 + lane] = hi;
                        q_lds[(KS + s) * 64 + lane] = lo;
                    }
                } else {
                    qh[s] = hi;
                    ql[s] = lo;
                }
            }
        } else {
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                f16x8 hi = *reinterpret_cast<const f16x8*>(qr + q_dim(s));
                if (!have) hi = f16x8{};
                if constexpr (QLDS) {
                    if (w == 0) q_lds[s * 64 + lane] = hi;
                } else {
                    qh[s] = hi;
                }
            }
        }
        if constexpr (QLDS) __syncthreads();
    }

    f32x4 o[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;  // m: reference exponent less kLift; -inf: nothing seen yet

    PageWindow pw;
    pw.row = a.p.table + (size_t)it.b * pg.table_stride;

    bool poison = false;           // V held an infinity or a NaN at a key that some row sees and some does not

    // Whether every row of the item sees all of the tile.
    auto all_seen = [&](const int (&pages)[T::GR], int t0) {
        bool whole = t0 + T::KEYS - 1 <= all_hi && t0 >= all_lo;
#pragma unroll
        for (int i = 0; i < T::GR; ++i) whole = whole && pages[i] >= 0;
        return whole;
    };

    Tile<HD, I8> t;
    int pages[T::GR], next[T::GR];
    // The tile at t0; the loads of the one at t1 take the registers as they fall
    // free.  One copy of this code, and no branch around the loads: a wave runs
    // it a few times per launch, so code that is fetched for one more copy costs
    // microseconds, and with a branch the compiler loses count of the loads and
    // waits for V where K would do.  (After its last tile a wave reads that tile
    // once more, from the caches.)
    auto step = [&](int t0, int t1) {
        // ---- 8-bit scales: a lane prepares one key's, all read theirs back (wave's own LDS)
        if constexpr (I8) {
            scales[w][0][lane] = LEAN && !F32 ? t.ks * a.c : t.ks;
            scales[w][1][lane] = log_v_scale(t.vs);
            if constexpr (LEAN) scales[w][2][lane] = least_v_scale(t.vs);
            wave_lds_order();
        }
        auto scale4 = [&](int what, int j) {  // of the lane's keys in block j
            return *reinterpret_cast<const f32x4*>(&scales[w][what][16 * g + 4 * j]);
        };
        // ---- scores
        f32x4 s[T::NB];
        f32x4 lv[LEAN ? T::NB : 1], vs[LEAN ? T::NB : 1];  // of the lane's keys: log2 of V's scale, and the scale
#pragma unroll
        for (int j = 0; j < T::NB; ++j) {
            s[j] = f32x4{0.f, 0.f, 0.f, 0.f};
            f32x4 sl = s[j];  // f16 pages: the products with q's second part
            auto& s2 = I8 ? s[j] : sl;
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                f16x8 kf;
                if constexpr (I8) {
                    const uint4 x = t.k[j][k >> 1];
                    kf = k & 1 ? i8x8_to_f16(x.z, x.w) : i8x8_to_f16(x.x, x.y);
                } else {
                    kf = __builtin_bit_cast(f16x8, t.k[j][k]);
                }
                if constexpr (QLDS) {
                    s[j] = mfma16(kf, q_lds[k * 64 + lane], s[j]);
                    if constexpr (F32) s2 = mfma16(kf, q_lds[(KS + k) * 64 + lane], s2);
                } else {
                    s[j] = mfma16(kf, qh[k], s[j]);
                    if constexpr (F32) s2 = mfma16(kf, ql[k], s2);
                }
            }
            if constexpr (F32 && !I8)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[j][i] += second_part(s[j][i], sl[i]);
            if constexpr (LEAN) {
                s[j] *= scale4(0, j);
                if constexpr (F32) s[j] *= qscale;
                lv[j] = scale4(1, j);
                vs[j] = scale4(2, j);
            } else if constexpr (I8) {
                const f32x4 ks = scale4(0, j), lv = scale4(1, j);
#pragma unroll
                for (int i = 0; i < 4; ++i) s[j][i] = fmaf(s[j][i] * ks[i], qscale, lv[i]);
            } else {
                s[j] *= qscale;
            }
        }
        // ---- mask: keys behind the row, before its window, in no page
        constexpr int QUART = T::KEYS / 4;
#pragma unroll
        for (int i = 0; i < T::GR; ++i) next[i] = pw.at(a.p, t1 + 16 * i);
        load_k<HD, I8>(a, next, it.h, t1, t);
        const bool whole = all_seen(pages, t0);
        uint32_t seen = 0xffffffffu;  // bit 4j + i: the lane's key 4j + i
        uint4 v_mask = {};            // f16, not whole: the lane's keys that some row sees
        if (!whole) {
            const int gran = I8 ? g : g >> 1;
            const int p0 = pages[0], p1 = pages[1];
            int page = gran & 1 ? p1 : p0;
            if constexpr (T::GR == 4) {
                const int p2 = pages[2], p3 = pages[3], q = gran & 1 ? p3 : p2;
                page = gran & 2 ? q : page;
            }
            const int key = t0 + QUART * g;
            if constexpr (!I8) v_mask = page >= 0 ? keys8_mask(any_lo - key, any_hi - key) : uint4{};
            seen = 0;
            if constexpr (SEEN) {
                if (page >= 0) seen = (uint32_t)sight.from(key) & ((1u << QUART) - 1);
            } else {
#pragma unroll
                for (int i = 0; i < QUART; ++i)
                    seen |= (uint32_t)(page >= 0 && key + i <= seen_hi && key + i >= seen_lo) << i;
            }
#pragma unroll
            for (int j = 0; j < T::NB; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (!(seen >> (4 * j + i) & 1)) {
                        s[j][i] = -INFINITY;
                        if constexpr (LEAN) lv[j][i] = vs[j][i] = 0.f;  // whatever the slot holds
                    }
        }
        // ---- the reference
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < T::NB; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) top = fmaxf(top, LEAN ? s[j][i] + lv[j][i] : s[j][i]);
        if (__ballot(top > m + (kSlack + kLift))) {  // m = -inf: any score
            top = max_groups(top);
            float mn = m;
            if (top > m + (kSlack + kLift)) mn = top - kLift;
            const float f = m == -INFINITY ? 0.f : fast_exp2(m - mn);
            l = m == -INFINITY ? 0.f : moved<I8>(l, m - mn);
            m = mn;
#pragma unroll
            for (int d = 0; d < DT; ++d) o[d] *= f;
        }
        // ---- weights
        const float ms = m == -INFINITY ? 0.f : m;
        f16x8 ph[T::NB / 2], pl[T::NB / 2];
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < T::NB; ++j) {
            f32x4 log_v;
            if constexpr (I8 && !LEAN) log_v = scale4(1, j);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x = s[j][i] - ms;
                float p = fast_exp2(x);
                if constexpr (I8 && !LEAN)
                    sum += seen >> (4 * j + i) & 1 ? fast_exp2(x - log_v[i]) : 0.f;
                else
                    sum += p;
                if constexpr (LEAN) p *= vs[j][i];
                const int at = 4 * (j & 1) + i;
                ph[j >> 1][at] = (f16)p;
                pl[j >> 1][at] = (f16)(p - (float)(f16)p);
            }
        }
        if constexpr (I8) wave_lds_order();  // the next tile's scales go where these were
        l += sum;
        // ---- O^T += V^T P^T
        if constexpr (!I8) {
            // An infinity or NaN in V would meet the zero weights of rows that
            // do not see its key (0 * inf): in tiles that hold such a key,
            // these elements stay out of the product, and the rows that do see
            // them get them after the loop.  What no row sees (slots behind the
            // sequence, pages that are none) is cleared and asks for nothing.
            if (!whole) {
                const uint4 on = v_mask;
                uint32_t bad = 0;
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    t.v[d] = uint4{t.v[d].x & on.x, t.v[d].y & on.y, t.v[d].z & on.z, t.v[d].w & on.w};
                    bad |= nonfinite2(t.v[d].x) | nonfinite2(t.v[d].y) | nonfinite2(t.v[d].z) | nonfinite2(t.v[d].w);
                    t.v[d] = uint4{finite2(t.v[d].x), finite2(t.v[d].y), finite2(t.v[d].z), finite2(t.v[d].w)};
                }
                poison = poison || __ballot(bad != 0) != 0;
            }
        }
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            if constexpr (I8) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const f16x8 vf = e ? i8x8_to_f16(t.v[d].z, t.v[d].w) : i8x8_to_f16(t.v[d].x, t.v[d].y);
                    o[d] = mfma16(vf, ph[e], o[d]);
                    o[d] = mfma16(vf, pl[e], o[d]);
                }
            } else {
                const f16x8 vf = __builtin_bit_cast(f16x8, t.v[d]);
                o[d] = mfma16(vf, ph[0], o[d]);
                o[d] = mfma16(vf, pl[0], o[d]);
            }
        }
        load_v<HD, I8>(a, next, it.h, t1, t);
#pragma unroll
        for (int i = 0; i < T::GR; ++i) pages[i] = next[i];
    };

    // A window of pages at a time (1024 keys and more): within it no lookup
    // waits, and the loads of two tiles stay counted apart.
    for (int k0 = key_lo; k0 < key_hi;) {
        pw.fill(a.p, k0);
        const int k1 = imin(key_hi, pw.end(a.p));
#pragma unroll
        for (int i = 0; i < T::GR; ++i) pages[i] = pw.at(a.p, k0 + 16 * i);
        load_k<HD, I8>(a, pages, it.h, k0, t);
        __builtin_amdgcn_sched_barrier(0);  // K's loads before V's, as in the loop
        load_v<HD, I8>(a, pages, it.h, k0, t);
        for (; k0 < k1; k0 += STEP) step(k0, k0 + STEP < k1 ? k0 + STEP : k0);
    }

    if constexpr (!I8) {
        float z = 0.f;  // NaN where an element of o is not finite
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int x = 0; x < 4; ++x) z = fmaf(o[d][x], 0.f, z);
        if (poison || __ballot(z != 0.f)) {
            // Rare: the infinities and NaN among V go to the rows that see
            // them (a product with a weight's parts made NaN of an infinity).
            f32x4 add[DT];
#pragma unroll
            for (int d = 0; d < DT; ++d) add[d] = f32x4{0.f, 0.f, 0.f, 0.f};
            pw.fill(a.p, key_lo);
            const size_t step = (size_t)1 << pg.ps_log2;
            for (int key = key_lo; key < key_hi; ++key) {
                if ((key - key_lo) % STEP == T::KEYS) key += STEP - T::KEYS;  // the other waves' tiles
                if (key >= key_hi) break;
                if (key >= pw.end(a.p)) pw.fill(a.p, key);
                const int page = pw.at(a.p, key);
                if (page < 0 || (SEEN ? !sight.sees(key) : key > seen_hi || key < seen_lo)) continue;
                const f16* e = reinterpret_cast<const f16*>(a.p.v) +
                               v_offset(a.p, page, it.h, key & ((1 << pg.ps_log2) - 1)) + ((4 * g) << pg.ps_log2);
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const float y = (float)*e;
                        if (!(fabsf(y) < INFINITY)) add[d][x] += y;
                        e += x < 3 ? step : 13 * step;  // dims 16d + 4g + x
                    }
            }
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int x = 0; x < 4; ++x)
                    if (!(fabsf(add[d][x]) < INFINITY)) o[d][x] = add[d][x];
        }
    }

    // ---- join the four waves
    l = sum_groups(l);
    float* const ex_m = reinterpret_cast<float*>(smem);  // [4][16]
    float* const ex_l = ex_m + 64;                       // [4][16]
    float* const ex_o = ex_m + 128;                      // [4][16][OP]
    if constexpr (QLDS) __syncthreads();                 // Q's place is taken over
    if (g == 0) {
        ex_m[w * 16 + c] = m;
        ex_l[w * 16 + c] = l;
    }
#pragma unroll
    for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4*>(&ex_o[(w * 16 + c) * OP + 16 * d + 4 * g]) = o[d];
    __syncthreads();
    const int rows = imin(kBM, it.s.n * pg.G - it.tile * kBM);
    const int item = it.first + it.split * it.stride;
    for (int i = tid; i < rows * (HD / 4); i += 256) {
        const int r = i / (HD / 4), d = 4 * (i % (HD / 4));
        const float m0 = ex_m[r], m1 = ex_m[16 + r], m2 = ex_m[32 + r], m3 = ex_m[48 + r];
        const float mm = fmaxf(fmaxf(m0, m1), fmaxf(m2, m3));
        const float ref = mm == -INFINITY ? 0.f : mm;
        f32x4 y = {0.f, 0.f, 0.f, 0.f};
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float f = join_weight(ex_m[16 * k + r] - ref);
            sum += moved<I8>(ex_l[16 * k + r], ex_m[16 * k + r] - ref);
            const f32x4 x = *reinterpret_cast<const f32x4*>(&ex_o[(k * 16 + r) * OP + d]);
            y += x * f;
        }
        if (it.splits > 1) {
            *reinterpret_cast<f32x4*>(a.part_o + ((size_t)item * kBM + r) * HD + d) = y;
            if (d == 0) *reinterpret_cast<f32x2*>(a.part_ml + ((size_t)item * kBM + r) * 2) = f32x2{mm, sum};
        } else {
            const int q = it.tile * kBM + r;
            y = sum == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : y * (1.f / sum);  // (y may hold infinities)
            QT* dst = static_cast<QT*>(a.out) +
                      ((size_t)(it.s.row0 + q / pg.G) * pg.Hkv * pg.G + it.h * pg.G + q % pg.G) * HD + d;
            if constexpr (F32)
                *reinterpret_cast<f32x4*>(dst) = y;
            else
                *reinterpret_cast<f16x4*>(dst) = f16x4{(f16)y[0], (f16)y[1], (f16)y[2], (f16)y[3]};
        }
    }
}

// Joins the splits of one query row: HD/4 columns x 1024/HD groups of splits.
// Latency: 4-6 us for the partials of 32 heads, most of it the launch.
// A workgroup for each row that a row tile can have (`rows` of them; tiles in
// find_item's order with one split each).
template <int HD, bool F32, bool I8>
__global__ __launch_bounds__(256) void paged_merge_kernel(AttnPagedArgs a, int bm, int rows) {
    using QT = std::conditional_t<F32, float, f16>;
    constexpr int C4 = HD / 4, NG = 256 / C4;
    __shared__ f32x4 ex[NG][C4];
    __shared__ float ex_m[NG], ex_l[NG];
    const PagedGeom& pg = a.p.g;
    Item it;
    if (!find_item(a, blockIdx.x / rows, bm, false, false, it)) return;
    const PagedSeq& s = it.s;
    const int h = it.h, row = it.tile * bm + blockIdx.x % rows;
    if (row >= s.n * pg.G || it.tile >= a.rt_max) return;
    const int4 info = a.rows[((size_t)it.b * pg.Hkv + h) * a.rt_max + it.tile];
    // written by this call's split 0; in range whatever it holds
    const int splits = imin(info.z, a.n_items);
    if (splits <= 1) return;
    const int col = threadIdx.x % C4, grp = threadIdx.x / C4;
    float m = -INFINITY, l = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    constexpr int U = 8;
    for (int s0 = grp; s0 < splits; s0 += NG * U) {
        f32x2 ml[U];
        f32x4 x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int sp = s0 + u * NG < splits ? s0 + u * NG : s0;
            // in range whatever the table of rows holds
            const size_t at = (size_t)imin(imax(info.x + sp * info.y, 0), a.n_items - 1) * bm + row % bm;
            ml[u] = *reinterpret_cast<const f32x2*>(a.part_ml + at * 2);
            x[u] = *reinterpret_cast<const f32x4*>(a.part_o + at * HD + 4 * col);
            if (s0 + u * NG >= splits) {
                ml[u] = f32x2{-INFINITY, 0.f};
                x[u] = f32x4{0.f, 0.f, 0.f, 0.f};
            }
        }
        float mn = m;
#pragma unroll
        for (int u = 0; u < U; ++u) mn = fmaxf(mn, ml[u][0]);
        const float ref = mn == -INFINITY ? 0.f : mn;
        const float f = join_weight(m - ref);
        l = moved<I8>(l, m - ref);
        o *= f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float fu = join_weight(ml[u][0] - ref);
            l += moved<I8>(ml[u][1], ml[u][0] - ref);
            o += x[u] * fu;
        }
        m = mn;
    }
    ex[grp][col] = o;
    if (col == 0) {
        ex_m[grp] = m;
        ex_l[grp] = l;
    }
    __syncthreads();
    if (grp) return;
    float mm = -INFINITY;
#pragma unroll
    for (int k = 0; k < NG; ++k) mm = fmaxf(mm, ex_m[k]);
    const float ref = mm == -INFINITY ? 0.f : mm;
    f32x4 y = {0.f, 0.f, 0.f, 0.f};
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < NG; ++k) {
        const float f = join_weight(ex_m[k] - ref);
        sum += moved<I8>(ex_l[k], ex_m[k] - ref);
        y += ex[k][col] * f;
    }
    y = sum == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : y * (1.f / sum);
    QT* dst = static_cast<QT*>(a.out) + ((size_t)(s.row0 + row / pg.G) * pg.Hkv * pg.G + h * pg.G + row % pg.G) * HD + 4 * col;
    if constexpr (F32)
        *reinterpret_cast<f32x4*>(dst) = y;
    else
        *reinterpret_cast<f16x4*>(dst) = f16x4{(f16)y[0], (f16)y[1], (f16)y[2], (f16)y[3]};
}

// The same for rows of masks: a wave a row, HD/4 columns x 256/HD groups of splits
// (two float4s a lane at 512 dims), joined across the lanes; four rows a workgroup.
// 32 sequences of up to 64 rows, 8 bits, 47 MB of partials: 8.7 us, with a workgroup a row 24.6.
template <int HD, bool F32, bool I8>
__global__ __launch_bounds__(256) void paged_merge_rows_kernel(AttnPagedArgs a, int bm, int per) {
    using QT = std::conditional_t<F32, float, f16>;
    constexpr int C4 = HD < 256 ? HD / 4 : 64, NG = 64 / C4, V = HD / 4 / C4, U = 4 / V;
    const PagedGeom& pg = a.p.g;
    Item it;
    if (!find_item(a, blockIdx.x / per, bm, false, false, it)) return;
    const int lane = threadIdx.x & 63, r = blockIdx.x % per * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = it.tile * bm + r;
    if (r >= bm || row >= it.s.n * pg.G || it.tile >= a.rt_max) return;
    const int4 info = a.rows[((size_t)it.b * pg.Hkv + it.h) * a.rt_max + it.tile];
    const int splits = imin(info.z, a.n_items);  // written by this call's split 0; in range whatever it holds
    if (splits <= 1) return;
    const int col = lane % C4, grp = lane / C4;
    float m = -INFINITY, l = 0.f;
    f32x4 o[V];
#pragma unroll
    for (int v = 0; v < V; ++v) o[v] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int s0 = grp; s0 < splits; s0 += NG * U) {
        f32x2 ml[U];
        f32x4 x[U][V];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int sp = s0 + u * NG < splits ? s0 + u * NG : s0;
            const size_t at = (size_t)imin(imax(info.x + sp * info.y, 0), a.n_items - 1) * bm + r;
            ml[u] = *reinterpret_cast<const f32x2*>(a.part_ml + at * 2);
#pragma unroll
            for (int v = 0; v < V; ++v) x[u][v] = *reinterpret_cast<const f32x4*>(a.part_o + at * HD + 4 * (col + C4 * v));
            if (s0 + u * NG >= splits) {
                ml[u] = f32x2{-INFINITY, 0.f};
#pragma unroll
                for (int v = 0; v < V; ++v) x[u][v] = f32x4{0.f, 0.f, 0.f, 0.f};
            }
        }
        float mn = m;
#pragma unroll
        for (int u = 0; u < U; ++u) mn = fmaxf(mn, ml[u][0]);
        const float ref = mn == -INFINITY ? 0.f : mn, f = join_weight(m - ref);
        l = moved<I8>(l, m - ref);
#pragma unroll
        for (int v = 0; v < V; ++v) o[v] *= f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float fu = join_weight(ml[u][0] - ref);
            l += moved<I8>(ml[u][1], ml[u][0] - ref);
#pragma unroll
            for (int v = 0; v < V; ++v) o[v] += x[u][v] * fu;
        }
        m = mn;
    }
#pragma unroll
    for (int d = C4; d < 64; d <<= 1) {  // the groups (then V is 1)
        const float m2 = shfl_xor(m, d), l2 = shfl_xor(l, d), mn = fmaxf(m, m2), ref = mn == -INFINITY ? 0.f : mn;
        const float f = join_weight(m - ref), f2 = join_weight(m2 - ref);
#pragma unroll
        for (int j = 0; j < 4; ++j) o[0][j] = o[0][j] * f + shfl_xor(o[0][j], d) * f2;
        l = moved<I8>(l, m - ref) + moved<I8>(l2, m2 - ref);
        m = mn;
    }
    if (grp) return;
    const float inv = 1.f / l;
    QT* dst = static_cast<QT*>(a.out) + ((size_t)(it.s.row0 + row / pg.G) * pg.Hkv * pg.G + it.h * pg.G + row % pg.G) * HD;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const f32x4 y = l == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : o[v] * inv;
        const int d = 4 * (col + C4 * v);
        if constexpr (F32)
            *reinterpret_cast<f32x4*>(dst + d) = y;
        else
            *reinterpret_cast<f16x4*>(dst + d) = f16x4{(f16)y[0], (f16)y[1], (f16)y[2], (f16)y[3]};
    }
}

// The same for chunks' row tiles: few splits, many rows.  A workgroup takes 32
// rows, a wave every fourth 8 of their dims, in the order that the chunk
// kernel's lanes hold them (part_at), so that a load is 1 KB in a row.  512 rows
// of 32 heads in 4 splits, 38 MB: 8.4 us, row by row 9.1 (and the chunk kernel 54 -> 52).
constexpr int kMergeRows = 32;
template <int HD, bool F32, bool I8>
__global__ __launch_bounds__(256) void paged_merge_tiles_kernel(AttnPagedArgs a, int bm) {
    using QT = std::conditional_t<F32, float, f16>;
    constexpr int V = HD / 32, U = V < 16 ? 16 / V : 1;  // float4s a lane; splits at once
    const PagedGeom& pg = a.p.g;
    const int per = bm / kMergeRows;
    Item it;
    if (!find_item(a, blockIdx.x / per, bm, false, false, it) || it.tile >= a.rt_max) return;
    const int4 info = a.rows[((size_t)it.b * pg.Hkv + it.h) * a.rt_max + it.tile];
    const int splits = imin(info.z, a.n_items);  // written by this call's split 0; in range whatever it holds
    if (splits <= 1) return;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, hh = lane >> 5;
    const int blk = blockIdx.x % per, r = blk * kMergeRows + (lane & 31), row = it.tile * bm + r;
    if (row >= it.s.n * pg.G) return;
    float m = -INFINITY, l = 0.f;
    f32x4 o[V];
#pragma unroll
    for (int v = 0; v < V; ++v) o[v] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < splits; s0 += U) {
        f32x2 ml[U];
        f32x4 x[U][V];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int sp = imin(s0 + u, splits - 1);
            const size_t at = (size_t)imin(imax(info.x + sp * info.y, 0), a.n_items - 1) * bm;
            ml[u] = *reinterpret_cast<const f32x2*>(a.part_ml + (at + r) * 2);
#pragma unroll
            for (int v = 0; v < V; ++v) x[u][v] = *reinterpret_cast<const f32x4*>(a.part_o + at * HD + part_at<HD>(blk, 4 * v + w, lane));
        }
        float mn = m;
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (s0 + u < splits) mn = fmaxf(mn, ml[u][0]);
        const float ref = mn == -INFINITY ? 0.f : mn, f = join_weight(m - ref);
        l = moved<I8>(l, m - ref);
#pragma unroll
        for (int v = 0; v < V; ++v) o[v] *= f;
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (s0 + u < splits) {
                const float fu = join_weight(ml[u][0] - ref);
                l += moved<I8>(ml[u][1], ml[u][0] - ref);
#pragma unroll
                for (int v = 0; v < V; ++v) o[v] += x[u][v] * fu;
            }
        m = mn;
    }
    const float inv = 1.f / l;
    QT* dst = static_cast<QT*>(a.out) +
              ((size_t)(it.s.row0 + row / pg.G) * pg.Hkv * pg.G + it.h * pg.G + row % pg.G) * HD + 4 * hh;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const f32x4 y = l == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : o[v] * inv;
        const int d = 8 * (4 * v + w);
        if constexpr (F32)
            *reinterpret_cast<f32x4*>(dst + d) = y;
        else
            *reinterpret_cast<f16x4*>(dst + d) = f16x4{(f16)y[0], (f16)y[1], (f16)y[2], (f16)y[3]};
    }
}

// ------------------------------------------------------------------- host --
// Items the rows kernel aims at: two rounds of the workgroups that the CUs hold
// (two a CU up to head_dim 128, else one), so that uneven sequences level out.
// Half as many: an 8-bit step of 32 sequences of 128-dim heads 112 -> 126 us, 4
// of 256 dims 117 -> 129; twice as many 112 and 128.  512-dim items, whose
// queries go through LDS first, come in one round: 16 sequences 139 us, in two
// 158.
constexpr int rows_target(int hd) { return hd <= 128 ? 1024 : hd == 256 ? 512 : 256; }
// 64-key units a split has at least.  Shorter splits (4 units) cost one token
// over 32k keys of 128 dims 29 -> 36 us and over 512 keys 9.7 -> 11.8 (a merge
// that it has no need of), longer ones (16) 29 -> 29.5; a 512-dim head, whose
// units take four times as long, gains: 32k keys, one kv head, 8 units 86 us, 4
// 65, 2 68.
constexpr int rows_least(int hd) { return hd <= 256 ? 8 : 4; }
constexpr int kCus = 256;          // compute units of the target (MI355X)
// The same for chunks; 512 rows on 4k keys take 64 us with 4, 8 and 16, eight
// sequences of 64 rows 54, 54 and 56.5.
constexpr int kChunkLeast = 8;
// Query rows a sequence may have per kv head for the rows kernel: its tiles of
// 16 each read the keys again, a chunk's tile of 128 wastes the rows that it
// has too many.  Eight sequences of 2000-8000 positions, us on the rows and on
// the chunk kernel (128 dims): 32 rows f16 46 and 50, 8 bits (f32 queries) 41
// and 63; 48 rows 64 and 67, 54 and 72; 64 rows 79 and 64, 65 and 73; 128 rows
// 135 and 58, 105 and 82.  256 dims, four sequences: 64 rows f16 94 and 105, 8
// bits 74 and 121; 128 rows 138 and 124, 104 and 127.  512 dims: 48 rows f16 141
// and 89, 8 bits 112 and 132.  (Both kernels before 8-bit sums took an exponential
// of their own, which costs the rows kernel 1% and the chunk kernel 4%.)
constexpr int rows_most(int hd, bool i8) { return hd == 256 ? (i8 ? 128 : 64) : i8 ? 64 : 32; }

// Workgroups of the chunk kernel that start at once.
static int chunk_slots(int hd, bool i8, bool f32) { return kCus * chunk_occ_of(hd, i8, f32); }

// One kernel's share of a call.
struct Part {
    bool on, splits;
    int bm, lo_rows, hi_rows, target, least, rt_max;
    int64_t items;  // workgroups: an upper bound of its items
    int64_t merge;  // workgroups of its merge
    int slots, fine;  // rows of masks: AttnPagedArgs'
    size_t o_bytes, ml_bytes, rows_bytes;
    size_t bytes() const { return o_bytes + ml_bytes + rows_bytes; }
    // 256 threads a workgroup are counted in 32 bits
    bool fits() const { return items < (1 << 24) && merge < (1 << 24); }
};
static Part make_part(const PagedGeom& g, int hd, int bm, int64_t tiles, int64_t seq_rows, bool splits, int target, int least) {
    Part r{};
    r.on = true;
    r.bm = bm;
    r.splits = splits && g.max_ctx > least * kUnit;  // else a single split reaches every key
    r.target = target;
    r.least = r.splits ? least : 1000000000;
    r.items = tiles * g.Hkv + (r.splits ? target : 0);
    r.rt_max = (int)((seq_rows + bm - 1) / bm);
    r.o_bytes = r.splits ? (size_t)r.items * bm * hd * 4 : 0;
    r.ml_bytes = r.splits ? (size_t)r.items * bm * 8 : 0;
    r.rows_bytes = r.splits ? ((size_t)g.n_seq * g.Hkv * r.rt_max * 16) : 0;
    r.hi_rows = 0x7fffffff;
    // a workgroup of the merge takes a row, of a chunk's tiles kMergeRows
    r.merge = r.splits ? tiles * g.Hkv * (bm == kBM ? std::min<int64_t>(bm, (int64_t)g.max_new * g.G) : bm / kMergeRows) : 0;
    return r;
}
struct Plan {
    Part rows, chunk;
};
// The rows kernel's share; it grows with each of n_seq, n_tokens, max_new and max_ctx.
static Part rows_part(const PagedGeom& g, int hd, bool i8) {
    const int seq_rows = (int)std::min<int64_t>((int64_t)g.max_new * g.G, rows_most(hd, i8));
    const int64_t tiles = std::min<int64_t>(row_tiles_bound(g, kBM), (int64_t)g.n_seq * ((seq_rows + kBM - 1) / kBM));
    Part r = make_part(g, hd, kBM, tiles, seq_rows, true, rows_target(hd), rows_least(hd));
    r.hi_rows = seq_rows;
    return r;
}
static Plan make_plan(const PagedGeom& g, int hd, bool i8, bool f32) {
    Plan p{};
    const int64_t most = (int64_t)g.max_new * g.G;  // rows of a sequence
    const int cm = chunk_rows(hd, i8, f32);
    const int few = rows_most(hd, i8);
    const bool chunks = most > few;
    if (!chunks || g.n_seq > 1) p.rows = rows_part(g, hd, i8);
    if (chunks) {
        const int64_t tiles = row_tiles_bound(g, cm);
        // Splits where two or more of them a tile still start at once (four in a
        // window, whose tiles meet parts of few splits): 512 rows on 4k keys 88 ->
        // 58 us, a prompt of 2048 with 8 heads of 256 120 -> 92, in a window of 1024
        // 75 -> 91.  Where tiles fill the CUs once, splits cost more than their
        // balance gives: two chunks in a window (256 dims) 114 -> 139 us, nine uneven
        // sequences 276 -> 292, the worst one (six of 256 dims) gains 1085 -> 979.
        const int slots = chunk_slots(hd, i8, f32);
        const bool cut = (g.window ? 4 : 2) * row_tiles_least(g, cm) * g.Hkv <= slots;
        p.chunk = make_part(g, hd, cm, tiles, most, cut, slots, kChunkLeast);
        if (p.rows.on) p.chunk.lo_rows = few;
    }
    return p;
}

// The most workspace that a plan of g or of any smaller geometry (n_seq, n_tokens,
// max_new, max_ctx at most g's) asks for.  Chunks are cut only while their tiles
// leave CUs idle, so their partials are largest at the most rows that are still
// cut; a prompt of more rows needs none.
static size_t most_workspace(const PagedGeom& g, int hd, bool i8, bool f32) {
    const int cm = chunk_rows(hd, i8, f32), slots = chunk_slots(hd, i8, f32);
    PagedGeom c = g;
    c.n_tokens = (int)std::min<int64_t>(g.n_tokens, (int64_t)(slots / (2 * g.Hkv)) * cm / g.G);
    c.max_new = std::min(g.max_new, c.n_tokens);
    const int64_t most = (int64_t)c.max_new * c.G;
    size_t bytes = rows_part(g, hd, i8).bytes();
    if (most > rows_most(hd, i8))
        bytes += make_part(c, hd, cm, row_tiles_bound(c, cm), most, true, slots, kChunkLeast).bytes();
    return bytes;
}

// ---- rows of masks.  A step's sequences bring about as many rows each, so that one
// kernel takes them all, and there is no launch for rows that turn out to be none's.
//
// Query rows a sequence may have per kv head for the rows kernel.  Eight sequences
// of 2000-8000 positions, 16 heads on 4, us on the rows and on the chunk kernel:
//   128 dims  f16            16 rows  30 and 32, 20 rows  49 and 34 (f32 q. 32 and 37, 51 and 38)
//             8 bits         64 rows  42 and 47, 80 rows  43 and 48, 96 rows  54 and 48
//             8 bits, f32 q. 64 rows  45 and 53, 80 rows  46 and 55, 96 rows  56 and 55
//             8 bits, 32 sequences of 4 to 64 rows and 16 to 8192 positions  124 and 163
//   64 dims   f16            16 rows  18 and 22, 20 rows  27 and 23
//             8 bits         64 rows  30 and 35, 80 rows  30 and 35, 96 rows  37 and 35 (f32 q. 32 and 38, 40 and 38)
//   256 dims  f16            16 rows  64 and 67, 20 rows 101 and 71 (f32 q. 68 and 79, 103 and 81)
//             8 bits         64 rows  80 and 135, 96 rows 99 and 138, 128 rows 114 and 140
//             8 bits, f32 q. 64 rows  94 and 99, 96 rows 115 and 103
//   512 dims  f16             4 rows 211 and 117, 16 rows 215 and 111; one sequence 58 and 77, 62 and 65
//             8 bits          4 rows 151 and 107, 16 rows 157 and 103; one sequence 47 and 81, 50 and 69
//             8 bits, f32 q.  4 rows 153 and 218, 16 rows 162 and 212
constexpr int seen_most(int hd, bool i8, bool f32, int n_seq) {
    if (hd == 512) return n_seq == 1 || (i8 && f32) ? kBM : 0;
    if (!i8) return kBM;
    return hd <= 128 ? 80 : f32 ? 64 : 128;
}
// 64-key units a split has at least where the work is short: one sequence of 6 rows
// (16 heads on 8, f32) on 518, 2048, 8192 and 32768 keys, splits of 2 units 12.0,
// 13.1, 19.9 and 46.8 us, of 4 units 13.3, 14.6, 17.2 and 37.1, of 8 units 14.6,
// 18.0, 18.7 and 38.5; so about half of target of them, up to 8 units.  (Even
// splits: 32 8-bit sequences 92 -> 84 us.)
constexpr int seen_fine(int hd) { return rows_least(hd) / 4; }
// Units of the longest sequence up to which nothing is split, and nothing merged, by
// the sequences times kv heads (`items`) that fill the CUs without.  (With weights of
// one part, which take 1 to 4% less time on either side.)  Not split and
// split, us, sequences of one length or up to it, 8 heads of 128 dims (4 of the others):
//   items 256 and more, 128 dims  1000 keys 22 and 28 (8 bits 14 and 23), 2000 keys 44 and
//                                 47 (21 and 29; one length 26 and 38), 4000 86 and 96 (46 and 58);
//                                 8192 as uneven 151 and 128.  One sequence among empty ones:
//                                 1000 keys 20 and 12, 2000 keys 34 and 13 (17 and 11), so f16 up to 1024
//                       256 dims  1000 keys 46 and 55 (23 and 34), 2000 keys 82 and 83 (40 and 55)
//                       64 dims   1000 keys 13 and 19 (10 and 19), 2000 keys 20 and 23 (14 and 21)
//   items 128, 128 dims           500 keys 14 and 17 (11 and 14), 1000 keys 21 and 18 (13 and 15)
//              256 dims           400 keys 21 and 25 (15 and 21), 1000 keys (21 and 33)
//   items 64,  128 dims           500 keys 13 and 13 (9 and 12), 1000 keys 20 and 15 (13 and 13)
//              256 dims           400 keys 21 and 20 (15 and 17), 1000 keys 37 and 20 (20 and 17)
//   items 8    128 dims           300 keys 10.0 and 10.4, 400 keys 11.4 and 10.4 (700 keys 10.2 and
//                                 10.4, 1000 keys 11.7 and 10.7)
//              256 dims           200 keys 14.7 and 14.7, 300 keys 17.5 and 14.7 (13.5 and 12.7)
//              64 dims            500 keys 8.1 and 9.7, 700 keys 9.4 and 9.1 (1000 keys 8.7 and 10.3)
//   512 dims (8 bits, f32 queries) 1000 keys, items 128 116 and 112
constexpr int kWholeLeast = 4;
constexpr int seen_whole(int hd, bool i8, int64_t items) {
    if (hd == 512) return kWholeLeast;
    if (items >= 256) return i8 ? 32 : 16;
    if (i8) return hd == 64 ? 16 : hd == 128 ? (items >= 64 ? 16 : 12) : items >= 128 ? 16 : items >= 64 ? 8 : kWholeLeast;
    return hd == 64 || items >= 128 ? 8 : hd == 128 ? 5 : kWholeLeast;
}
static Part seen_rows_part(const PagedGeom& g, int hd, int most, int whole) {
    const int rows = (int)std::min<int64_t>((int64_t)g.max_new * g.G, most);
    const int64_t tiles = std::min<int64_t>(row_tiles_bound(g, kBM), (int64_t)g.n_seq * ((rows + kBM - 1) / kBM));
    Part r = make_part(g, hd, kBM, tiles, rows, true, rows_target(hd), whole);
    r.least = r.splits ? 1 : r.least;
    r.fine = r.splits ? seen_fine(hd) : 0;
    r.merge = r.splits ? tiles * g.Hkv * ((std::min(kBM, rows) + 3) / 4) : 0;
    return r;
}
static Part seen_chunk_part(const PagedGeom& g, int hd, bool i8, bool f32) {
    const int cm = chunk_rows(hd, i8, f32), slots = chunk_slots(hd, i8, f32);
    const bool cut = (g.window ? 4 : 2) * row_tiles_least(g, cm) * g.Hkv <= slots;
    Part r = make_part(g, hd, cm, row_tiles_bound(g, cm), (int64_t)g.max_new * g.G, cut, slots, kChunkLeast);
    r.slots = slots;
    return r;
}
static Plan seen_plan(const PagedGeom& g, int hd, bool i8, bool f32) {
    Plan p{};
    const int most = seen_most(hd, i8, f32, g.n_seq);
    if ((int64_t)g.max_new * g.G > most) p.chunk = seen_chunk_part(g, hd, i8, f32);
    else p.rows = seen_rows_part(g, hd, most, seen_whole(hd, i8, (int64_t)g.n_seq * g.Hkv));
    return p;
}
// The most of any smaller geometry, as most_workspace: of few rows (split, as fewer
// sequences may be where these are not), or of chunks.
static size_t seen_most_workspace(const PagedGeom& g, int hd, bool i8, bool f32) {
    size_t bytes = seen_rows_part(g, hd, seen_most(hd, i8, f32, 1), kWholeLeast).bytes();
    if ((int64_t)g.max_new * g.G > seen_most(hd, i8, f32, g.n_seq)) {
        const int cm = chunk_rows(hd, i8, f32), slots = chunk_slots(hd, i8, f32);
        PagedGeom c = g;
        c.n_tokens = (int)std::min<int64_t>(g.n_tokens, (int64_t)(slots / (2 * g.Hkv)) * cm / g.G);
        c.max_new = std::min(g.max_new, c.n_tokens);
        if (c.n_tokens > 0)
            bytes = std::max(bytes, make_part(c, hd, cm, row_tiles_bound(c, cm), (int64_t)c.max_new * c.G, true, slots, kChunkLeast).bytes());
    }
    return bytes;
}

static PagedGeom attn_geom(const lmxp_pool* p, const lmxp_batch* b, const lmxp_attn_desc* d) {
    PagedGeom g = paged_args(p, b).g;
    g.G = (int)(d->n_heads / p->n_kv_heads);
    g.window = d->window < b->max_ctx ? (int)d->window : 0;  // a wider one hides nothing
    return g;
}

static Plan plan_of(const PagedGeom& g, int hd, bool i8, bool f32, bool seen) {
    return seen ? seen_plan(g, hd, i8, f32) : make_plan(g, hd, i8, f32);
}
// The workspace that one call needs; false where launches of either type could not name their work.
bool paged_attn_need(const lmxp_pool* p, const lmxp_batch* b, const lmxp_attn_desc* d, bool is_f32, bool seen, size_t* bytes) {
    bool fits = true;
    for (bool f32 : {false, true}) {
        const Plan pl = plan_of(attn_geom(p, b, d), (int)p->head_dim, p->store == LMXP_I8, f32, seen);
        fits = fits && pl.rows.fits() && pl.chunk.fits();
        if (f32 == is_f32) *bytes = pl.rows.bytes() + pl.chunk.bytes();
    }
    return fits;
}
// What serves calls of either type, with any window, on this batch and on every smaller one.
size_t paged_attn_workspace(const lmxp_pool* p, const lmxp_batch* b, const lmxp_attn_desc* d, bool seen) {
    size_t need, bytes = 0;
    if (!paged_attn_need(p, b, d, true, seen, &need)) return 0;
    const PagedGeom g = attn_geom(p, b, d);
    const bool i8 = p->store == LMXP_I8;
    for (bool f32 : {false, true})
        bytes = std::max(bytes, seen ? seen_most_workspace(g, (int)p->head_dim, i8, f32) : most_workspace(g, (int)p->head_dim, i8, f32));
    return bytes;
}

template <int HD>
static lmx_status launch_part(AttnPagedArgs a, const Part& r, bool chunk, bool i8, bool f32, char* ws, hipStream_t st) {
    if (!r.on) return LMX_OK;
    a.part_o = reinterpret_cast<float*>(ws);
    a.part_ml = reinterpret_cast<float*>(ws + r.o_bytes);
    a.rows = reinterpret_cast<int4*>(ws + r.o_bytes + r.ml_bytes);
    a.n_items = (int)r.items;
    a.target = r.target;
    a.least = r.least;
    a.rt_max = r.splits ? r.rt_max : 0;
    a.lo_rows = r.lo_rows;
    a.hi_rows = r.hi_rows;
    a.slots = r.slots;
    a.even = a.seen != nullptr;
    a.fine = r.fine;
    const dim3 grid((unsigned)r.items);
    if (chunk) {
        launch_chunk(a, HD, i8, f32, grid.x, st);
    } else {
        auto go = [&](auto i8_tag, auto f32_tag) {
            constexpr bool I8 = decltype(i8_tag)::value, F32 = decltype(f32_tag)::value;
            if (a.seen) hipLaunchKernelGGL((paged_rows_kernel<HD, I8, F32, true>), grid, dim3(256), 0, st, a);
            else hipLaunchKernelGGL((paged_rows_kernel<HD, I8, F32, false>), grid, dim3(256), 0, st, a);
        };
        const std::true_type yes;
        const std::false_type no;
        if (i8) f32 ? go(yes, yes) : go(yes, no);
        else f32 ? go(no, yes) : go(no, no);
    }
    LMX_CHECK_LAUNCH();
    if (r.splits) {
        if (chunk) {
            const dim3 mgrid((unsigned)r.merge);
            if (i8) {
                if (f32) hipLaunchKernelGGL((paged_merge_tiles_kernel<HD, true, true>), mgrid, dim3(256), 0, st, a, r.bm);
                else hipLaunchKernelGGL((paged_merge_tiles_kernel<HD, false, true>), mgrid, dim3(256), 0, st, a, r.bm);
            } else {
                if (f32) hipLaunchKernelGGL((paged_merge_tiles_kernel<HD, true, false>), mgrid, dim3(256), 0, st, a, r.bm);
                else hipLaunchKernelGGL((paged_merge_tiles_kernel<HD, false, false>), mgrid, dim3(256), 0, st, a, r.bm);
            }
            LMX_CHECK_LAUNCH();
            return LMX_OK;
        }
        const int rows = (int)std::min<int64_t>(r.bm, (int64_t)a.p.g.max_new * a.p.g.G);
        const dim3 mgrid((unsigned)r.merge);
        if (a.seen) {
            auto go = [&](auto i8_tag, auto f32_tag) {
                hipLaunchKernelGGL((paged_merge_rows_kernel<HD, decltype(f32_tag)::value, decltype(i8_tag)::value>), mgrid, dim3(256),
                                   0, st, a, r.bm, (rows + 3) / 4);
            };
            const std::true_type yes;
            const std::false_type no;
            if (i8) f32 ? go(yes, yes) : go(yes, no);
            else f32 ? go(no, yes) : go(no, no);
            LMX_CHECK_LAUNCH();
            return LMX_OK;
        }
        if (i8) {
            if (f32) hipLaunchKernelGGL((paged_merge_kernel<HD, true, true>), mgrid, dim3(256), 0, st, a, r.bm, rows);
            else hipLaunchKernelGGL((paged_merge_kernel<HD, false, true>), mgrid, dim3(256), 0, st, a, r.bm, rows);
        } else {
            if (f32) hipLaunchKernelGGL((paged_merge_kernel<HD, true, false>), mgrid, dim3(256), 0, st, a, r.bm, rows);
            else hipLaunchKernelGGL((paged_merge_kernel<HD, false, false>), mgrid, dim3(256), 0, st, a, r.bm, rows);
        }
        LMX_CHECK_LAUNCH();
    }
    return LMX_OK;
}

// seen NULL: causal.
static lmx_status attend(const lmxp_pool* p, const lmxp_batch* b, const lmxp_attn_desc* d, const uint64_t* seen,
                         uint32_t words, const int32_t* at, const void* q, lmx_dtype dt, void* out, void* ws,
                         hipStream_t st) {
    AttnPagedArgs a{};
    a.seen = seen;
    a.words = (int)words;
    a.at = at;
    a.p = paged_args(p, b);
    a.p.g = attn_geom(p, b, d);
    a.q = q;
    a.out = out;
    a.q_head_stride = d->q_head_stride ? d->q_head_stride : p->head_dim;
    a.q_row_stride = d->q_row_stride ? d->q_row_stride : a.q_head_stride * d->n_heads;
    a.c = d->scale * kLog2e;
    const bool i8 = p->store == LMXP_I8, f32 = dt == LMX_F32;
    const Plan pl = plan_of(a.p.g, (int)p->head_dim, i8, f32, seen != nullptr);
    (void)hipGetLastError();
    auto go = [&](auto tag) {
        constexpr int HD = decltype(tag)::value;
        const lmx_status s = launch_part<HD>(a, pl.chunk, true, i8, f32, static_cast<char*>(ws) + pl.rows.bytes(), st);
        return s != LMX_OK ? s : launch_part<HD>(a, pl.rows, false, i8, f32, static_cast<char*>(ws), st);
    };
    switch (p->head_dim) {
        case 64: return go(std::integral_constant<int, 64>{});
        case 128: return go(std::integral_constant<int, 128>{});
        case 256: return go(std::integral_constant<int, 256>{});
        default: return go(std::integral_constant<int, 512>{});
    }
}
lmx_status paged_attn(const lmxp_pool* p, const lmxp_batch* b, const lmxp_attn_desc* d, const void* q, lmx_dtype dt,
                      void* out, void* ws, hipStream_t st) {
    return attend(p, b, d, nullptr, 0, nullptr, q, dt, out, ws, st);
}
lmx_status paged_attn_seen(const lmxp_pool* p, const lmxp_batch* b, const lmxp_attn_desc* d, const uint64_t* seen,
                           uint32_t words, const int32_t* pos, const void* q, lmx_dtype dt, void* out, void* ws,
                           hipStream_t st) {
    return attend(p, b, d, seen, words, pos, q, dt, out, ws, st);
}

}  // namespace lmx
