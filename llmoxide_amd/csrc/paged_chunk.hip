// Attention of prompt chunks over pages on gfx950 (MFMA-bound).
//
// A workgroup takes a tile of 128 query rows of one kv head (row r: token
// r / G, head r % G, so that all heads of a group share the tile's keys) and
// walks its 64- or 32-key tiles; four waves of 32 rows share each K/V tile in
// LDS (512-dim heads: two or four waves share 32 rows as well).  As in the rows kernel the products are computed transposed,
//   S^T = K Q^T, O^T += V^T P^T   on v_mfma_f32_32x32x16_f16,
// Q^T in registers for the whole walk.  The keys that MFMA row r of a 32-key
// block stands for are chosen so that a lane's scores are 8 consecutive keys
// of each 16, the B operand of the second product; and V lies transposed in
// the pages, so both A operands are 16-byte LDS reads and nothing is shuffled
// or turned.  K rows and V columns sit in LDS in 16-byte chunks, those of row
// r permuted by an XOR with swizzle(r): what 16 neighbouring rows have at one
// chunk then covers the 64 banks once.
//
// f16 pages go from memory straight to LDS (the chunk permutation is made on
// the addresses that the lanes read); 8-bit pages go through registers, where
// they become f16 (exact), and their scales stay apart: K's multiplies the
// score, V's joins the exponent as its logarithm, so that weights are weighed
// against each other with it, row by row; the sum leaves it out.
//
// Bound by MFMA: 4 * hd operations a query row and key, for 4 * hd bytes a key
// that 128 rows share.  Measured (a large matrix product reaches 1.18 PFLOP/s):
//   prompt of 8192, 32 heads on 8 of 128 dims, f16   560-575 us, 955-980 TFLOP/s
//   (MFMA busy 52% of the cycles; without its softmax, operand reads and copies
//   the loop takes 400 us); 512 rows on 4k keys 57 us, 640 TFLOP/s with the merge
//   8-bit pages and fp32 queries, nine sequences     297 us, 353 TFLOP/s, twice
//   that with the queries' and weights' second parts
//   256 dims, a window of 1024                       106 us, 558 TFLOP/s
//   512 dims, 1024 rows of 16 heads on 2048 keys     158 us, 327 TFLOP/s
// Steps on the way, prompt: 128-row tiles of two workgroups a CU, conflict-free
// places and loops of one tile kind 859 -> 625 us; one base address a tile 578.
// Waves of 64 rows (half the LDS reads a product, one workgroup a CU) take 677.
// Counters: profiles/paged_cache.md.
#include <algorithm>

#include "lds_dma.hpp"
#include "paged_attn.hpp"

namespace lmx {

__device__ __forceinline__ f32x16 mfma32(f16x8 a, f16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// Operand reads in flight ahead of their product (2, 3, 4, 6: 121, 116, 116, 116
// us for a window of 1024 at 256 dims; 3 to 6 alike at 128).
constexpr int kAhead = 6;

// Weights are exp2(arg), arg = score - m, with m kLift below the largest score
// that set it; a tile with an arg above kMost moves m.  f16 queries, of 11 bits
// themselves, take weights rounded once to f16's 11, and least 2^-24 of the scale
// 2^6 of a weight at m; fp32 queries two parts of 22 bits together.  Two parts
// for f16 queries as well double the second product: the prompt of 8192 588 ->
// 793 us, 512 rows on 4k keys 57 -> 73, the 256-dim window 108 -> 148, 8-bit
// chunks 361 -> 454.  The error of a result against 64 bits (root mean square, of
// the result) is 2.7e-4, 2.9e-4, 2.8e-4 and 2.5e-4 with one part, 2.1e-4 with two,
// as that of the exact result rounded to f16.  By masks f16 queries have two parts
// all the same, as they have in the rows kernel: eight trees of 64 rows 72 -> 88 us.
template <bool TWO>
struct Lift {
    static constexpr float lift = TWO ? 10.f : 6.f, most = 14.f;
};

// Place of row r's chunk c is c ^ swizzle(r): rows of 256 bytes and more start
// at the same bank, of rows of 128 (64) bytes every second (fourth) one does.
template <int ROW_BYTES>
__device__ __forceinline__ int swizzle(int r) {
    return ROW_BYTES >= 256 ? r & 15 : ROW_BYTES == 128 ? (r >> 1) & 7 : (r >> 2) & 3;
}

// 16 bytes of LDS at a byte address.
__device__ __forceinline__ f16x8 lds16(uint32_t at) {
    return *reinterpret_cast<const __attribute__((address_space(3))) f16x8*>(at);
}

// lo: a of the lower 32 lanes, b of the lower in the upper lanes; hi: a of the
// upper lanes in the lower, b of the upper.
__device__ __forceinline__ void swap_halves(uint32_t a, uint32_t b, uint32_t& lo, uint32_t& hi) {
    const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    lo = r[0];
    hi = r[1];
}

template <int HD, int BN, int DS>
struct ChunkTile {
    static constexpr int KS = HD / 16;   // k-steps of QK
    static constexpr int NB = HD / 32 / DS;  // 32-dim blocks of the output, a wave
    static constexpr int BM = 128 / DS;  // rows a workgroup
    static constexpr int KB = BN / 32;   // 32-key blocks a tile
    static constexpr int ST = BN / 16;   // k-steps of PV
    static constexpr int GR = BN / 16;   // 16-key granules a tile, each in one page
    static constexpr int CH = HD / 8;    // 16-byte chunks of a K row
    static constexpr int CV = BN / 8;    // 16-byte chunks of a V column
    static constexpr int LOADS = BN * HD / 2048;  // 1 KB transfers a wave makes of a tile's K, and of its V
    static constexpr int STAGE = 2 * BN * HD;     // halfs: K then V
};

// BN: keys a tile.  DS: waves that share rows, each with its part of the
// output's dims (the scores are made by all of them).  OCC: workgroups a CU.
// SEEN: rows see each other by a mask, and all what lies before them.
template <int HD, bool I8, bool F32, int BN, int DS, int OCC, bool SEEN>
__global__ __launch_bounds__(256, OCC) void paged_chunk_kernel(AttnPagedArgs a) {
    using T = ChunkTile<HD, BN, DS>;
    using QT = std::conditional_t<F32, float, f16>;
    constexpr int KS = T::KS, NB = T::NB, BM = T::BM, CH = T::CH, KB = T::KB, ST = T::ST, GR = T::GR, CV = T::CV;
    constexpr bool TWO = F32 || SEEN;  // parts of a weight
    constexpr float kLift = Lift<TWO>::lift, kMost = Lift<TWO>::most;
    __shared__ __align__(1024) f16 tiles[2][T::STAGE];
    __shared__ __align__(16) float scales[I8 ? 2 : 1][2][BN];  // K's, log2 of V's

    Item it;
    // longest first: eight uneven 8-bit sequences of 100-12000 positions 812 -> 757 us
    if (!find_item(a, blockIdx.x, BM, true, true, it)) return;
    const PagedGeom& pg = a.p.g;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l32 = lane & 31, hh = lane >> 5;
    if (it.split == 0 && tid == 0 && it.tile < a.rt_max)
        a.rows[((size_t)it.b * pg.Hkv + it.h) * a.rt_max + it.tile] = make_int4(it.first, it.stride, it.splits, 0);

    // ---- rows, and the keys they see
    const int n_rows = it.s.n * pg.G, first_pos = it.s.first;
    const int r0 = it.tile * BM, r1 = imin(r0 + BM, n_rows) - 1;
    auto pos_of = [&](int r) { return first_pos + r / pg.G; };
    auto low_of = [&](int pos) { return pg.window ? imax(pos - pg.window + 1, 0) : 0; };
    const int split_lo = it.splits > 1 ? it.w.lo + it.split * it.per * kUnit : it.w.lo;
    const int split_hi = it.splits > 1 ? split_lo + it.per * kUnit : 0x7fffffff;
    // a tile's first and last position (by a mask: the least and the largest)
    auto least = [&](int r) { return SEEN ? first_pos : pos_of(r); };
    auto most = [&](int r) { return SEEN ? first_pos + it.s.n - 1 : pos_of(r); };
    auto held = [&](int pos) { return imin(pos, it.s.ctx - 1); };  // the last key up to there
    const int k_lo = imax(low_of(least(r0)) & ~(BN - 1), split_lo);
    const int k_hi = imin(held(most(r1)) + 1, split_hi);  // one behind the last key
    const int n_t = k_hi > k_lo ? (k_hi - k_lo + BN - 1) / BN : 0;
    // the wave's: keys some row sees, keys all rows see
    const int w0 = r0 + w / DS * 32, w1 = imin(w0 + 32, n_rows) - 1;
    const int nb0 = w % DS * NB;  // the wave's first block of dims
    const bool live = w0 <= r1;
    const int any_hi = live ? held(most(w1)) : -1, all_hi = live ? held(least(w0) - SEEN) : -1;
    const int any_lo = live ? low_of(least(w0)) : 0, all_lo = live ? low_of(most(w1)) : 0;

    f16x8 qh[KS], ql[F32 ? KS : 1];
    const int row = w0 + l32;
    const bool have = row < n_rows;
    const int tok = have ? row / pg.G : 0, head = it.h * pg.G + (have ? row % pg.G : 0);
    const int pos = have ? first_pos + tok : -1, seen_lo = low_of(pos), seen_hi = held(pos);
    Sight sight;
    if constexpr (SEEN) sight = sight_of(a, it.s, have, tok);
    float qs = a.c;  // what a score is multiplied by
    const QT* qr = static_cast<const QT*>(a.q) + (size_t)(it.s.row0 + tok) * a.q_row_stride + head * a.q_head_stride + 8 * hh;
    if constexpr (F32) {
        float m = 0.f;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            float x[8];
            load_f32<8>(qr + 16 * k, x);
#pragma unroll
            for (int j = 0; j < 8; ++j) m = fmaxf(m, finite_or_0(fabsf(x[j])));
        }
        m = fmaxf(m, shfl_xor(m, 32));
        int e = 0;  // the row's largest element to [2^14, 2^15), as in the rows kernel
        if (m > 0.f) e = 15 - __builtin_amdgcn_frexp_expf(m);
        e = imin(imax(e, -120), 120);
        const float up = ldexpf(1.f, e);
        qs = ldexpf(a.c, -e);
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            float x[8];
            load_f32<8>(qr + 16 * k, x);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float y = have ? x[j] * up : 0.f;
                qh[k][j] = (f16)y;
                ql[k][j] = (f16)finite_or_0(y - (float)(f16)y);
            }
        }
    } else {
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            qh[k] = *reinterpret_cast<const f16x8*>(qr + 16 * k);
            if (!have) qh[k] = f16x8{};
        }
    }

    // ---- copies.  Granule j of a tile: its keys 16j .. 16j+15, in one page.
    const int psm = (1 << pg.ps_log2) - 1;
    PageWindow pw;
    pw.row = a.p.table + (size_t)it.b * pg.table_stride;
    pw.fill(a.p, k_lo);
    int pages[GR], next_pages[GR];
    auto look_up = [&](int t0, int (&p)[GR]) {
        if (t0 >= pw.end(a.p)) pw.fill(a.p, t0);
#pragma unroll
        for (int j = 0; j < GR; ++j) p[j] = pw.at(a.p, t0 + 16 * j);
    };
    auto slab = [&](int page) {  // positions of the pool before the page's
        return ((size_t)imax(page, 0) * pg.Hkv + it.h) << pg.ps_log2;
    };
    constexpr int RL = BN * HD / 4096;  // 16-byte loads a thread makes of an 8-bit tile's K, and of its V
    static_assert(!I8 || RL >= 1, "8-bit tile split");
    uint4 rk[I8 ? RL : 1], rv[I8 ? RL : 1];
    float rs = 0.f;
    // Of four values, or two, the one at j.
    auto pick = [&](const int (&p)[GR], int j) {
        const int p0 = p[0], p1 = p[1];
        int x = j & 1 ? p1 : p0;
        if constexpr (GR == 4) {
            const int p2 = p[2], p3 = p[3], y = j & 1 ? p3 : p2;
            x = j & 2 ? y : x;
        }
        return x;
    };
    // Offsets of the lane's chunks in transfer 0 from a wave's base; transfer i's
    // differ by the swizzle's bits that i moves (an XOR, as the bits of rows
    // within a transfer and of transfers are apart).  V's: where a tile lies in
    // one page.
    constexpr int RPT = 64 / CH, DPT = 64 / CV;  // rows of K, dims of V a transfer
    const int k_row0 = w * (BN / 4) + lane / CH;
    const uint32_t k_off = (lane / CH) * (HD * 2) + (((lane % CH) ^ swizzle<HD * 2>(k_row0)) * 16);
    const uint32_t v_off = ((lane / CV) << (pg.ps_log2 + 1)) + (((lane % CV) ^ swizzle<BN * 2>(lane / CV)) * 16);
    // f16: a wave copies BN / 4 rows of K and HD / 4 columns of V; lane l of a
    // transfer fills place l % CH (CV) of its row (column) l / CH (CV).
    auto fetch = [&](int t0, const int (&p)[GR], int stage) {
        if constexpr (!I8) {
            const uint32_t lds = lds_addr(&tiles[stage][0]);
            const char* kb = a.p.k + (slab(pick(p, w * GR / 4)) + ((t0 + w * (BN / 4)) & psm)) * (HD * 2);
#pragma unroll
            for (int i = 0; i < T::LOADS; ++i)
                dma16(kb + i * 1024, k_off ^ (swizzle<HD * 2>(RPT * i) * 16), lds + w * (BN / 4) * (HD * 2) + i * 1024);
            const uint32_t v_lds = lds + BN * HD * 2 + w * (HD / 4) * (BN * 2);
            if ((16 << pg.ps_log2) >= 16 * BN) {  // the tile lies in one page: a base for the wave, offsets that stay
                const char* vb = a.p.v + (slab(p[0]) * HD + ((size_t)(w * (HD / 4)) << pg.ps_log2) + (t0 & psm)) * 2;
#pragma unroll
                for (int i = 0; i < T::LOADS; ++i)
                    dma16(vb + ((size_t)(DPT * i) << (pg.ps_log2 + 1)), v_off ^ (swizzle<BN * 2>(DPT * i) * 16), v_lds + i * 1024);
            } else {
                // (of 64-key tiles, every other transfer's dims swap the halves of the keys)
                const char* vb[2];
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const int c = (lane % CV) ^ swizzle<BN * 2>(DPT * x + lane / CV);
                    const int pv = pw.lane_at(a.p, t0 + 8 * c);
                    vb[x] = a.p.v + (slab(pv) * HD + ((t0 + 8 * c) & psm) + ((size_t)(w * (HD / 4) + lane / CV) << pg.ps_log2)) * 2;
                }
#pragma unroll
                for (int i = 0; i < T::LOADS; ++i)
                    dma16_lane(vb[i & 1] + ((size_t)(DPT * i) << (pg.ps_log2 + 1)), v_lds + i * 1024);
            }
        } else {
            // K: 16 dims of a key a load; V: the 16 keys of a granule of one dim
#pragma unroll
            for (int i = 0; i < RL; ++i) {
                const int x = tid + 256 * i, key = x / (HD / 16), c = x % (HD / 16);
                rk[i] = *reinterpret_cast<const uint4*>(a.p.k + (slab(pick(p, key >> 4)) + ((t0 + key) & psm)) * HD + 16 * c);
                const int dim = x / GR, g = x % GR;
                rv[i] = *reinterpret_cast<const uint4*>(a.p.v + slab(pick(p, g)) * HD + ((size_t)dim << pg.ps_log2) + ((t0 + 16 * g) & psm));
            }
            if (w < 2 && lane < BN)
                rs = (w ? a.p.v_scale : a.p.k_scale)[slab(pick(p, lane >> 4)) + ((t0 + lane) & psm)];
        }
    };
    auto stash = [&](int stage) {  // 8-bit tiles: registers to LDS as f16
        if constexpr (I8) {
            f16* Ks = tiles[stage];
            f16* Vs = tiles[stage] + BN * HD;
            auto put = [&](f16* row, int c, int sw, const uint4& x) {  // chunks c and c + 1 of a row
                *reinterpret_cast<f16x8*>(&row[(c ^ sw) * 8]) = i8x8_to_f16(x.x, x.y);
                *reinterpret_cast<f16x8*>(&row[((c + 1) ^ sw) * 8]) = i8x8_to_f16(x.z, x.w);
            };
#pragma unroll
            for (int i = 0; i < RL; ++i) {
                const int x = tid + 256 * i, key = x / (HD / 16);
                put(&Ks[key * HD], 2 * (x % (HD / 16)), swizzle<HD * 2>(key), rk[i]);
                const int dim = x / GR;
                put(&Vs[dim * BN], 2 * (x % GR), swizzle<BN * 2>(dim), rv[i]);
            }
            if (lane < BN) {
                if (w == 0) scales[stage][0][lane] = rs;
                if (w == 1) scales[stage][1][lane] = log_v_scale(rs);
            }
        }
    };

    f32x16 o[NB];
    float m = pos < 0 ? 0.f : -INFINITY, l = 0.f;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[nb][i] = 0.f;
    bool poison = false;

    // MFMA row l32 of a 32-key block stands for this key of it
    const int krow = 16 * (l32 >> 4) + 8 * ((l32 >> 2) & 1) + 4 * ((l32 >> 3) & 1) + (l32 & 3);

    const uint32_t k_lane = krow * (HD * 2) + ((hh ^ swizzle<HD * 2>(krow)) * 16);
    const uint32_t v_lane = BN * HD * 2 + nb0 * (32 * BN * 2) + l32 * (BN * 2) + ((hh ^ swizzle<BN * 2>(l32)) * 16);

    // WHOLE: every row of the wave sees every key of the tile.
    auto compute = [&](auto whole_tag, int t0, const int (&p)[GR], int stage) {
        constexpr bool WHOLE = decltype(whole_tag)::value;
        // Operand addresses: of k-step 0; a k-step's chunk moves bits that an XOR
        // reaches, blocks of rows lie constants apart.  (Opaque, so that they
        // are made from one register here, not held in many across the loop.)
        uint32_t k_at = lds_addr(&tiles[0][0]) + stage * (T::STAGE * 2) + k_lane;
        uint32_t v_at = lds_addr(&tiles[0][0]) + stage * (T::STAGE * 2) + v_lane;
        opaque(k_at);
        opaque(v_at);
        f32x16 s[KB];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            f32x16 sl;  // f16 pages: the products with q's second part
            auto& s2 = I8 ? s[kb] : sl;
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                const f16x8 kf = lds16((k_at ^ (32 * (k & 7))) + 256 * (k >> 3) + kb * (32 * HD * 2));
                s[kb] = mfma32(kf, qh[k], k ? s[kb] : f32x16{});
                if constexpr (F32) s2 = mfma32(kf, ql[k], I8 || k ? s2 : f32x16{});
            }
            if constexpr (F32 && !I8)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[kb][i] += second_part(s[kb][i], sl[i]);
        }
        {
            constexpr int N = KB * KS, PER = F32 ? 2 : 1, AHEAD = N < kAhead ? N : kAhead;
            __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x8, PER, 0);
                if (i + AHEAD < N) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            }
        }
        // register i of block kb is key 32 kb + 16 (i / 8) + 8 hh + i % 8: granule 2 kb + i / 8
        f16x8 ph[ST], pl[TWO ? ST : 1];
        float mb = m == -INFINITY ? 0.f : m;
        float top = -INFINITY;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int q = 0; q < 4; ++q) {  // four registers: keys 32 kb + 16 (q/2) + 8 hh + 4 (q%2) ..
                f32x4 ks, lv;
                if constexpr (I8) {
                    const int at = 32 * kb + 16 * (q >> 1) + 8 * hh + 4 * (q & 1);
                    ks = *reinterpret_cast<const f32x4*>(&scales[stage][0][at]);
                    lv = *reinterpret_cast<const f32x4*>(&scales[stage][1][at]);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float x = s[kb][4 * q + e];
                    if constexpr (I8)
                        s[kb][4 * q + e] = fmaf(x * ks[e], qs, lv[e] - mb);
                    else
                        s[kb][4 * q + e] = fmaf(x, qs, -mb);
                }
            }
        if constexpr (!WHOLE) {
            uint64_t seen = 0;  // bit k: key t0 + 8 hh + k
            if constexpr (SEEN) seen = sight.from(t0 + 8 * hh);
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int at = 32 * kb + 16 * (i >> 3) + (i & 7), key = t0 + 8 * hh + at;
                    const bool on = p[2 * kb + (i >> 3)] >= 0 && (SEEN ? seen >> at & 1 : key <= seen_hi && key >= seen_lo);
                    if (!on) s[kb][i] = -INFINITY;
                }
        }
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, s[kb][i]);
        if (__ballot(top > kMost || m == -INFINITY)) {
            top = fmaxf(top, shfl_xor(top, 32));
            float mn = m;
            if (mn == -INFINITY)
                mn = top > -INFINITY ? top - kLift : -INFINITY;  // mb = 0
            else if (top > kMost)
                mn = mb + top - kLift;
            const float f = m == -INFINITY ? 0.f : fast_exp2(m - mn);
            l = m == -INFINITY ? 0.f : moved<I8>(l, m - mn);
            const float delta = mn == -INFINITY ? 0.f : mn - mb;
            m = mn;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) o[nb] *= f;
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) s[kb] -= delta;
        }
        float sum = 0.f;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
                const float p0 = fast_exp2(s[kb][i]), p1 = fast_exp2(s[kb][i + 1]);
                const f16x2 hi = __builtin_convertvector(f32x2{p0, p1}, f16x2);
                ph[2 * kb + (i >> 3)][i & 7] = hi[0];
                ph[2 * kb + (i >> 3)][(i & 7) + 1] = hi[1];
                if constexpr (TWO) {
                    const f16x2 lo = __builtin_convertvector(f32x2{p0 - (float)hi[0], p1 - (float)hi[1]}, f16x2);
                    pl[2 * kb + (i >> 3)][i & 7] = lo[0];
                    pl[2 * kb + (i >> 3)][(i & 7) + 1] = lo[1];
                }
                if constexpr (I8) {
                    const float* lv = &scales[stage][1][32 * kb + 16 * (i >> 3) + 8 * hh + (i & 7)];
                    // (an unseen key's scale may be anything)
                    const float x0 = s[kb][i], x1 = s[kb][i + 1];
                    sum += WHOLE || x0 != -INFINITY ? fast_exp2(x0 - lv[0]) : 0.f;
                    sum += WHOLE || x1 != -INFINITY ? fast_exp2(x1 - lv[1]) : 0.f;
                } else if constexpr (TWO) {
                    sum += p0 + p1;
                } else {
                    sum = __builtin_amdgcn_fdot2(hi, f16x2{(f16)1.f, (f16)1.f}, sum, false);
                }
            }
        l += sum;
        uint32_t bad = 0;
#pragma unroll
        for (int st = 0; st < ST; ++st)
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                f16x8 vf = lds16((v_at ^ (32 * st)) + nb * (32 * BN * 2));
                if constexpr (!I8 && !WHOLE) {  // as in the rows kernel: infinities and NaN that not all rows see
                    uint4 u = __builtin_bit_cast(uint4, vf);
                    bad |= nonfinite2(u.x) | nonfinite2(u.y) | nonfinite2(u.z) | nonfinite2(u.w);
                    u = uint4{finite2(u.x), finite2(u.y), finite2(u.z), finite2(u.w)};
                    vf = __builtin_bit_cast(f16x8, u);
                }
                o[nb] = mfma32(vf, ph[st], o[nb]);
                if constexpr (TWO) o[nb] = mfma32(vf, pl[st], o[nb]);
                if constexpr (!WHOLE) __builtin_amdgcn_sched_barrier(0);  // few operands in flight: registers
            }
        if constexpr (WHOLE && !I8) {
            // the first operands are on their way during the first weights'
            // exponentials; the others' run beside the products
            constexpr int N = ST * NB, PER = TWO ? 2 : 1, AHEAD = N < kAhead ? N : kAhead;
            constexpr int FIRST = TWO ? 24 : 14, EACH = (TWO ? 24 : 13) * ST / N;
            __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);
            __builtin_amdgcn_sched_group_barrier(0x2, FIRST, 0);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x8, PER, 0);
                if (i + AHEAD < N) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x2, EACH, 0);
            }
        }
        if constexpr (!I8 && !WHOLE) {
            if (__ballot(bad != 0)) {
                // Again, without the keys that no row of the wave sees (slots
                // behind the sequence, pages that are none): they ask for
                // nothing.  (Masked above, they cost a 256-dim window 107 -> 145 us.)
                bad = 0;
#pragma unroll 1
                for (int st = 0; st < ST; ++st) {
                    const int key = t0 + 16 * st + 8 * hh;
                    int page = p[0];
#pragma unroll
                    for (int j = 1; j < GR; ++j) page = st == j ? p[j] : page;
                    const uint4 on = page >= 0 ? keys8_mask(any_lo - key, any_hi - key) : uint4{};
#pragma unroll 1
                    for (int nb = 0; nb < NB; ++nb) {
                        const uint4 u = __builtin_bit_cast(uint4, lds16((v_at ^ (32 * st)) + nb * (32 * BN * 2)));
                        bad |= nonfinite2(u.x & on.x) | nonfinite2(u.y & on.y) | nonfinite2(u.z & on.z) | nonfinite2(u.w & on.w);
                    }
                }
                poison = poison || __ballot(bad != 0) != 0;
            }
        }
    };

    if (n_t > 0) {
        look_up(k_lo, pages);
        fetch(k_lo, pages, 0);
        stash(0);
        // Tiles of one kind run in a loop of their own: with a branch inside one
        // loop the output's registers are copied at every join.
        int t = 0;
        auto begin = [&]() {  // the tile is in LDS, the next one on its way
            if constexpr (!I8) wait_dma<0>();
            __syncthreads();
            if (t + 1 < n_t) {
                look_up(k_lo + (t + 1) * BN, next_pages);
                fetch(k_lo + (t + 1) * BN, next_pages, (t + 1) & 1);
            }
        };
        auto end = [&]() {
            if (t + 1 < n_t) stash((t + 1) & 1);
#pragma unroll
            for (int j = 0; j < GR; ++j) pages[j] = next_pages[j];
            ++t;
        };
        auto whole = [&]() {
            const int t0 = k_lo + t * BN;
            bool all = t < n_t && t0 + BN - 1 <= all_hi && t0 >= all_lo;
#pragma unroll
            for (int j = 0; j < GR; ++j) all = all && pages[j] >= 0;
            return all;
        };
        while (t < n_t) {
            while (whole()) {
                begin();
                compute(std::true_type{}, k_lo + t * BN, pages, t & 1);
                end();
            }
            if (t >= n_t) break;
            begin();
            const int t0 = k_lo + t * BN;
            if (t0 <= any_hi && t0 + BN - 1 >= any_lo) compute(std::false_type{}, t0, pages, t & 1);
            end();
        }
    }

    // ---- results
    if constexpr (!I8) {
        float z = 0.f;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int i = 0; i < 16; ++i) z = fmaf(o[nb][i], 0.f, z);
        if (poison || __ballot(z != 0.f)) {
            // rare, as in the rows kernel: V's infinities and NaN go to the rows that see them
            const size_t step = (size_t)1 << pg.ps_log2;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                f32x16 add;
#pragma unroll
                for (int i = 0; i < 16; ++i) add[i] = 0.f;
                pw.fill(a.p, k_lo);
                for (int key = k_lo; key < k_hi; ++key) {
                    if (key >= pw.end(a.p)) pw.fill(a.p, key);
                    const int page = pw.at(a.p, key);
                    if (page < 0 || (SEEN ? !sight.sees(key) : key > seen_hi || key < seen_lo)) continue;
                    const f16* e = reinterpret_cast<const f16*>(a.p.v) + v_offset(a.p, page, it.h, key & psm) +
                                   ((32 * (nb0 + nb) + 4 * hh) << pg.ps_log2);
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float y = (float)*e;
                        if (!(fabsf(y) < INFINITY)) add[i] += y;
                        e += (i & 3) < 3 ? step : 5 * step;  // dims 32 (nb0 + nb) + 8 (i/4) + 4 hh + i%4
                    }
                }
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (!(fabsf(add[i]) < INFINITY)) o[nb][i] = add[i];
            }
        }
    }
    float sum = l + shfl_xor(l, 32);
    if (row >= n_rows) return;
    if (it.splits > 1) {
        const size_t at = (size_t)(it.first + it.split * it.stride) * BM;
        float* dst = a.part_o + at * HD;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                *reinterpret_cast<f32x4*>(dst + part_at<HD>(w / DS, 4 * (nb0 + nb) + q, lane)) =
                    f32x4{o[nb][4 * q], o[nb][4 * q + 1], o[nb][4 * q + 2], o[nb][4 * q + 3]};
        if (hh == 0 && nb0 == 0) *reinterpret_cast<f32x2*>(a.part_ml + (at + row - r0) * 2) = f32x2{m, sum};
    } else {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        if constexpr (!I8)
            if (sum == 0.f)  // (o may hold infinities)
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) o[nb] = f32x16{};
        QT* dst = static_cast<QT*>(a.out) +
                  ((size_t)(it.s.row0 + row / pg.G) * pg.Hkv * pg.G + it.h * pg.G + row % pg.G) * HD + 32 * nb0;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
            if constexpr (F32) {
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    *reinterpret_cast<f32x4*>(dst + 32 * nb + 8 * q + 4 * hh) =
                        f32x4{o[nb][4 * q], o[nb][4 * q + 1], o[nb][4 * q + 2], o[nb][4 * q + 3]} * inv;
            } else {
                // the row's two lanes trade, so that each stores 8 dims: the lower
                // those of q, the upper those of q + 1
#pragma unroll
                for (int q = 0; q < 4; q += 2) {
                    uint32_t x[2][2];
#pragma unroll
                    for (int e = 0; e < 2; ++e)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const float y0 = o[nb][4 * (q + e) + 2 * i] * inv, y1 = o[nb][4 * (q + e) + 2 * i + 1] * inv;
                            x[e][i] = __builtin_bit_cast(uint32_t, f16x2{(f16)y0, (f16)y1});
                        }
                    uint4 y;
                    swap_halves(x[0][0], x[1][0], y.x, y.z);
                    swap_halves(x[0][1], x[1][1], y.y, y.w);
                    *reinterpret_cast<uint4*>(dst + 32 * nb + 8 * (q + hh)) = y;
                }
            }
    }
}

// Keys a tile, waves to a row and workgroups a CU, by what fits the registers
// (two workgroups a CU leave 256, one 512) and the LDS.  With both sides
// measured: f32 queries at 128 dims 64 keys and one workgroup 768 us, 32 keys and
// two 386 (nine 8-bit sequences); f16 at 256 dims 64 keys and one 135 us, 32 keys
// and two, though registers spilled (129 then; 63 now), 119 (a window of 1024;
// 106 now), two waves to a row 139; 8 bits at 256 dims 64 keys and one 366, two
// waves to a row 585.  512 dims (queries of 128 registers, outputs of 256) need
// waves that share rows: f16 two 157 us, four 207; 8 bits, whose tiles pass the
// registers too, two 354, four 263; f32 queries two 478, four 297.
constexpr int chunk_bn(int hd, bool i8, bool f32) { return hd == 512 || (hd == 256 && (f32 || !i8)) || (hd == 128 && f32) ? 32 : 64; }
constexpr int chunk_occ(int hd, bool i8, bool f32) { return hd <= 128 || (hd == 256 && !f32 && !i8) ? 2 : 1; }
constexpr int chunk_ds(int hd, bool i8, bool f32) { return hd <= 256 ? 1 : i8 || f32 ? 4 : 2; }
int chunk_rows(int hd, bool i8, bool f32) { return 128 / chunk_ds(hd, i8, f32); }
int chunk_occ_of(int hd, bool i8, bool f32) { return chunk_occ(hd, i8, f32); }

template <int HD, bool I8, bool F32>
static void go_chunk(const AttnPagedArgs& a, unsigned items, hipStream_t st) {
    auto launch = [&](auto seen) {
        hipLaunchKernelGGL((paged_chunk_kernel<HD, I8, F32, chunk_bn(HD, I8, F32), chunk_ds(HD, I8, F32), chunk_occ(HD, I8, F32), decltype(seen)::value>), dim3(items), dim3(256), 0, st, a);
    };
    a.seen ? launch(std::true_type{}) : launch(std::false_type{});
}
void launch_chunk(const AttnPagedArgs& a, int hd, bool i8, bool f32, unsigned items, hipStream_t st) {
    auto by = [&](auto tag) {
        constexpr int HD = decltype(tag)::value;
        if (i8) f32 ? go_chunk<HD, true, true>(a, items, st) : go_chunk<HD, true, false>(a, items, st);
        else f32 ? go_chunk<HD, false, true>(a, items, st) : go_chunk<HD, false, false>(a, items, st);
    };
    if (hd == 64) by(std::integral_constant<int, 64>{});
    else if (hd == 128) by(std::integral_constant<int, 128>{});
    else if (hd == 256) by(std::integral_constant<int, 256>{});
    else by(std::integral_constant<int, 512>{});
}

}  // namespace lmx
