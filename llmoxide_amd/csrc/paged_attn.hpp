// Attention over pages: what its kernels share.
#pragma once

#include "paged.hpp"

namespace lmx {

struct AttnPagedArgs {
    PagedArgs p;
    const void* q;
    void* out;
    size_t q_row_stride, q_head_stride;
    float c;              // scale * log2(e)
    float* part_o;        // [items][bm][hd]   partial outputs, unnormalised (chunks: in part_at's order)
    float* part_ml;       // [items][bm][2]    (reference exponent, sum)
    int4* rows;           // [n_seq][Hkv][rt_max]  (first item, item stride, splits, 0)
    int n_items;          // workgroups, and slots in part_o
    int target;           // items aimed at where splits help
    int least;            // units a split has at least
    int rt_max;           // entries of `rows` a (sequence, head)
    int lo_rows, hi_rows; // this kernel takes sequences with lo_rows < rows * G <= hi_rows
};

// paged_chunk.hip: rows of its workgroups, and the launch.
int chunk_rows(int hd, bool i8, bool f32);
int chunk_occ_of(int hd, bool i8, bool f32);  // workgroups a CU holds
void launch_chunk(const AttnPagedArgs& a, int hd, bool i8, bool f32, unsigned items, hipStream_t st);

// Where a chunk's partial output keeps the dims 8c + 4 (lane / 32) .. of row
// 32 blk + lane % 32 of its tile.
template <int HD>
__device__ __forceinline__ int part_at(int blk, int c, int lane) {
    return ((blk * (HD / 8) + c) * 64 + lane) * 4;
}

// One work item: a row tile of one sequence and kv head, over one split.
struct Item {
    int b, tile, h, split, splits;
    int first, stride;  // item index of split 0, and from one split to the next
    PagedSeq s;
    SeqWork w;
    int per;
};

// Sequence b's rows and work; no work where it has none or another kernel's
// share of them.
__device__ __forceinline__ void load_work(const AttnPagedArgs& a, int b, int bm, PagedSeq& s, SeqWork& w) {
    s = PagedSeq{0, 0, 0};
    w = SeqWork{0, 0, 0};
    if (b < a.p.g.n_seq) {
        s = paged_seq(a.p.g, a.p.cu[b], a.p.cu[b + 1], a.p.ctx[b]);
        w = seq_work(a.p.g, s, bm);
        const int64_t rows = (int64_t)s.n * a.p.g.G;
        if (rows <= a.lo_rows || rows > a.hi_rows) w.rt = 0;
    }
}

// Item `id` of the batch, by every wave for itself: the lengths are read from
// the device in the call, so a replayed graph splits by the lengths of that
// replay.  Each lane takes a sequence (64 at a time); the total of units x
// row tiles decides how long a split is, a scan over the sequences' item
// counts finds the one that holds `id`.  False: no such item.
// `longest_first`: of 64 sequences, those with the longest reach come first.
__device__ __forceinline__ bool find_item(const AttnPagedArgs& a, int id, int bm, bool splits_on, bool longest_first,
                                          Item& o) {
    const int lane = __lane_id(), Hkv = a.p.g.Hkv;
    PagedSeq s;
    SeqWork w;
    int b;
    auto load = [&](int c0) {
        b = c0 + lane;
        load_work(a, b, bm, s, w);
        const int n = min(64, a.p.g.n_seq - c0);
        if (!longest_first || n == 1) return;
        int rank = 0;
        for (int j = 0; j < n; ++j) {
            const int u = __builtin_amdgcn_readlane(w.units, j);
            rank += u > w.units || (u == w.units && j < lane);
        }
        // lanes behind the last sequence, of no work, stay where they are
        const int to = 4 * (lane < n ? rank : lane);
        auto put = [&](int& x) { x = __builtin_amdgcn_ds_permute(to, x); };
        put(b), put(s.row0), put(s.n), put(s.ctx), put(w.rt), put(w.lo), put(w.units);
    };
    load(0);
    o.per = 1000000000;
    if (splits_on) {
        float work = (float)w.rt * (float)w.units;
        for (int c0 = 64; c0 < a.p.g.n_seq; c0 += 64) {
            PagedSeq s2;
            SeqWork w2;
            load_work(a, c0 + lane, bm, s2, w2);
            work += (float)w2.rt * (float)w2.units;
        }
        o.per = units_per_split(wave_sum64(work) * (float)Hkv, a.target, a.least);
    }
    int base = 0;
    for (int c0 = 0;; ) {
        const int n = w.rt * Hkv * seq_splits(w, o.per);
        const int upto = a.p.g.n_seq == 1 ? n : wave_scan(n);
        const uint64_t has = __ballot(base + upto > id);
        if (has) {
            const int l = __builtin_ctzll(has);
            auto get = [&](int x) { return __builtin_amdgcn_readlane(x, l); };
            o.b = get(b);
            o.s = PagedSeq{get(s.row0), get(s.n), get(s.ctx)};
            o.w = SeqWork{get(w.rt), get(w.lo), get(w.units)};
            o.splits = seq_splits(o.w, o.per);
            const int first = base + get(upto) - get(n);
            // item order within a sequence: split, then row tile, then kv head
            // (with 8 heads every XCD keeps to one, and the row tiles that
            // share its keys meet in that XCD's L2)
            const int i = id - first;
            o.h = i % Hkv;
            const int at = (i / Hkv) % o.w.rt;
            o.tile = o.w.rt - 1 - at;  // the last rows, which see the most keys, first
            o.split = i / Hkv / o.w.rt;
            o.first = first + at * Hkv + o.h;
            o.stride = Hkv * o.w.rt;
            return true;
        }
        base += __builtin_amdgcn_readlane(upto, 63);
        c0 += 64;
        if (c0 >= a.p.g.n_seq) return false;
        load(c0);
    }
}

// Two f16 in a word: the sign bit of each half that is infinite or NaN (an
// exponent of all ones carries into it), and the word without those halves.
__device__ __forceinline__ uint32_t nonfinite2(uint32_t x) { return ((x & 0x7c007c00u) + 0x04000400u) & 0x80008000u; }
__device__ __forceinline__ uint32_t finite2(uint32_t x) {
    const uint32_t m = nonfinite2(x);
    return x & ~(m | (m - (m >> 15)));
}

// Of eight f16, those lo .. hi (any integers) all ones.
__device__ __forceinline__ uint4 keys8_mask(int lo, int hi) {
    auto word = [&](int i) {
        return (lo <= 2 * i && 2 * i <= hi ? 0xffffu : 0u) | (lo <= 2 * i + 1 && 2 * i + 1 <= hi ? 0xffff0000u : 0u);
    };
    return uint4{word(0), word(1), word(2), word(3)};
}

// f32 queries are two f16 parts, hi and lo.  Where K or q holds an infinity the
// score is hi's alone: lo's product would be inf - inf, or 0 * inf, beside it.
// (In f16 pages K may; the two products have a sum each there.)
__device__ __forceinline__ float finite_or_0(float x) { return fabsf(x) < INFINITY ? x : 0.f; }
__device__ __forceinline__ float second_part(float hi, float lo) { return fabsf(hi) < INFINITY ? lo : 0.f; }

// 8-bit values: a key's V scale joins its score's exponent as its logarithm, so
// the running reference m is that of score + log2(scale).  In the sum of the
// softmax a key counts exp2(score - m), without its scale, by an exponential of
// its own.  (The weight divided by the scale would cost one multiplication, and
// 1 to 7% less time, but beside a scale 2^130 times as large a weight lies below
// f32's range where its key may have half of the sum.)  With scales of 2^-90 to
// 2^100 that term is in range wherever it matters: no score is above m + 14 + 90,
// and the largest is at least m + 6 - 100, 2^32 above what f32 loses.
//
// log2 of a V scale, of 2^-90 at least: finite, and values below 1e-24 are all
// that notices.
__device__ __forceinline__ float log_v_scale(float s) { return __builtin_amdgcn_logf(s < 0x1p-90f ? 0x1p-90f : s); }
// The weight of a partial output in a join, d below the highest reference.  Never
// 0, which would make NaN of an infinity among V: 2^-126 of a finite output is
// far below the last place of the weights beside it.
__device__ __forceinline__ float join_weight(float d) { return fmaxf(fast_exp2(d), 0x1p-126f); }
// A sum brought to a reference -d above its own (d <= 0).  I8: a step down to
// -240, as scales alone make it, in two factors that f32 holds; above
// -120 the second is 1.
template <bool I8>
__device__ __forceinline__ float moved(float l, float d) {
    if constexpr (I8) return l * fast_exp2(fmaxf(d, -120.f)) * fast_exp2(fminf(d + 120.f, 0.f));
    return l * fast_exp2(d);
}

// Two int8 words -> f16: x's bytes 0, 1 (lo) and 2, 3 (hi) as f16 pairs.  A
// byte b + 128 set under 0x6400 is the f16 1024 + b + 128: exact, so is the
// difference.
__device__ __forceinline__ void i8x4_to_f16(uint32_t x, f16x2& lo, f16x2& hi) {
    x ^= 0x80808080u;
    const uint32_t a = __builtin_amdgcn_perm(0x64646464u, x, 0x04010400u);
    const uint32_t b = __builtin_amdgcn_perm(0x64646464u, x, 0x04030402u);
    const f16x2 k = {(f16)1152.f, (f16)1152.f};
    lo = __builtin_bit_cast(f16x2, a) - k;
    hi = __builtin_bit_cast(f16x2, b) - k;
}
// Eight int8 in two words as eight f16.
__device__ __forceinline__ f16x8 i8x8_to_f16(uint32_t x, uint32_t y) {
    f16x2 a, b, c, d;
    i8x4_to_f16(x, a, b);
    i8x4_to_f16(y, c, d);
    return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// The pages of a run of keys, 64 table entries in the wave's lanes, so that
// lookups in a loop wait on no memory.  at() and lane_at() take keys of the
// entries that fill() was given; keys of a tile whose first key is a multiple
// of 64 never straddle two fills that begin at such a key.
struct PageWindow {
    const int32_t* row;  // the sequence's table
    int first;           // entry in lane 0
    int ids;             // the lane's page, -1: none
    __device__ __forceinline__ void fill(const PagedArgs& a, int key) {
        first = key >> a.g.ps_log2;
        const int e = first + (int)__lane_id();
        ids = e < a.g.table_stride ? paged_page(a.g, row[e]) : -1;
    }
    // One behind the last key of the window (a multiple of 64 where fill's was).
    __device__ __forceinline__ int end(const PagedArgs& a) const { return (first + 64) << a.g.ps_log2; }
    // Page of key k (wave-uniform).
    __device__ __forceinline__ int at(const PagedArgs& a, int k) const {
        return __builtin_amdgcn_readlane(ids, (k >> a.g.ps_log2) - first);
    }
    // Page of the lane's own key.
    __device__ __forceinline__ int lane_at(const PagedArgs& a, int k) const {
        return __shfl(ids, (k >> a.g.ps_log2) - first, 64);
    }
};

}  // namespace lmx
