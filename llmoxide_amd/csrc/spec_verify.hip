// Which drafted rows a target model accepts, and the token behind them.
//
// The walk has all rows' p(c), q(c) and u in LDS, so that accepting and refusing
// reads no memory; only sums over the vocabulary that a second sibling asks for
// (drafts that were sampled), or the largest scores (greedy), are passes over a
// row of p, by one workgroup of the request.  Then the last row's distribution is
// weighed, 256 entries a sum; and one wave adds the sums up, finds the one where the
// running sum passes r times the whole, and goes through its 256 entries.  Up to 32768
// entries all of this is one launch, a workgroup a request.  Longer rows are weighed by
// a workgroup for 4096 entries; chosen drafts and chains, which need no passes, are
// then walked by every workgroup that weighs, which saves a launch.
//
// What is left of p after refusals needs one number: with w = p - a q wherever
// that is above 0, and W its sum, the next refusal's w / W - q is, times W,
// p - (a + W) q.  So no distribution is ever written.
//
// Sums are in 64 bits: two entries of a vocabulary of 131072 may lie 1e-7 apart
// in the running sum, which is where a 32-bit sum's own rounding lies.  Each is
// made in an order that the shapes alone decide.
//
// Bound by latency: the last rows (4 or 8 bytes an entry) are 8 MB for 16 requests of
// 131072 entries, chosen drafts: 8.8 us from a graph (weights 8.3, token 4.5 by
// themselves), 15 from the host.  A pass takes a workgroup 9.7 us for 100003 entries of
// p and q (82 GB/s of one CU; conversions to 64 bits are what it costs): eight sampled
// trees of up to 24 rows 44 us.
#include <type_traits>

#include "spec.hpp"

namespace lmx {

constexpr int kGroup = 256;            // entries of the vocabulary a sum
constexpr int kGroups = 16;            // sums a workgroup makes, four a wave
constexpr int kOne = 1 << 15;          // most entries that one workgroup goes through

// Where the walk ended.
struct Last {
    int row;       // of the batch; -1: the request has none
    int at;        // of the request
    int children;  // of that row: all were refused
    int pad;
    double a;
};

struct VerifyArgs {
    int n_seq, n_tokens, max_new, vocab;
    int n_groups, n_blocks;  // sums a request, workgroups that make them
    size_t p_stride, q_stride;
    const int32_t* cu;
    const int32_t* tokens;
    const int32_t* parent;
    const void* p;
    const void* q;
    const float* u;
    const float* r;
    int32_t* path;
    int32_t* accepted;
    int32_t* token;
    int32_t* lens;
    double* sums;   // [n_seq][n_groups]
    Last* last;     // [n_seq]
};

// A probability; what is not above 0 and finite is 0.
__device__ __forceinline__ double prob(float x) {
    const bool on = __builtin_bit_cast(uint32_t, x) - 1u < 0x7f7fffffu;  // the bits of 0 < x < inf
    return (double)(on ? x : 0.f);
}

// A row's parent within the request, -1 for a root.
__device__ __forceinline__ int parent_of(const VerifyArgs& a, int row0, int i) {
    const int p = a.parent ? a.parent[row0 + i] : i - 1;
    return p >= 0 && p < i ? p : -1;
}

// Four consecutive entries of a row, which need not be aligned to more than one.
template <typename T>
struct Four {
    typedef T type __attribute__((ext_vector_type(4), aligned(sizeof(T))));
};
template <typename T>
__device__ __forceinline__ f32x4 four(const T* p) {
    const typename Four<T>::type x = *reinterpret_cast<const typename Four<T>::type*>(p);
    return f32x4{(float)x[0], (float)x[1], (float)x[2], (float)x[3]};
}
// Entries t .. t+3 of a row of n, `none` behind its end.
template <typename T>
__device__ __forceinline__ f32x4 four_of(const T* p, int t, int n, float none) {
    if (t + 4 <= n) return four(p + t);
    f32x4 x = {none, none, none, none};
#pragma unroll
    for (int j = 0; j < 3; ++j)
        if (t + j < n) x[j] = (float)p[t + j];
    return x;
}

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) x += __shfl_xor(x, m, 64);
    return x;
}
// Sum of the lanes before this one.
__device__ __forceinline__ double wave_before(double x) {
    const int lane = __lane_id();
    double y = x;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const double z = __shfl_up(y, d, 64);
        y += lane >= d ? z : 0.0;
    }
    const double z = __shfl_up(y, 1, 64);
    return lane ? z : 0.0;
}
__device__ __forceinline__ double lane_value(double x, int lane) { return __shfl(x, lane, 64); }

// CHAIN: sampled, each row the next one's parent.
enum Drafts { CHOSEN, CHAIN, SAMPLED, GREEDY };

// A request's rows in LDS.
struct Rows {
    int up[LMXS_MAX_ROWS], tok[LMXS_MAX_ROWS];  // parent (-1: none), token (-1: none, or no parent)
    float p[LMXS_MAX_ROWS], q[LMXS_MAX_ROWS], u[LMXS_MAX_ROWS];
};

template <typename T, Drafts D, int NT>
__device__ __forceinline__ void load_rows(const VerifyArgs& a, const SpecRows& s, Rows& r) {
    const T* const p = static_cast<const T*>(a.p);
    const T* const q = static_cast<const T*>(a.q);
    for (int i = threadIdx.x; i < s.n; i += NT) {
        const int above = parent_of(a, s.row0, i), t = a.tokens[s.row0 + i];
        const bool on = above >= 0 && (uint32_t)t < (uint32_t)a.vocab;
        r.up[i] = above;
        r.tok[i] = on ? t : -1;
        if (D != GREEDY && on) {
            r.p[i] = (float)p[(size_t)(s.row0 + above) * a.p_stride + t];
            if (D != CHOSEN) r.q[i] = (float)q[(size_t)(s.row0 + above) * a.q_stride + t];
            r.u[i] = a.u[s.row0 + i];
        }
    }
    __syncthreads();
}

// The walk, by every wave for itself over the same LDS (so that passes' barriers
// meet).  mass(row, c): sum of (p - c q)+; best_of(row): its largest entry's index.
// path: where to note the accepted rows, or NULL.
struct Walk {
    int cur, count, children, best;
    double a;
};
template <Drafts D, typename M, typename B>
__device__ __forceinline__ Walk walk(const SpecRows& s, const Rows& r, int32_t* path, const M& mass, const B& best_of) {
    const int lane = threadIdx.x & 63;
    Walk w{0, s.n ? 1 : 0, 0, -1, 0.0};
    double W = 1.0;
    bool known = D != GREEDY;  // SAMPLED: W is that of w.a; GREEDY: best is cur's
    for (int from = 1;;) {
        int i = -1;
        for (int c0 = from & ~63; c0 < s.n && i < 0; c0 += 64) {
            const int k = c0 + lane;
            const uint64_t hit = __ballot(k >= from && k < s.n && r.up[k < s.n ? k : 0] == w.cur);
            if (hit) i = c0 + __builtin_ctzll(hit);
        }
        if (i < 0) break;
        from = i + 1;
        ++w.children;
        const int t = r.tok[i];
        bool pass = false;
        if constexpr (D == GREEDY) {
            if (!known) w.best = best_of(w.cur);
            known = true;
            pass = t >= 0 && t == w.best;
        } else if (t >= 0) {
            double x = prob(r.p[i]);
            if constexpr (D != CHOSEN) {
                if (!known) W = mass(w.cur, w.a);
                known = true;
                const double y = prob(r.q[i]);
                x = fmax(x - w.a * y, 0.0);
                pass = (double)r.u[i] * W * y < x;
                if (!pass) {
                    w.a += W;
                    known = false;
                }
            } else {
                bool twice = false;  // an earlier sibling was the same token
                for (int c0 = (w.cur + 1) & ~63; c0 < i; c0 += 64) {
                    const int k = c0 + lane;
                    twice = twice || __ballot(k < i && k > w.cur && r.up[k < s.n ? k : 0] == w.cur && r.tok[k < s.n ? k : 0] == t);
                }
                if (twice) x = 0.0;
                pass = (double)r.u[i] * W < x;
                if (!pass) W -= x;
            }
        }
        if (pass) {
            if (path && threadIdx.x == 0) path[w.count] = i;
            ++w.count;
            w.cur = i;
            w.children = 0;
            w.a = 0.0;
            W = 1.0;
            known = D != GREEDY;
        }
    }
    if (D == GREEDY && s.n && !known) w.best = best_of(w.cur);
    return w;
}
// What the walk found, by the request's first workgroup.
template <Drafts D, int NT>
__device__ __forceinline__ void write_walk(const VerifyArgs& a, int b, const SpecRows& s, const Walk& w) {
    int32_t* path = a.path + (size_t)b * a.max_new;
    for (int j = w.count + threadIdx.x; j < a.max_new; j += NT) path[j] = -1;
    if (threadIdx.x == 0) {
        if (w.count) path[0] = 0;
        a.accepted[b] = w.count;
        if (a.lens) a.lens[b] += w.count;
        if (D == GREEDY || !s.n) a.token[b] = w.best;
        if (D != GREEDY && a.last) a.last[b] = Last{s.n ? s.row0 + w.cur : -1, w.cur, w.children, 0, w.a};
    }
}

// ---- the last row's weights
//
// Weights behind the walk: (p - a q)+, or p, of which the tokens of refused children
// are taken by their readers.
template <typename T, bool Q>
struct Weights {
    const T* p;
    const T* q;
    double a;
    int vocab;
    __device__ __forceinline__ void load(int t, f32x4& x, f32x4& y) const {
        x = four_of(p, t, vocab, 0.f);
        if (Q) y = four_of(q, t, vocab, 0.f);
    }
    __device__ __forceinline__ double of(float x, float y) const {
        return Q ? fmax(prob(x) - a * prob(y), 0.0) : prob(x);
    }
};
template <typename T, bool Q>
__device__ __forceinline__ Weights<T, Q> weights_of(const VerifyArgs& a, int row, double c) {
    // (behind a leaf a is 0 and q says nothing: p is read in its place)
    const T* const p = static_cast<const T*>(a.p) + (size_t)row * a.p_stride;
    return Weights<T, Q>{p, Q && c != 0.0 ? static_cast<const T*>(a.q) + (size_t)row * a.q_stride : p, c, a.vocab};
}

// Where the walk's children are: child(k) is the token of row k if it continues row
// `at`, else -1; `drop`: their tokens weigh nothing.
template <typename C>
struct Refused {
    bool drop;
    int at, n;
    const C& child;
    // The lanes' entries 4 lane .. of W groups from g0 on that are such tokens: 0.
    template <int W>
    __device__ __forceinline__ void clear(int g0, f32x4 (&x)[W]) const {
        if (!drop) return;
        const int lane = __lane_id();
        for (int c0 = (at + 1) & ~63; c0 < n; c0 += 64) {
            const int t = child(c0 + lane);
            for (uint64_t left = __ballot(t >= g0 * kGroup && t < (g0 + W) * kGroup); left; left &= left - 1) {
                const int e0 = __builtin_amdgcn_readlane(t, __builtin_ctzll(left)) - g0 * kGroup;
#pragma unroll
                for (int g = 0; g < W; ++g)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (e0 == g * kGroup + 4 * lane + e) x[g][e] = 0.f;
            }
        }
    }
};

// A wave's W sums from group g0 on, of whose weights x and y are loaded.
template <int W, typename T, bool Q, typename C>
__device__ __forceinline__ void weigh(const Weights<T, Q>& wt, const Refused<C>& refused, int g0, int n_groups,
                                      f32x4 (&x)[W], const f32x4 (&y)[W], double* sums) {
    const int lane = __lane_id();
    refused.clear(g0, x);
    double sum[W];
#pragma unroll
    for (int g = 0; g < W; ++g) {
        sum[g] = 0.0;
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[g] += wt.of(x[g][e], Q ? y[g][e] : 0.f);
    }
    // Over the lanes: while there are several sums a lane hands half of them to its
    // partner, so that lane l ends with sum l % W.
#pragma unroll
    for (int m = 1, n = W; m < 64; m <<= 1) {
        if (n > 1) {
            n >>= 1;
#pragma unroll
            for (int g = 0; g < n; ++g) {
                // (sum 2g is the even lanes')
                const double give = lane & m ? sum[2 * g] : sum[2 * g + 1], keep = lane & m ? sum[2 * g + 1] : sum[2 * g];
                sum[g] = keep + __shfl_xor(give, m, 64);
            }
        } else {
            sum[0] += __shfl_xor(sum[0], m, 64);
        }
    }
    if (lane < W && g0 + lane < n_groups) sums[g0 + lane] = sum[0];
}

// The token, from the groups' sums, by a wave.
template <typename T, bool Q, typename C>
__device__ __forceinline__ int find_token(Weights<T, Q> wt, Refused<C> refused, int n_groups, const double* sums, double r) {
    const int lane = __lane_id();
    // Of 64 lanes' values, those of which `some` count: the first whose running sum
    // passes the target, or else the last that counts, or else -1.
    auto choose = [&](bool passes, bool some) {
        const uint64_t p = __ballot(passes && some), s = __ballot(some);
        return p ? (int)__builtin_ctzll(p) : s ? 63 - (int)__builtin_clzll(s) : -1;
    };
    // The entry of group g at which the running sum, `before` at its start, passes the target.
    auto search = [&](int g, double before, double target) {
        const int t0 = g * kGroup + 4 * lane;
        f32x4 x[1], y = {};
        wt.load(t0, x[0], y);
        refused.clear(g, x);
        double v[4], sum = 0.0;
#pragma unroll
        for (int e = 0; e < 4; ++e) sum += v[e] = wt.of(x[0][e], y[e]);
        double run = before + wave_before(sum);
        int hit = -1, any = -1;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            run += v[e];
            if (v[e] > 0.0) {
                any = t0 + e;
                if (run > target && hit < 0) hit = any;
            }
        }
        const int at = choose(hit >= 0, any >= 0);
        return at < 0 ? -1 : __builtin_amdgcn_readlane(hit >= 0 ? hit : any, at);
    };

    // ---- the sums: a run of them a lane
    const int per = (n_groups + 63) / 64, first = lane * per;
    constexpr int U = 8;
    double part = 0.0;
    for (int k0 = 0; k0 < per; k0 += U) {
        double v[U];
#pragma unroll
        for (int k = 0; k < U; ++k) v[k] = k0 + k < per && first + k0 + k < n_groups ? sums[first + k0 + k] : 0.0;
#pragma unroll
        for (int k = 0; k < U; ++k) part += v[k];
    }
    const double before = wave_before(part), total = lane_value(before + part, 63);
    int token = -1;
    if (total > 0.0) {
        const double target = r * total;
        const int at = choose(before + part > target, part > 0.0);
        // that lane's run, by all lanes alike
        const int g1 = at * per;
        double run = lane_value(before, at), below = run;
        int group = -1;
        for (int k = 0; k < per && g1 + k < n_groups; ++k) {
            const double x = sums[g1 + k];
            if (x > 0.0) {
                group = g1 + k;
                below = run;
                if (run + x > target) break;  // uniform
            }
            run += x;
        }
        token = search(group, below, target);
    } else {
        // Nothing is left (the drafts had all of p): from p itself, twice through the row,
        // 256 entries a step that waits for the one before: rare, and slow (131072 entries
        // 93 us, where something is left 7.7).
        wt.a = 0.0;
        refused.drop = false;
        double all = 0.0;
        for (int g = 0; g < n_groups; ++g) {
            f32x4 x, y = {};
            wt.load(g * kGroup + 4 * lane, x, y);
#pragma unroll
            for (int e = 0; e < 4; ++e) all += prob(x[e]);
        }
        all = wave_sum(all);
        const double target = r * all;
        double run = 0.0;
        for (int g = 0; all > 0.0 && g < n_groups; ++g) {
            f32x4 x, y = {};
            wt.load(g * kGroup + 4 * lane, x, y);
            double sum = 0.0;
#pragma unroll
            for (int e = 0; e < 4; ++e) sum += prob(x[e]);
            sum = wave_sum(sum);
            if (sum > 0.0) token = search(g, run, target);
            if (run + sum > target) break;  // uniform
            run += sum;
        }
    }
    return token;
}

// ---- a request in one workgroup, from its rows to its token
template <typename T, Drafts D>
__device__ __forceinline__ void token_here(const VerifyArgs& a, int b, const SpecRows& s, const Rows& rows, const Walk& k,
                                           double* sums) {
    constexpr bool Q = D != CHOSEN;
    constexpr int W = Q ? 4 : 8;  // groups of a wave on the way
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const Weights<T, Q> wt = weights_of<T, Q>(a, s.row0 + k.cur, k.a);
    auto child = [&](int i) { return i > k.cur && i < s.n && rows.up[i < s.n ? i : 0] == k.cur ? rows.tok[i] : -1; };
    const Refused<decltype(child)> refused{D == CHOSEN && k.children > 0, k.cur, s.n, child};
    for (int g0 = w * W; g0 < a.n_groups; g0 += 16 * W) {
        f32x4 x[W], y[W];
#pragma unroll
        for (int g = 0; g < W; ++g) wt.load((g0 + g) * kGroup + 4 * lane, x[g], y[g]);
        weigh<W>(wt, refused, g0, a.n_groups, x, y, sums);
    }
    __syncthreads();
    if (w) return;
    const int token = find_token(wt, refused, a.n_groups, sums, fmax((double)a.r[b], 0.0));
    if (lane == 0) a.token[b] = token;
}

// A workgroup a request: the walk, and where TOKEN what follows from it.
template <typename T, Drafts D, bool TOKEN>
__global__ __launch_bounds__(1024) void spec_walk_kernel(VerifyArgs a) {
    constexpr int NT = 1024, U = 4;  // fours a thread has on the way
    __shared__ Rows rows;
    __shared__ double sums[TOKEN ? kOne / kGroup : 1];
    __shared__ double ex[NT / 64];
    __shared__ float ex_x[NT / 64];
    __shared__ int ex_t[NT / 64];
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
    const SpecRows s = spec_rows(a.cu, b, a.n_tokens, a.max_new);
    load_rows<T, D, NT>(a, s, rows);
    // Sum of (p - c q)+ over a row, in 64 bits throughout: terms rounded to 32 leave a
    // W of few entries off by 2^-24 of itself, which decides a test beside its border
    // (and take 7.9 us a pass for 9.7).
    // Entries that are no probabilities show in the largest of all bits, and ask for a
    // careful pass.
    auto block = [&](double sum) {
        sum = wave_sum(sum);
        __syncthreads();
        if (lane == 0) ex[tid >> 6] = sum;
        __syncthreads();
        sum = 0.0;
#pragma unroll
        for (int k = 0; k < NT / 64; ++k) sum += ex[k];
        return sum;
    };
    auto mass = [&](int row, double c) {
        const T* pr = static_cast<const T*>(a.p) + (size_t)(s.row0 + row) * a.p_stride;
        const T* qr = static_cast<const T*>(a.q) + (size_t)(s.row0 + row) * a.q_stride;
        double sum = 0.0;
        uint32_t top = 0;
        auto bits = [](float x) { return __builtin_bit_cast(uint32_t, x); };
        for (int t0 = 4 * tid; t0 < a.vocab; t0 += 4 * U * NT) {
            f32x4 x[U], y[U];
#pragma unroll
            for (int k = 0; k < U; ++k) x[k] = four_of(pr, t0 + 4 * k * NT, a.vocab, 0.f);
#pragma unroll
            for (int k = 0; k < U; ++k) y[k] = four_of(qr, t0 + 4 * k * NT, a.vocab, 0.f);
#pragma unroll
            for (int k = 0; k < U; ++k)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t u = bits(x[k][j]), v = bits(y[k][j]), w = u > v ? u : v;
                    top = top > w ? top : w;
                    sum += fmax((double)x[k][j] - c * (double)y[k][j], 0.0);
                }
        }
        sum = block(top >= 0x7f800000u ? (double)__builtin_nanf("") : sum);
        if (sum != sum) {
            sum = 0.0;
            for (int t = tid; t < a.vocab; t += NT) sum += fmax(prob((float)pr[t]) - c * prob((float)qr[t]), 0.0);
            sum = block(sum);
        }
        return sum;
    };
    // The largest score's index, the lowest of equals; -1 where all are NaN.  A pass by
    // one workgroup for each accepted row: a chain of 6 rows 31 us (32000 entries) and 69
    // (131072).
    auto best_of = [&](int row) {
        const T* pr = static_cast<const T*>(a.p) + (size_t)(s.row0 + row) * a.p_stride;
        float top = -INFINITY;
        int at = 0x7fffffff;
        auto take = [&](float x, int t) {
            if (x > top || (x == top && t < at)) top = x, at = t;
        };
        for (int t0 = 4 * tid; t0 < a.vocab; t0 += 4 * U * NT) {
            f32x4 x[U];
#pragma unroll
            for (int k = 0; k < U; ++k) x[k] = four_of(pr, t0 + 4 * k * NT, a.vocab, __builtin_nanf(""));
            // a thread's entries come in order: of equals the first one stays
#pragma unroll
            for (int k = 0; k < U; ++k)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const bool up = x[k][j] > top || (at == 0x7fffffff && x[k][j] == top);
                    top = up ? x[k][j] : top;
                    at = up ? t0 + 4 * k * NT + j : at;
                }
        }
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) take(__shfl_xor(top, m, 64), __shfl_xor(at, m, 64));
        __syncthreads();
        if (lane == 0) ex_x[tid >> 6] = top, ex_t[tid >> 6] = at;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < NT / 64; ++k) take(ex_x[k], ex_t[k]);
        return at == 0x7fffffff ? -1 : at;
    };
    const Walk w = walk<D>(s, rows, a.path + (size_t)b * a.max_new, mass, best_of);
    write_walk<D, NT>(a, b, s, w);
    if constexpr (TOKEN)
        if (s.n) token_here<T, D>(a, b, s, rows, w, sums);  // uniform
}

// ---- the last row's weights and the token, where a workgroup of the request would
// take too long
//
// WALK: the workgroup walks for itself (CHOSEN, CHAIN); else the walk is there.
template <typename T, Drafts D>
__global__ __launch_bounds__(256) void spec_weigh_kernel(VerifyArgs a) {
    constexpr bool WALK = D == CHOSEN || D == CHAIN, Q = D != CHOSEN;
    constexpr int W = kGroups / 4;  // sums a wave
    __shared__ std::conditional_t<WALK, Rows, int> rows;
    const int b = blockIdx.x / a.n_blocks, block = blockIdx.x % a.n_blocks;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Last l;
    SpecRows s{0, 0};
    if constexpr (WALK) {
        s = spec_rows(a.cu, b, a.n_tokens, a.max_new);
        load_rows<T, D, 256>(a, s, rows);
        const Walk k = walk<D>(s, rows, block ? nullptr : a.path + (size_t)b * a.max_new,
                               [](int, double) { return 0.0; }, [](int) { return -1; });
        if (block == 0) write_walk<D, 256>(a, b, s, k);
        l = Last{s.n ? s.row0 + k.cur : -1, k.cur, k.children, 0, k.a};
    } else {
        l = a.last[b];
    }
    if (l.row < 0) return;
    const Weights<T, Q> wt = weights_of<T, Q>(a, l.row, l.a);
    const int g0 = block * kGroups + w * W;
    f32x4 x[W], y[W];
#pragma unroll
    for (int g = 0; g < W; ++g) wt.load((g0 + g) * kGroup + 4 * lane, x[g], y[g]);
    auto child = [&](int i) {
        if constexpr (WALK) return i > l.at && i < s.n && rows.up[i < s.n ? i : 0] == l.at ? rows.tok[i] : -1;
        else return -1;
    };
    const Refused<decltype(child)> refused{D == CHOSEN && l.children > 0, l.at, s.n, child};
    weigh<W>(wt, refused, g0, a.n_groups, x, y, a.sums + (size_t)b * a.n_groups);
}

// The token: a wave a request.
template <typename T, Drafts D>
__global__ __launch_bounds__(64) void spec_find_kernel(VerifyArgs a) {
    constexpr bool Q = D != CHOSEN;
    const int b = blockIdx.x;
    const Last l = a.last[b];
    if (l.row < 0) return;
    const SpecRows s = spec_rows(a.cu, b, a.n_tokens, a.max_new);
    auto child = [&](int k) { return k > l.at && k < s.n && parent_of(a, s.row0, k) == l.at ? a.tokens[s.row0 + k] : -1; };
    const Refused<decltype(child)> refused{D == CHOSEN && l.children > 0, l.at, s.n, child};
    const int token = find_token(weights_of<T, Q>(a, l.row, l.a), refused, a.n_groups, a.sums + (size_t)b * a.n_groups,
                                 fmax((double)a.r[b], 0.0));
    if (threadIdx.x == 0) a.token[b] = token;
}

// ------------------------------------------------------------------- host --
static size_t align16(size_t x) { return (x + 15) & ~(size_t)15; }
static int groups_of(const lmxs_verify_desc* d) { return (int)((d->vocab + kGroup - 1) / kGroup); }
static int blocks_of(const lmxs_verify_desc* d) { return (groups_of(d) + kGroups - 1) / kGroups; }
// One launch, a workgroup a request, or two and three with many, us (a step's calls
// from a graph; from the host, which then waits for no launch): 16 requests of 32 rows
// and 32000 entries, chosen drafts 7.8 and 7.9 (9.0 and 11.1 from the host), sampled
// chains 12.9 and 10.2 (12.9 and 11.2; one request 9.8 and 7.2, 9.9 and 11.3), sampled
// trees 21.3 and 21.4; 65536 entries 10.2 and 8.2, 15.3 and 8.9, 19.4 and 15.4; 4096
// entries 6.5 and 7.8, 7.3 and 8.5, 14.9 and 18.4.
static bool one_workgroup(const lmxs_verify_desc* d) { return d->vocab <= kOne; }
size_t spec_verify_workspace(const lmxs_verify_desc* d) {
    if (d->greedy || one_workgroup(d)) return 0;
    return align16((size_t)d->n_seq * groups_of(d) * sizeof(double)) + align16(d->n_seq * sizeof(Last));
}
// A launch names its workgroups' threads in 32 bits.
bool spec_verify_fits(const lmxs_verify_desc* d) { return (uint64_t)d->n_seq * blocks_of(d) < (1u << 24); }

template <typename T, Drafts D>
static void launch(const VerifyArgs& a, hipStream_t st) {
    const dim3 seqs((unsigned)a.n_seq), blocks((unsigned)(a.n_seq * a.n_blocks));
    if constexpr (D != GREEDY)
        if (!a.last) {
            hipLaunchKernelGGL((spec_walk_kernel<T, D, true>), seqs, dim3(1024), 0, st, a);
            return;
        }
    if constexpr (D == SAMPLED || D == GREEDY)
        hipLaunchKernelGGL((spec_walk_kernel<T, D, false>), seqs, dim3(1024), 0, st, a);
    if constexpr (D != GREEDY) {
        hipLaunchKernelGGL((spec_weigh_kernel<T, D>), blocks, dim3(256), 0, st, a);
        hipLaunchKernelGGL((spec_find_kernel<T, D>), seqs, dim3(64), 0, st, a);
    }
}
template <typename T>
static void launch_by(const VerifyArgs& a, bool greedy, hipStream_t st) {
    if (greedy) launch<T, GREEDY>(a, st);
    else if (!a.q) launch<T, CHOSEN>(a, st);
    else if (!a.parent) launch<T, CHAIN>(a, st);  // one child a row: no second sibling asks for a sum
    else launch<T, SAMPLED>(a, st);
}

lmx_status spec_verify(const lmxs_verify_desc* d, const int32_t* cu, const int32_t* tokens, const int32_t* parent,
                       const void* p, const void* q, lmx_dtype dt, const float* u, const float* r, int32_t* path,
                       int32_t* accepted, int32_t* token, int32_t* lens, void* ws, hipStream_t st) {
    VerifyArgs a{};
    a.n_seq = (int)d->n_seq;
    a.n_tokens = (int)d->n_tokens;
    a.max_new = (int)d->max_new;
    a.vocab = (int)d->vocab;
    a.n_groups = groups_of(d);
    a.n_blocks = blocks_of(d);
    a.p_stride = d->p_stride ? d->p_stride : d->vocab;
    a.q_stride = d->q_stride ? d->q_stride : d->vocab;
    a.cu = cu;
    a.tokens = tokens;
    a.parent = parent;
    a.p = p;
    a.q = q;
    a.u = u;
    a.r = r;
    a.path = path;
    a.accepted = accepted;
    a.token = token;
    a.lens = lens;
    if (spec_verify_workspace(d)) {
        a.sums = static_cast<double*>(ws);
        a.last = reinterpret_cast<Last*>(static_cast<char*>(ws) + align16((size_t)d->n_seq * a.n_groups * sizeof(double)));
    }
    (void)hipGetLastError();
    if (dt == LMX_F32) launch_by<float>(a, d->greedy != 0, st);
    else launch_by<f16>(a, d->greedy != 0, st);
    LMX_CHECK_LAUNCH();
    return LMX_OK;
}

}  // namespace lmx
