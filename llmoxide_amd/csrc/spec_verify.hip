// Which drafted rows a target model accepts, and the token behind them.
//
// Two launches.  The walk: a workgroup a request, with all of its rows' p(c),
// q(c) and u in LDS, so that accepting and refusing chosen drafts reads no
// memory at all; only sums over the vocabulary that a second sibling asks for
// (drafts that were sampled), or the largest scores (greedy), are passes over a
// row of p, by the whole workgroup.  The sample: the last row's distribution in
// chunks of 4096 entries, a workgroup each; the one that finishes last adds the
// chunks up, finds the one where the sum passes r times the whole, and goes
// through it.
//
// What is left of p after refusals needs one number: with w = p - a q wherever
// that is above 0, and W its sum, the next refusal's w / W - q is, times W,
// p - (a + W) q.  So no distribution is ever written.
//
// Sums are in 64 bits: two entries of a vocabulary of 131072 may lie 1e-7 apart
// in the running sum, which is where a 32-bit sum's own rounding lies.  Each is
// made in an order that the shapes alone decide.
//
// Bound by HBM in the sample (the last rows once: 4 or 8 bytes an entry), by
// latency elsewhere.
#include "spec.hpp"

namespace lmx {

constexpr int kChunk = 4096;   // entries of the vocabulary a workgroup of the sample

// What the walk leaves for the sample.
struct Last {
    int row;       // of the batch; -1: the request has none
    int at;        // of the request
    int children;  // of that row: all were refused
    int pad;
    double a;
};

struct VerifyArgs {
    int n_seq, n_tokens, max_new, vocab, n_chunks;
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
    double* sums;   // [n_seq][n_chunks]
    Last* last;     // [n_seq]
    int* done;      // [n_seq] chunks whose sums are there
};

// A probability; what is not above 0 and finite is 0.
__device__ __forceinline__ double prob(float x) { return x > 0.f && x < INFINITY ? (double)x : 0.0; }

// A row's parent within the request, -1 for a root.
__device__ __forceinline__ int parent_of(const VerifyArgs& a, int row0, int i) {
    const int p = a.parent ? a.parent[row0 + i] : i - 1;
    return p >= 0 && p < i ? p : -1;
}

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) x += __shfl_xor(x, m, 64);
    return x;
}
// Sum over a workgroup of NT threads, in every thread.  ex: NT / 64 doubles.
template <int NT>
__device__ __forceinline__ double block_sum(double x, double* ex) {
    x = wave_sum(x);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) ex[threadIdx.x >> 6] = x;
    __syncthreads();
    double s = 0.0;
#pragma unroll
    for (int k = 0; k < NT / 64; ++k) s += ex[k];
    return s;
}

enum Drafts { CHOSEN, SAMPLED, GREEDY };

template <typename T, Drafts D>
__global__ __launch_bounds__(D == CHOSEN ? 256 : 1024) void spec_walk_kernel(VerifyArgs a) {
    constexpr int NT = D == CHOSEN ? 256 : 1024;
    __shared__ int up[LMXS_MAX_ROWS], tok[LMXS_MAX_ROWS];
    __shared__ float ps[LMXS_MAX_ROWS], qs[LMXS_MAX_ROWS], us[LMXS_MAX_ROWS];
    __shared__ double ex[NT / 64];
    __shared__ float ex_x[NT / 64];
    __shared__ int ex_t[NT / 64];
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
    const SpecRows s = spec_rows(a.cu, b, a.n_tokens, a.max_new);
    const T* const p = static_cast<const T*>(a.p);
    const T* const q = static_cast<const T*>(a.q);

    for (int i = tid; i < s.n; i += NT) {
        const int above = parent_of(a, s.row0, i), t = a.tokens[s.row0 + i];
        const bool on = above >= 0 && (uint32_t)t < (uint32_t)a.vocab;
        up[i] = above;
        tok[i] = on ? t : -1;
        if (D != GREEDY && on) {
            ps[i] = (float)p[(size_t)(s.row0 + above) * a.p_stride + t];
            if (D == SAMPLED) qs[i] = (float)q[(size_t)(s.row0 + above) * a.q_stride + t];
            us[i] = a.u[s.row0 + i];
        }
    }
    __syncthreads();

    // Sum of (p - c q)+ over a row.
    auto mass = [&](int row, double c) {
        const T* pr = p + (size_t)(s.row0 + row) * a.p_stride;
        const T* qr = q + (size_t)(s.row0 + row) * a.q_stride;
        constexpr int U = 8;
        double sum = 0.0;
        for (int t0 = tid; t0 < a.vocab; t0 += U * NT) {
            float x[U], y[U];
#pragma unroll
            for (int k = 0; k < U; ++k) {
                const int t = t0 + k * NT < a.vocab ? t0 + k * NT : t0;
                x[k] = t0 + k * NT < a.vocab ? (float)pr[t] : 0.f;
                y[k] = (float)qr[t];
            }
#pragma unroll
            for (int k = 0; k < U; ++k) sum += fmax(prob(x[k]) - c * prob(y[k]), 0.0);
        }
        return block_sum<NT>(sum, ex);
    };
    // Index of a row's largest score, the lowest of equals; -1 where all are NaN.
    auto best_of = [&](int row) {
        const T* pr = p + (size_t)(s.row0 + row) * a.p_stride;
        constexpr int U = 8;
        float top = -INFINITY;
        int at = 0x7fffffff;
        auto take = [&](float x, int t) {
            if (x > top || (x == top && t < at)) top = x, at = t;
        };
        for (int t0 = tid; t0 < a.vocab; t0 += U * NT) {
            float x[U];
#pragma unroll
            for (int k = 0; k < U; ++k) x[k] = (float)pr[t0 + k * NT < a.vocab ? t0 + k * NT : t0];
#pragma unroll
            for (int k = 0; k < U; ++k)
                if (t0 + k * NT < a.vocab) take(x[k], t0 + k * NT);
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

    // Every wave walks by itself, over the same LDS: the passes' barriers meet.
    int cur = 0, count = s.n ? 1 : 0, children = 0;
    double c = 0.0, W = 1.0;
    bool known = D != GREEDY;  // SAMPLED: W is that of c; GREEDY: best is cur's
    int best = -1;
    for (int from = 1;;) {
        int i = -1;
        for (int c0 = from & ~63; c0 < s.n && i < 0; c0 += 64) {
            const int k = c0 + lane;
            const uint64_t hit = __ballot(k >= from && k < s.n && up[k < s.n ? k : 0] == cur);
            if (hit) i = c0 + __builtin_ctzll(hit);
        }
        if (i < 0) break;
        from = i + 1;
        ++children;
        const int t = tok[i];
        bool pass = false;
        if constexpr (D == GREEDY) {
            if (!known) best = best_of(cur);
            known = true;
            pass = t >= 0 && t == best;
        } else if (t >= 0) {
            double w = prob(ps[i]);
            if constexpr (D == SAMPLED) {
                if (!known) W = mass(cur, c);
                known = true;
                const double y = prob(qs[i]);
                w = fmax(w - c * y, 0.0);
                pass = (double)us[i] * W * y < w;
                if (!pass) {
                    c += W;
                    known = false;
                }
            } else {
                bool twice = false;  // an earlier sibling was the same token
                for (int c0 = (cur + 1) & ~63; c0 < i; c0 += 64) {
                    const int k = c0 + lane;
                    twice = twice || __ballot(k < i && k > cur && up[k < s.n ? k : 0] == cur && tok[k < s.n ? k : 0] == t);
                }
                if (twice) w = 0.0;
                pass = (double)us[i] * W < w;
                if (!pass) W -= w;
            }
        }
        if (pass) {
            if (tid == 0) a.path[(size_t)b * a.max_new + count] = i;
            ++count;
            cur = i;
            children = 0;
            c = 0.0;
            W = 1.0;
            known = D != GREEDY;
        }
    }
    if (D == GREEDY && s.n && !known) best = best_of(cur);
    for (int j = count + tid; j < a.max_new; j += NT) a.path[(size_t)b * a.max_new + j] = -1;
    if (tid == 0) {
        if (count) a.path[(size_t)b * a.max_new] = 0;
        a.accepted[b] = count;
        if (a.lens) a.lens[b] += count;
        if (D == GREEDY || !s.n) a.token[b] = best;
        if (D != GREEDY) {
            a.last[b] = Last{s.n ? s.row0 + cur : -1, cur, children, 0, c};
            a.done[b] = 0;
        }
    }
}

// The weight of entry t: what is left of p behind the refused drafts.
template <typename T, bool Q>
struct Weights {
    const T* p;
    const T* q;
    double a;
    const uint32_t* gone;  // bits of the chunk's entries that chosen drafts took
    __device__ __forceinline__ double at(int t, int in_chunk) const {
        const double x = prob((float)p[t]);
        if constexpr (Q) return fmax(x - a * prob((float)q[t]), 0.0);
        return gone && (gone[in_chunk >> 5] >> (in_chunk & 31) & 1) ? 0.0 : x;
    }
};

template <typename T, bool Q>
__global__ __launch_bounds__(256) void spec_sample_kernel(VerifyArgs a) {
    constexpr int PER = kChunk / 256;
    __shared__ double ex[4], ex_scan[4];
    __shared__ uint32_t gone[kChunk / 32];
    __shared__ int found, finishing;
    const int b = blockIdx.x / a.n_chunks, mine = blockIdx.x % a.n_chunks, tid = threadIdx.x, lane = tid & 63;
    const Last l = a.last[b];
    if (l.row < 0) return;
    const SpecRows s = spec_rows(a.cu, b, a.n_tokens, a.max_new);
    // (behind a leaf a is 0 and q says nothing: p is read in its place)
    const T* const pr = static_cast<const T*>(a.p) + (size_t)l.row * a.p_stride;
    Weights<T, Q> w{pr, Q && l.a != 0.0 ? static_cast<const T*>(a.q) + (size_t)l.row * a.q_stride : pr, l.a, nullptr};
    const bool some_gone = !Q && l.children > 0;

    // The chunk's entries that refused drafts took.
    auto mark = [&](int chunk) {
        w.gone = some_gone ? gone : nullptr;
        if (!some_gone) return;
        __syncthreads();
        if (tid < kChunk / 32) gone[tid] = 0;
        __syncthreads();
        for (int i = l.at + 1 + tid; i < s.n; i += 256) {
            if (parent_of(a, s.row0, i) != l.at) continue;
            const uint32_t t = (uint32_t)a.tokens[s.row0 + i] - (uint32_t)chunk * kChunk;
            if (t < kChunk) atomicOr(&gone[t >> 5], 1u << (t & 31));
        }
        __syncthreads();
    };
    auto chunk_sum = [&](int chunk) {
        const int t0 = chunk * kChunk, n = imin(kChunk, a.vocab - t0);
        double x[PER], sum = 0.0;
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const int i = tid + 256 * k;
            x[k] = i < n ? w.at(t0 + i, i) : 0.0;
        }
#pragma unroll
        for (int k = 0; k < PER; ++k) sum += x[k];
        return block_sum<256>(sum, ex);
    };
    // Sum over the threads before this one, and of all.
    auto scan = [&](double x, double& total) {
        double y = x;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const double z = __shfl_up(y, d, 64);
            y += lane >= d ? z : 0.0;
        }
        __syncthreads();
        if (lane == 63) ex_scan[tid >> 6] = y;
        __syncthreads();
        double before = 0.0;
        total = 0.0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (k == (tid >> 6)) before = total;
            total += ex_scan[k];
        }
        return before + y - x;
    };
    // The least entry of the chunk whose sum, with `before`, passes the target; the
    // last one with a weight where rounding keeps the sum below it; -1: no weight.
    auto search = [&](int chunk, double before, double target) {
        const int t0 = chunk * kChunk, n = imin(kChunk, a.vocab - t0);
        double x[PER], sum = 0.0, total;
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const int i = tid * PER + k;
            x[k] = i < n ? w.at(t0 + i, i) : 0.0;
            sum += x[k];
        }
        double run = before + scan(sum, total);
        int hit = 0x7fffffff, any = -1;
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            run += x[k];
            if (x[k] > 0.0) {
                any = t0 + tid * PER + k;
                if (run > target && hit == 0x7fffffff) hit = any;
            }
        }
        if (tid == 0) found = 0x7fffffff;
        __syncthreads();
        if (hit != 0x7fffffff) atomicMin(&found, hit);
        __syncthreads();
        const int first = found;
        if (first != 0x7fffffff) return first;
        __syncthreads();
        if (tid == 0) found = -1;
        __syncthreads();
        if (any >= 0) atomicMax(&found, any);
        __syncthreads();
        return found;
    };

    mark(mine);
    const double sum = chunk_sum(mine);
    if (tid == 0) {
        __hip_atomic_store(&a.sums[(size_t)b * a.n_chunks + mine], sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        finishing = __hip_atomic_fetch_add(&a.done[b], 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == a.n_chunks - 1;
    }
    __syncthreads();
    if (!finishing) return;  // uniform
    __threadfence();

    // ---- the last workgroup of the request: every sum is there
    const int per = (a.n_chunks + 255) / 256;
    double part = 0.0, total;
    auto chunk_at = [&](int c) {
        return __hip_atomic_load(&a.sums[(size_t)b * a.n_chunks + c], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    };
    for (int k = 0; k < per; ++k)
        if (tid * per + k < a.n_chunks) part += chunk_at(tid * per + k);
    const double before = scan(part, total);
    const double r = fmax((double)a.r[b], 0.0);
    int token = -1;
    if (total > 0.0) {
        const double target = r * total;
        double run = before;
        int hit = 0x7fffffff, any = -1;
        for (int k = 0; k < per; ++k)
            if (tid * per + k < a.n_chunks) {
                const double x = chunk_at(tid * per + k);
                run += x;
                if (x > 0.0) {
                    any = tid * per + k;
                    if (run > target && hit == 0x7fffffff) hit = any;
                }
            }
        if (tid == 0) found = 0x7fffffff;
        __syncthreads();
        if (hit != 0x7fffffff) atomicMin(&found, hit);
        __syncthreads();
        int chunk = found;
        if (chunk == 0x7fffffff) {  // (r of 1, or rounding): the last chunk with a weight
            __syncthreads();
            if (tid == 0) found = -1;
            __syncthreads();
            if (any >= 0) atomicMax(&found, any);
            __syncthreads();
            chunk = found;
        }
        // the sum of the chunks before it
        double x = 0.0;
        for (int k = 0; k < per; ++k)
            if (tid * per + k < chunk) x += chunk_at(tid * per + k);
        const double below = block_sum<256>(x, ex);
        mark(chunk);
        token = search(chunk, below, target);
    } else {
        // Nothing is left (the drafts had all of p): from p itself, by this
        // workgroup alone, twice through the row.
        w.a = 0.0;
        w.gone = nullptr;
        double all = 0.0;
        for (int c = 0; c < a.n_chunks; ++c) all += chunk_sum(c);
        const double target = r * all;
        double run = 0.0;
        for (int c = 0; c < a.n_chunks; ++c) {
            const double x = chunk_sum(c);
            if (x > 0.0) {
                const int t = search(c, run, target);
                if (t >= 0) token = t;
                if (run + x > target) break;  // uniform
            }
            run += x;
        }
    }
    if (tid == 0) a.token[b] = token;
}

// ------------------------------------------------------------------- host --
static size_t align16(size_t x) { return (x + 15) & ~(size_t)15; }
static int chunks_of(const lmxs_verify_desc* d) { return (int)((d->vocab + kChunk - 1) / kChunk); }
size_t spec_verify_workspace(const lmxs_verify_desc* d) {
    if (d->greedy) return 0;
    return align16((size_t)d->n_seq * chunks_of(d) * sizeof(double)) + d->n_seq * sizeof(Last) +
           align16((size_t)d->n_seq * sizeof(int));
}
// A launch names its workgroups' threads in 32 bits.
bool spec_verify_fits(const lmxs_verify_desc* d) { return (uint64_t)d->n_seq * chunks_of(d) < (1u << 24); }

template <typename T>
static void launch(const VerifyArgs& a, bool greedy, hipStream_t st) {
    const dim3 seqs((unsigned)a.n_seq), chunks((unsigned)(a.n_seq * a.n_chunks));
    if (greedy) {
        hipLaunchKernelGGL((spec_walk_kernel<T, GREEDY>), seqs, dim3(1024), 0, st, a);
    } else if (a.q) {
        hipLaunchKernelGGL((spec_walk_kernel<T, SAMPLED>), seqs, dim3(1024), 0, st, a);
        hipLaunchKernelGGL((spec_sample_kernel<T, true>), chunks, dim3(256), 0, st, a);
    } else {
        hipLaunchKernelGGL((spec_walk_kernel<T, CHOSEN>), seqs, dim3(256), 0, st, a);
        hipLaunchKernelGGL((spec_sample_kernel<T, false>), chunks, dim3(256), 0, st, a);
    }
}

lmx_status spec_verify(const lmxs_verify_desc* d, const int32_t* cu, const int32_t* tokens, const int32_t* parent,
                       const void* p, const void* q, lmx_dtype dt, const float* u, const float* r, int32_t* path,
                       int32_t* accepted, int32_t* token, int32_t* lens, void* ws, hipStream_t st) {
    VerifyArgs a{};
    a.n_seq = (int)d->n_seq;
    a.n_tokens = (int)d->n_tokens;
    a.max_new = (int)d->max_new;
    a.vocab = (int)d->vocab;
    a.n_chunks = chunks_of(d);
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
    char* at = static_cast<char*>(ws);
    a.sums = reinterpret_cast<double*>(at);
    at += align16((size_t)d->n_seq * a.n_chunks * sizeof(double));
    a.last = reinterpret_cast<Last*>(at);
    a.done = reinterpret_cast<int*>(at + d->n_seq * sizeof(Last));
    (void)hipGetLastError();
    if (dt == LMX_F32) launch<float>(a, d->greedy != 0, st);
    else launch<f16>(a, d->greedy != 0, st);
    LMX_CHECK_LAUNCH();
    return LMX_OK;
}

}  // namespace lmx
