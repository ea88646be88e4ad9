// What the kernels of a step with drafted tokens (lmx/spec.h) share.
#pragma once

#include "lmx/spec.h"
#include "paged.hpp"

namespace lmx {

// a + b of numbers from 0 to 2^30 - 1, kept there: whatever the device holds,
// sums of counts stay in range.
constexpr int kMost = (1 << 30) - 1;
__device__ __forceinline__ int add_sat(int a, int b) { return imin(a + b, kMost); }

// A request's rows of the batch, forced into range.
struct SpecRows {
    int row0, n;
};
__device__ __forceinline__ SpecRows spec_rows(const int32_t* cu, int b, int n_tokens, int most) {
    SpecRows r;
    r.row0 = imin(imax(cu[b], 0), n_tokens);
    r.n = imin(imin(imax(cu[b + 1], r.row0), n_tokens) - r.row0, most);
    return r;
}

}  // namespace lmx
