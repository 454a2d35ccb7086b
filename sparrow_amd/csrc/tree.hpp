// tree.hpp -- the drafted tokens of a sequence, as the kernels that take them see
// them: token t stands at position pos0 + t of the cache and hangs below token
// parent[t] < t (-1: below the text before pos0); without parents below token t - 1.
#pragma once

#include "internal.hpp"

namespace vmlm {

// A sequence's tokens: n of them (0: it is idle, or refused by the device guard), the
// first position, and lane t's parent where there are parents.
struct TreeRows {
    int n, pos0, parent;
};

// Called by whole waves. Refused: tokens that leave the cache, parents that are no
// earlier token; `report`: this workgroup trips the guard.
__device__ __forceinline__ TreeRows tree_rows(const int32_t *pos0, const int32_t *count,
                                              const int32_t *parent, int S, int cap, int b,
                                              int *guard, bool report) {
    const int lane = threadIdx.x & 63;
    TreeRows r{0, pos0[b], -1};
    if (r.pos0 < 0) return r;
    const int n = count ? min(max(count[b], 0), S) : S;
    bool bad = n > 0 && r.pos0 > cap - n;
    if (parent && lane < n) {
        r.parent = parent[(size_t)b * S + lane];
        bad |= r.parent < -1 || r.parent >= lane;
    }
    if (__any(bad)) {
        if (report && threadIdx.x == 0) atomicOr(guard, 1);
        return r;
    }
    r.n = n;
    return r;
}

// Token t and those above it, a bit each; `parent` as tree_rows gives it. Called by whole
// waves, t the same in all lanes.
__device__ __forceinline__ unsigned long long tree_ancestors(int parent, int t) {
    unsigned long long seen = 0;
    for (int at = t; at >= 0; at = __builtin_amdgcn_readlane(parent, at)) seen |= 1ull << at;
    return seen;
}

}  // namespace vmlm
