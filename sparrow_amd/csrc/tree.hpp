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
    // (all loads at once: they are the start of every kernel that takes drafted tokens)
    const int listed = count ? count[b] : S, up = parent && lane < S ? parent[(size_t)b * S + lane] : -1;
    TreeRows r{0, pos0[b], -1};
    if (r.pos0 < 0) return r;
    const int n = min(max(listed, 0), S);
    bool bad = n > 0 && r.pos0 > cap - n;
    if (parent && lane < n) {
        r.parent = up;
        bad |= up < -1 || up >= lane;
    }
    if (__any(bad)) {
        if (report && threadIdx.x == 0) atomicOr(guard, 1);
        return r;
    }
    r.n = n;
    return r;
}

}  // namespace vmlm
