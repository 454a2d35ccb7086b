// k_rope.hip -- positions rotated into the query and key heads
// (vmlm_hip_rope_qk): both layouts of the pairs, a part of the head, frequencies
// from a table.
//
// (x_a, x_b) -> m (x_a c - x_b s, x_a s + x_b c), c and s the cosine and sine of pos * freq[i],
// for the pairs i of the first `rot` channels: (i, i + rot / 2), or (2i, 2i + 1).
//
// A thread turns V neighbouring pairs of a head (16-byte loads where rot and the head allow
// V = 4). Bound by the rows' bytes, read once and written once: 2048 rows of 32 + 8 heads of 128,
// half of each turned, 84 MB in 16.0 us (5.2 TB/s); one row of 36 + 36 heads of 64 5.2 us, a
// launch.
//
// Angles: pos * freq / 2 pi is formed in 64 bits and its whole turns dropped there; a
// 32-bit product would be off by 2^-24 of the angle itself (0.006 at position 100000). What
// the fraction of a turn loses in f32 (up to 2^-25 of it) is turned by afterwards.
#include <algorithm>

#include "internal.hpp"

namespace vmlm {
namespace {

struct RopeParams {
    const float *q, *k;
    float *qo, *ko;
    size_t ldq, ldk, ldqo, ldko;
    const int32_t *pos;
    const double *freq;
    int H, Hkv, hd, rot, units;  // units: of 2 V channels a head, the rotated ones first
    int y0;                      // of the launch, in workgroups along a row
    float m;
};

template <int V, bool INTER>
__global__ __launch_bounds__(256) void rope_kernel(RopeParams p) {
    typedef float vec __attribute__((ext_vector_type(V), aligned(4)));  // from any float on
    const int row = blockIdx.x;
    const int id = (p.y0 + blockIdx.y) * 256 + threadIdx.x;
    const int h = id / p.units, u = id % p.units;
    if (h >= p.H + p.Hkv) return;
    const int pos = p.pos[row];
    if (pos < 0) return;  // an idle row
    const bool isq = h < p.H, turned = u * 2 * V < p.rot;
    // the unit's two vectors: of a pair each, or 2 V neighbours
    const int a = !turned || INTER ? u * 2 * V : u * V, b = !turned || INTER ? a + V : a + p.rot / 2;
    const size_t head = (size_t)(isq ? h : h - p.H) * p.hd;
    const float *src = (isq ? p.q + row * p.ldq : p.k + row * p.ldk) + head;
    float *dst = (isq ? p.qo + row * p.ldqo : p.ko + row * p.ldko) + head;
    if (!turned && src == dst) return;
    vec x = *(const vec *)(src + a), y = *(const vec *)(src + b);
    if (turned) {
        float v[2 * V], w[2 * V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            v[e] = x[e];
            v[V + e] = y[e];
        }
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const double t = (double)pos * (p.freq[u * V + e] * 0.15915494309189533577);  // 1 / 2 pi
            const double turn = t - __builtin_rint(t);
            const float hi = (float)turn, rest = (float)(turn - (double)hi) * 6.28318531f;
            float s0, c0;
            sincospif(2.0f * hi, &s0, &c0);
            const float s = p.m * __builtin_fmaf(c0, rest, s0), c = p.m * __builtin_fmaf(-s0, rest, c0);
            const int ia = INTER ? 2 * e : e, ib = INTER ? 2 * e + 1 : V + e;
            w[ia] = v[ia] * c - v[ib] * s;
            w[ib] = v[ia] * s + v[ib] * c;
        }
#pragma unroll
        for (int e = 0; e < V; ++e) {
            x[e] = w[e];
            y[e] = w[V + e];
        }
    }
    *(vec *)(dst + a) = x;
    *(vec *)(dst + b) = y;
}

template <int V>
int launch_t(RopeParams p, int rows, bool inter, hipStream_t st) {
    // (a grid has at most 65535 workgroups along y; a row up to 2 x 65535 heads of 510 channels)
    const int all = (int)cdiv((size_t)(p.H + p.Hkv) * p.units, 256);
    for (p.y0 = 0; p.y0 < all; p.y0 += 65535) {
        const dim3 grid((unsigned)rows, (unsigned)std::min(65535, all - p.y0));
        if (inter)
            rope_kernel<V, true><<<grid, 256, 0, st>>>(p);
        else
            rope_kernel<V, false><<<grid, 256, 0, st>>>(p);
        VMLM_HIP_CHECK(hipGetLastError());
    }
    return VMLM_OK;
}

}  // namespace

int launch_rope_qk(const RopeArgs &a, hipStream_t st) {
    // (a grid has at most 2^32 - 1 threads along its rows)
    constexpr int ROWS = 1 << 23;
    for (int r = 0; r < a.rows; r += ROWS) {
        const int rows = std::min(ROWS, a.rows - r);
        const bool wide = a.rot % 8 == 0 && a.hd % 8 == 0;
        const RopeParams p{a.q + r * a.ldq,
                           a.k + r * a.ldk,
                           a.qo + r * a.ldqo,
                           a.ko + r * a.ldko,
                           a.ldq,
                           a.ldk,
                           a.ldqo,
                           a.ldko,
                           a.pos + r,
                           a.freq,
                           a.H,
                           a.Hkv,
                           a.hd,
                           a.rot,
                           a.hd / (wide ? 8 : 2),
                           0,
                           a.m};
        const int rc = wide ? launch_t<4>(p, rows, a.inter, st) : launch_t<1>(p, rows, a.inter, st);
        if (rc) return rc;
    }
    return VMLM_OK;
}

}  // namespace vmlm
