// k_rope.hip -- positions rotated into the query and key heads
// (vmlm_hip_rope_qk): both layouts of the pairs, a part of the head, frequencies
// from a table.
//
// (x_a, x_b) -> m (x_a c - x_b s, x_a s + x_b c), c and s the cosine and sine of pos * freq[i],
// for the pairs i of the first `rot` channels: (i, i + rot / 2), or (2i, 2i + 1).
//
// A thread turns V neighbouring pairs (16-byte loads where rot and the head allow V =
// 4) of up to NH heads, whose sines and cosines it forms once. Bound by the rows' bytes,
// read once and written once.
//
// Angles: pos * freq / 2 pi is formed in 64 bits and its whole turns dropped there; a
// 32-bit product would be off by 2^-24 of the angle itself (0.006 at position 100000).
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
    int H, Hkv, hd, rot, units;  // units: of V pairs a head, the rotated ones first
    float m;
};

// V values from any float on.
template <int V>
struct Vec {
    typedef float t __attribute__((ext_vector_type(V), aligned(4)));
};
template <>
struct Vec<1> {
    typedef float t __attribute__((ext_vector_type(1), aligned(4)));
};

template <int V, bool INTER, int NH>
__global__ __launch_bounds__(256) void rope_kernel(RopeParams p) {
    using vec = typename Vec<V>::t;
    const int row = blockIdx.x, heads = p.H + p.Hkv;
    const int id = blockIdx.y * 256 + threadIdx.x;
    const int g = id / p.units, u = id % p.units, h0 = g * NH;
    if (h0 >= heads) return;
    const int pos = p.pos[row];
    if (pos < 0) return;  // an idle row
    const bool turned = u * 2 * V < p.rot;
    // the unit's two vectors: of a pair each, or 2 V neighbours
    const int a = !turned || INTER ? u * 2 * V : u * V, b = !turned || INTER ? a + V : a + p.rot / 2;
    vec x[NH], y[NH];
    auto at = [&](int h, bool out) {
        const bool isq = h < p.H;
        const size_t c = (size_t)(isq ? h : h - p.H) * p.hd;
        if (out) return (isq ? p.qo + row * p.ldqo : p.ko + row * p.ldko) + c;
        return const_cast<float *>((isq ? p.q + row * p.ldq : p.k + row * p.ldk) + c);
    };
#pragma unroll
    for (int i = 0; i < NH; ++i) {
        const float *src = at(min(h0 + i, heads - 1), false);
        x[i] = *(const vec *)(src + a);
        y[i] = *(const vec *)(src + b);
    }
    if (turned) {
        float s[V], c[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const double t = (double)pos * (p.freq[u * V + e] * 0.15915494309189533577);  // 1 / 2 pi
            sincospif(2.0f * (float)(t - __builtin_rint(t)), &s[e], &c[e]);
            s[e] *= p.m;
            c[e] *= p.m;
        }
#pragma unroll
        for (int i = 0; i < NH; ++i) {
            float v[2 * V], w[2 * V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                v[e] = x[i][e];
                v[V + e] = y[i][e];
            }
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const int ia = INTER ? 2 * e : e, ib = INTER ? 2 * e + 1 : V + e;
                w[ia] = v[ia] * c[e] - v[ib] * s[e];
                w[ib] = v[ia] * s[e] + v[ib] * c[e];
            }
#pragma unroll
            for (int e = 0; e < V; ++e) {
                x[i][e] = w[e];
                y[i][e] = w[V + e];
            }
        }
    }
#pragma unroll
    for (int i = 0; i < NH; ++i) {
        if (h0 + i >= heads) break;
        float *dst = at(h0 + i, true);
        *(vec *)(dst + a) = x[i];
        *(vec *)(dst + b) = y[i];
    }
}

template <int V, int NH>
int launch_t(const RopeParams &p, int rows, bool inter, hipStream_t st) {
    const size_t threads = (size_t)cdiv((size_t)(p.H + p.Hkv), NH) * p.units;
    const dim3 grid((unsigned)rows, cdiv(threads, 256));
    if (inter)
        rope_kernel<V, true, NH><<<grid, 256, 0, st>>>(p);
    else
        rope_kernel<V, false, NH><<<grid, 256, 0, st>>>(p);
    VMLM_HIP_CHECK(hipGetLastError());
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
                           a.m};
        const int rc = wide ? launch_t<4, 1>(p, rows, a.inter, st) : launch_t<1, 1>(p, rows, a.inter, st);
        if (rc) return rc;
    }
    return VMLM_OK;
}

}  // namespace vmlm
