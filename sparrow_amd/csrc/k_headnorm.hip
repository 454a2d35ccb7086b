// k_headnorm.hip -- RMSNorm of every query and key head with the position
// rotation in the same pass (vmlm_hip_qk_norm_rope).
//
// y = x / sqrt(mean(x^2) + eps) * g over a head's hd values, then the pairs
// (i, i + hd/2) turned by pos * theta^(-2i/hd).
//
// A head is held by LH lanes (the power of two from hd/8), each with four values
// of the first half and the four that they are turned with: two 16-byte loads,
// no exchange between lanes but the sum of squares. A wave takes 64 / LH of a
// row's heads, each lane its four sines and cosines.
//
// Bound by the rows' bytes, read once and written once: 2048 rows of 36 + 36 heads of 64
// take 14.7 us, 5.1 TB/s (as a large copy). One row takes 2.8 us, a launch and a latency.
//
// Angles: pos * theta^(-2i/hd) / 2 pi is formed in 64 bits and its whole turns
// dropped there; a 32-bit product would be off by 2^-24 of the angle itself (0.006 at
// position 100000), more than the values' own rounding from a few positions on.
#include <algorithm>

#include "internal.hpp"

namespace vmlm {
namespace {

// Rows may start at any float: the 16-byte loads of gfx950 take any 4-byte
// alignment.
typedef float f32x4a __attribute__((ext_vector_type(4), aligned(4)));

struct HeadNormParams {
    const float *q, *k, *gq, *gk;
    float *qo, *ko;
    size_t ldq, ldk, ldqo, ldko;
    const int32_t *pos;
    int rows, H, Hkv, hd;
    float eps;
    // theta^(-2i/hd) / 2 pi = coarse[i / 16] * fine[i % 16] (256 bytes of arguments: with the
    // table itself, 2 KB of them, a call of one row took 6.2 us instead of 5.0)
    double coarse[HEADNORM_MAX_HD / 32], fine[16];
};

// TURN: with positions. (A pair is turned there only: an infinity or a NaN of one channel
// is not its partner's in the norm alone.)
template <int LH, bool TURN>
__global__ __launch_bounds__(256) void headnorm_kernel(HeadNormParams p) {
    constexpr int HW = 64 / LH;  // heads of a wave at a time
    const int row = blockIdx.x;
    const int wave = blockIdx.y * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int l = lane % LH, half = p.hd / 2, heads = p.H + p.Hkv;
    if (wave * HW >= heads) return;
    const bool in = 4 * l < half;
    const int i0 = in ? 4 * l : 0;
    float s[4], c[4];
    if constexpr (TURN) {
        const int pos = p.pos[row];
        if (pos < 0) return;  // an idle row
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const double t = (double)pos * (p.coarse[i0 / 16] * p.fine[i0 % 16 + e]);
            sincospif(2.0f * (float)(t - __builtin_rint(t)), &s[e], &c[e]);
        }
    }
    const f32x4a gq0 = *(const f32x4a *)(p.gq + i0), gq1 = *(const f32x4a *)(p.gq + half + i0);
    const f32x4a gk0 = *(const f32x4a *)(p.gk + i0), gk1 = *(const f32x4a *)(p.gk + half + i0);
    const int hh = wave * HW + lane / LH, hc = min(hh, heads - 1);
    const bool live = in && hh < heads, isq = hc < p.H;
    const float *src = isq ? p.q + row * p.ldq + (size_t)hc * p.hd
                           : p.k + row * p.ldk + (size_t)(hc - p.H) * p.hd;
    float *dst = isq ? p.qo + row * p.ldqo + (size_t)hc * p.hd
                     : p.ko + row * p.ldko + (size_t)(hc - p.H) * p.hd;
    f32x4a x0 = *(const f32x4a *)(src + i0), x1 = *(const f32x4a *)(src + half + i0);
    float ss = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) ss = __builtin_fmaf(x0[e], x0[e], __builtin_fmaf(x1[e], x1[e], ss));
    if (!in) ss = 0.0f;
#pragma unroll
    for (int o = LH / 2; o > 0; o >>= 1) ss += __shfl_xor(ss, o, 64);
    const float inv = 1.0f / sqrtf(ss / (float)p.hd + p.eps);
    f32x4a y0, y1;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float a = x0[e] * inv * (isq ? gq0[e] : gk0[e]);
        const float b = x1[e] * inv * (isq ? gq1[e] : gk1[e]);
        if constexpr (TURN) {
            y0[e] = a * c[e] - b * s[e];
            y1[e] = a * s[e] + b * c[e];
        } else {
            y0[e] = a;
            y1[e] = b;
        }
    }
    if (live) {
        *(f32x4a *)(dst + i0) = y0;
        *(f32x4a *)(dst + half + i0) = y1;
    }
}

template <int LH>
int launch_lh(const HeadNormParams &p, hipStream_t st) {
    const unsigned waves = cdiv((size_t)(p.H + p.Hkv), 64 / LH);
    const dim3 grid((unsigned)p.rows, cdiv(waves, 4));
    if (p.pos)
        headnorm_kernel<LH, true><<<grid, 256, 0, st>>>(p);
    else
        headnorm_kernel<LH, false><<<grid, 256, 0, st>>>(p);
    VMLM_HIP_CHECK(hipGetLastError());
    return VMLM_OK;
}

}  // namespace

int launch_headnorm(const HeadNormArgs &a, hipStream_t st) {
    HeadNormParams p;
    // (a grid has at most 2^32 - 1 threads along its rows)
    constexpr int ROWS = 1 << 23;
    if (a.rows > ROWS) {
        for (int r = 0; r < a.rows;) {
            HeadNormArgs part = a;
            part.rows = std::min(ROWS, a.rows - r);
            part.q = a.q + r * a.ldq;
            part.k = a.k + r * a.ldk;
            part.qo = a.qo + r * a.ldqo;
            part.ko = a.ko + r * a.ldko;
            part.pos = a.pos ? a.pos + r : nullptr;
            const int rc = launch_headnorm(part, st);
            if (rc) return rc;
            r += part.rows;
        }
        return VMLM_OK;
    }
    p.q = a.q;
    p.k = a.k;
    p.gq = a.gq ? a.gq : a.gk;
    p.gk = a.gk ? a.gk : a.gq;
    p.qo = a.qo;
    p.ko = a.ko;
    p.ldq = a.ldq;
    p.ldk = a.ldk;
    p.ldqo = a.ldqo;
    p.ldko = a.ldko;
    p.pos = a.pos;
    p.rows = a.rows;
    p.H = a.H;
    p.Hkv = a.Hkv;
    p.hd = a.hd;
    p.eps = a.eps;
    const double ratio = pow((double)a.theta, -2.0 / a.hd);
    p.fine[0] = 1.0;
    for (int i = 1; i < 16; ++i) p.fine[i] = p.fine[i - 1] * ratio;
    p.coarse[0] = 0.15915494309189533577;  // 1 / 2 pi
    for (int i = 1; i < HEADNORM_MAX_HD / 32; ++i)
        p.coarse[i] = p.coarse[i - 1] * (p.fine[15] * ratio);
    int lh = 1;
    while (lh * 8 < a.hd) lh *= 2;
    switch (lh) {
    case 1: return launch_lh<1>(p, st);
    case 2: return launch_lh<2>(p, st);
    case 4: return launch_lh<4>(p, st);
    case 8: return launch_lh<8>(p, st);
    case 16: return launch_lh<16>(p, st);
    case 32: return launch_lh<32>(p, st);
    default: return launch_lh<64>(p, st);
    }
}

}  // namespace vmlm
