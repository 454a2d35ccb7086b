// k_int4.hip -- C[m][j] = sum over groups g of scale[j][g] * (A[m] . Q[j]) over
// the group's k, Q in 4 bits (vmlm_hip_gemm_nt_int4).
//
// Q is [N][K/2] bytes, byte i of a row holding k = 2i (low nibble) and 2i + 1,
// two's complement. K is a multiple of 32; the last group may be short.
//
// A nibble in the high half of a byte is 16 q as a signed byte: a lane's 16-byte load
// of a row becomes two int8 operands (even and odd k) with 12 operations and no
// conversion. The activations of a run of 128 k are 31-bit fixed-point numbers
// below the row's largest value there, as four signed bytes, so every product and
// sum over a group is exact in int32 and four conversions, three FMAs and one scale make
// an f32 of it: errors are those of K/128 f32 additions.
//
// D = A . B^T per v_mfma_i32_16x16x64_i8, B the nibbles of 16 weight rows, the 16
// rows of A the four bytes of
//   G a multiple of 128:  4 activation rows (a run lies in one group),
//   G = 64:               2 activation rows x 2 groups of the run,
//   G = 32:               1 activation row x 4 groups,
// zero outside their group, so that a lane's four registers are one row's four
// bytes over one group, whose scale the lane loads.
#include <algorithm>

#include "internal.hpp"

namespace vmlm {
namespace {

typedef __attribute__((__vector_size__(4 * sizeof(int)))) int i32x4;
// rows may start anywhere: gfx950's 16-byte loads take any alignment
typedef uint32_t u32x4a __attribute__((ext_vector_type(4), aligned(1)));
typedef float f32x4a __attribute__((ext_vector_type(4), aligned(4)));

constexpr int I4_RUN = 128;  // k of a run
constexpr int I4_WAVES = 8;  // of a workgroup
constexpr int int4_wave_bytes(int rows) { return (rows * 516 + 15) / 16 * 16; }

struct Int4Params {
    const float *A, *scale;
    const uint8_t *Q;
    float *C;
    int M, N, K, G, ng, runs;
};

// Four integers' bytes transposed: byte i of out[t] is digit t (highest first) of v[i].
__device__ __forceinline__ void digit_planes(const uint32_t (&v)[4], uint32_t (&out)[4]) {
    const uint32_t a = __builtin_amdgcn_perm(v[1], v[0], 0x05010400u);  // v0.0 v1.0 v0.1 v1.1
    const uint32_t b = __builtin_amdgcn_perm(v[3], v[2], 0x05010400u);
    const uint32_t c = __builtin_amdgcn_perm(v[1], v[0], 0x07030602u);  // v0.2 v1.2 v0.3 v1.3
    const uint32_t d = __builtin_amdgcn_perm(v[3], v[2], 0x07030602u);
    out[3] = __builtin_amdgcn_perm(b, a, 0x05040100u);
    out[2] = __builtin_amdgcn_perm(b, a, 0x07060302u);
    out[1] = __builtin_amdgcn_perm(d, c, 0x05040100u);
    out[0] = __builtin_amdgcn_perm(d, c, 0x07060302u);
}

__device__ __forceinline__ float row16_max(float v) {
    v = fmaxf(v, dpp_mov<0xB1>(v));
    v = fmaxf(v, dpp_mov<0x4E>(v));
    v = fmaxf(v, dpp_mov<0x124>(v));
    return fmaxf(v, dpp_mov<0x128>(v));
}

// One element in f32, group by group: rows with a NaN or an infinity.
__device__ float int4_f32(const Int4Params &p, int m, int j) {
    const float *a = p.A + (size_t)m * p.K;
    const uint8_t *q = p.Q + (size_t)j * (p.K / 2);
    float c = 0.0f;
    for (int g = 0; g < p.ng; ++g) {
        float s = 0.0f;
        for (int k = g * p.G; k < min(p.K, (g + 1) * p.G); ++k)
            s = __builtin_fmaf(a[k], (float)((int8_t)(q[k / 2] << (k & 1 ? 0 : 4)) >> 4), s);
        c = __builtin_fmaf(s, p.scale[(size_t)j * p.ng + g], c);
    }
    return c;
}

// GM: 128 (any multiple of it), 64 or 32; MT tiles of GM / 32 rows; TN tiles of 16
// columns. A workgroup's waves share out the runs and meet in LDS.
template <int GM, int MT, int TN>
__global__ __launch_bounds__(64 * I4_WAVES) void gemm_int4_kernel(Int4Params p) {
    constexpr int RM = GM / 32, ROWS = RM * MT;
    extern __shared__ __align__(16) uint8_t lds[];
    const int tid = threadIdx.x, w = tid >> 6, W = blockDim.x >> 6, lane = tid & 63;
    const int kb = lane >> 4, n = lane & 15;
    const int n0 = blockIdx.x * (16 * TN), m0 = blockIdx.y * ROWS;
    // a wave's terms [row][byte][parity][64] and its rows' factors
    constexpr int WSZ = int4_wave_bytes(ROWS);
    uint8_t *buf = lds + w * WSZ;
    float *fac = (float *)(buf + ROWS * 512);
    const int per = (p.runs + W - 1) / W, r0 = w * per, r1 = min(p.runs, r0 + per);

    // the lane's place in the A operand: row n = (group, row, byte)
    const int byte = n & 3, row = GM == 128 ? n >> 2 : GM == 64 ? (n >> 2) & 1 : 0;
    const bool mine = GM == 128 || (GM == 64 ? n >> 3 == kb >> 1 : n >> 2 == kb);
    // and what its D registers are: row and group of quad kb
    const int drow = GM == 128 ? kb : GM == 64 ? kb & 1 : 0;
    const int dgrp = GM == 128 ? 0 : GM == 64 ? kb >> 1 : kb;

    const uint8_t *qrow[TN];
    const float *srow[TN];
#pragma unroll
    for (int t = 0; t < TN; ++t) {
        const size_t j = min(n0 + t * 16 + n, p.N - 1);
        qrow[t] = p.Q + j * (p.K / 2) + kb * 16;
        srow[t] = p.scale + j * p.ng;
    }
    float acc[TN][MT];
#pragma unroll
    for (int t = 0; t < TN; ++t)
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[t][i] = 0.0f;

    u32x4 wq[TN];
    float sc[TN];
    auto fetch = [&](int r) {
        const bool in = r * I4_RUN + kb * 32 < p.K;
        const int g = min(GM == 128 ? r * I4_RUN / p.G : r * (I4_RUN / GM) + dgrp, p.ng - 1);
#pragma unroll
        for (int t = 0; t < TN; ++t) {
            wq[t] = u32x4{0, 0, 0, 0};
            if (in) wq[t] = __builtin_bit_cast(u32x4, *(const u32x4a *)(qrow[t] + (size_t)r * 64));
            sc[t] = srow[t][g];
        }
    };
    if (r0 < r1) fetch(r0);
    for (int r = r0; r < r1; ++r) {
        // the run's activations: 16 lanes a row, 8 values a lane
        const int k = r * I4_RUN + n * 8;
#pragma unroll
        for (int i = 0; i < (ROWS + 3) / 4; ++i) {
            const int mr = i * 4 + kb;
            if (ROWS % 4 && mr >= ROWS) continue;
            if (m0 + mr >= p.M) continue;
            f32x4a x0 = {0, 0, 0, 0}, x1 = x0;
            if (k < p.K) {
                const float *a = p.A + (size_t)(m0 + mr) * p.K + k;
                x0 = *(const f32x4a *)a;
                x1 = *(const f32x4a *)(a + 4);
            }
            const float x[8] = {x0[0], x0[1], x0[2], x0[3], x1[0], x1[1], x1[2], x1[3]};
            float mx = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) mx = fmaxf(mx, q8_mag(x[e]));
            mx = row16_max(mx);
            const bool ok = mx <= 3.40282347e38f;
            // (below 2^-112 the factor's range leaves fewer bits)
            const int e2 = ok && mx > 0.0f ? min(29 - ilogbf(mx), 141) : 0;
            uint32_t d[8];
#pragma unroll
            for (int e = 0; e < 8; ++e)
                d[e] = ((uint32_t)(ok ? (int)rintf(ldexpf(x[e], e2)) : 0) + 0x808080u) ^ 0x808080u;
            uint32_t ev[4], od[4];
            digit_planes({d[0], d[2], d[4], d[6]}, ev);
            digit_planes({d[1], d[3], d[5], d[7]}, od);
            uint8_t *o = buf + mr * 512 + n * 4;
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                *(uint32_t *)(o + t * 128) = ev[t];
                *(uint32_t *)(o + t * 128 + 64) = od[t];
            }
            // 2^-4 for the nibble's place in its byte
            if (n == 0) fac[mr] = ok ? ldexpf(1.0f, -e2 - 4) : __builtin_nanf("");
        }
        u32x4 cq[TN];
        float cs[TN];
#pragma unroll
        for (int t = 0; t < TN; ++t) {
            cq[t] = wq[t];
            cs[t] = sc[t];
        }
        if (r + 1 < r1) fetch(r + 1);
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const uint8_t *a = buf + (i * RM + row) * 512 + byte * 128 + kb * 16;
            i32x4 a0 = *(const i32x4 *)a, a1 = *(const i32x4 *)(a + 64);
            if (!mine) a0 = a1 = i32x4{0, 0, 0, 0};
            const float f = fac[i * RM + drow];
#pragma unroll
            for (int t = 0; t < TN; ++t) {
                const i32x4 lo = __builtin_bit_cast(i32x4, (cq[t] << 4) & 0xf0f0f0f0u);
                const i32x4 hi = __builtin_bit_cast(i32x4, cq[t] & 0xf0f0f0f0u);
                i32x4 d = {0, 0, 0, 0};
                d = __builtin_amdgcn_mfma_i32_16x16x64_i8(a0, lo, d, 0, 0, 0);
                d = __builtin_amdgcn_mfma_i32_16x16x64_i8(a1, hi, d, 0, 0, 0);
                float v = (float)d[0];
#pragma unroll
                for (int b = 1; b < 4; ++b) v = __builtin_fmaf(v, 256.0f, (float)d[b]);
                acc[t][i] = __builtin_fmaf(v * f, cs[t], acc[t][i]);
            }
        }
        __builtin_amdgcn_wave_barrier();
    }

    // the waves' sums, and of a row's groups, in order
    __syncthreads();
    float *red = (float *)lds;
#pragma unroll
    for (int t = 0; t < TN; ++t)
#pragma unroll
        for (int i = 0; i < MT; ++i) red[((w * TN + t) * MT + i) * 64 + lane] = acc[t][i];
    __syncthreads();
    for (int i = tid; i < ROWS * TN * 16; i += blockDim.x) {
        const int mr = i / (TN * 16), col = i % (TN * 16), t = col / 16, m = m0 + mr, j = n0 + col;
        if (m >= p.M || j >= p.N) continue;
        const int tile = mr / RM, q0 = GM == 32 ? 0 : mr % RM;
        float v = 0.0f;
        for (int x = 0; x < W; ++x) {
            const float *s = red + ((x * TN + t) * MT + tile) * 64 + col % 16;
#pragma unroll
            for (int g = 0; g < 128 / GM; ++g) v += s[(q0 + g * RM) * 16];
        }
        if (v != v) v = int4_f32(p, m, j);
        p.C[(size_t)m * p.N + j] = v;
    }
}

template <int GM, int MT, int TN>
int launch_t(const Int4Params &p, int W, hipStream_t st) {
    constexpr int ROWS = GM / 32 * MT;
    // the terms, then the sums
    constexpr size_t wave = std::max(int4_wave_bytes(ROWS), TN * MT * 256);
    const size_t lds = W * wave;
    int rc = allow_lds((const void *)gemm_int4_kernel<GM, MT, TN>, lds, I4_WAVES * wave);
    if (rc) return rc;
    const dim3 grid(cdiv((size_t)p.N, 16 * TN), cdiv((size_t)p.M, ROWS));
    gemm_int4_kernel<GM, MT, TN><<<grid, 64 * W, lds, st>>>(p);
    VMLM_HIP_CHECK(hipGetLastError());
    return VMLM_OK;
}

template <int GM, int MT>
int launch_mt(const Int4Params &p, int W, hipStream_t st) {
    const size_t slabs = cdiv((size_t)p.M, GM / 32 * MT);
    const size_t tiles = cdiv((size_t)p.N, 16) * slabs;
    if (tiles >= 2048) return launch_t<GM, MT, 4>(p, W, st);
    if (tiles >= 1024) return launch_t<GM, MT, 2>(p, W, st);
    return launch_t<GM, MT, 1>(p, W, st);
}

template <int GM>
int launch_gm(const Int4Params &p, int W, hipStream_t st) {
    const int tiles = cdiv((size_t)p.M, GM / 32);
    if (tiles == 1) return launch_mt<GM, 1>(p, W, st);
    if (tiles == 2) return launch_mt<GM, 2>(p, W, st);
    return launch_mt<GM, 4>(p, W, st);
}

}  // namespace

int launch_gemm_int4(const Int4Args &a, hipStream_t st) {
    Int4Params p;
    p.A = a.A;
    p.Q = a.Q;
    p.scale = a.scale;
    p.C = a.C;
    p.M = a.M;
    p.N = a.N;
    p.K = a.K;
    p.G = a.G;
    p.ng = (a.K + a.G - 1) / a.G;
    p.runs = (a.K + I4_RUN - 1) / I4_RUN;
    const int each = (p.runs + I4_WAVES - 1) / I4_WAVES, W = (p.runs + each - 1) / each;
    if (a.G == 32) return launch_gm<32>(p, W, st);
    if (a.G == 64) return launch_gm<64>(p, W, st);
    return launch_gm<128>(p, W, st);
}

}  // namespace vmlm
