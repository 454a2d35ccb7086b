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
// sum over a group is exact in int32 and two conversions, an FMA and two products make
// an f32 of it: errors are the split's (2^-29 of that largest value) and those of K/128 f32
// additions.
//
// D = A . B^T per v_mfma_i32_16x16x64_i8, B the nibbles of 16 weight rows, the 16
// rows of A the four bytes of
//   G a multiple of 128:  4 activation rows (a run lies in one group),
//   G = 64:               2 activation rows x 2 groups of the run,
//   G = 32:               1 activation row x 4 groups,
// zero outside their group, so that a lane's four registers are one row's four
// bytes over one group, and one lane needs one scale.
//
// Codes and scales come in pairs of runs, eight lanes to 128 bytes of a row, and take
// their places for the B operand through LDS that belongs to the wave: read straight
// from the rows, 16 neighbouring lanes want 16 rows, and the address unit, which takes
// them line by line, was what the time went to (LM head 47 us so, 36.5 this way).
//
// Bound, and measured (kernel times): one row of 122753 x 2304 in groups of 64 takes 36.5
// us, 4.4 TB/s of codes and scales against 5.1 of a large copy. Up to a tile a CU the
// launch and one latency through the K / 256 pairs are the time: 1 x 2304 x 2304 in 5 us,
// where a call's issue takes 3.8. Many rows: see gemm_int4_rows_kernel.
#include <algorithm>
#include <type_traits>

#include "internal.hpp"

namespace vmlm {
namespace {

typedef __attribute__((__vector_size__(4 * sizeof(int)))) int i32x4;
// rows may start anywhere: gfx950's 16-byte loads take any alignment
typedef uint32_t u32x4a __attribute__((ext_vector_type(4), aligned(1)));
typedef float f32x4a __attribute__((ext_vector_type(4), aligned(4)));

constexpr int I4_RUN = 128;  // k of a run
constexpr int I4_ROWB = 144;  // LDS bytes of a row's pair of runs: 128, and 16 against bank conflicts
constexpr int I4_LDS = 160 * 1024;

struct Int4Params {
    const float *A, *scale;
    const uint8_t *Q;
    float *C;
    int M, N, K, G, ng, runs;
    size_t ldc;
    int rg;  // runs of a group (G a multiple of 128)
    // the activations as planes (int4_planes_kernel), or null
    const uint8_t *planes;
    const float *fac;
    int rows;  // of fac
};

// Codes and scales of 16 columns over a pair of runs, as loaded and in LDS. The
// addresses are 32-bit offsets from the workgroup's first column, fixed for its whole
// run over K. Behind K the row's last codes are read again: the activations are zero
// there.
template <int GM>
struct Pair {
    static constexpr int S = 256 / GM;             // scales of a row
    static constexpr int SL = (S * 16 + 63) / 64;  // loads of them
    static constexpr int BYTES = 16 * I4_ROWB + 16 * (S + 1) * 4;
    uint32_t qo[2], so[SL];
    u32x4 q[2];
    float s[SL];
    // 16 columns from n0 + 16 t on
    __device__ __forceinline__ void place(const Int4Params &p, int n0, int t, int lane) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            qo[i] = (uint32_t)(min(n0 + t * 16 + i * 8 + (lane >> 3), p.N - 1) - n0) * (p.K / 2);
#pragma unroll
        for (int i = 0; i < SL; ++i) {
            const int x = (lane + i * 64) & (S * 16 - 1);
            so[i] = (uint32_t)(min(n0 + t * 16 + x / S, p.N - 1) - n0) * p.ng;
        }
    }
    // g0, g1: the groups of the two runs (GM = 128)
    __device__ __forceinline__ void load(const Int4Params &p, int n0, int pair, int g0, int g1,
                                         int lane) {
        const uint8_t *qb = p.Q + (size_t)n0 * (p.K / 2);
        const float *sb = p.scale + (size_t)n0 * p.ng;
        const uint32_t k = min(pair * 128 + (lane & 7) * 16, p.K / 2 - 16);
#pragma unroll
        for (int i = 0; i < 2; ++i)
            q[i] = __builtin_bit_cast(u32x4, *(const u32x4a *)(qb + (size_t)(qo[i] + k)));
#pragma unroll
        for (int i = 0; i < SL; ++i) {
            const int e = (lane + i * 64) & (S - 1);
            const int g = GM == 128 ? (e ? g1 : g0) : min(pair * S + e, p.ng - 1);
            s[i] = sb[so[i] + (uint32_t)g];
        }
    }
    __device__ __forceinline__ void store(uint8_t *b, int lane) const {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            *(u32x4 *)(b + (i * 8 + (lane >> 3)) * I4_ROWB + (lane & 7) * 16) = q[i];
        float *f = (float *)(b + 16 * I4_ROWB);
#pragma unroll
        for (int i = 0; i < SL; ++i) {
            const int x = (lane + i * 64) & (S * 16 - 1);
            f[x / S * (S + 1) + x % S] = s[i];
        }
    }
    // the lane's B codes of run u (0, 1) and its group's scale
    static __device__ __forceinline__ u32x4 codes(const uint8_t *b, int u, int lane) {
        return *(const u32x4 *)(b + (lane & 15) * I4_ROWB + u * 64 + (lane >> 4) * 16);
    }
    static __device__ __forceinline__ float scale(const uint8_t *b, int u, int lane, int grp) {
        return ((const float *)(b + 16 * I4_ROWB))[(lane & 15) * (S + 1) + u * (S / 2) + grp];
    }
};

// The group of a run, walked along (runs of a group: G / 128).
struct RunGroup {
    int g, left, each, last;
    __device__ __forceinline__ RunGroup(int run, int each, int ng) : each(each), last(ng - 1) {
        g = run / each;
        left = each - run % each;
    }
    __device__ __forceinline__ int next() {
        const int now = min(g, last);
        if (--left == 0) {
            ++g;
            left = each;
        }
        return now;
    }
};

// Planes: for each run and four rows, [parity][kb][row % 4][byte][16]: an A operand of
// 4 x 4 rows is 1 KB in lane order. `rows` is padded to whole slabs.
constexpr int I4_SLAB = 16;
__device__ __forceinline__ size_t plane_at(int runs, int m, int r) {
    return ((size_t)(m >> 2) * runs + r) * 2048 + (m & 3) * 64;
}

// over each row of 16 lanes; a NaN stays
__device__ __forceinline__ float row16_maximum(float v) {
    v = __builtin_elementwise_maximum(v, dpp_mov<0xB1>(v));
    v = __builtin_elementwise_maximum(v, dpp_mov<0x4E>(v));
    v = __builtin_elementwise_maximum(v, dpp_mov<0x124>(v));
    return __builtin_elementwise_maximum(v, dpp_mov<0x128>(v));
}

// Eight neighbouring values of a run's row, 16 lanes a row, as digit planes of the
// even and the odd ones; the factor that takes the sums back, NaN for a row with
// one, is the same in all 16 lanes.
__device__ __forceinline__ float split8(const float *row, int k, int K, uint32_t (&ev)[4],
                                        uint32_t (&od)[4]) {
    const float *a = row + min(k, K - 8);
    const bool in = k < K;
    const f32x4a x0 = *(const f32x4a *)a, x1 = *(const f32x4a *)(a + 4);
    const float x[8] = {x0[0], x0[1], x0[2], x0[3], x1[0], x1[1], x1[2], x1[3]};
    float mx = 0.0f;  // a NaN stays
#pragma unroll
    for (int e = 0; e < 8; ++e) mx = __builtin_elementwise_maximum(mx, fabsf(x[e]));
    mx = row16_maximum(in ? mx : 0.0f);
    const bool ok = mx <= 3.40282347e38f;
    // (below 2^-112 the factor's range leaves fewer bits)
    const int e2 = ok && mx > 0.0f ? min(29 - ilogbf(mx), 141) : 0;
    const int es = in && ok ? e2 : -1000;  // none behind K, nor of a row without a factor
    uint32_t d[8];
#pragma unroll
    for (int e = 0; e < 8; ++e)  // signed_bytes of an integer at most one step off: the sum has
                                 // f32's 24 bits, and the conversion cuts a fraction off
        d[e] = (uint32_t)(int)(ldexpf(x[e], es) + (float)0x808080) ^ 0x808080u;
    transpose_bytes({d[0], d[2], d[4], d[6]}, ev);
    transpose_bytes({d[1], d[3], d[5], d[7]}, od);
    // 2^-4 for the nibble's place in its byte
    return ok ? ldexpf(1.0f, -e2 - 4) : __builtin_nanf("");
}

// 4 x 4 dwords transposed over four neighbouring lanes: r[i] of lane k becomes r[k] of
// lane i.
__device__ __forceinline__ void transpose_quad(uint32_t (&r)[4], int lane) {
    auto swap = [&](uint32_t &a, uint32_t &b, auto ctrl, bool odd) {
        const uint32_t give = odd ? a : b;
        const uint32_t got = __float_as_uint(dpp_mov<decltype(ctrl)::value>(__uint_as_float(give)));
        (odd ? a : b) = got;
    };
    using Xor1 = std::integral_constant<int, 0xB1>;
    using Xor2 = std::integral_constant<int, 0x4E>;
    swap(r[0], r[1], Xor1{}, lane & 1);
    swap(r[2], r[3], Xor1{}, lane & 1);
    swap(r[0], r[2], Xor2{}, lane & 2);
    swap(r[1], r[3], Xor2{}, lane & 2);
}

// The rows' planes and factors [runs][rows]; 16 lanes a (row, run), four of them 64
// bytes of a plane. One pass: 4 bytes read and 4 written a value; 100 x 5760 in 4.5 us, most
// of it a launch and one latency.
__global__ __launch_bounds__(256) void int4_planes_kernel(const float *A, int M, int K, int runs,
                                                          int rows, uint8_t *planes, float *fac) {
    const int rb = (runs + 15) / 16, m = blockIdx.x / rb;
    const int l = threadIdx.x & 15, r = (blockIdx.x - m * rb) * 16 + (threadIdx.x >> 4);
    if (r >= runs) return;
    const int k = r * I4_RUN + l * 8;
    uint32_t ev[4], od[4];
    const float f = split8(A + (size_t)m * K, k, K, ev, od);
    transpose_quad(ev, l);  // byte l & 3 (lowest first) of 16 k
    transpose_quad(od, l);
    uint8_t *o = planes + plane_at(runs, m, r) + (l >> 2) * 256 + (3 - (l & 3)) * 16;
    *(u32x4 *)o = u32x4{ev[0], ev[1], ev[2], ev[3]};
    *(u32x4 *)(o + 1024) = u32x4{od[0], od[1], od[2], od[3]};
    if (l == 0) fac[(size_t)r * rows + m] = f;
}

// The sum over one lane's group of an A operand (even k, odd k) and 16 rows' codes.
__device__ __forceinline__ float product(const i32x4 &a0, const i32x4 &a1, u32x4 q) {
    i32x4 d = {0, 0, 0, 0};
    d = __builtin_amdgcn_mfma_i32_16x16x64_i8(a0, __builtin_bit_cast(i32x4, (q << 4) & 0xf0f0f0f0u),
                                              d, 0, 0, 0);
    d = __builtin_amdgcn_mfma_i32_16x16x64_i8(a1, __builtin_bit_cast(i32x4, q & 0xf0f0f0f0u), d, 0, 0,
                                              0);
    // each below 2^21: two of them fit an int32
    const int hi = d[0] * 256 + d[1], lo = d[2] * 256 + d[3];
    return __builtin_fmaf((float)hi, 65536.0f, (float)lo);
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

// A workgroup's place: COLS columns of ROWS rows. Every XCD gets one stretch of the
// places in column order: the slabs of a column group read the same weights through
// one L2.
template <int COLS, int ROWS>
__device__ __forceinline__ bool int4_place(const Int4Params &p, int *n0, int *m0) {
    const int slabs = (p.M + ROWS - 1) / ROWS, all = (p.N + COLS - 1) / COLS * slabs;
    const int at = (int)(blockIdx.x & 7) * ((all + 7) / 8) + (int)(blockIdx.x >> 3);
    *n0 = at / slabs * COLS;
    *m0 = at % slabs * ROWS;
    return at < all;
}

// The waves' sums, and of a row's groups, in order.
template <int GM, int MT, int TN>
__device__ __forceinline__ void int4_finish(const Int4Params &p, const float (&acc)[TN][MT],
                                            float *red, int n0, int m0) {
    constexpr int RM = GM / 32, ROWS = RM * MT;
    const int tid = threadIdx.x, w = tid >> 6, W = blockDim.x >> 6, lane = tid & 63;
    __syncthreads();
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
        p.C[m * p.ldc + j] = v;
    }
}

// LDS of a wave: the terms [run][row][byte][parity][64] of `cr` runs, the rows'
// factors, the columns' pairs; then its sums.
constexpr int int4_conv_runs(int rows) { return rows <= 2 ? 2 : 1; }
template <int GM, int MT, int TN>
constexpr int int4_wave_bytes() {
    constexpr int rows = GM / 32 * MT, cr = int4_conv_runs(rows);
    const int conv = (cr * rows * 516 + 15) / 16 * 16 + TN * Pair<GM>::BYTES;
    return (std::max(conv, TN * MT * 256) + 15) / 16 * 16;
}

// GM: 128 (any multiple of it), 64 or 32; MT tiles of GM / 32 rows; TN tiles of 16
// columns. A workgroup's waves share out the pairs of runs and meet in LDS. Each
// wave splits its runs' rows itself.
template <int GM, int MT, int TN>
__global__ __launch_bounds__(TN == 4 ? 256 : 1024) void gemm_int4_kernel(Int4Params p) {
    constexpr int RM = GM / 32, ROWS = RM * MT, CR = int4_conv_runs(ROWS);
    extern __shared__ __align__(16) uint8_t lds[];
    const int tid = threadIdx.x, w = tid >> 6, W = blockDim.x >> 6, lane = tid & 63;
    const int kb = lane >> 4, n = lane & 15;
    int n0, m0;
    if (!int4_place<16 * TN, ROWS>(p, &n0, &m0)) return;
    uint8_t *buf = lds + w * int4_wave_bytes<GM, MT, TN>();
    float *fac = (float *)(buf + CR * ROWS * 512);
    uint8_t *cols = buf + (CR * ROWS * 516 + 15) / 16 * 16;
    const int pairs = p.runs / 2, per = (pairs + W - 1) / W;
    const int p0 = w * per, p1 = min(pairs, p0 + per);

    // the lane's place in the A operand: row n = (group, row, byte)
    const int byte = n & 3, row = GM == 128 ? n >> 2 : GM == 64 ? (n >> 2) & 1 : 0;
    const bool mine = GM == 128 || (GM == 64 ? n >> 3 == kb >> 1 : n >> 2 == kb);
    // and what its D registers are: row and group of quad kb
    const int drow = GM == 128 ? kb : GM == 64 ? kb & 1 : 0;
    const int dgrp = GM == 128 ? 0 : GM == 64 ? kb >> 1 : kb;

    float acc[TN][MT];
#pragma unroll
    for (int t = 0; t < TN; ++t)
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[t][i] = 0.0f;

    Pair<GM> next[TN];
    RunGroup rg(p0 * 2, p.rg, p.ng);
    auto fetch_cols = [&](int pr) {
        const int g0 = rg.next(), g1 = rg.next();
#pragma unroll
        for (int t = 0; t < TN; ++t) next[t].load(p, n0, min(pr, pairs - 1), g0, g1, lane);
    };
#pragma unroll
    for (int t = 0; t < TN; ++t) next[t].place(p, n0, t, lane);
    fetch_cols(p0);
    for (int pr = p0; pr < p1; ++pr) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int r = pr * 2 + u;
            if (u % CR == 0) {
                // the activations of CR runs: 16 lanes a row of a run, 8 values a lane
#pragma unroll
                for (int i = 0; i < (CR * ROWS + 3) / 4; ++i) {
                    const int x = i * 4 + kb, mr = x % ROWS, rr = x / ROWS;
                    if (rr >= CR || m0 + mr >= p.M) continue;
                    const int k = (r + rr) * I4_RUN + n * 8;
                    uint32_t ev[4], od[4];
                    const float f = split8(p.A + (size_t)(m0 + mr) * p.K, k, p.K, ev, od);
                    uint8_t *o = buf + x % (CR * ROWS) * 512 + n * 4;
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        *(uint32_t *)(o + t * 128) = ev[3 - t];
                        *(uint32_t *)(o + t * 128 + 64) = od[3 - t];
                    }
                    if (n == 0) fac[rr * ROWS + mr] = f;
                }
            }
            if (u == 0) {
#pragma unroll
                for (int t = 0; t < TN; ++t)
                    next[t].store(cols + t * Pair<GM>::BYTES, lane);
                fetch_cols(pr + 1);
            }
            __builtin_amdgcn_wave_barrier();
            u32x4 q[TN];
            float sc[TN];
#pragma unroll
            for (int t = 0; t < TN; ++t) {
                q[t] = Pair<GM>::codes(cols + t * Pair<GM>::BYTES, u, lane);
                sc[t] = Pair<GM>::scale(cols + t * Pair<GM>::BYTES, u, lane, dgrp);
            }
            const int at = u % CR * ROWS;
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const uint8_t *a = buf + (at + i * RM + row) * 512 + byte * 128 + kb * 16;
                i32x4 a0 = *(const i32x4 *)a, a1 = *(const i32x4 *)(a + 64);
                const float f = fac[at + i * RM + drow];
                if (!mine) a0 = a1 = i32x4{0, 0, 0, 0};
#pragma unroll
                for (int t = 0; t < TN; ++t)
                    acc[t][i] = __builtin_fmaf(product(a0, a1, q[t]) * f, sc[t], acc[t][i]);
            }
            __builtin_amdgcn_wave_barrier();
        }
    }

    int4_finish<GM, MT, TN>(p, acc, (float *)lds, n0, m0);
}

// Many rows, the activations as planes: a wave takes 4 tiles of rows and 64 columns
// over its share of the pairs, A operands straight from the planes (1 KB in lane
// order), one run ahead. 100 x 2304 x 5760 in groups of 128: planes 4.5 us, this 15, 0.18
// POP/s (0.7 on the matrix units: four bytes a value). Bound by the A operands, which every
// 64 columns read again through the caches, at two waves a SIMD.
constexpr int I4_TM = 4, I4_TN = 4;

template <int GM>
__global__ __launch_bounds__(512) void gemm_int4_rows_kernel(Int4Params p) {
    constexpr int RM = GM / 32, ROWS = RM * I4_TM, MT = I4_TM, TN = I4_TN, PB = Pair<GM>::BYTES;
    extern __shared__ __align__(16) uint8_t lds[];
    const int tid = threadIdx.x, w = tid >> 6, W = blockDim.x >> 6, lane = tid & 63;
    const int kb = lane >> 4, n = lane & 15;
    int n0, m0;
    if (!int4_place<16 * TN, ROWS>(p, &n0, &m0)) return;
    uint8_t *cols = lds + w * std::max(TN * PB, TN * MT * 256);
    const int pairs = p.runs / 2, per = (pairs + W - 1) / W;
    const int p0 = w * per, p1 = min(pairs, p0 + per);

    const int byte = n & 3, row = GM == 128 ? n >> 2 : GM == 64 ? (n >> 2) & 1 : 0;
    const bool mine = GM == 128 || (GM == 64 ? n >> 3 == kb >> 1 : n >> 2 == kb);
    const int drow = GM == 128 ? kb : GM == 64 ? kb & 1 : 0;
    const int dgrp = GM == 128 ? 0 : GM == 64 ? kb >> 1 : kb;

    uint32_t plane[MT], fat[MT];  // from the slab's first row
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        plane[i] = (uint32_t)plane_at(p.runs, (m0 & 3) + i * RM + row, 0) + kb * 256 + byte * 16;
        fat[i] = i * RM + drow;
    }
    float acc[TN][MT];
#pragma unroll
    for (int t = 0; t < TN; ++t)
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[t][i] = 0.0f;

    Pair<GM> next[TN];
    struct {
        i32x4 a[MT][2];
        float f[MT];
    } op[2];
    auto fetch = [&](int r, auto &o) {
        r = min(r, p.runs - 1);
        const uint8_t *a = p.planes + plane_at(p.runs, m0 & ~3, r);
        const float *f = p.fac + (size_t)r * p.rows + m0;
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            o.a[i][0] = *(const i32x4 *)(a + (size_t)plane[i]);
            o.a[i][1] = *(const i32x4 *)(a + (size_t)plane[i] + 1024);
            o.f[i] = f[fat[i]];
        }
    };
    RunGroup rg(p0 * 2, p.rg, p.ng);
    auto fetch_cols = [&](int pr) {
        const int g0 = rg.next(), g1 = rg.next();
#pragma unroll
        for (int t = 0; t < TN; ++t) next[t].load(p, n0, min(pr, pairs - 1), g0, g1, lane);
    };
#pragma unroll
    for (int t = 0; t < TN; ++t) next[t].place(p, n0, t, lane);
    fetch_cols(p0);
    fetch(p0 * 2, op[0]);
    for (int pr = p0; pr < p1; ++pr) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            if (u == 0) {
#pragma unroll
                for (int t = 0; t < TN; ++t) next[t].store(cols + t * PB, lane);
                fetch_cols(pr + 1);
            }
            fetch(pr * 2 + u + 1, op[1 - u]);
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int t = 0; t < TN; ++t) {
                const u32x4 q = Pair<GM>::codes(cols + t * PB, u, lane);
                const float sc = Pair<GM>::scale(cols + t * PB, u, lane, dgrp);
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    const i32x4 z = {0, 0, 0, 0};
                    acc[t][i] = __builtin_fmaf(product(mine ? op[u].a[i][0] : z,
                                                       mine ? op[u].a[i][1] : z, q) * op[u].f[i],
                                               sc, acc[t][i]);
                }
            }
            __builtin_amdgcn_wave_barrier();
        }
    }
    int4_finish<GM, MT, TN>(p, acc, (float *)lds, n0, m0);
}

template <int GM, int MT, int TN>
int launch_t(Int4Params p, hipStream_t st) {
    constexpr int wave = int4_wave_bytes<GM, MT, TN>();
    // few columns: as many waves as pairs, a workgroup's time is one latency; many: three
    // or four waves with some pairs each, so that loads run ahead (LM head 39.5 us with
    // five waves, 36.5 with three)
    constexpr int most = std::min(TN == 4 ? 4 : 16, I4_LDS / wave);
    const int pairs = p.runs / 2, each = (pairs + most - 1) / most;
    const int W = (pairs + each - 1) / each;
    int rc = allow_lds((const void *)gemm_int4_kernel<GM, MT, TN>, W * wave, most * wave);
    if (rc) return rc;
    const size_t all = (size_t)cdiv((size_t)p.N, 16 * TN) * cdiv((size_t)p.M, GM / 32 * MT);
    gemm_int4_kernel<GM, MT, TN><<<cdiv(all, 8) * 8, 64 * W, W * wave, st>>>(p);
    VMLM_HIP_CHECK(hipGetLastError());
    return VMLM_OK;
}

template <int GM>
int launch_rows(const Int4Params &p, hipStream_t st) {
    constexpr int wave = I4_TN * std::max(Pair<GM>::BYTES, I4_TM * 256);
    const int pairs = p.runs / 2, each = (pairs + 7) / 8, W = (pairs + each - 1) / each;
    int rc = allow_lds((const void *)gemm_int4_rows_kernel<GM>, W * wave, 8 * wave);
    if (rc) return rc;
    const size_t all = (size_t)cdiv((size_t)p.N, 16 * I4_TN) * cdiv((size_t)p.M, GM / 32 * I4_TM);
    gemm_int4_rows_kernel<GM><<<cdiv(all, 8) * 8, 64 * W, W * wave, st>>>(p);
    VMLM_HIP_CHECK(hipGetLastError());
    return VMLM_OK;
}

template <int GM, int MT>
int launch_mt(const Int4Params &p, hipStream_t st) {
    const size_t slabs = cdiv((size_t)p.M, GM / 32 * MT);
    const size_t tiles = cdiv((size_t)p.N, 16) * slabs;
    // Up to a tile a CU each for itself (2304 columns, one row: 4.8 us against 5.2 with two
    // together); more share the rows' split (5760 columns, one row 6.0 and 5.2, 16 rows 17.4 and
    // 10.2); with many, loads run ahead in long workgroups (24 rows of 20000 45 and 42).
    if (tiles >= 2048) return launch_t<GM, MT, 4>(p, st);
    if (tiles > 256) return launch_t<GM, MT, 2>(p, st);
    return launch_t<GM, MT, 1>(p, st);
}

template <int GM>
int launch_gm(const Int4Params &p, hipStream_t st) {
    if constexpr (GM > 32) {  // (no planes for groups of 32)
        if (p.planes) return launch_rows<GM>(p, st);
    }
    const int tiles = cdiv((size_t)p.M, GM / 32);
    if (tiles == 1) return launch_mt<GM, 1>(p, st);
    if (tiles == 2) return launch_mt<GM, 2>(p, st);
    return launch_mt<GM, 4>(p, st);
}

// The planes' rows: whole slabs of 16, so that every lane's row exists.
size_t plane_rows(int M) { return ((size_t)M + I4_SLAB - 1) / I4_SLAB * I4_SLAB; }

// Columns and rows of a launch, so that its threads stay below 2^32 (a grid's limit): there are at
// most 64 for each 4 rows x 64 columns (256 where there are no more than 4 rows), and in the
// planes' launch 256 for each 16 runs of a row.
constexpr int I4_COLS = 1 << 26;
int piece_rows(int M, int N, int runs) {
    const int n = std::min(N, I4_COLS), by_tiles = (1 << 30) / n / I4_SLAB * I4_SLAB;
    const int by_runs = (1 << 23) / (int)cdiv((size_t)runs, 16) / I4_SLAB * I4_SLAB;
    return std::min(M, std::max((int)I4_SLAB, std::min(by_tiles, by_runs)));
}
int pair_runs(int K) { return (K + 2 * I4_RUN - 1) / (2 * I4_RUN) * 2; }  // whole pairs

}  // namespace

// Planes cost a launch and their bytes, splitting in place the split again for every
// 16 to 64 columns. (K = 2304, planes and in place, us; group 128: 16 rows of 5760 columns 10.2 and
// 8.7, 20 rows 10.7 and 15.6, 32 rows of 2304 10.4 and 8.7, 64 rows 10.9 and 15.8, 6 rows of
// 20000 16.8 and 16.9, 12 rows 17.4 and 21.6; group 64: 8 rows of 5760 9.3 and 7.0, 12 rows 9.7
// and 12.2, 20 rows of 2304 9.5 and 7.0, 32 rows 9.6 and 12.0). With groups of 32 a slab is
// four rows either way: 64 rows of 2304 21.9 and 21.7, of 20000 122 and 113. Other K were not
// measured.)
size_t gemm_int4_work_bytes(int M, int N, int K, int G) {
    if (G == 32 || M <= 4 || (size_t)M * N <= (G == 64 ? 60000 : 100000)) return 0;
    const int runs = pair_runs(K);
    return plane_rows(piece_rows(M, N, runs)) * runs * (512 + 4);
}

int launch_gemm_int4(const Int4Args &a, hipStream_t st) {
    Int4Params p;
    p.K = a.K;
    p.G = a.G;
    p.ng = (a.K + a.G - 1) / a.G;
    p.runs = pair_runs(a.K);
    p.rg = std::max(1, a.G / I4_RUN);
    p.ldc = a.N;
    p.planes = nullptr;
    p.fac = nullptr;
    p.rows = 0;
    const int each = piece_rows(a.M, a.N, p.runs);
    for (int m = 0; m < a.M; m += each) {  // (one piece of nearly any call)
        p.A = a.A + (size_t)m * a.K;
        p.M = std::min(each, a.M - m);
        if (a.work) {
            const int rows = (int)plane_rows(p.M);
            uint8_t *planes = (uint8_t *)a.work;
            float *fac = (float *)(planes + (size_t)rows * p.runs * 512);
            const unsigned wgs = (unsigned)p.M * cdiv((size_t)p.runs, 16);
            int4_planes_kernel<<<wgs, 256, 0, st>>>(p.A, p.M, a.K, p.runs, rows, planes, fac);
            VMLM_HIP_CHECK(hipGetLastError());
            p.planes = planes;
            p.fac = fac;
            p.rows = rows;
        }
        for (int n = 0; n < a.N; n += p.N) {
            p.N = std::min(I4_COLS, a.N - n);
            p.Q = a.Q + (size_t)n * (a.K / 2);
            p.scale = a.scale + (size_t)n * p.ng;
            p.C = a.C + (size_t)m * a.N + n;
            const int rc = a.G == 32   ? launch_gm<32>(p, st)
                           : a.G == 64 ? launch_gm<64>(p, st)
                                       : launch_gm<128>(p, st);
            if (rc) return rc;
        }
    }
    return VMLM_OK;
}

}  // namespace vmlm
