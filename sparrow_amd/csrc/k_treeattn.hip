// k_treeattn.hip -- attention of several tokens a sequence over the 4-bit KV cache
// (vmlm_hip_attention_tree_kv4); the format is in kv4.hpp.
//
// Token t of a sequence stands at position pos0 + t, its row already in the cache. It sees
// the positions before pos0, and of the tokens itself and its ancestors (a tree) or those
// before it (a chain): s_p = scale * q . k_p over the positions seen, o = sum_p exp(s_p - m) v_p /
// sum_p exp(s_p - m).
//
// With tens of queries a cached position the vector units would bound it, so what a
// (query, position) pair costs beside the matrix products is kept to a dozen operations:
//  * scale * (u - 8) is EXACT in f16: 8 significant bits times at most 8 are 11. So a key
//    channel is one f16 (a shift, a mask and a fused multiply-add for two of them), and a group's
//    middle, min + 8 scale, two more: k . q = sum_c f16(scale (u - 8)) q_c + sum_g
//    (min + 8 scale)_g Q_g, Q_g the sum of q over group g: one more step of the same
//    product. No scale is applied to a score. (Sums of min and of 8 scale apart would
//    cancel: 9e-6 off where 65463 values average out, 2e-6 in f32.)
//  * q, Q_g, the middles and the weights are two f16 terms, 22 bits; products of f16 are exact, sums f32.
//  * The same for V, whose middles come out as 2 extra "channels" a group.
//  * S^T = K q^T, then O^T = V^T P^T: the lane that holds a query's column of scores holds
//    its weights' operand too, since the rows of K are dealt so that a lane's eight
//    positions are the eight of a V dword. Nothing crosses lanes but the maximum.
// Range: a query's 16-bit terms stand below its own power of two, a key's below its
// position's, channels groups weighed by the tile's queries (keys may be large just where queries are
// small); a value's power of two goes to its weight, and the running maximum is that of
// weight times value. It is kept an integer: the rescalings are exact, and the exponent
// score * log2(e) - maximum is one fused operation that rounds at its own small size.
// 16-bit terms hold 11 bits down to 2^-28 of the largest and round at 2^-39 of it below.
#include <algorithm>

#include "kv4.hpp"
#include "tree.hpp"

namespace vmlm {
namespace {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2m __attribute__((ext_vector_type(2), aligned(4)));
typedef uint32_t u32x4m __attribute__((ext_vector_type(4), aligned(4)));
typedef float f32x4l __attribute__((ext_vector_type(4)));
typedef int i32x4l __attribute__((ext_vector_type(4)));

constexpr int TA_W = 4;  // waves of a workgroup
constexpr float TA_NONE = -3.40282347e38f;  // the maximum of no score yet
constexpr int TA_NO_GROUP = -1000;          // the weight of channels where all queries are 0

struct TreeAttnParams {
    Kv4View c;
    const float *q;
    size_t ldq, ldo;
    const int32_t *pos0, *count, *parent;
    int S, H, G;
    int tiles, shares;  // of queries; of the positions
    float *out, *work;
    float scale;  // of the scores: scale * 2^scale_e, |scale| in [1/2, 1), times log2(e)
    int scale_e;
    int *guard;
};

__device__ __forceinline__ float ta_swap16(float v, float (*f)(float, float)) {
    const auto t = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return f(__uint_as_float(t[0]), __uint_as_float(t[1]));
}
__device__ __forceinline__ float ta_swap32(float v, float (*f)(float, float)) {
    const auto t = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return f(__uint_as_float(t[0]), __uint_as_float(t[1]));
}
__device__ __forceinline__ float ta_add(float a, float b) { return a + b; }
__device__ __forceinline__ float ta_max(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ float ta_row16(float v, float (*f)(float, float)) {
    v = f(v, dpp_mov<0xB1>(v));
    v = f(v, dpp_mov<0x4E>(v));
    v = f(v, dpp_mov<0x124>(v));
    return f(v, dpp_mov<0x128>(v));
}

__device__ __forceinline__ uint32_t f16_pair(float a, float b) {
    const hw_f32x2 v = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
}
__device__ __forceinline__ float f16_low(uint32_t v) { return (float)__builtin_bit_cast(f16x2, v)[0]; }
__device__ __forceinline__ float f16_high(uint32_t v) { return (float)__builtin_bit_cast(f16x2, v)[1]; }

// x as two f16 terms
__device__ __forceinline__ uint32_t two_terms(float x) {
    const _Float16 hi = (_Float16)x;
    const f16x2 v = {hi, (_Float16)(x - (float)hi)};
    return __builtin_bit_cast(uint32_t, v);
}

// The exponent e of a magnitude below 2^e (of numbers that are not normal -126).
__device__ __forceinline__ int exp_of(float mag) { return (int)(__float_as_uint(mag) >> 23) - 126; }

// Eight codes of a dword as f16 scale (u - 8): of nibbles (k, k + 4) in register k. s and c
// hold the scale and -24 times it: the nibbles lie in the mantissa of 16 + u.
struct Codes8 {
    f16x8 v;
    __device__ __forceinline__ Codes8(uint32_t w, const uint32_t (&s)[4], const uint32_t (&c)[4]) {
        w ^= 0x88888888u;
        const uint32_t t[4] = {w << 6, w << 2, w >> 2, w >> 6};
        uint32_t r[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t x = (t[k] & 0x03C003C0u) | 0x4C004C00u;
            r[k] = __builtin_bit_cast(
                uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(f16x2, x),
                                                    __builtin_bit_cast(f16x2, s[k]),
                                                    __builtin_bit_cast(f16x2, c[k])));
        }
        v = __builtin_bit_cast(f16x8, u32x4{r[0], r[1], r[2], r[3]});
    }
};
__device__ __forceinline__ uint32_t minus24(uint32_t s) {
    const f16x2 k = {(_Float16)-24.0f, (_Float16)-24.0f};
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, s) * k);
}
// where position or channel o of eight stands in the registers' order
__device__ __forceinline__ int slot8(int o) { return o < 4 ? 2 * o : 2 * o - 7; }

// LDS of a workgroup: the queries' operands [tile][step and term, then the sums][lane][8], for each
// wave its block's V middles as f16 [16][32], scales [8][32] and three numbers for each position, for each
// query its power of two and the tokens it sees, for each group the queries' weight; the waves' results
// then lie over it all.
template <int HD, int MT>
struct TreeLds {
    static constexpr int KS = HD / 32, NG = HD / 32;
    static constexpr int FR = 2 * KS + 1;
    static constexpr int Q = 0;
    static constexpr int WAVE = Q + MT * FR * 1024;
    static constexpr int SC = 1024, N = SC + 512;  // scales [8][32], numbers
    static constexpr int WB = N + 3 * 128;
    static constexpr int F = WAVE + TA_W * WB;
    static constexpr int MASK = F + MT * 64;  // u64
    static constexpr int E = MASK + MT * 128;
    static constexpr int END = E + 64;
    static constexpr int RO = 0;  // [wave][16 MT][HD], then maxima and sums
    static constexpr int RM = RO + TA_W * 16 * MT * HD * 4;
    static constexpr int REND = RM + TA_W * 16 * MT * 8;
    static constexpr int OFF = END > REND ? END : REND;  // [wave][16 MT][8] the middles' sums
    static constexpr int SIZE = OFF + TA_W * 16 * MT * 32;
};

// What a wave reads of a block of 32 positions.
template <int HD>
struct RawBlock {
    static constexpr int NG = HD / 32, KD = HD / 32, GX = NG < 4 ? NG : 4;
    static constexpr int OWN = HD == 256 ? 2 : 1, VM = NG < 2 ? 1 : NG / 2;
    uint32_t k[2][KD], km[2][GX], own[2][OWN], v[HD / 16], vm[VM];
    __device__ __forceinline__ void load(const Kv4View &c, size_t head, int blk, int lane) {
        const int r = lane & 15, j = lane >> 4;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const size_t row = head * c.cap + blk * KV4_BLOCK + 8 * (r >> 2) + (r & 3) + 4 * x;
            const uint8_t *kp = c.k + row * (HD / 2) + j * (HD / 8);
            const uint32_t *mp = c.km + row * NG;
            if constexpr (HD == 32) {
                k[x][0] = *(const uint32_t *)kp;
                km[x][0] = own[x][0] = mp[0];
            } else if constexpr (HD == 64) {
                const u32x2m a = *(const u32x2m *)kp, b = *(const u32x2m *)mp;
                k[x][0] = a[0];
                k[x][1] = a[1];
                km[x][0] = b[0];
                km[x][1] = b[1];
                own[x][0] = j < 2 ? b[0] : b[1];
            } else {
#pragma unroll
                for (int i = 0; i < KD; i += 4) {
                    const u32x4m a = *(const u32x4m *)(kp + i * 4);
#pragma unroll
                    for (int e = 0; e < 4; ++e) k[x][i + e] = a[e];
                }
                const u32x4m b = *(const u32x4m *)(mp + (NG == 8 ? 4 * (j & 1) : 0));
#pragma unroll
                for (int e = 0; e < 4; ++e) km[x][e] = b[e];
#pragma unroll
                for (int e = 0; e < OWN; ++e) own[x][e] = mp[j * OWN + e];
            }
        }
        const uint32_t *vp = (const uint32_t *)(c.v + (head * (c.cap / KV4_BLOCK) + blk) * (size_t)(HD * 16));
#pragma unroll
        for (int n = 0; n < HD / 16; ++n) v[n] = vp[(n * 16 + r) * 4 + j];
        const uint32_t *mp = c.vm + (head * c.cap + blk * KV4_BLOCK + (lane & 31)) * NG + (lane >> 5) * (NG / 2);
#pragma unroll
        for (int i = 0; i < VM; ++i) vm[i] = mp[i];
    }
};

// A tile of 16 MT (token, head) pairs of one sequence and kv head, and one share of the positions.
template <int HD, int MT>
__global__ __launch_bounds__(64 * TA_W, 2) void tree_attn_kernel(TreeAttnParams p) {
    using M = TreeLds<HD, MT>;
    using Raw = RawBlock<HD>;
    constexpr int NG = HD / 32, KS = HD / 32, NT = HD / 16, CL = HD / 4, ROWS = 16 * MT;
    extern __shared__ __align__(16) uint8_t lds[];
    const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63, col = lane & 15, j = lane >> 4;
    // the tiles that read the same positions lie 8 workgroups apart: on one XCD
    const int x8 = blockIdx.x / 8, stream = x8 / p.tiles * 8 + (int)(blockIdx.x % 8), tile = x8 % p.tiles;
    const int share = stream % p.shares, pair = stream / p.shares, kvh = pair % p.c.Hkv, b = pair / p.c.Hkv;
    if (b >= p.c.B) return;
    const TreeRows tr = tree_rows(p.pos0, p.count, p.parent, p.S, p.c.cap, b, p.guard,
                                  kvh == 0 && tile == 0 && share == 0);
    const int row0 = tile * ROWS, rows = min(ROWS, tr.n * p.G - row0);
    if (rows <= 0) return;
    const int t_lo = row0 / p.G, t_hi = (row0 + rows - 1) / p.G;
    const int last = tr.pos0 + t_hi;                               // the last position seen
    const int zone = tr.pos0 + (p.parent ? 0 : t_lo + 1);  // from here on not by all
    const int blocks = last / KV4_BLOCK + 1;
    const int b0 = (int)((long long)share * blocks / p.shares), b1 = (int)((long long)(share + 1) * blocks / p.shares);
    const size_t head = (size_t)b * p.c.Hkv + kvh;

    // 1. the queries' operands
    int *fe = (int *)(lds + M::F), *ge = (int *)(lds + M::E);
    unsigned long long *mask = (unsigned long long *)(lds + M::MASK);
    for (int i = tid; i < MT * 64; i += 64 * TA_W)  // the sums' step: zeros where there is no group
        *(u32x4 *)(lds + M::Q + ((i >> 6) * M::FR + 2 * KS) * 1024 + (i & 63) * 16) = u32x4{0, 0, 0, 0};
    for (int i = tid; i < TA_W * 64; i += 64 * TA_W)
        *(u32x4 *)(lds + M::WAVE + (i >> 6) * M::WB + (i & 63) * 16) = u32x4{0, 0, 0, 0};
    if (tid < 16) ge[tid] = TA_NO_GROUP;
    __syncthreads();
    constexpr int CW = (HD + 63) / 64;
    auto query = [&](int r, float (&x)[CW]) {
        const int R = row0 + min(r, rows - 1), t = R / p.G;
        const float *q = p.q + ((size_t)b * p.S + t) * p.ldq + ((size_t)kvh * p.G + R % p.G) * HD;
#pragma unroll
        for (int i = 0; i < CW; ++i) {
            const int c = i * 64 + lane;
            x[i] = c < HD && r < rows ? q[c] : 0.0f;
        }
    };
    for (int r = w; r < ROWS; r += TA_W) {
        float x[CW], mx[CW], most = 0.0f;
        int bad = 0;
        query(r, x);
#pragma unroll
        for (int i = 0; i < CW; ++i) {
            mx[i] = ta_swap16(ta_row16(fabsf(x[i]), ta_max), ta_max);  // of its 32 channels
            most = fmaxf(most, mx[i]);
            bad |= !(fabsf(x[i]) <= 3.40282347e38f);
        }
        most = ta_swap32(most, ta_max);
        bad = __any(bad);
        const int F = most > 0.0f && !bad ? ilogbf(most) : 0;
        if (lane == 0) fe[r] = F - 8 + p.scale_e;
#pragma unroll
        for (int i = 0; i < CW; ++i)
            if ((lane & 31) == 0 && i * 64 + lane < HD && mx[i] > 0.0f && !bad)
                atomicMax(&ge[i * 2 + lane / 32], ilogbf(mx[i]) - F);
    }
    if (p.parent) {
        if (w == 0) {  // ancestors by doubling: of 2, 4, 8 .. tokens at once
            int up = tr.parent;
            unsigned long long seen = 1ull << lane;
#pragma unroll
            for (int i = 0; i < 6; ++i) {
                const int at = max(up, 0);
                const uint32_t lo = __shfl((uint32_t)seen, at, 64), hi = __shfl((uint32_t)(seen >> 32), at, 64);
                const int next = __shfl(up, at, 64);
                if (up >= 0) {
                    seen |= (unsigned long long)hi << 32 | lo;
                    up = next;
                }
            }
            for (int r = lane; r < ROWS; r += 64) mask[r] = 0;
            __builtin_amdgcn_wave_barrier();
            // (the tokens of the tile, G rows each)
            if (lane >= t_lo && lane <= t_hi)
                for (int r = max(lane * p.G - row0, 0); r < min((lane + 1) * p.G - row0, rows); ++r) mask[r] = seen;
        }
    }
    __syncthreads();
    int group_e[NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) group_e[g] = __builtin_amdgcn_readfirstlane(ge[g]);
    for (int r = w; r < ROWS; r += TA_W) {
        float x[CW];
        int bad = 0;
        query(r, x);
        const int F = fe[r] + 8 - p.scale_e;
#pragma unroll
        for (int i = 0; i < CW; ++i) bad |= !(fabsf(x[i]) <= 3.40282347e38f);
        bad = __any(bad);
        uint8_t *at = lds + M::Q + (r / 16) * M::FR * 1024 + (r % 16) * 16;
#pragma unroll
        for (int i = 0; i < CW; ++i) {
            const int c = i * 64 + lane, g = min(c / 32, NG - 1);
            const float y = bad ? __builtin_nanf("") : ldexpf(x[i], 8 - F - ge[g]);  // below 2^9
            const _Float16 hi = (_Float16)y, lo = (_Float16)(y - (float)hi);
            const float sum = ta_swap16(ta_row16((float)hi + (float)lo, ta_add), ta_add);
            if (c >= HD) continue;
            _Float16 *o = (_Float16 *)(at + (2 * (c % CL / 8)) * 1024 + c / CL * 256) + slot8(c % 8);
            o[0] = hi;
            o[512] = lo;
            if ((c & 31) == 0) {
                const _Float16 sh = (_Float16)sum, sl = (_Float16)(sum - (float)sh);
                _Float16 *s = (_Float16 *)(at + 2 * KS * 1024 + g / 4 * 256) + g % 4 * 2;
                s[0] = s[1] = sh;
                s[256] = s[257] = sl;
            }
        }
    }
    __syncthreads();

    float m[MT], l[MT];
    f32x4 O[MT][NT + 1];
    int fq[MT], lim[MT];
    unsigned long long see[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int r = t * 16 + col;
        m[t] = TA_NONE;
        l[t] = 0.0f;
#pragma unroll
        for (int n = 0; n <= NT; ++n) O[t][n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        fq[t] = fe[r];
        see[t] = p.parent ? mask[r] : 0;
        lim[t] = tr.pos0 + (row0 + min(r, rows - 1)) / p.G;
    }
    uint8_t *wl = lds + M::WAVE + w * M::WB;
    int *ek = (int *)(wl + M::N);
    float *ev = (float *)(wl + M::N + 128), *iev = ev + 32;
    const uint8_t *qf = lds + M::Q + lane * 16;
    const float cs = p.scale;
    // group g's number, g the same in all lanes or not
    auto pick = [&](int g) {
        int e = group_e[0];
#pragma unroll
        for (int i = 1; i < NG; ++i) e = g == i ? group_e[i] : e;
        return e;
    };

    Raw next;
    if (b0 + w < b1) next.load(p.c, head, b0 + w, lane);
    for (int blk = b0 + w; blk < b1; blk += TA_W) {
        const Raw raw = next;
        if (blk + TA_W < b1) next.load(p.c, head, blk + TA_W, lane);
        const int p0 = blk * KV4_BLOCK;
        const bool edge = p0 + KV4_BLOCK > zone || p0 + KV4_BLOCK > last + 1;

        // 2. keys: rows of S^T, 4 j' + i of tile x is position 8 j' + 4 x + i
        f16x8 kf[2][KS + 1];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int at = 8 * (col >> 2) + (col & 3) + 4 * x;
            const bool in = !edge || p0 + at <= last;
            float mid[Raw::GX];
            int e = -0x1000;
            const int gb = NG == 8 ? 4 * (j & 1) : 0;
            int eg[Raw::GX];
#pragma unroll
            for (int g = 0; g < Raw::GX; ++g) {
                const uint32_t meta = in ? raw.km[x][g] : 0u;
                mid[g] = __builtin_fmaf(8.0f, kv4_scale(meta), kv4_min(meta));
                eg[g] = NG == 8 ? (j & 1 ? group_e[NG > 4 ? 4 + g : g] : group_e[g]) : group_e[g];
                e = max(e, exp_of(fmaxf(fabsf(mid[g]) * 0.125f, kv4_scale(meta))) + eg[g]);
            }
            if (NG == 8) e = max(e, __shfl_xor(e, 16, 64));
            e -= 11;
            if (j == 0) ek[at] = e;
            uint32_t ex[4] = {0, 0, 0, 0};
#pragma unroll
            for (int g = 0; g < Raw::GX; ++g)
                ex[g] = two_terms(ldexpf(mid[g], eg[g] - e));
            if (NG <= 4 && (j & 1)) ex[0] = ex[1] = ex[2] = ex[3] = 0;  // (no group 4 ..)
            kf[x][KS] = __builtin_bit_cast(f16x8, u32x4{ex[0], ex[1], ex[2], ex[3]});
#pragma unroll
            for (int o = 0; o < Raw::OWN; ++o) {
                const int g = NG == 1 ? 0 : NG == 2 ? j >> 1 : j * Raw::OWN + o;
                const float s = in ? ldexpf(kv4_scale(raw.own[x][o]), pick(g) - e) : 0.0f;
                const uint32_t sp = f16_pair(s, s), cp = minus24(sp);
                const uint32_t s4[4] = {sp, sp, sp, sp}, c4[4] = {cp, cp, cp, cp};
                constexpr int D = KS / Raw::OWN;
#pragma unroll
                for (int i = 0; i < D; ++i) kf[x][o * D + i] = Codes8(raw.k[x][o * D + i], s4, c4).v;
            }
        }
        // 3. values' meta: lane (position, half of the groups)
        unsigned long long nan_p[Raw::VM];  // lanes whose meta is a NaN
        {
            const int at = lane & 31;
            float mid[Raw::VM], sc[Raw::VM], mag = 0.0f;
#pragma unroll
            for (int i = 0; i < Raw::VM; ++i) {
                const uint32_t meta = !edge || p0 + at <= last ? raw.vm[i] : 0u;
                sc[i] = kv4_scale(meta);
                mid[i] = __builtin_fmaf(8.0f, sc[i], kv4_min(meta));
                nan_p[i] = 0;
                if (edge) {  // what some queries see and others do not: told below
                    const bool bad = !(mid[i] == mid[i]);
                    nan_p[i] = __ballot(bad);
                    if (bad) mid[i] = sc[i] = 0.0f;
                }
                mag = fmaxf(mag, fmaxf(fabsf(mid[i]) * 0.125f, sc[i]));
            }
            if (NG > 1) mag = ta_swap32(mag, ta_max);
            const int e = max(exp_of(mag) - 11, -105);
            _Float16 *o = (_Float16 *)wl + (at & ~7) + slot8(at & 7);
            if (NG > 1 || lane < 32) {
#pragma unroll
                for (int i = 0; i < Raw::VM; ++i) {
                    const int g = (lane >> 5) * (NG / 2) + i;
                    const f16x2 t = __builtin_bit_cast(f16x2, two_terms(ldexpf(mid[i], -e)));
                    o[g * 64] = t[0];
                    o[g * 64 + 32] = t[1];
                    o[M::SC / 2 + g * 32] = (_Float16)ldexpf(sc[i], -e);
                }
            }
            if (lane < 32) {
                ev[at] = (float)e;
                iev[at] = ldexpf(1.0f, -e - 14);
            }
        }
        __builtin_amdgcn_wave_barrier();
        // 4. values: rows of O^T
        f16x8 vf[NT + 1];
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const u32x4 s = *(const u32x4 *)(wl + M::SC + g * 64 + j * 16);
            const uint32_t s4[4] = {s[0], s[1], s[2], s[3]};
            const uint32_t c4[4] = {minus24(s[0]), minus24(s[1]), minus24(s[2]), minus24(s[3])};
            vf[2 * g] = Codes8(raw.v[2 * g], s4, c4).v;
            vf[2 * g + 1] = Codes8(raw.v[2 * g + 1], s4, c4).v;
        }
        vf[NT] = *(const f16x8 *)(wl + col * 64 + j * 16);
        const i32x4l ka = *(const i32x4l *)(ek + 8 * j), kb = *(const i32x4l *)(ek + 8 * j + 4);
        const f32x4l va = *(const f32x4l *)(ev + 8 * j), vb = *(const f32x4l *)(ev + 8 * j + 4);
        const f32x4l ia = *(const f32x4l *)(iev + 8 * j), ib = *(const f32x4l *)(iev + 8 * j + 4);
        __builtin_amdgcn_wave_barrier();

#pragma unroll
        for (int t = 0; t < MT; ++t) {
            // 5. scores of 16 queries at 32 positions
            f32x4 sa = {0.0f, 0.0f, 0.0f, 0.0f}, sb = sa;
#pragma unroll
            for (int i = 0; i < 2 * KS + 1; ++i) {
                const f16x8 qv = *(const f16x8 *)(qf + (t * M::FR + i) * 1024);
                const int k = i == 2 * KS ? KS : i / 2;
                sa = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[0][k], qv, sa, 0, 0, 0);
                sb = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[1][k], qv, sb, 0, 0, 0);
            }
            // 6. their powers of two, what is seen, the maximum of weight times value
            float y[8], mx = TA_NONE;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                y[i] = ldexpf(i < 4 ? sa[i] : sb[i - 4], (i < 4 ? ka[i] : kb[i - 4]) + fq[t]);
            }
            bool seen[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) seen[i] = true;
            if (edge) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int at = p0 + 8 * j + i, own = at - tr.pos0;
                    seen[i] = p.parent ? own < 0 || (own < 64 && (see[t] >> (own & 63) & 1)) : at <= lim[t];
                }
            }
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[i] = __builtin_fmaf(y[i], cs, i < 4 ? va[i] : vb[i - 4]);
                if (!seen[i]) x[i] = -__builtin_inff();
                mx = fmaxf(mx, x[i]);
            }
            mx = __builtin_ceilf(ta_swap32(ta_swap16(mx, ta_max), ta_max));
            if (__any(mx > m[t])) {
                const float to = fmaxf(m[t], mx), corr = __builtin_amdgcn_exp2f(m[t] - to);
                m[t] = to;
                l[t] *= corr;
#pragma unroll
                for (int n = 0; n <= NT; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) O[t][n][i] *= corr;
            }
            // 7. weights (2^14 of them at the maximum), two f16 terms
            const float top = m[t] - 14.0f;
            float P[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float d = __builtin_fmaf(y[i], cs, (i < 4 ? va[i] : vb[i - 4]) - top);
                P[i] = __builtin_amdgcn_exp2f(d);
                if (!seen[i]) P[i] = 0.0f;
            }
            // scores of millions: their rounding is larger than a weight's
            const bool far = fabsf(m[t]) >= 4194304.0f && m[t] > TA_NONE;
            if (__builtin_expect(__any(far), 0)) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float e = __builtin_amdgcn_exp2f((x[i] - m[t]) + 14.0f);
                    P[i] = far ? e : P[i];
                }
            }
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                l[t] = __builtin_fmaf(P[i], ia[i], l[t]);
                l[t] = __builtin_fmaf(P[i + 4], ib[i], l[t]);
                hi[i] = f16_pair(P[i], P[i + 4]);
                lo[i] = f16_pair(__builtin_fmaf(f16_low(hi[i]), -1.0f, P[i]),
                                 __builtin_fmaf(f16_high(hi[i]), -1.0f, P[i + 4]));
            }
            const f16x8 ph = __builtin_bit_cast(f16x8, u32x4{hi[0], hi[1], hi[2], hi[3]});
            const f16x8 pl = __builtin_bit_cast(f16x8, u32x4{lo[0], lo[1], lo[2], lo[3]});
            // 8. the outputs
#pragma unroll
            for (int n = 0; n <= NT; ++n) {
                O[t][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[n], ph, O[t][n], 0, 0, 0);
                O[t][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[n], pl, O[t][n], 0, 0, 0);
            }
            if (edge) {  // values that are NaN, to the queries that see them: through the middles' sums
#pragma unroll
                for (int i = 0; i < Raw::VM; ++i) {
                    for (unsigned long long left = nan_p[i]; left; left &= left - 1) {
                        const int at = __builtin_ctzll(left), pos = p0 + (at & 31), own = pos - tr.pos0;
                        const int g = NG == 1 ? 0 : (at >> 5) * (NG / 2) + i;
                        const bool hit = p.parent ? own < 0 || (own < 64 && (see[t] >> (own & 63) & 1))
                                                  : pos <= lim[t];
                        if (hit && j == g / 2) O[t][NT][0] = g % 2 ? O[t][NT][0] : __builtin_nanf("");
                        if (hit && j == g / 2) O[t][NT][2] = g % 2 ? __builtin_nanf("") : O[t][NT][2];
                    }
                }
            }
        }
    }

    // 9. the waves' results
    float *off = (float *)(lds + M::OFF) + w * ROWS * 8;
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        l[t] = ta_swap32(ta_swap16(l[t], ta_add), ta_add);
        if (2 * j < NG) off[(t * 16 + col) * 8 + 2 * j] = O[t][NT][0] + O[t][NT][1];
        if (2 * j + 1 < NG) off[(t * 16 + col) * 8 + 2 * j + 1] = O[t][NT][2] + O[t][NT][3];
    }
    __syncthreads();  // the operands are read; the results lie over them
    float *ro = (float *)(lds + M::RO) + w * ROWS * HD, *rm = (float *)(lds + M::RM);
#pragma unroll
    for (int t = 0; t < MT; ++t) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const float mid = off[(t * 16 + col) * 8 + n / 2];
            *(f32x4l *)(ro + (t * 16 + col) * HD + n * 16 + 4 * j) =
                f32x4l{O[t][n][0] + mid, O[t][n][1] + mid, O[t][n][2] + mid, O[t][n][3] + mid};
        }
        if (j == 0) {
            rm[(w * ROWS + t * 16 + col) * 2] = m[t];
            rm[(w * ROWS + t * 16 + col) * 2 + 1] = l[t];
        }
    }
    __syncthreads();
    for (int i = tid; i < rows * HD; i += 64 * TA_W) {
        const int r = i / HD, c = i % HD;
        float mx = TA_NONE, L = 0.0f, o = 0.0f;
#pragma unroll
        for (int x = 0; x < TA_W; ++x) mx = fmaxf(mx, rm[(x * ROWS + r) * 2]);
#pragma unroll
        for (int x = 0; x < TA_W; ++x) {
            const float f = __builtin_amdgcn_exp2f(rm[(x * ROWS + r) * 2] - mx);
            L = __builtin_fmaf(f, rm[(x * ROWS + r) * 2 + 1], L);
            o = __builtin_fmaf(f, ((const float *)(lds + M::RO))[(x * ROWS + r) * HD + c], o);
        }
        if (p.shares == 1) {
            const int R = row0 + r;
            p.out[((size_t)b * p.S + R / p.G) * p.ldo + ((size_t)kvh * p.G + R % p.G) * HD + c] = o * 0x1p-14f / L;
        } else {
            float *pw = p.work + (((size_t)pair * p.tiles + tile) * p.shares + share) * (ROWS * (HD + 2));
            pw[r * HD + c] = o;
            if (c == 0) {
                pw[ROWS * HD + 2 * r] = mx;
                pw[ROWS * HD + 2 * r + 1] = L;
            }
        }
    }
}

// The shares of a query, in order.
template <int HD>
__global__ __launch_bounds__(HD < 64 ? 64 : HD) void tree_merge_kernel(TreeAttnParams p, int ROWS) {
    const int r = blockIdx.x % ROWS, tile = blockIdx.x / ROWS, kvh = blockIdx.y, b = blockIdx.z, c = threadIdx.x;
    const TreeRows tr = tree_rows(p.pos0, p.count, p.parent, p.S, p.c.cap, b, p.guard, false);
    const int R = tile * ROWS + r;
    if (R >= tr.n * p.G || c >= HD) return;
    const size_t pair = (size_t)b * p.c.Hkv + kvh, ld = (size_t)ROWS * (HD + 2);
    const float *pw = p.work + (pair * p.tiles + tile) * p.shares * ld;
    float mx = TA_NONE, L = 0.0f, o = 0.0f;
    for (int s = 0; s < p.shares; ++s) mx = fmaxf(mx, pw[s * ld + ROWS * HD + 2 * r]);
    for (int s = 0; s < p.shares; ++s) {
        const float f = __builtin_amdgcn_exp2f(pw[s * ld + ROWS * HD + 2 * r] - mx);
        L = __builtin_fmaf(f, pw[s * ld + ROWS * HD + 2 * r + 1], L);
        o = __builtin_fmaf(f, pw[s * ld + r * HD + c], o);
    }
    p.out[((size_t)b * p.S + R / p.G) * p.ldo + ((size_t)kvh * p.G + R % p.G) * HD + c] = o * 0x1p-14f / L;
}

struct TreePlan {
    int mt, tiles, shares;
};
TreePlan tree_plan(const Kv4View &c, int H, int S) {
    const long long rows = (long long)S * (H / c.Hkv);
    const int most = c.hd <= 64 ? 4 : c.hd == 128 ? 2 : 1;
    TreePlan pl;
    pl.mt = rows <= 16 ? 1 : rows <= 32 ? std::min(2, most) : most;
    pl.tiles = (int)((rows + 16 * pl.mt - 1) / (16 * pl.mt));
    // workgroups for two a CU, where the capacity gives each wave of a share two blocks
    const long long streams = (long long)c.B * c.Hkv * pl.tiles;
    const long long by_length = c.cap / KV4_BLOCK / (2 * TA_W);
    pl.shares = (int)std::max(1ll, std::min(std::min(512 / streams, by_length), 64ll));
    return pl;
}

template <int HD, int MT>
int launch_t(const TreeAttnParams &p, hipStream_t st) {
    using M = TreeLds<HD, MT>;
    int rc = allow_lds((const void *)tree_attn_kernel<HD, MT>, M::SIZE, M::SIZE);
    if (rc) return rc;
    const size_t streams = (size_t)p.c.B * p.c.Hkv * p.shares;
    tree_attn_kernel<HD, MT><<<(unsigned)((streams + 7) / 8 * 8 * p.tiles), 64 * TA_W, M::SIZE, st>>>(p);
    VMLM_HIP_CHECK(hipGetLastError());
    if (p.shares == 1) return VMLM_OK;
    tree_merge_kernel<HD><<<dim3((unsigned)p.tiles * 16 * MT, (unsigned)p.c.Hkv, (unsigned)p.c.B),
                            HD < 64 ? 64 : HD, 0, st>>>(p, 16 * MT);
    VMLM_HIP_CHECK(hipGetLastError());
    return VMLM_OK;
}

template <int HD>
int launch_hd(const TreeAttnParams &p, int mt, hipStream_t st) {
    if (mt == 1) return launch_t<HD, 1>(p, st);
    if constexpr (HD <= 128) {
        if (mt == 2) return launch_t<HD, 2>(p, st);
    }
    if constexpr (HD <= 64) return launch_t<HD, 4>(p, st);
    return VMLM_OK;
}

}  // namespace

size_t tree_attn_work_floats(const Kv4View &c, int H, int S) {
    if (c.B == 0 || c.Hkv == 0 || c.cap == 0 || H == 0 || S == 0) return 0;
    const TreePlan pl = tree_plan(c, H, S);
    if (pl.shares == 1) return 0;
    return (size_t)c.B * c.Hkv * pl.tiles * pl.shares * (16 * pl.mt) * (c.hd + 2);
}

int launch_tree_attn(const TreeAttnArgs &a, hipStream_t st) {
    const TreePlan pl = tree_plan(a.c, a.H, a.S);
    TreeAttnParams p;
    p.c = a.c;
    p.q = a.q;
    p.ldq = a.ldq;
    p.ldo = a.ldo;
    p.pos0 = a.pos0;
    p.count = a.count;
    p.parent = a.parent;
    p.S = a.S;
    p.H = a.H;
    p.G = a.H / a.c.Hkv;
    p.tiles = pl.tiles;
    p.shares = pl.shares;
    p.out = a.out;
    p.work = a.work;
    p.scale = frexpf(a.scale, &p.scale_e) * 1.44269504f;
    p.guard = guard_flag_ptr();
    VMLM_GUARD(p.shares == 1 || p.work, "kv4 tree attention: split positions need a workspace");
    switch (a.c.hd) {
    case 32: return launch_hd<32>(p, pl.mt, st);
    case 64: return launch_hd<64>(p, pl.mt, st);
    case 128: return launch_hd<128>(p, pl.mt, st);
    default: return launch_hd<256>(p, pl.mt, st);
    }
}

}  // namespace vmlm
