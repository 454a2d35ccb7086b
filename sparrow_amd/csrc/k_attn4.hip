// k_attn4.hip -- decode attention over the 4-bit KV cache
// (vmlm_hip_attention_decode_kv4); the format is in kv4.hpp.
//
// For each head, s_p = scale * q . k_p over positions 0 .. pos and
// o = sum_p exp(s_p - m) v_p / sum_p exp(s_p - m).
//
// Bound by the cache's bytes: 5 bits a value, read once for all query heads of a
// group. What keeps the arithmetic out of the way is that both products run on int8
// matrix instructions over the nibbles as they lie:
//  * A nibble in the high half of a byte is 16 (u - 8) as a signed byte, so a
//    16-byte load becomes two int8 operands (low and high nibbles) with 12
//    operations. q, and for the output the weights times V's scale, are 31-bit fixed-point
//    numbers below the largest of their group (32 channels of q, a chunk's positions
//    for the weights), as four signed bytes: with 16 (u - 8) every product and sum is
//    exact in int32, and two conversions and an FMA put the terms together. 32-bit
//    sums, then, at 8-bit rates. (Three bytes left the many small weights 2^-22 of the
//    largest: 1.4e-6 off where f32 sums are 4e-7.)
//  * Scores: a wave takes 128 positions. Lane (row kb, column n) loads the 32
//    channels of group kb mod NG at one position. The A operand has a row (j, t) for
//    each kb = j and term t that is zero outside kb = j, so D's rows 4 kb + t at column n
//    -- the registers of that very lane -- hold its own 32 channels' product, and
//    the lane applies the scale and minimum that it loaded beside them. The groups of a
//    position meet by lane swaps that leave each position's sum, and its exponential,
//    to one lane.
//  * Output: o[c] = sum_p (P_p scale_p,g) 16 (u - 8) / 16 + sum_p P_p (min + 8 scale)_p,g.
//    The lanes that hold (p, g) write P_p scale_p,g as four bytes to LDS, from where
//    they are the A operand (rows: head, term) against V's nibbles, which lie along
//    positions; the second sum is a lane's own.
//  * The maximum and sum of the softmax run along in the wave; the waves of a
//    workgroup meet in LDS, the workgroups of a split head in a second launch.
// The new token's row is quantised by the wave that holds its position, put into
// its registers and stored from there: no read back, no second launch.
//
// Measured (kernel times; a large copy moves 5.1 TB/s): 65500 positions of 36 heads of 64,
// one sequence, 39 us, 4.8 TB/s, and 4.7 us of merging; 8 sequences of up to 16000 with 8 kv
// heads of 128 and 4 queries each 36 us, 3.3 TB/s: there the softmax and the bytes of
// 4 queries' weights keep the vector units as busy as the memory, at two waves a SIMD.
// 1024 positions: 7.0 us, a launch and a few latencies.
#include <algorithm>

#include "kv4.hpp"

namespace vmlm {
namespace {

typedef float f32x4a __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x4m __attribute__((ext_vector_type(4), aligned(4)));
typedef __attribute__((__vector_size__(4 * sizeof(int)))) int i32x4;

// Positions of a wave at a time: what the registers hold. (64 for heads of 128 too, more
// waves at once: 36.0 us instead of 34.3, then, for 8 sequences of 16000 with 4 queries a kv head.)
constexpr int attn4_ch(int hd) { return hd <= 128 ? 128 : 64; }
// The maximum of no score yet, or of scores that all left f32 downwards: finite, so that
// its distance from itself is none (not -inf - -inf).
constexpr float A4_NONE = -3.40282347e38f;
constexpr int A4_MAX_GH = 4;   // query heads of a workgroup (rows of the A operand / 4)
constexpr int A4_MAX_W = 8;    // waves of a workgroup
constexpr int A4_MAX_SPLIT = 64;  // shares of a sequence

struct Attn4Params {
    Kv4View c;
    const float *q, *k_new, *v_new;
    size_t ldq, ldkv, ldo;
    const int32_t *pos;
    float *out, *work;
    int H, G, ch, W;
    int shares;  // of a split launch (0: one workgroup a pair of head and sequence)
    int parts;  // workgroups that share a kv head's queries
    float scale;  // of the scores: scale * 2^scale_e, |scale| in [1/2, 1)
    int scale_e;
    int *guard;
};

__device__ __forceinline__ float swap16(float v, float (*f)(float, float)) {
    const auto t = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                    false);
    return f(__uint_as_float(t[0]), __uint_as_float(t[1]));
}
__device__ __forceinline__ float swap32(float v, float (*f)(float, float)) {
    const auto t = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                    false);
    return f(__uint_as_float(t[0]), __uint_as_float(t[1]));
}
// log2(e) multiplies scores' distances from the maximum: in the score scale it would
// round at a score's own magnitude, 2^-10 of a weight at scores of 16000.
__device__ __forceinline__ float a4_exp(float x) {
    return __builtin_amdgcn_exp2f(x * 1.44269504f);
}
__device__ __forceinline__ float add_f(float a, float b) { return a + b; }
__device__ __forceinline__ float max_f(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ float row16_max(float v) {
    v = fmaxf(v, dpp_mov<0xB1>(v));
    v = fmaxf(v, dpp_mov<0x4E>(v));
    v = fmaxf(v, dpp_mov<0x124>(v));
    return fmaxf(v, dpp_mov<0x128>(v));
}
__device__ __forceinline__ float row16_sum(float v) {
    v += dpp_mov<0xB1>(v);
    v += dpp_mov<0x4E>(v);
    v += dpp_mov<0x124>(v);
    return v + dpp_mov<0x128>(v);
}
// over the rows of lanes that hold other positions of the same group
template <int GR>
__device__ __forceinline__ float rows_red(float v, float (*f)(float, float)) {
    if (GR == 1) v = swap16(v, f);
    if (GR <= 2) v = swap32(v, f);
    return v;
}

__device__ __forceinline__ i32x4 nib_lo(u32x4 w) {
    return __builtin_bit_cast(i32x4, (w << 4) & 0xf0f0f0f0u);
}
__device__ __forceinline__ i32x4 nib_hi(u32x4 w) {
    return __builtin_bit_cast(i32x4, w & 0xf0f0f0f0u);
}
// Sums of an integer's four bytes, highest first, put together again.
__device__ __forceinline__ float undigits(const i32x4 &d) {
    // each is below 2^22: two of them fit an int32
    return __builtin_fmaf((float)(d[0] * 256 + d[1]), 65536.0f, (float)(d[2] * 256 + d[3]));
}
// The power of two that brings values up to mx below 2^30 (0 for none).
__device__ __forceinline__ int fixed_exp(float mx) {
    return mx > 0.0f && mx <= 3.40282347e38f ? 29 - ilogbf(mx) : 0;
}

// A lane's V codes of one channel: CH / 4 positions, and their product with the
// weights' bytes.
template <int CH>
struct VCodes {  // 128: 32 positions, low nibbles (even ones), then high ones
    u32x4 w;
    __device__ __forceinline__ void load(const uint8_t *v) { w = *(const u32x4 *)v; }
    __device__ __forceinline__ i32x4 product(const uint8_t *a) const {
        i32x4 d = {0, 0, 0, 0};
        d = __builtin_amdgcn_mfma_i32_16x16x64_i8(*(const i32x4 *)a, nib_lo(w), d, 0, 0, 0);
        return __builtin_amdgcn_mfma_i32_16x16x64_i8(*(const i32x4 *)(a + 64), nib_hi(w), d, 0, 0, 0);
    }
};
typedef __attribute__((__vector_size__(2 * sizeof(uint32_t)))) uint32_t u32x2;
template <>
struct VCodes<64> {  // 16 positions: both nibbles in one operand
    u32x2 w;
    __device__ __forceinline__ void load(const uint8_t *v) { w = *(const u32x2 *)v; }
    __device__ __forceinline__ i32x4 product(const uint8_t *a) const {
        const u32x2 lo = (w << 4) & 0xf0f0f0f0u, hi = w & 0xf0f0f0f0u;
        const u32x4 v = {lo[0], lo[1], hi[0], hi[1]};
        return __builtin_amdgcn_mfma_i32_16x16x64_i8(*(const i32x4 *)a, __builtin_bit_cast(i32x4, v),
                                                     i32x4{0, 0, 0, 0}, 0, 0, 0);
    }
};

// Sums over the GR rows of lanes that hold a position's groups; of each GR steps a
// row keeps its own (GR = 4: row kb of step 4 j + kb; 2: row g of step 2 j + g).
template <int GR, int NS>
__device__ __forceinline__ void sum_groups(const float (&x)[NS], float (&s)[NS / GR]) {
    auto pair16 = [](float a, float b) {
        const auto t = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false,
                                                        false);
        return __uint_as_float(t[0]) + __uint_as_float(t[1]);
    };
    auto pair32 = [](float a, float b) {
        const auto t = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false,
                                                        false);
        return __uint_as_float(t[0]) + __uint_as_float(t[1]);
    };
#pragma unroll
    for (int j = 0; j < NS / GR; ++j) {
        if constexpr (GR == 4)
            s[j] = pair16(pair32(x[4 * j], x[4 * j + 2]), pair32(x[4 * j + 1], x[4 * j + 3]));
        else if constexpr (GR == 2)
            s[j] = pair16(x[2 * j], x[2 * j + 1]);
        else
            s[j] = x[j];
    }
}
// The way back: every step's value in all of its rows.
template <int GR, int NO, int NS>
__device__ __forceinline__ void to_groups(const float (&s)[NO], float (&x)[NS]) {
#pragma unroll
    for (int j = 0; j < NO; ++j) {
        const uint32_t v = __float_as_uint(s[j]);
        if constexpr (GR == 4) {
            const auto t = __builtin_amdgcn_permlane32_swap(v, v, false, false);
            const auto a = __builtin_amdgcn_permlane16_swap(t[0], t[0], false, false);
            const auto b = __builtin_amdgcn_permlane16_swap(t[1], t[1], false, false);
            x[4 * j] = __uint_as_float(a[0]);
            x[4 * j + 1] = __uint_as_float(a[1]);
            x[4 * j + 2] = __uint_as_float(b[0]);
            x[4 * j + 3] = __uint_as_float(b[1]);
        } else if constexpr (GR == 2) {
            const auto t = __builtin_amdgcn_permlane16_swap(v, v, false, false);
            x[2 * j] = __uint_as_float(t[0]);
            x[2 * j + 1] = __uint_as_float(t[1]);
        } else {
            x[j] = s[j];
        }
    }
}

// 4 x 4 dwords transposed over the four rows of lanes: r[i] of row k becomes r[k] of row i.
__device__ __forceinline__ void transpose_rows(uint32_t (&r)[4]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const auto t = __builtin_amdgcn_permlane32_swap(r[i], r[i + 2], false, false);
        r[i] = t[0];
        r[i + 2] = t[1];
    }
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
        const auto t = __builtin_amdgcn_permlane16_swap(r[i], r[i + 1], false, false);
        r[i] = t[0];
        r[i + 1] = t[1];
    }
}

// The meta dwords of the lane's positions: 16 bytes a load, its neighbours in the
// other rows of lanes given theirs by a transpose when they are used (it waits for
// the loads). Past `pos`: of positions up to it.
template <int HD, int NS, int GL>
struct Meta {
    static constexpr int NG = HD / 32, PN = attn4_ch(HD) / 16, L = NG == 1 ? NS : NS * GL / 4;
    uint32_t raw[L][NG == 1 ? 1 : 4];
    __device__ __forceinline__ void load(const uint32_t *m, int p0, int n, int kb, int pos) {
#pragma unroll
        for (int s = 0; s < L; ++s) {
            if constexpr (NG == 1) {
                raw[s][0] = m[min(p0 + n * PN + 2 * ((kb >> 1) * NS + s) + (kb & 1), pos)];
            } else {
                // row kb loads what step kb (of each parity, HD = 128; of each half, 256) needs
                size_t at;
                if (NG == 2)
                    at = (size_t)min(p0 + n * PN + 2 * kb, pos & ~1) * 2;  // both parities' groups
                else if (NG == 4)
                    at = (size_t)min(p0 + n * PN + 2 * kb + s, pos) * 4;
                else
                    at = (size_t)min(p0 + n * PN + 2 * (kb & 1) + (kb >> 1), pos) * 8 + 4 * s;
                const u32x4m v = *(const u32x4m *)(m + at);
#pragma unroll
                for (int i = 0; i < 4; ++i) raw[s][i] = v[i];
            }
        }
    }
    __device__ __forceinline__ void spread(uint32_t (&out)[NS][GL]) {
#pragma unroll
        for (int s = 0; s < L; ++s) {
            if constexpr (NG == 1) {
                out[s][0] = raw[s][0];
            } else {
                transpose_rows(raw[s]);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (NG == 8)
                        out[i][s] = raw[s][i];
                    else
                        out[s * 4 + i][0] = raw[s][i];
                }
            }
        }
    }
};

// The bytes of the lane's weights into the terms (highest first, TB bytes each).
template <int HD, int NS>
__device__ __forceinline__ void store_terms(uint8_t *o, int n, int kb, const uint32_t (&d)[NS]) {
    constexpr int TB = attn4_ch(HD);
    if constexpr (HD == 64 || HD == 128) {  // four of one parity
#pragma unroll
        for (int s = 0; s < NS / 4; ++s) {
            uint32_t t[4];
            transpose_bytes({d[s * 4], d[s * 4 + 1], d[s * 4 + 2], d[s * 4 + 3]}, t);
            uint8_t *at = o + (HD == 128 ? s : kb >> 1) * 64 + n * 4;
#pragma unroll
            for (int k = 0; k < 4; ++k) *(uint32_t *)(at + k * TB) = t[3 - k];
        }
    } else {  // two
#pragma unroll
        for (int s = 0; s < NS / 2; ++s) {
            const uint32_t a = __builtin_amdgcn_perm(d[s * 2 + 1], d[s * 2], 0x07030602u);
            const uint32_t b = __builtin_amdgcn_perm(d[s * 2 + 1], d[s * 2], 0x05010400u);
            uint8_t *at = HD == 32 ? o + (kb & 1) * 64 + n * 4 + (kb >> 1) * 2
                                   : o + (n >> 2) * 16 + s * 8 + (n & 3) * 2;
            *(uint16_t *)at = (uint16_t)(a >> 16);
            *(uint16_t *)(at + TB) = (uint16_t)a;
            *(uint16_t *)(at + 2 * TB) = (uint16_t)(b >> 16);
            *(uint16_t *)(at + 3 * TB) = (uint16_t)b;
        }
    }
}

// Shares of a split launch. The positions are known on the device alone and differ
// between sequences: every workgroup works out from all of them how many chunks a share
// takes so that about `shares` of them cover all sequences, and which one is its own.
// A sequence has one share for every `each` chunks, at most A4_MAX_SPLIT.
struct Shares {
    int each;
    int b, pos, count, first;  // a sequence, its shares and the number of the first
};
__device__ __forceinline__ int chunks_of(const Attn4Params &p, int b, int *pos) {
    *pos = b < p.c.B ? p.pos[b] : -1;
    if (*pos >= p.c.cap) {
        atomicOr(p.guard, 1);
        return 0;
    }
    return *pos < 0 ? 0 : *pos / p.ch + 1;
}
// The sequence of share number `at`, or (want_b >= 0) that sequence; count 0: there is none.
// Called by whole waves.
__device__ __forceinline__ Shares shares_of(const Attn4Params &p, int at, int want_b) {
    const int lane = threadIdx.x & 63;
    int pos;
    float all = 0.0f, most = 0.0f;
    for (int b0 = 0; b0 < p.c.B; b0 += 64) {
        const float n = (float)chunks_of(p, b0 + lane, &pos);
        all += wave_sum_dpp(n);
        most = fmaxf(most, wave_max_nonneg(n));
    }
    Shares r;
    const int want = max((int)ceilf(all / (float)p.shares), (int)ceilf(most / A4_MAX_SPLIT));
    r.each = __builtin_amdgcn_readfirstlane(max(1, (want + p.W - 1) / p.W)) * p.W;
    r.count = 0;
    int before = 0;
    for (int b0 = 0; b0 < p.c.B; b0 += 64) {
        const int n = chunks_of(p, b0 + lane, &pos), mine = (n + r.each - 1) / r.each;
        int to = mine;  // shares up to this lane's sequence
#pragma unroll
        for (int o = 1; o < 64; o *= 2) {
            const int v = __shfl_up(to, o, 64);
            to += lane >= o ? v : 0;
        }
        const unsigned long long hit =
            __ballot(want_b >= 0 ? b0 + lane == want_b : before + to > at);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            r.b = b0 + l;
            r.pos = __builtin_amdgcn_readlane(pos, l);
            r.count = __builtin_amdgcn_readlane(mine, l);
            r.first = before + __builtin_amdgcn_readlane(to, l) - r.count;
            return r;
        }
        before += __builtin_amdgcn_readlane(to, 63);
    }
    return r;
}

// LDS of a workgroup: the query terms [head][term][group][32], zeros, the heads' powers of two,
// a factor and a sum for each head and group, the new token's codes and meta, a number for each wave, head and group (the weight
// terms' power of two, then the V offset), and one region
// that holds the waves' weight terms, then their results.
template <int HD, int HEADS>
struct Lds {
    static constexpr int NG = HD / 32;
    static constexpr int Q = 0;
    static constexpr int Z = Q + HEADS * 4 * HD;  // as many zeros
    static constexpr int F = Z + HEADS * 4 * HD;
    static constexpr int S = F + HEADS * 4;
    static constexpr int NK = (S + HEADS * NG * 8 + 15) / 16 * 16;
    static constexpr int NV = NK + HD / 2;
    static constexpr int NM = NV + HD;
    static constexpr int OFF = NM + 2 * NG * 4;
    static constexpr int R0 = OFF + A4_MAX_W * HEADS * NG * 4;
    static constexpr int R = (R0 + 15) / 16 * 16;
};

// GH query heads of one kv head.
template <int HD, int GH>
__global__ __launch_bounds__(64 * A4_MAX_W) void attn4_kernel(Attn4Params p) {
    constexpr int NG = HD / 32, GR = NG < 4 ? NG : 4, GL = NG / GR;
    constexpr int CH = attn4_ch(HD), PN = CH / 16, NS = PN * GR / 4, CT = HD / 16;
    constexpr int TB = CH;  // bytes of a term
    using M = Lds<HD, GH>;
    extern __shared__ __align__(16) uint8_t lds[];
    const int tid = threadIdx.x, w = tid >> 6, W = blockDim.x >> 6, lane = tid & 63;
    const int kb = lane >> 4, n = lane & 15, g0 = kb % GR;
    // The parts of a kv head lie 8 workgroups apart: on one XCD, whose L2 then gives the
    // later ones the cache. (Single ones go round the XCDs: 36 heads bound to them are
    // five on four of them.)
    int kvh = blockIdx.x, part = 0;
    if (p.parts > 1) {
        const int x8 = blockIdx.x / 8;
        kvh = x8 / p.parts * 8 + (int)(blockIdx.x % 8);
        part = x8 % p.parts;
    }
    if (kvh >= p.c.Hkv) return;
    const int h0 = part * GH, G = min(GH, p.G - h0);  // of the kv head's queries
    int b = blockIdx.y, pos = 0, c0 = 0, c1 = 0, count = 1;
    if (p.shares) {
        const Shares sh = shares_of(p, blockIdx.y, -1);
        if (sh.count == 0) return;
        const int n = sh.pos / CH + 1, s = (int)blockIdx.y - sh.first;
        b = sh.b;
        pos = sh.pos;
        count = sh.count;
        c0 = (int)((long long)s * n / count);
        c1 = (int)((long long)(s + 1) * n / count);
    } else {
        pos = p.pos[b];
        if (pos < 0) return;  // an idle sequence
        if (pos >= p.c.cap) {
            if (tid == 0 && blockIdx.x == 0) atomicOr(p.guard, 1);
            return;
        }
        c1 = pos / CH + 1;
    }
    const size_t head = (size_t)b * p.c.Hkv + kvh, row0 = head * p.c.cap;
    const int last = pos / CH;

    // 1. the new token's codes, by the wave that will put them in place; the query heads as
    // fixed-point terms
    if (p.k_new && last < c1 && (last - c0) % W == w) {
        uint32_t *nm = (uint32_t *)(lds + M::NM);
        const int c4 = min(lane, HD / 4 - 1) * 4;
        const size_t at = b * p.ldkv + (size_t)kvh * HD + c4;
        const f32x4a rk = *(const f32x4a *)(p.k_new + at), rv = *(const f32x4a *)(p.v_new + at);
        const float k[4] = {rk[0], rk[1], rk[2], rk[3]}, v[4] = {rv[0], rv[1], rv[2], rv[3]};
        const uint32_t mk = kv4_meta8(k), mv = kv4_meta8(v);
        uint32_t ck[4], cv[4];
        kv4_codes(k, mk, ck);
        kv4_codes(v, mv, cv);
        if (lane < HD / 4) {
            *(uint16_t *)(lds + M::NK + c4 / 2) = kv4_nibbles(ck);
            *(uint32_t *)(lds + M::NV + c4) = kv4_bytes(cv);
            if ((lane & 7) == 0) {
                nm[lane / 8] = mk;
                nm[NG + lane / 8] = mv;
            }
        }
    }
    for (int i = tid; i < GH * HD / 4; i += W * 64) ((u32x4 *)(lds + M::Z))[i] = u32x4{0, 0, 0, 0};
    int *qe = (int *)(lds + M::F);
    float *qs = (float *)(lds + M::S);
    for (int h = w; h < GH; h += W) {
        const float *q = p.q + b * p.ldq + ((size_t)kvh * p.G + h0 + min(h, G - 1)) * HD;
        constexpr int CL = (HD + 63) / 64;
        float x[CL], mx[CL], most = 0.0f;
        int bad = 0;
#pragma unroll
        for (int i = 0; i < CL; ++i) {
            const int c = i * 64 + lane;
            x[i] = c < HD ? q[c] : 0.0f;
            mx[i] = swap16(row16_max(fabsf(x[i])), max_f);  // of its 32 channels
            most = fmaxf(most, mx[i]);
            bad |= !(fabsf(x[i]) <= 3.40282347e38f);
        }
        most = swap32(most, max_f);
        bad = __any(bad);
        // Each group's fixed point lies below its own largest value: keys may be small just
        // where queries are large. The sums come in units that keep them below 2^-5 of the
        // largest key value (2^eh takes them back): no step between leaves f32.
        const int eh = bad || most == 0.0f ? 0 : ilogbf(most) + 14;
#pragma unroll
        for (int i = 0; i < CL; ++i) {
            const int c = i * 64 + lane, e = fixed_exp(mx[i]);
            const int f = bad ? 0 : (int)rintf(ldexpf(x[i], e));
            const float s = swap16(row16_sum((float)f), add_f);
            if (c >= HD) continue;
            const uint32_t d = signed_bytes(f);
            uint8_t *t = lds + M::Q + ((h * 4) * NG + c / 32) * 32 + (c & 1) * 16 + c % 32 / 2;
#pragma unroll
            for (int k = 0; k < 4; ++k) t[k * NG * 32] = (uint8_t)(d >> (24 - 8 * k));
            if ((c & 31) == 0) {
                float *o = qs + (h * NG + c / 32) * 2;
                o[0] = mx[i] > 0.0f && !bad ? ldexpf(1.0f, -4 - e - eh) : 0.0f;
                o[1] = bad ? __builtin_nanf("") : ldexpf(s, -e - eh);
            }
        }
        if (lane == 0) qe[h] = eh + p.scale_e;
    }
    __syncthreads();

    // the A operand of head h: row (j, t), nonzero where kb = j
    const int term = n & 3;
    const uint8_t *qt = lds + (n >> 2 == kb ? M::Q + (term * NG + g0) * 32 : M::Z);
    auto qa = [&](int h, int e, int par) {
        return *(const i32x4 *)(qt + (h * 4 * NG + 4 * e) * 32 + par * 16);
    };
    // Column n of the scores is PN neighbouring positions, and the lane's are NS of them,
    // of one parity (or, with a group each for the four kb, first the even ones, then the
    // odd ones): their bytes lie side by side in the weights' terms.
    auto place = [&](int i) {
        if (GR == 4) return n * PN + 2 * (i % (PN / 2)) + i / (PN / 2);
        if (GR == 2) return n * PN + 2 * i + (kb >> 1);
        return n * PN + 2 * ((kb >> 1) * NS + i) + (kb & 1);
    };
    // the positions whose score is summed here (sum_groups)
    auto own_place = [&](int j) {
        if (GR == 4) return n * PN + 2 * ((j * 4 + kb) % (PN / 2)) + (j * 4 + kb) / (PN / 2);
        if (GR == 2) return n * PN + 2 * (j * 2 + (kb & 1)) + (kb >> 1);
        return place(j);
    };

    // the new token's meta, from LDS, in the lanes that hold its position
    auto new_meta = [&](uint32_t (&m)[NS][GL], int at) {
        const uint32_t *nm = (const uint32_t *)(lds + M::NM) + at;
#pragma unroll
        for (int i = 0; i < NS; ++i)
#pragma unroll
            for (int e = 0; e < GL; ++e)
                if (last * CH + place(i) == pos) m[i][e] = nm[g0 + 4 * e];
    };

    float m[GH], l[GH], off[GH][GL], O[CT];
#pragma unroll
    for (int h = 0; h < GH; ++h) {
        m[h] = A4_NONE;
        l[h] = 0.0f;
#pragma unroll
        for (int e = 0; e < GL; ++e) off[h][e] = 0.0f;
    }
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) O[ct] = 0.0f;
    uint8_t *pb = lds + M::R + w * (GH * NG * 4 * TB);
    int *ex = (int *)(lds + M::OFF) + w * GH * NG;  // the terms' powers of two; in the end V offsets

    for (int ch = c0 + w; ch < c1; ch += W) {
        const int p0 = ch * CH;
        // 2. everything of the CH positions; past the last one, that one again. (K a chunk
        // ahead gained nothing: the loads of the CU's other waves fill the time.)
        u32x4 kc[NS][GL];
        Meta<HD, NS, GL> kmeta, vmeta;
        VCodes<CH> vc[CT];
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            const size_t row = row0 + min(p0 + place(i), pos);
#pragma unroll
            for (int e = 0; e < GL; ++e)
                kc[i][e] = *(const u32x4 *)(p.c.k + row * (HD / 2) + (g0 + 4 * e) * 16);
        }
        kmeta.load(p.c.km + row0 * NG, p0, n, kb, pos);
        // lane (kb, n): the kb-th quarter of the positions, channel 16 ct + n
        const int vblk = min((p0 + kb * (CH / 4)) / KV4_BLOCK, pos / KV4_BLOCK);
        uint8_t *vb = p.c.v + ((head * (p.c.cap / KV4_BLOCK) + vblk) * HD + n) * 16 +
                      (CH == 128 ? 0 : (kb & 1) * 8);
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) vc[ct].load(vb + ct * 256);
        vmeta.load(p.c.vm + row0 * NG, p0, n, kb, pos);

        const bool put = p.k_new && ch == last;
        if (put) {  // 3. the new token: put in place and stored
            const uint32_t *nm = (const uint32_t *)(lds + M::NM);
#pragma unroll
            for (int i = 0; i < NS; ++i) {
                if (p0 + place(i) != pos) continue;
#pragma unroll
                for (int e = 0; e < GL; ++e) {
                    const int g = g0 + 4 * e;
                    const size_t row = row0 + pos;
                    kc[i][e] = *(const u32x4 *)(lds + M::NK + g * 16);
                    if (part) continue;
                    *(u32x4 *)(p.c.k + row * (HD / 2) + g * 16) = kc[i][e];
                    p.c.km[row * NG + g] = nm[g];
                    p.c.vm[row * NG + g] = nm[NG + g];
                }
            }
            if ((p0 + kb * (CH / 4)) / (CH / 4) == pos / (CH / 4)) {
                const int d = pos % (CH / 4) / 8, sh = pos % 8 * 4;
#pragma unroll
                for (int ct = 0; ct < CT; ++ct) {
                    const uint32_t nib = (uint32_t)lds[M::NV + ct * 16 + n] << sh;
#pragma unroll
                    for (int x = 0; x < CH / 32; ++x)
                        if (x == d) {
                            vc[ct].w[x] = (vc[ct].w[x] & ~(15u << sh)) | nib;
                            if (part == 0) *(uint32_t *)(vb + ct * 256 + x * 4) = vc[ct].w[x];
                        }
                }
            }
        }

        // 4. scores, each position's in one of the lanes that hold it
        float s[GH][NS / GR];
        {
            uint32_t km[NS][GL];
            kmeta.spread(km);
            if (put) new_meta(km, 0);
            float ks[NS][GL], ko[NS][GL];
#pragma unroll
            for (int i = 0; i < NS; ++i)
#pragma unroll
                for (int e = 0; e < GL; ++e) {
                    ks[i][e] = kv4_scale(km[i][e]);
                    ko[i][e] = __builtin_fmaf(8.0f, ks[i][e], kv4_min(km[i][e]));
                }
#pragma unroll
            for (int h = 0; h < GH; ++h) {
                float part_s[NS], unit[GL], sum[GL];
#pragma unroll
                for (int e = 0; e < GL; ++e) {
                    const float *o = qs + (h * NG + g0 + 4 * e) * 2;
                    unit[e] = o[0];
                    sum[e] = o[1];
                }
#pragma unroll
                for (int i = 0; i < NS; ++i) {
                    part_s[i] = 0.0f;
#pragma unroll
                    for (int e = 0; e < GL; ++e) {
                        i32x4 d = {0, 0, 0, 0};
                        d = __builtin_amdgcn_mfma_i32_16x16x64_i8(qa(h, e, 0), nib_lo(kc[i][e]), d, 0, 0, 0);
                        d = __builtin_amdgcn_mfma_i32_16x16x64_i8(qa(h, e, 1), nib_hi(kc[i][e]), d, 0, 0, 0);
                        part_s[i] = __builtin_fmaf(ko[i][e], sum[e], part_s[i]);
                        part_s[i] = __builtin_fmaf(undigits(d) * unit[e], ks[i][e], part_s[i]);
                    }
                }
                sum_groups<GR>(part_s, s[h]);
            }
        }

        uint32_t vm[NS][GL];
        vmeta.spread(vm);
        if (put) new_meta(vm, NG);
        // 5. V's scales and middles (none past the last position)
        float vs[NS][GL], vo[NS][GL];
#pragma unroll
        for (int e = 0; e < GL; ++e)
#pragma unroll
            for (int i = 0; i < NS; ++i) {
                const bool in = p0 + place(i) <= pos;
                vs[i][e] = in ? kv4_scale(vm[i][e]) : 0.0f;
                vo[i][e] = in ? __builtin_fmaf(8.0f, vs[i][e], kv4_min(vm[i][e])) : 0.0f;
            }

        float corr[GH];
#pragma unroll
        for (int h = 0; h < GH; ++h) {
            // 6. the running maximum, the weights and their bytes
            float mx = m[h];
#pragma unroll
            for (int j = 0; j < NS / GR; ++j) {
                s[h][j] = p0 + own_place(j) <= pos ? ldexpf(s[h][j] * p.scale, qe[h])
                                                   : -__builtin_inff();
                mx = fmaxf(mx, s[h][j]);
            }
            mx = swap32(swap16(row16_max(mx), max_f), max_f);
            corr[h] = a4_exp(m[h] - mx);
            m[h] = mx;
            l[h] *= corr[h];
#pragma unroll
            for (int j = 0; j < NS / GR; ++j) {
                s[h][j] = a4_exp(s[h][j] - mx);
                l[h] += s[h][j];
            }
            float P[NS];
            to_groups<GR>(s[h], P);
#pragma unroll
            for (int e = 0; e < GL; ++e) {
                off[h][e] *= corr[h];
                // The fixed point lies below the largest weight times scale, not below the
                // largest scale: a value row that stands out and is not attended would take
                // the others' bits.
                float wt[NS], mw = 0.0f;
#pragma unroll
                for (int i = 0; i < NS; ++i) {
                    off[h][e] = __builtin_fmaf(P[i], vo[i][e], off[h][e]);
                    wt[i] = P[i] * vs[i][e];
                    mw = fmaxf(mw, wt[i]);
                }
                const int ev = fixed_exp(rows_red<GR>(row16_max(mw), max_f));
                if (n == 0 && kb < GR) ex[h * NG + kb + 4 * e] = ev;
                // (the power of two of a product below 2^-98 is no f32)
                if (__any(ev > 127)) {
#pragma unroll
                    for (int i = 0; i < NS; ++i) wt[i] = ldexpf(wt[i], max(ev - 127, 0));
                }
                const float up = ldexpf(1.0f, min(ev, 127));
                uint32_t d[NS];
#pragma unroll
                for (int i = 0; i < NS; ++i) {
                    // signed_bytes of the product (below 2^30), the sum rounded to an integer
                    // (or to f32's 24 bits)
                    d[i] = (uint32_t)__builtin_fmaf(wt[i], up, (float)0x808080) ^ 0x808080u;
                }
                store_terms<HD>(pb + (h * NG + g0 + 4 * e) * 4 * TB, n, kb, d);
            }
        }
        __builtin_amdgcn_wave_barrier();
        // 7. the output's product over the positions
        float cq = corr[0];
#pragma unroll
        for (int h = 1; h < GH; ++h) cq = kb == h ? corr[h] : cq;
        const int hq = min(n >> 2, GH - 1), hd4 = min(kb, GH - 1);
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
            const int g = ct / 2;
            const i32x4 d = vc[ct].product(pb + ((hq * NG + g) * 4 + term) * TB + kb * 16);
            O[ct] = __builtin_fmaf(O[ct], cq, ldexpf(undigits(d), -4 - ex[hd4 * NG + g]));
        }
        __builtin_amdgcn_wave_barrier();
    }

    // 8. the waves' results
#pragma unroll
    for (int h = 0; h < GH; ++h) {
        l[h] = rows_red<1>(row16_sum(l[h]), add_f);
#pragma unroll
        for (int e = 0; e < GL; ++e) {
            const float o = rows_red<GR>(row16_sum(off[h][e]), add_f);
            if (n == 0 && kb < GR) ex[h * NG + kb + 4 * e] = __float_as_int(o);
        }
    }
    __syncthreads();  // the weights' bytes are read; the region is the results' now
    float *mo = (float *)(lds + M::R), *ml = mo + W * GH * HD;
    if (kb < G) {
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
            mo[(w * GH + kb) * HD + ct * 16 + n] = O[ct] + __int_as_float(ex[kb * NG + ct / 2]);
    }
#pragma unroll
    for (int h = 0; h < GH; ++h)
        if (lane == 0) {
            ml[(w * GH + h) * 2] = m[h];
            ml[(w * GH + h) * 2 + 1] = l[h];
        }
    __syncthreads();
    for (int i = tid; i < G * HD; i += blockDim.x) {
        const int h = i / HD, c = i % HD;
        float mx = A4_NONE, L = 0.0f, o = 0.0f;
        for (int x = 0; x < W; ++x) mx = fmaxf(mx, ml[(x * GH + h) * 2]);
        for (int x = 0; x < W; ++x) {
            const float f = a4_exp(ml[(x * GH + h) * 2] - mx);
            L = __builtin_fmaf(f, ml[(x * GH + h) * 2 + 1], L);
            o = __builtin_fmaf(f, mo[(x * GH + h) * HD + c], o);
        }
        if (count == 1) {
            p.out[b * p.ldo + ((size_t)kvh * p.G + h0 + h) * HD + c] = o / L;
        } else {
            float *pw = p.work + ((size_t)blockIdx.y * p.H + (size_t)kvh * p.G + h0 + h) * (HD + 4);
            pw[c] = o;
            if (c == 0) {
                pw[HD] = mx;
                pw[HD + 1] = L;
            }
        }
    }
}

// The shares of a head, in order: the lanes of the first wave take one's maximum and sum
// each, the threads eight of their rows at a time.
__global__ __launch_bounds__(KV4_MAX_HD) void attn4_merge_kernel(Attn4Params p) {
    __shared__ float weight[A4_MAX_SPLIT], sum;
    const int h = blockIdx.x, c = threadIdx.x, hd = p.c.hd;
    const Shares sh = shares_of(p, 0, blockIdx.y);
    const int live = sh.count, b = sh.b;
    if (live <= 1) return;  // idle, or written already
    const size_t ld = (size_t)p.H * (hd + 4);
    const float *pw = p.work + (size_t)sh.first * ld + (size_t)h * (hd + 4);
    const int cc = min(c, hd - 1);
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = pw[min(i, live - 1) * ld + cc];
    if (c < 64) {
        const int s = min(c, live - 1);
        const float m = pw[s * ld + hd], l = pw[s * ld + hd + 1];
        const float mx = swap32(swap16(row16_max(m), max_f), max_f);
        const float e = a4_exp(m - mx), f = c < live ? e : 0.0f;
        weight[c] = f;
        const float t = wave_sum_dpp(c < live ? f * l : 0.0f);
        if (c == 0) sum = t;
    }
    __syncthreads();
    if (c >= hd) return;
    float o = 0.0f;
    for (int s = 0; s < live; s += 8) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            o = s + i < live ? __builtin_fmaf(weight[s + i], x[i], o) : o;
        if (s + 8 >= live) break;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = pw[min(s + 8 + i, live - 1) * ld + c];
    }
    p.out[b * p.ldo + (size_t)h * hd + c] = o / sum;
}

// Where the sequences can be long and the pairs of head and sequence are fewer than
// the workgroups that the chip holds, the pairs are split into about as many shares: 512
// of eight waves where a wave keeps to 128 registers, else of four. As many sequences as
// shares or more stay whole, whatever their lengths: of 16 with 36 heads one of 60000 positions
// runs on 36 workgroups, 114 us where it takes 35 alone. (768 for heads of
// 128: one sequence of 16000, 8 kv heads of 4 queries 21.0 us instead of 18.8, four of 30000, 8
// heads 36.8 instead of 38.2.) Short ones: a wave a chunk, up to eight, and no second launch.
struct Attn4Plan {
    int W, parts, shares;
};
Attn4Plan attn4_plan(const Kv4View &c, int H) {
    const int ch = attn4_ch(c.hd), chunks = (c.cap + ch - 1) / ch, per = H / c.Hkv;
    Attn4Plan pl;
    pl.parts = (per + A4_MAX_GH - 1) / A4_MAX_GH;
    pl.W = std::min(A4_MAX_W, chunks);
    pl.shares = 0;
    const long long heads = (long long)c.Hkv * pl.parts;
    const long long room = 512 / heads;
    if (chunks > A4_MAX_W && room > c.B) {
        // a sequence's last share is half one in the mean
        pl.shares = (int)(room - c.B / 2);
        pl.W = c.hd <= 64 && per == 1 ? 8 : 4;
    }
    return pl;
}
// The shares that there can be: `each` is at least their part of the chunks, and a
// sequence has one more for what is left.
int attn4_rows(const Attn4Plan &pl, int B) { return pl.shares + B + 1; }

template <int HD, int GH>
int launch_t(const Attn4Params &p, int W, int rows, hipStream_t st) {
    using M = Lds<HD, GH>;
    // a wave's weight terms, or its results
    constexpr size_t region = std::max(GH * M::NG * 4 * attn4_ch(HD), GH * (HD + 2) * 4);
    const size_t bytes = M::R + W * region;
    int rc = allow_lds((const void *)attn4_kernel<HD, GH>, bytes, M::R + A4_MAX_W * region);
    if (rc) return rc;
    const dim3 grid(p.parts > 1 ? cdiv((size_t)p.c.Hkv, 8) * 8 * p.parts : (unsigned)p.c.Hkv,
                    (unsigned)rows);
    attn4_kernel<HD, GH><<<grid, 64 * W, bytes, st>>>(p);
    VMLM_HIP_CHECK(hipGetLastError());
    return VMLM_OK;
}

template <int HD>
int launch_hd(const Attn4Params &p, int W, int rows, hipStream_t st) {
    if (p.G == 1) return launch_t<HD, 1>(p, W, rows, st);
    if (p.G == 2) return launch_t<HD, 2>(p, W, rows, st);
    return launch_t<HD, A4_MAX_GH>(p, W, rows, st);
}

}  // namespace

size_t attn4_work_floats(const Kv4View &c, int H) {
    if (c.B == 0 || c.Hkv == 0 || c.cap == 0 || H == 0) return 0;
    const Attn4Plan pl = attn4_plan(c, H);
    return pl.shares ? (size_t)attn4_rows(pl, c.B) * H * (c.hd + 4) : 0;
}

int launch_attn4(const Attn4Args &a, hipStream_t st) {
    const Attn4Plan pl = attn4_plan(a.c, a.H);
    Attn4Params p;
    p.c = a.c;
    p.q = a.q;
    p.k_new = a.k_new;
    p.v_new = a.v_new;
    p.ldq = a.ldq;
    p.ldkv = a.ldkv;
    p.ldo = a.ldo;
    p.pos = a.pos;
    p.out = a.out;
    p.work = a.work;
    p.H = a.H;
    p.G = a.H / a.c.Hkv;
    p.shares = pl.shares;
    p.W = pl.W;
    p.parts = pl.parts;
    p.ch = attn4_ch(a.c.hd);
    p.scale = frexpf(a.scale, &p.scale_e);
    p.guard = guard_flag_ptr();
    VMLM_GUARD(!p.shares || p.work, "kv4 attention: split positions need a workspace");
    const int rows = p.shares ? attn4_rows(pl, a.c.B) : a.c.B;
    int rc;
    switch (a.c.hd) {
    case 32: rc = launch_hd<32>(p, pl.W, rows, st); break;
    case 64: rc = launch_hd<64>(p, pl.W, rows, st); break;
    case 128: rc = launch_hd<128>(p, pl.W, rows, st); break;
    default: rc = launch_hd<256>(p, pl.W, rows, st); break;
    }
    if (rc || !p.shares) return rc;
    attn4_merge_kernel<<<dim3((unsigned)p.H, (unsigned)p.c.B), std::max(64, p.c.hd), 0, st>>>(p);
    VMLM_HIP_CHECK(hipGetLastError());
    return VMLM_OK;
}

}  // namespace vmlm
