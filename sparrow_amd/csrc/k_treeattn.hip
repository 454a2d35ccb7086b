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
// 16-bit terms stand below 2^11 and hold 11 bits down to 2^-14 and steps of 2^-24 below it.
//
// Bound by its instructions: with 63 tokens over 65463 positions, 36 heads of 64, 117 us, vector
// instructions 59 % of the cycles and matrix instructions 37 %, which do not run beside each other; 190 MB of
// cache at 1.6 TB/s. 333 tokens of 3 sequences after 4000 positions, 32 heads over 8 of 128: 156 us, 64 % and
// 34 %. A wave makes a block's operands for 64 queries (heads up to 64), 32 or 48 (128): the registers there are.
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
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

constexpr int TA_W = 4;  // waves of a workgroup
constexpr float TA_NONE = -3.40282347e38f;  // the maximum of no score yet
constexpr int TA_NO_GROUP = -1000;          // the weight of channels where all queries are 0
// Keys' and values' f16 stand below 2^TA_TOP_E (8 scale and the middle of a group do); positions of
// like size are within 2^TA_SPAN of that: their smallest middles keep 22 bits.
constexpr int TA_TOP_E = 11, TA_SPAN = 14;
constexpr float TA_TOP = 1 << TA_TOP_E;
// A weight is 2^TA_BASE at the maximum that its wave knew when it last raised it, which it
// does where one is 2^TA_SLACK larger: with 64 queries some maximum grows in nearly every block
// (63 tokens, 65463 positions, 36 heads of 64: 192 us when each was followed, 158 otherwise).
constexpr int TA_BASE = 9, TA_SLACK = 6;
constexpr float TA_UNBASE = 1.0f / (1 << TA_BASE);
constexpr float TA_FAR = 4194304.0f;        // scores whose f32 steps are no longer small
// The weights' sum. A position adds 2^score to it whatever its values; the weight that the products take is that times the
// value's power of two, so that of positions with scores alike those of small values weigh least. Three ways to sum:
//  * by the product, whose 16-bit terms end 2^-34 below the largest weight: where values are within 2^TA_SUM16 of the
//    largest that the wave has met, n of them are off by n 2^-24 at most, as a sum in f32 is;
//  * of the f32 weights over the values' powers of two: within 2^TA_SUM32, and 2^TA_RISE for values that come after
//    smaller ones (weights below 2^-126, and sums rescaled by less, are lost; below n 2^-24 of the sum up to there);
//  * by exponents of the scores alone: beyond, as with zeros among large values. And for blocks that not all queries
//    see, so that what a query does not see has no say in how its sum is formed.
// (All scores' exponents alone: 8 more exponentials a tile and block.)
constexpr int TA_SUM16 = 10, TA_SUM32 = 110, TA_RISE = 85;

struct TreeAttnParams {
    Kv4View c;
    const float *q;
    size_t ldq, ldo;
    const int32_t *pos0, *count, *parent;
    int S, G;
    // tiles of queries; whether positions are dealt out in shares: `per` is the number of workgroups that a
    // tile of all sequences may have, 0 if each takes all of a sequence's
    int tiles, per;
    int apart;    // a stream's tiles lie so many workgroups apart
    float *out;
    int *dealt;   // [B][2]: where a sequence's shares' results begin, how many shares it has
    float *work;  // [..][tile]: the results, of sequences of more than one share
    float scale, sign;  // of the scores: sign * scale * 2^scale_e, scale in [1/2, 1) (or 0), times log2(e)
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
// v times 2^e for integers e of any size (the weights' sums go below what a factor can be)
__device__ __forceinline__ float ta_scale(float v, float e) { return ldexpf(v, (int)fmaxf(e, -1000.0f)); }
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
// x less an f16, rounded to f16: one operation where the factor -1 is not known to the
// compiler, which else converts, subtracts and converts.
struct Rest {
    float minus_one = -1.0f;
    __device__ __forceinline__ Rest() { asm("" : "+s"(minus_one)); }
    __device__ __forceinline__ _Float16 operator()(float x, _Float16 h) const {
        return (_Float16)__builtin_fmaf((float)h, minus_one, x);
    }
};
// x as two f16 terms
__device__ __forceinline__ uint32_t two_terms(float x, const Rest &rest) {
    const _Float16 hi = (_Float16)x;
    const f16x2 v = {hi, rest(x, hi)};
    return __builtin_bit_cast(uint32_t, v);
}

// A number that is the same in all lanes, in a scalar register.
__device__ __forceinline__ float uniform(float v) {
    return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(v)));
}
__device__ __forceinline__ int uniform(int v) {
    asm volatile("" : "+v"(v));  // (else what comes after it is done before it, in vector registers)
    return __builtin_amdgcn_readfirstlane(v);
}

// The exponent e of a magnitude below 2^e (of numbers that are not normal -126).
__device__ __forceinline__ int exp_of(float mag) { return (int)(__float_as_uint(mag) >> 23) - 126; }

// Eight codes of a dword as f16 scale (u - 8): of nibbles (k, k + 4) in register k. s and c
// hold the scale and -24 times it: the nibbles lie in the mantissa of 16 + u.
struct Codes8 {
    f16x8 v;
    __device__ __forceinline__ Codes8(uint32_t w, const uint32_t (&s)[4], const uint32_t (&c)[4]) {
        const uint32_t t[4] = {w << 6, w << 2, w >> 2, w >> 6};
        uint32_t r[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t x = (t[k] & 0x03C003C0u) ^ 0x4E004E00u;  // (nibble ^ 8)
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
// wave its block's meta and three numbers for each position (V's middles as f16 [16][32]), for each
// query its power of two and the tokens it sees, for each group the queries' weight; the waves' results
// then lie over it all.
template <int HD, int MT>
struct TreeLds {
    static constexpr int KS = HD / 32, NG = HD / 32;
    static constexpr int FR = 2 * KS + 1;
    static constexpr bool ONES = NG < 8;  // the middles' rows leave one for the weights' sum
    static constexpr int Q = 0;
    static constexpr int WAVE = Q + MT * FR * 1024;
    static constexpr int SC = 1024, N = SC + 512;  // V's scales [8][32], numbers
    static constexpr int KG = 8;  // (zeros where there is no group)
    static constexpr int KM = N + 3 * 128, KSC = KM + 32 * KG * 4;  // K's middles [32][KG], scales [group][32]
    static constexpr int WB = KSC + NG * 64;
    static constexpr int F = WAVE + TA_W * WB;
    static constexpr int MASK = F + MT * 64;  // u64
    static constexpr int E = MASK + MT * 128;
    static constexpr int LM = E + 64;
    static constexpr int END = LM + TA_W * MT * 64;
    // [wave][16 MT][channels] (rows of other banks), then maxima and sums; half of the channels at a time
    // where two workgroups a CU would not fit
    static constexpr int PARTS = TA_W * 16 * MT * HD * 4 > 72 * 1024 ? 2 : 1, RC = HD / PARTS, RS = RC + 4;
    static constexpr int RO = 0;
    static constexpr int RM = RO + TA_W * 16 * MT * RS * 4;
    static constexpr int REND = RM + TA_W * 16 * MT * 8;
    static constexpr int OFF = END > REND ? END : REND;  // [wave][16 MT][8] the middles' sums
    static constexpr int SIZE = OFF + TA_W * 16 * MT * 32;
};

// What a wave reads of a block of 32 positions.
template <int HD>
struct RawBlock {
    static constexpr int NG = HD / 32, KD = HD / 32;
    static constexpr int OWN = HD == 256 ? 2 : 1, VM = NG < 2 ? 1 : NG / 2;
    uint32_t k[2][KD], v[HD / 16], km[VM], vm[VM];  // meta: of position lane % 32, half of the groups
    // (addresses: the same for all lanes, and 32 bits of a lane's own)
    __device__ __forceinline__ static uint32_t key_row(int r, int x) { return 8 * (r >> 2) + (r & 3) + 4 * x; }
    __device__ __forceinline__ void load_meta(const Kv4View &c, size_t row0, int lane) {
        const uint32_t m = (lane & 31) * NG + (lane >> 5) * (NG / 2);
        const uint32_t *kp = c.km + row0 * NG + m, *vp = c.vm + row0 * NG + m;
        if constexpr (VM == 1) {
            km[0] = kp[0];
            vm[0] = vp[0];
        } else {
            typedef uint32_t vec __attribute__((ext_vector_type(VM), aligned(4)));
            const vec a = *(const vec *)kp, b = *(const vec *)vp;
#pragma unroll
            for (int i = 0; i < VM; ++i) {
                km[i] = a[i];
                vm[i] = b[i];
            }
        }
    }
    __device__ __forceinline__ void load_k(const Kv4View &c, size_t row0, int lane) {
        const int r = lane & 15, j = lane >> 4;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const uint8_t *kp = c.k + row0 * (HD / 2) + (key_row(r, x) * (HD / 2) + j * (HD / 8));
            if constexpr (HD == 32) {
                k[x][0] = *(const uint32_t *)kp;
            } else if constexpr (HD == 64) {
                const u32x2m a = *(const u32x2m *)kp;
                k[x][0] = a[0];
                k[x][1] = a[1];
            } else {
#pragma unroll
                for (int i = 0; i < KD; i += 4) {
                    const u32x4m a = *(const u32x4m *)(kp + i * 4);
#pragma unroll
                    for (int e = 0; e < 4; ++e) k[x][i + e] = a[e];
                }
            }
        }
    }
    __device__ __forceinline__ void load_v(const Kv4View &c, size_t row0, int lane) {
        const uint32_t *vp = (const uint32_t *)(c.v + row0 * (HD / 2));
#pragma unroll
        for (int n = 0; n < HD / 16; ++n) v[n] = vp[(uint32_t)((n * 16 + (lane & 15)) * 4 + (lane >> 4))];
    }
};

// How the positions are dealt out where there are fewer tiles than the card takes workgroups, or a long
// sequence among short ones: in proportion to a sequence's blocks, which only the card knows. (One of
// 32700 positions beside 15 of 600, 8 tokens each: 36 heads of 64 44 us, 246 with shares that the capacity
// sets alike for all; 32 heads over 8 of 128 47 and 127. 16 of 2600, where nothing is gained: 48 and 47, 34 and 34.)
// At most (a lane of the merging wave each; 8 tokens over 65000 positions, 4 heads over one of 64: 25 us, 32 with 32 shares);
// blocks of a share (us with 4, 8 and 16: 8 tokens over 1000 positions, 36 heads of 64 11.3, 11.3, 13.1, over 600 11.3,
// 12.2, 12.5; 4 sequences of 2000, 8 heads over 2 of 128 19.0, 19.1, 24.0).
constexpr int TA_SHARES = 64, TA_LEAST = 2 * TA_W;
__device__ __forceinline__ float share_blocks(float blocks, int per) {
    return fmaxf(blocks / (float)per, (float)TA_LEAST);
}
__device__ __forceinline__ int shares_of(int blocks, float each) {
    return min(max((int)((float)blocks / each), 1), TA_SHARES);
}
struct Dealt {
    int b, shares, rest, at;  // rest: share * Hkv + kv head; at: where its shares' results begin
};
// The sequence and share of a stream, b < 0 if it has none; every wave finds them by itself.
__device__ __forceinline__ Dealt deal(const TreeAttnParams &p, int stream, bool first_tile) {
    const int lane = threadIdx.x & 63;
    auto blocks_of = [&](int b, bool *bad) {
        *bad = false;
        if (b >= p.c.B) return 0;
        const int at = p.pos0[b], n = p.count ? min(max(p.count[b], 0), p.S) : p.S;
        if (at < 0 || n == 0) return 0;
        *bad = at > p.c.cap - n;
        return *bad ? 0 : (at + n - 1) / KV4_BLOCK + 1;
    };
    bool bad = false;
    int blocks = blocks_of(lane, &bad);
    float sum = (float)blocks;
    for (int at = 64; at < p.c.B; at += 64) {
        bool more;
        sum += (float)blocks_of(at + lane, &more);
        bad |= more;
    }
    const bool tell = stream == 0 && first_tile && __builtin_amdgcn_readfirstlane(threadIdx.x) == 0;
    if (tell && __any(bad) && lane == 0) atomicOr(p.guard, 1);
    const float each = share_blocks(wave_sum_dpp(sum) * (float)p.c.Hkv, p.per);
    Dealt d{-1, 1, 0, 0};
    uint32_t before = 0;
    // (streams, 2^21 at most, below those whose results are kept, `per` at most: shares of two and more)
    constexpr int KEPT = 22;
    for (int at = 0; at < p.c.B; at += 64) {
        if (at) blocks = blocks_of(at + lane, &bad);
        const int s = blocks ? shares_of(blocks, each) : 0, n = s * p.c.Hkv;
        const uint32_t both = (uint32_t)n + (s > 1 ? (uint32_t)n << KEPT : 0u);
        uint32_t upto = both;  // of the sequences up to the lane's
#pragma unroll
        for (int i = 1; i < 64; i *= 2) {
            const uint32_t v = __shfl_up(upto, i, 64);
            if (lane >= i) upto += v;
        }
        const uint32_t first = before + upto - both;
        const int from = (int)(first & ((1u << KEPT) - 1)), kept = (int)(first >> KEPT);
        if (tell && at + lane < p.c.B) {
            p.dealt[2 * (at + lane)] = kept;
            p.dealt[2 * (at + lane) + 1] = s;
        }
        const unsigned long long here = __ballot(stream >= from && stream < from + n);
        if (here) {
            const int i = __builtin_ctzll(here);
            d.b = at + i;
            d.shares = __builtin_amdgcn_readlane(s, i);
            d.rest = stream - __builtin_amdgcn_readlane(from, i);
            d.at = __builtin_amdgcn_readlane(kept, i);
            if (!tell) break;
        }
        before += __builtin_amdgcn_readlane(upto, 63);
    }
    return d;
}

// A tile of 16 MT (token, head) pairs of one sequence and kv head, and one share of the positions.
// (Registers for two waves a SIMD: 8 sequences of 16000 positions, 4 heads over each of 4 of 256 and 16 tokens,
// 121 us, 167 with registers for one. <128, 3> spills 5 and <256, 1> 3, two of which the products read.)
template <int HD, int MT>
__global__ __launch_bounds__(64 * TA_W, 2) void tree_attn_kernel(TreeAttnParams p) {
    using M = TreeLds<HD, MT>;
    using Raw = RawBlock<HD>;
    constexpr int NG = HD / 32, KS = HD / 32, NT = HD / 16, CL = HD / 4, ROWS = 16 * MT;
    extern __shared__ __align__(16) uint8_t lds[];
    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int col = lane & 15, j = lane >> 4;
    // the tiles that read the same positions lie 8 workgroups apart: on one XCD. Fewer streams than 8 take all XCDs, with
    // no workgroups that have nothing to do (2048 tokens of 32 heads over one of 64: 86 us, 473 on one XCD).
    const int x8 = blockIdx.x / p.apart, stream = x8 / p.tiles * p.apart + (int)(blockIdx.x % p.apart),
              tile = x8 % p.tiles;
    int b, kvh = stream % p.c.Hkv, share = 0, shares = 1, kept = stream;
    if (p.per == 0) {
        b = stream / p.c.Hkv;
        if (b >= p.c.B) return;
    } else if (p.c.B == 1) {
        b = 0;
        share = stream / p.c.Hkv;
    } else {
        const Dealt d = deal(p, stream, tile == 0);
        if (d.b < 0) return;
        b = d.b;
        shares = d.shares;
        kvh = d.rest % p.c.Hkv;
        share = d.rest / p.c.Hkv;
        kept = d.at + d.rest;
    }
    // 16 queries a wave, loaded before anything is known of the sequence: lane (column, j) holds
    // channels CL j .. of its column's
    constexpr int GL = CL < 32 ? 1 : CL / 32;  // groups of the lane's channels
    const int row0 = tile * ROWS;
    const bool mine = w < MT;
    float x[CL];
    if (mine) {
        const int R = min(row0 + w * 16 + col, p.S * p.G - 1), t = R / p.G;
        const float *q = p.q + ((size_t)b * p.S + t) * p.ldq + ((size_t)kvh * p.G + R % p.G) * HD + CL * j;
#pragma unroll
        for (int c = 0; c < CL; c += 4) {
            const f32x4u v = *(const f32x4u *)(q + c);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[c + e] = v[e];
        }
    }
    const TreeRows tr = tree_rows(p.pos0, p.count, p.parent, p.S, p.c.cap, b, p.guard,
                                  kvh == 0 && tile == 0 && share == 0);
    if (p.per && p.c.B == 1) {
        const int all = tr.n ? (tr.pos0 + tr.n - 1) / KV4_BLOCK + 1 : 0;
        shares = __builtin_amdgcn_readfirstlane(shares_of(all, share_blocks((float)all * (float)p.c.Hkv, p.per)));
        if (stream == 0 && tile == 0 && tid < 2) p.dealt[tid] = tid * shares;
    }
    const int rows = min(ROWS, tr.n * p.G - row0);
    if (rows <= 0) return;
    const int t_lo = row0 / p.G, t_hi = (row0 + rows - 1) / p.G;
    const int last = tr.pos0 + t_hi;                               // the last position seen
    const int zone = tr.pos0 + (p.parent ? 0 : t_lo + 1);  // from here on not by all
    const int blocks = last / KV4_BLOCK + 1;
    if (share >= shares) return;
    const int b0 = (int)((long long)share * blocks / shares), b1 = (int)((long long)(share + 1) * blocks / shares);
    const size_t head = (size_t)b * p.c.Hkv + kvh;

    // 1. the queries' operands
    int *fe = (int *)(lds + M::F), *ge = (int *)(lds + M::E);
    unsigned long long *mask = (unsigned long long *)(lds + M::MASK);
    for (int i = tid; i < TA_W * 64; i += 64 * TA_W)
        *(u32x4 *)(lds + M::WAVE + (i >> 6) * M::WB + (i & 63) * 16) =
            M::ONES && (i & 63) >= 60 ? u32x4{0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u} : u32x4{0, 0, 0, 0};
    if (NG < 8)
        for (int i = tid; i < TA_W * 64; i += 64 * TA_W)
            *(u32x4 *)(lds + M::WAVE + (i >> 6) * M::WB + M::KM + (i & 63) * 16) = u32x4{0, 0, 0, 0};
    if (tid < 16) ge[tid] = TA_NO_GROUP;
    __syncthreads();
    int own_e = 0;  // the query's power of two
    bool bad = false;
    auto group_of = [&](int g) { return CL < 32 ? j * CL / 32 : j * GL + g; };  // the lane's g-th
    if (mine) {
        float mx[GL], most = 0.0f;
        int fine = 1;
#pragma unroll
        for (int g = 0; g < GL; ++g) {
            mx[g] = 0.0f;
#pragma unroll
            for (int c = 0; c < CL / GL; ++c) {
                float &v = x[g * 32 + c];
                if (w * 16 + col >= rows) v = 0.0f;
                mx[g] = fmaxf(mx[g], fabsf(v));
                fine &= fabsf(v) <= 3.40282347e38f;
            }
            if (CL <= 16) mx[g] = ta_swap16(mx[g], ta_max);
            if (CL <= 8) mx[g] = ta_swap32(mx[g], ta_max);
            most = fmaxf(most, mx[g]);
        }
        most = ta_swap32(ta_swap16(most, ta_max), ta_max);
        bad = ta_swap32(ta_swap16(fine ? 0.0f : 1.0f, ta_max), ta_max) > 0.0f;
        own_e = most > 0.0f && !bad ? ilogbf(most) : 0;
        if (j == 0) fe[w * 16 + col] = own_e - 8 + p.scale_e;
#pragma unroll
        for (int g = 0; g < GL; ++g) {
            const float e = mx[g] > 0.0f && !bad ? (float)(ilogbf(mx[g]) - own_e) : (float)TA_NO_GROUP;
            const float all = ta_row16(e, ta_max);
            if (col == 0) atomicMax(&ge[group_of(g)], (int)all);
        }
    }
    if (p.parent) {
        if (w == TA_W - 1) {  // ancestors by doubling: of 2, 4, 8 .. tokens at once
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
    } else if (tid < ROWS) {
        mask[tid] = (uint32_t)(tr.pos0 + (row0 + min(tid, rows - 1)) / p.G);  // the last position
    }
    __syncthreads();
    if (mine) {
        uint8_t *at = lds + M::Q + w * M::FR * 1024 + lane * 16;
        const Rest rest;
        float sum[GL];
#pragma unroll
        for (int g = 0; g < GL; ++g) sum[g] = 0.0f;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int e = 8 - own_e - ge[group_of(s / 4)];
            _Float16 hi[8], lo[8];
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                const float y = bad ? __builtin_nanf("") : ldexpf(x[8 * s + c] * p.sign, e);  // below 2^9
                hi[c] = (_Float16)y;
                lo[c] = rest(y, hi[c]);
                sum[CL < 32 ? 0 : s / 4] += (float)hi[c] + (float)lo[c];
            }
            *(f16x8 *)(at + 2 * s * 1024) = f16x8{hi[0], hi[4], hi[1], hi[5], hi[2], hi[6], hi[3], hi[7]};
            *(f16x8 *)(at + (2 * s + 1) * 1024) = f16x8{lo[0], lo[4], lo[1], lo[5], lo[2], lo[6], lo[3], lo[7]};
        }
#pragma unroll
        for (int g = 0; g < GL; ++g) {
            if (CL <= 16) sum[g] = ta_swap16(sum[g], ta_add);
            if (CL <= 8) sum[g] = ta_swap32(sum[g], ta_add);
        }
        // the sums' step: of lane j twice the upper terms of groups 4 (j & 1) .. where j < 2, else the lower
        uint32_t e[4] = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int g = 4 * (j & 1) + i;
            const int from = col + 16 * (NG == 8 ? (g >> 1) & 3 : NG == 4 ? i : NG == 2 ? (i & 1) * 2 : 0);
            float v = __shfl(sum[0], from, 64);
            if (GL == 2) {
                const float v1 = __shfl(sum[GL - 1], from, 64);
                v = g & 1 ? v1 : v;
            }
            const _Float16 h = (_Float16)v, l = rest(v, h), o = j < 2 ? h : l;
            if (g < NG) e[i] = __builtin_bit_cast(uint32_t, f16x2{o, o});
        }
        *(u32x4 *)(at + 2 * KS * 1024) = u32x4{e[0], e[1], e[2], e[3]};
    }
    __syncthreads();

    float m[MT], l[MT], cq[MT];
    f32x4 O[MT][NT + 1];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        m[t] = TA_NONE;
        l[t] = 0.0f;
#pragma unroll
        for (int n = 0; n <= NT; ++n) O[t][n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    uint8_t *wl = lds + M::WAVE + w * M::WB;
    int *ek = (int *)(wl + M::N);
    float *ev = (float *)(wl + M::N + 128), *iev = ev + 32;
    const uint8_t *qf = lds + M::Q + lane * 16;
    const float cs = p.scale;
    const Rest rest;
    // Blocks that all queries see and whose positions are of like size share their powers of
    // two: keys stand below 2^ek, values below 2^ev, those of the block that they were taken from with
    // room above. kg and vg bring scales to them, cq scores back.
    int ek_run = 0, ev_run = 0;
    int ev_top = -1000, ev_low = 1000;  // the values' powers of two so far, of what all queries see
    // The weights' sum by the scores alone from here on (no block is shared then), in units of 2^lm, which is in LDS:
    // in a register it costs every block.
    int alone = 0, wide = 0;
    float *lm = (float *)(lds + M::LM) + w * ROWS;
    constexpr int VM = Raw::VM;
    float kg[VM], vg = 0.0f;
#pragma unroll
    for (int i = 0; i < VM; ++i) kg[i] = 0.0f;
    bool far_any = false;

    // (nothing is moved over it, nor kept in registers for what comes after: fewer of them)
    auto apart = [] {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    const int lp = lane & 31, hf = lane >> 5;
    // the group of the lane's i-th meta, and of its o-th K codes
    auto group = [&](int i) { return NG == 1 ? 0 : hf * VM + i; };
    auto own_group = [&](int o) { return NG == 1 ? 0 : NG == 2 ? j >> 1 : j * Raw::OWN + o; };

    // What the products take of a block's meta: middles as two f16 terms, scales.
    uint32_t kmid[VM], vmid[VM];
    float kscale[VM], vscale[VM];
    unsigned long long nan_p[VM];  // lanes whose value's meta is a NaN

    // 2. by the shared powers of two; false where a position is too large for them, or its keys or a
    // group of its values smaller than 2^-TA_SPAN of them. (Zeros lose nothing; but where all of a position's
    // values are, its weight would be taken for that of the others' size, and small ones beside it lost.)
    auto shared_meta = [&](const Raw &raw) {
        float kmost = 0.0f, hi = 0.0f, lo = __builtin_inff();
#pragma unroll
        for (int i = 0; i < VM; ++i) {
            kscale[i] = kv4_scale(raw.km[i]) * kg[i];
            const float k8 = 8.0f * kscale[i], km = __builtin_fmaf(kv4_min(raw.km[i]), kg[i], k8);
            kmost = fmaxf(kmost, fmaxf(fabsf(km), k8));
            kmid[i] = two_terms(km, rest);
            vscale[i] = kv4_scale(raw.vm[i]) * vg;
            const float v8 = 8.0f * vscale[i], vm = __builtin_fmaf(kv4_min(raw.vm[i]), vg, v8);
            const float v = fmaxf(fabsf(vm), v8);
            hi = fmaxf(hi, v);
            lo = fminf(lo, v == 0.0f ? TA_TOP : v);
            vmid[i] = two_terms(vm, rest);
            nan_p[i] = 0;
        }
        if (NG > 1) {
            kmost = ta_swap32(kmost, ta_max);
            hi = ta_swap32(hi, ta_max);
        }
        lo = fminf(lo, kmost == 0.0f && kg[0] > 0.0f ? TA_TOP : kmost);
        return __all(fmaxf(kmost, hi) < TA_TOP && lo >= TA_TOP / (1 << TA_SPAN) && hi > 0.0f);
    };
    // the sums of weights that stand in O, in units of 2^ev, to the others
    auto join_sums = [&] {
        if (M::ONES) {
#pragma unroll
            for (int t = 0; t < MT; ++t)
                if (j == 3) {
                    l[t] += ldexpf(O[t][NT][3], TA_TOP_E - ev_run - TA_BASE);
                    O[t][NT][3] = 0.0f;
                }
        }
    };
    auto share_nothing = [&] {  // until the next choice
#pragma unroll
        for (int i = 0; i < VM; ++i) kg[i] = 0.0f;
    };
    auto also = [&](int top, int low) {  // values of these powers of two besides those so far
        const int rises = top > ev_top;
        ev_top = max(ev_top, top);
        ev_low = min(ev_low, low);
        wide |= (int)(ev_top - ev_low > TA_SUM32) | (rises & (int)(ev_top - ev_low > TA_RISE));
        wide = uniform(wide);
    };
    // 3. the powers of two of a block whose positions did not suit the ones there were; false
    // where they leave the range that the shared form keeps to
    auto choose = [&](const Raw &raw) {
        int e = -0x1000;
        float v = 0.0f;
#pragma unroll
        for (int i = 0; i < VM; ++i) {
            const float s = kv4_scale(raw.km[i]), mid = __builtin_fmaf(0.125f, kv4_min(raw.km[i]), s);
            e = max(e, exp_of(fmaxf(fabsf(mid), s)) + ge[group(i)]);
            const float sv = kv4_scale(raw.vm[i]);
            v = fmaxf(v, fmaxf(fabsf(__builtin_fmaf(0.125f, kv4_min(raw.vm[i]), sv)), sv));
        }
        const float ke = ta_swap32(ta_swap16(ta_row16((float)e, ta_max), ta_max), ta_max);
        v = ta_swap32(ta_swap16(ta_row16(v, ta_max), ta_max), ta_max);
        // (a group's middle / 8 and its scale are below 2^e; 8 times that, with two bits of room)
        join_sums();
        ek_run = __builtin_amdgcn_readfirstlane((int)ke) + 5;
        ev_run = __builtin_amdgcn_readfirstlane(exp_of(v)) + 5;
        bool fits = ev_run >= -90 && ev_run <= 120 && ek_run >= -90 && ek_run <= 120;
#pragma unroll
        for (int i = 0; i < VM; ++i) {
            const int g = ge[group(i)], f = g - ek_run;
            kg[i] = ldexpf(1.0f, f + TA_TOP_E);
            fits &= g == TA_NO_GROUP || (f <= 100 && f >= -100);
        }
        vg = uniform(ldexpf(1.0f, TA_TOP_E - ev_run));
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const int f = fe[t * 16 + col] + ek_run - TA_TOP_E;
            cq[t] = ldexpf(cs, f);
            fits &= f <= 100;
        }
        const int at = uniform(ev_run - TA_TOP_E);
        fits = __all(fits) && (!M::ONES || at >= ev_top - TA_SUM16);
        if (fits) also(at, at);
        fits &= wide == 0;
        if (!fits) share_nothing();
        return fits;
    };
    // 2'. by a power of two for every position, which the other lanes find in LDS; nothing past
    // the last position
    auto own_meta = [&](const Raw &raw, int p0, bool edge) {
        const bool in = !edge || p0 + lp <= last;
        float km[VM], vm[VM], mag = 0.0f;
        int e = -0x1000;
#pragma unroll
        for (int i = 0; i < VM; ++i) {
            const uint32_t mk = in ? raw.km[i] : 0u, mv = in ? raw.vm[i] : 0u;
            kscale[i] = kv4_scale(mk);
            km[i] = __builtin_fmaf(0.125f, kv4_min(mk), kscale[i]);
            e = max(e, exp_of(fmaxf(fabsf(km[i]), kscale[i])) + ge[group(i)]);
            vscale[i] = kv4_scale(mv);
            vm[i] = __builtin_fmaf(0.125f, kv4_min(mv), vscale[i]);
            nan_p[i] = 0;
            if (edge) {  // what some queries see and others do not: told at the end
                const bool bad = !(vm[i] == vm[i]);
                nan_p[i] = __ballot(bad);
                if (bad) vm[i] = vscale[i] = 0.0f;
            }
            mag = fmaxf(mag, fmaxf(fabsf(vm[i]), vscale[i]));
        }
        if (NG > 1) {
            e = (int)ta_swap32((float)e, ta_max);
            mag = ta_swap32(mag, ta_max);
        }
        e += 3 - TA_TOP_E;
        const int ve = max(exp_of(mag) + 3 - TA_TOP_E, -105);
#pragma unroll
        for (int i = 0; i < VM; ++i) {
            const int f = ge[group(i)] - e;
            kmid[i] = two_terms(ldexpf(km[i], f + 3), rest);
            kscale[i] = ldexpf(kscale[i], f);
            vmid[i] = two_terms(ldexpf(vm[i], 3 - ve), rest);
            vscale[i] = ldexpf(vscale[i], -ve);
        }
        if (!edge) {
            const float top = ta_swap16(ta_row16((float)ve, ta_max), ta_max);
            const float low = ta_swap16(ta_row16((float)-ve, ta_max), ta_max);
            const int from = ev_low, to = ev_top;
            also(uniform((int)top), -uniform((int)low));
            if (ev_top != to || ev_low != from) share_nothing();
        }
        if (lane < 32) {
            ek[lane] = e;
            ev[lane] = (float)ve;
            iev[lane] = ldexpf(1.0f, -ve - TA_BASE);
        }
    };

    // What follows a block's meta. (One copy of the products for both kinds of blocks: with
    // two, the accumulators took their registers twice.)
    auto block = [&](Raw &raw, int blk, size_t next, bool edge, bool shared) {
        const int p0 = blk * KV4_BLOCK;
        // (kept from splitting the code after it in two)
        auto is_shared = [&] {
            int v = __builtin_amdgcn_readfirstlane(shared);
            asm volatile("" : "+s"(v));
            return v != 0;
        };
        // 4. the meta, where the lanes that hold the codes find it
        if (NG > 1 || lane < 32) {
            _Float16 *o = (_Float16 *)wl + (lane & 24) + slot8(lane & 7);
#pragma unroll
            for (int i = 0; i < VM; ++i) {
                const int g = group(i);
                const f16x2 t = __builtin_bit_cast(f16x2, vmid[i]);
                o[g * 64] = t[0];
                o[g * 64 + 32] = t[1];
                o[M::SC / 2 + g * 32] = (_Float16)vscale[i];
                ((uint32_t *)(wl + M::KM))[lp * M::KG + g] = kmid[i];
                ((_Float16 *)(wl + M::KSC))[g * 32 + lp] = (_Float16)kscale[i];
            }
        }
        __builtin_amdgcn_wave_barrier();
        // 5. scores: rows of S^T, 4 j' + i of tile x is position 8 j' + 4 x + i
        f32x4 S[MT][2];
        f16x8 kf[2][KS + 1];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int at = (int)Raw::key_row(col, x);
            kf[x][KS] = *(const f16x8 *)(wl + M::KM + (at * M::KG + 4 * (j & 1)) * 4);
#pragma unroll
            for (int o = 0; o < Raw::OWN; ++o) {
                const _Float16 sk = ((const _Float16 *)(wl + M::KSC))[own_group(o) * 32 + at];
                const uint32_t sp = __builtin_bit_cast(uint32_t, f16x2{sk, sk}), cp = minus24(sp);
                const uint32_t s4[4] = {sp, sp, sp, sp}, c4[4] = {cp, cp, cp, cp};
                constexpr int D = KS / Raw::OWN;
#pragma unroll
                for (int i = 0; i < D; ++i) kf[x][o * D + i] = Codes8(raw.k[x][o * D + i], s4, c4).v;
            }
        }
        raw.load_k(p.c, next, lane);
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            apart();
            S[t][0] = S[t][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < 2 * KS + 1; ++i) {
                const f16x8 qv = *(const f16x8 *)(qf + (t * M::FR + i) * 1024);
                const int k = i == 2 * KS ? KS : i / 2;
                S[t][0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[0][k], qv, S[t][0], 0, 0, 0);
                S[t][1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[1][k], qv, S[t][1], 0, 0, 0);
            }
        }
        __builtin_amdgcn_wave_barrier();
        // 6. the running maximum of weight times value
        // the block's positions that query t of the lane sees
        auto sees = [&](int t) {
            const unsigned long long v = mask[t * 16 + col];
            const int own = tr.pos0 - p0, n = (int)(uint32_t)v - p0;  // the tokens' first; the last seen
            if (p.parent)
                return own >= 32 ? ~0u : own < 0 ? (own > -64 ? (uint32_t)(v >> -own) : 0u) : (uint32_t)(v << own) | ((1u << own) - 1);
            return n >= 31 ? ~0u : n < 0 ? 0u : (2u << n) - 1;
        };
        // whether the query's scores are in the millions: their rounding is larger than a weight's
        auto far = [&](int t) { return fabsf(m[t]) >= TA_FAR && m[t] > TA_NONE; };
        float top[MT];
        uint32_t seen = 0;  // a byte a tile
        if (is_shared()) {
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                float a = fmaxf(fmaxf(S[t][0][0], S[t][0][1]), S[t][0][2]);
                a = fmaxf(fmaxf(a, S[t][0][3]), S[t][1][0]);
                a = fmaxf(fmaxf(a, S[t][1][1]), S[t][1][2]);
                top[t] = __builtin_fmaf(fmaxf(a, S[t][1][3]), cq[t], (float)(ev_run - TA_TOP_E));
            }
        } else {
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const int f = fe[t * 16 + col];
                const uint32_t in8 = edge ? sees(t) >> (8 * j) & 255u : 255u;
                seen |= in8 << (8 * t);
                top[t] = TA_NONE;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float y = ldexpf(S[t][i / 4][i % 4], ek[8 * j + i] + f);
                    S[t][i / 4][i % 4] = y;
                    const float v = __builtin_fmaf(y, cs, ev[8 * j + i]);
                    top[t] = fmaxf(top[t], in8 >> i & 1 ? v : TA_NONE);
                }
                apart();
            }
        }
        bool more = false;
#pragma unroll
        for (int t = 0; t < MT; ++t) more |= top[t] > m[t] + TA_SLACK;
        if (__any(more)) {
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const float mx = __builtin_ceilf(ta_swap32(ta_swap16(top[t], ta_max), ta_max));
                // (each query by its own scores: nothing that only others see shows in it)
                const float to = mx > m[t] + TA_SLACK ? mx : m[t], corr = __builtin_amdgcn_exp2f(m[t] - to);
                m[t] = to;
                l[t] *= alone ? 1.0f : corr;
#pragma unroll
                for (int n = 0; n <= NT; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) O[t][n][i] *= corr;
                far_any |= __any(far(t));
            }
        }
        // 7. weights, in S's place
        if (is_shared()) {
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const float v = (float)(ev_run - TA_TOP_E), base = v - (m[t] - TA_BASE);
                if (far_any) {
                    const bool is_far = far(t);  // (the exponents themselves, none above TA_BASE + TA_SLACK)
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        float d = __builtin_fmaf(S[t][i / 4][i % 4], cq[t], base);
                        if (is_far) d = (__builtin_fmaf(S[t][i / 4][i % 4], cq[t], v) - m[t]) + TA_BASE;
                        S[t][i / 4][i % 4] = __builtin_amdgcn_exp2f(d);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        S[t][i / 4][i % 4] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[t][i / 4][i % 4], cq[t], base));
                }
                if (!M::ONES) {
                    float sum = 0.0f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) sum += S[t][i / 4][i % 4];
                    l[t] = __builtin_fmaf(sum, uniform(ldexpf(1.0f, TA_TOP_E - ev_run - TA_BASE)), l[t]);
                }
            }
        } else {
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const float base = m[t] - TA_BASE;
                const bool is_far = far_any && far(t);
                if (alone) {
                    float a = TA_NONE;
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        a = fmaxf(a, seen >> (8 * t + i) & 1 ? S[t][i / 4][i % 4] * cs : TA_NONE);
                    a = __builtin_ceilf(ta_swap32(ta_swap16(a, ta_max), ta_max));
                    // (far: the maximum itself, from which the weights are taken; a score's own rounding is another step)
                    const float old = lm[t * 16 + col], to = is_far ? m[t] : a > old + TA_SLACK ? a : old;
                    l[t] = ta_scale(l[t], old - to);
                    lm[t * 16 + col] = to;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float v = ev[8 * j + i];
                        float d = __builtin_fmaf(S[t][i / 4][i % 4], cs, -to);
                        if (is_far) d = (__builtin_fmaf(S[t][i / 4][i % 4], cs, v) - to) - v;
                        l[t] += __builtin_amdgcn_exp2f(seen >> (8 * t + i) & 1 ? d : -1000.0f);
                    }
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float v = ev[8 * j + i];
                    float d = __builtin_fmaf(S[t][i / 4][i % 4], cs, v - base);
                    if (is_far) d = (__builtin_fmaf(S[t][i / 4][i % 4], cs, v) - m[t]) + TA_BASE;
                    const float w8 = seen >> (8 * t + i) & 1 ? __builtin_amdgcn_exp2f(d) : 0.0f;
                    S[t][i / 4][i % 4] = w8;
                }
                if (!alone) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) l[t] = __builtin_fmaf(S[t][i / 4][i % 4], iev[8 * j + i], l[t]);
                }
                apart();
            }
        }
        f16x8 ph[MT], pl[MT];
#pragma unroll
        for (int t = 0; t < MT; ++t) {  // two f16 terms
            f16x2 hi[4], lo[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float a = S[t][0][i], c = S[t][1][i];
                hi[i] = __builtin_bit_cast(f16x2, f16_pair(a, c));
                lo[i] = f16x2{rest(a, hi[i][0]), rest(c, hi[i][1])};
            }
            ph[t] = __builtin_shufflevector(__builtin_shufflevector(hi[0], hi[1], 0, 1, 2, 3),
                                            __builtin_shufflevector(hi[2], hi[3], 0, 1, 2, 3), 0, 1, 2, 3, 4, 5, 6, 7);
            pl[t] = __builtin_shufflevector(__builtin_shufflevector(lo[0], lo[1], 0, 1, 2, 3),
                                            __builtin_shufflevector(lo[2], lo[3], 0, 1, 2, 3), 0, 1, 2, 3, 4, 5, 6, 7);
        }
        // 8. outputs: rows of O^T
#pragma unroll
        for (int n = 0; n <= NT; ++n) {
            f16x8 vf;
            if (n == NT) {  // the middles, and ones where the weights' sum is in shared units
                u32x4 e = *(const u32x4 *)(wl + col * 64 + j * 16);
                if (M::ONES && !is_shared() && col == 15) e = u32x4{0, 0, 0, 0};
                vf = __builtin_bit_cast(f16x8, e);
            } else {
                const u32x4 s = *(const u32x4 *)(wl + M::SC + n / 2 * 64 + j * 16);
                const uint32_t s4[4] = {s[0], s[1], s[2], s[3]};
                const uint32_t c4[4] = {minus24(s[0]), minus24(s[1]), minus24(s[2]), minus24(s[3])};
                vf = Codes8(raw.v[n], s4, c4).v;
            }
#pragma unroll
            for (int t = 0; t < MT; ++t) O[t][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, ph[t], O[t][n], 0, 0, 0);
#pragma unroll
            for (int t = 0; t < MT; ++t) O[t][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pl[t], O[t][n], 0, 0, 0);
        }
        raw.load_v(p.c, next, lane);
        // 9. values that are NaN, to the queries that see them: through the middles' sums
        unsigned long long any_nan = 0;
#pragma unroll
        for (int i = 0; i < VM; ++i) any_nan |= nan_p[i];
        if (any_nan) {
#pragma unroll
            for (int i = 0; i < VM; ++i) {
                for (unsigned long long left = nan_p[i]; left; left &= left - 1) {
                    const int at = __builtin_ctzll(left);
                    const int g = NG == 1 ? 0 : (at >> 5) * VM + i;
#pragma unroll
                    for (int t = 0; t < MT; ++t)
                        if ((sees(t) >> (at & 31) & 1) && j == g / 2) {
                            O[t][NT][0] = g % 2 ? O[t][NT][0] : __builtin_nanf("");
                            O[t][NT][2] = g % 2 ? __builtin_nanf("") : O[t][NT][2];
                        }
                }
            }
        }
        __builtin_amdgcn_wave_barrier();
    };

    const int whole = min(b1, min(zone, last + 1) / KV4_BLOCK);  // blocks that all queries see
    int share_end = whole;                                       // that may share powers of two
    Raw raw;
    const size_t first = head * p.c.cap;
    if (b0 + w < b1) {
        raw.load_meta(p.c, first + (b0 + w) * KV4_BLOCK, lane);
        raw.load_k(p.c, first + (b0 + w) * KV4_BLOCK, lane);
        raw.load_v(p.c, first + (b0 + w) * KV4_BLOCK, lane);
    }
    for (int blk = b0 + w; blk < b1; blk += TA_W) {
        const bool edge = blk >= whole;
        bool shared = blk < share_end;
        if (shared && !shared_meta(raw)) shared = choose(raw) && shared_meta(raw);
        if (!shared) {
            own_meta(raw, blk * KV4_BLOCK, edge);
            if (!alone && (edge || wide)) {
                alone = 1;
                share_end = 0;
                join_sums();
#pragma unroll
                for (int t = 0; t < MT; ++t) lm[t * 16 + col] = m[t];
            }
        }
        // what comes next into the same registers, as soon as they are read (the last block again at the end)
        const size_t next = first + (blk + TA_W < b1 ? blk + TA_W : blk) * KV4_BLOCK;
        raw.load_meta(p.c, next, lane);
        block(raw, blk, next, edge, shared);
    }
    if (alone) {
#pragma unroll
        for (int t = 0; t < MT; ++t) l[t] = ta_scale(l[t], lm[t * 16 + col] - m[t]);
    } else {
        join_sums();
    }

    // 10. the waves' results
    float *off = (float *)(lds + M::OFF) + w * ROWS * 8;
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        l[t] = ta_swap32(ta_swap16(l[t], ta_add), ta_add);
        if (2 * j < NG) off[(t * 16 + col) * 8 + 2 * j] = O[t][NT][0] + O[t][NT][1];
        if (2 * j + 1 < NG) off[(t * 16 + col) * 8 + 2 * j + 1] = O[t][NT][2] + O[t][NT][3];
    }
    __syncthreads();  // the operands are read; the results lie over them
    constexpr int RC = M::RC, RS = M::RS, NP = NT / M::PARTS;
    float *ro = (float *)(lds + M::RO) + w * ROWS * RS, *rm = (float *)(lds + M::RM);
#pragma unroll
    for (int part = 0; part < M::PARTS; ++part) {
        if (part) __syncthreads();
#pragma unroll
        for (int t = 0; t < MT; ++t) {
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                const int n = part * NP + i;
                const float mid = off[(t * 16 + col) * 8 + n / 2];
                *(f32x4l *)(ro + (t * 16 + col) * RS + i * 16 + 4 * j) =
                    f32x4l{O[t][n][0] + mid, O[t][n][1] + mid, O[t][n][2] + mid, O[t][n][3] + mid};
            }
            if (j == 0 && part == 0) {
                rm[(w * ROWS + t * 16 + col) * 2] = m[t];
                rm[(w * ROWS + t * 16 + col) * 2 + 1] = l[t];
            }
        }
        __syncthreads();
        for (int i = tid; i < rows * (RC / 4); i += 64 * TA_W) {
            const int r = i / (RC / 4), ci = i % (RC / 4) * 4, c = part * RC + ci;
            float mx = TA_NONE, L = 0.0f, f[TA_W];
#pragma unroll
            for (int x = 0; x < TA_W; ++x) mx = fmaxf(mx, rm[(x * ROWS + r) * 2]);
#pragma unroll
            for (int x = 0; x < TA_W; ++x) {
                f[x] = __builtin_amdgcn_exp2f(rm[(x * ROWS + r) * 2] - mx);
                L += ta_scale(rm[(x * ROWS + r) * 2 + 1], rm[(x * ROWS + r) * 2] - mx);
            }
            f32x4u o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int x = 0; x < TA_W; ++x) {
                const f32x4l v = *(const f32x4l *)((const float *)(lds + M::RO) + (x * ROWS + r) * RS + ci);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(f[x], v[e], o[e]);
            }
            if (shares == 1) {
                const int R = row0 + r;
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = o[e] * TA_UNBASE / L;
                *(f32x4u *)(p.out + ((size_t)b * p.S + R / p.G) * p.ldo + ((size_t)kvh * p.G + R % p.G) * HD + c) = o;
            } else {
                float *pw = p.work + ((size_t)kept * p.tiles + tile) * (ROWS * (HD + 2));
                *(f32x4u *)(pw + r * HD + c) = o;
                if (c == 0) {
                    pw[ROWS * HD + 2 * r] = mx;
                    pw[ROWS * HD + 2 * r + 1] = L;
                }
            }
        }
    }
}

// The shares of a query, in order: lane s takes the s-th one's maximum and sum, the threads
// eight of their rows at a time.
template <int HD>
__global__ __launch_bounds__(HD < 64 ? 64 : HD) void tree_merge_kernel(TreeAttnParams p, int ROWS) {
    const int r = blockIdx.x % ROWS, tile = blockIdx.x / ROWS, kvh = blockIdx.y, b = blockIdx.z;
    const int lane = threadIdx.x & 63, c = min((int)threadIdx.x, HD - 1);
    const int shares = p.dealt[2 * b + 1];
    if (shares <= 1) return;
    const size_t one = (size_t)ROWS * (HD + 2), ld = (size_t)p.c.Hkv * p.tiles * one;
    const float *pw = p.work + ((size_t)(p.dealt[2 * b] + kvh) * p.tiles + tile) * one;
    const float *px = pw + r * HD + c, *pm = pw + min(lane, shares - 1) * ld + ROWS * HD + 2 * r;
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = px[min(i, shares - 1) * ld];
    const float m = pm[0], l = pm[1];
    const TreeRows tr = tree_rows(p.pos0, p.count, p.parent, p.S, p.c.cap, b, p.guard, false);
    const int R = tile * ROWS + r;
    if (R >= tr.n * p.G) return;  // (what was read is not this query's)
    const float mx = ta_swap32(ta_swap16(ta_row16(m, ta_max), ta_max), ta_max);
    const float f = lane < shares ? __builtin_amdgcn_exp2f(m - mx) : 0.0f;
    const float L = wave_sum_dpp(lane < shares ? ta_scale(l, m - mx) : 0.0f);
    float o = 0.0f;
    for (int s = 0; s < shares; s += 8) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float w = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(f), min(s + i, 63)));
            o = s + i < shares ? __builtin_fmaf(w, x[i], o) : o;
        }
        if (s + 8 >= shares) break;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = px[min(s + 8 + i, shares - 1) * ld];
    }
    if (threadIdx.x < HD)
        p.out[((size_t)b * p.S + R / p.G) * p.ldo + ((size_t)kvh * p.G + R % p.G) * HD + c] = o * TA_UNBASE / L;
}

struct TreePlan {
    int mt, rows, tiles, per;
    size_t streams, work;  // work: floats
};
TreePlan tree_plan(const Kv4View &c, int H, int S) {
    const long long rows = (long long)S * (H / c.Hkv);
    const int most = c.hd <= 64 ? 4 : c.hd == 128 ? 2 : 1;
    TreePlan pl;
    // Rows of a tile (us with 16, 32 and 64; 16 sequences of 960 positions, 36 heads of 64: 16 tokens 21.7, 28.0, 50.8; 32
    // 32.4, 29.3, 52.1; 64 53, 48, 56; one of 65000: 24 tokens 100, 76, 113; 40 167, 137, 114. The widest, for what is
    // read often, costs a sixth after short contexts. Heads of 128, with 16 and 32: 8 sequences of 16000, 4 heads over
    // each of 8: 3 tokens 43, 55; 8 74, 58; 16 133, 99.)
    pl.mt = rows <= 16 ? 1 : rows <= 32 ? std::min(2, most) : most;
    // Heads of 128: 48 rows fill the registers, but a round of workgroups that is not full costs more (us with 48 and 32,
    // 4 heads over each of 8: 2 x 2048 tokens after 2048 positions 507 and 547, 4 x 400 184 and 189, 2 x 1024 242 both; below
    // the limit 4 x 300 146 and 138, 3 x 333 after 4000 201 and 186, 512 of one 80 and 62).
    if (c.hd == 128 && (long long)c.B * c.Hkv * ((rows + 47) / 48) >= 1024) pl.mt = 3;
    pl.rows = 16 * pl.mt;
    pl.tiles = (int)((rows + pl.rows - 1) / pl.rows);
    // Workgroups for two a CU, where a sequence's length gives each wave of a share two blocks. Where there are as
    // many without shares, only a cache of 8192 positions and more (16 sequences of 36 heads of 64, 8 tokens: where one
    // has 8100 positions and 15 have 600, 24 us, 66 without; where all have 600, 20 and 16), and only where the workgroups
    // that each look over all sequences are few beside the positions of one that is long. (4 queries over each kv
    // head of 64, 4 tokens, all of 600 positions, and one of the whole capacity; us with shares and without:
    // 512 sequences of 2 kv heads, 8192: 32 and 21, 39 and 64; of 8, 8192: 112 and 72, 115 and 77; 32768: 113 and 73, 120
    // and 239; 1024 of 2, 8192: 69 and 37, 72 and 65; 32768: 72 and 38, 79 and 235; 16384 of 1 of 32, 8192: 1850 and 87.)
    const size_t pairs = (size_t)c.B * c.Hkv, groups = pairs * pl.tiles, slots = 512;
    pl.per = groups < slots || c.cap >= 8192 ? (int)(slots / pl.tiles) : 0;
    const size_t longest = (size_t)c.cap / KV4_BLOCK / TA_LEAST;  // shares of the longest sequence
    if (longest <= 1 || (c.B == 1 && pl.per < 2 * c.Hkv)) pl.per = 0;
    // (what a workspace is asked for depends on the sequences' number by their table alone)
    pl.work = pl.per == 0 ? 0 : ((size_t)c.B * 2 + 63) / 64 * 64 + (size_t)pl.per * pl.tiles * pl.rows * (c.hd + 2);
    if (groups >= slots && (groups > (size_t)c.cap / 8 || c.B > c.cap / 16)) pl.per = 0;
    // (all shares of sequences of more than one are `per` at most; of several sequences each may round up to one)
    pl.streams = pl.per == 0 ? pairs : std::min(c.B == 1 ? (size_t)pl.per : pairs + pl.per, pairs * longest);
    return pl;
}

template <int HD, int MT>
int launch_t(const TreeAttnParams &p, const TreePlan &pl, hipStream_t st) {
    using M = TreeLds<HD, MT>;
    int rc = allow_lds((const void *)tree_attn_kernel<HD, MT>, M::SIZE, M::SIZE);
    if (rc) return rc;
    const size_t grid = (pl.streams + p.apart - 1) / p.apart * p.apart * p.tiles;
    tree_attn_kernel<HD, MT><<<(unsigned)grid, 64 * TA_W, M::SIZE, st>>>(p);
    VMLM_HIP_CHECK(hipGetLastError());
    if (p.per == 0) return VMLM_OK;
    tree_merge_kernel<HD><<<dim3((unsigned)(p.tiles * pl.rows), (unsigned)p.c.Hkv, (unsigned)p.c.B),
                            HD < 64 ? 64 : HD, 0, st>>>(p, pl.rows);
    VMLM_HIP_CHECK(hipGetLastError());
    return VMLM_OK;
}

template <int HD>
int launch_hd(const TreeAttnParams &p, const TreePlan &pl, hipStream_t st) {
    if (pl.mt == 1) return launch_t<HD, 1>(p, pl, st);
    if constexpr (HD <= 128) {
        if (pl.mt == 2) return launch_t<HD, 2>(p, pl, st);
    }
    if constexpr (HD == 128) return launch_t<HD, 3>(p, pl, st);
    if constexpr (HD <= 64) return launch_t<HD, 4>(p, pl, st);
    return VMLM_OK;
}

}  // namespace

size_t tree_attn_work_floats(const Kv4View &c, int H, int S) {
    if (c.B == 0 || c.Hkv == 0 || c.cap == 0 || H == 0 || S == 0) return 0;
    return tree_plan(c, H, S).work;
}

bool tree_attn_splits(const Kv4View &c, int H, int S) { return tree_plan(c, H, S).per != 0; }

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
    p.G = a.H / a.c.Hkv;
    p.tiles = pl.tiles;
    p.per = pl.per;
    p.apart = (int)std::min(pl.streams, (size_t)8);
    p.out = a.out;
    p.dealt = (int *)a.work;
    p.work = a.work + ((size_t)a.c.B * 2 + 63) / 64 * 64;
    p.scale = frexpf(fabsf(a.scale), &p.scale_e) * 1.44269504f;
    p.sign = a.scale < 0.0f ? -1.0f : 1.0f;
    p.guard = guard_flag_ptr();
    VMLM_GUARD(p.per == 0 || a.work, "kv4 tree attention: split positions need a workspace");
    switch (a.c.hd) {
    case 32: return launch_hd<32>(p, pl, st);
    case 64: return launch_hd<64>(p, pl, st);
    case 128: return launch_hd<128>(p, pl, st);
    default: return launch_hd<256>(p, pl, st);
    }
}

}  // namespace vmlm
