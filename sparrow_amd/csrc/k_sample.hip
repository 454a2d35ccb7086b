// k_sample.hip -- one token of each row of logits, drawn with a given random number
// (vmlm_hip_sample).
//
// The tokens stand in the order of their logits, the largest first, of equal ones the
// lowest index; token j has the weight w_j = exp((l_j - l_max) / T). Kept are the first k of
// them, of those the ones before which the weights sum to less than p of the k's, of those
// the ones with w_j >= min_p. The token is the first whose weights up to it sum to more
// than u times the kept ones'.
//
// Nothing is sorted but what can be kept: -l / T falls into bins of 1/64, and every question
// (the k-th token, the mass p, the token drawn) is answered by the bins' counts and masses
// down to one bin. Where the bins up to the last one that can matter hold few tokens, those are
// gathered and sorted together; else one bin is, for each question. 2048 bins from the largest logit's
// reach weights of 2^-46; what lies behind counts as none (a million tokens of that are 2^-26 of the first).
//
// Next to a border between two tokens 32 bits are too few: with 122753 tokens of like weight
// a sum off by 2^-24 takes the neighbour's token once in 50 rows. So l / T is formed in 64 bits, and a
// token's weight is exp(-bin / 64) (1 - d), d = 1 - exp(-r) < 1/64 of the rest r, held as an
// integer in units of 2^-30: a bin's sum of d and its count are one 64-bit atomic add in
// LDS, whose order changes nothing. A token's bin and rest depend on its logit and T alone.
//
// A row is read once for its bins (a larger logit than those before moves them along), and as a rule once more,
// by f32 comparisons, for the tokens to sort. Where a bin that a question ends in holds more tokens than are sorted at
// once, as in flat rows and those of few values, it is narrowed by two readings a time, for each such question, and min_p
// may count its tokens in one of its own (a row of 122753 within a hundredth of each other 0.5 ms, of equal logits 0.8, with
// top_k and top_p 2.4; 512 of them 1.1, 1.7 and 4.8). Few rows are cut into slices, which also list the tokens of their first bins, so
// that the second reading is seldom needed.
//
// 512 rows of 122753 (251 MB): 52 us greedy, HBM's rate; 98 with top_k 50 and 118 without a filter, the first
// reading bound by two dozen vector instructions a token and its LDS addition. One row 25 us (35 without a
// filter): a slice's 9 and its end's 16, latencies.
#include <algorithm>

#include "internal.hpp"

namespace vmlm {
namespace {

constexpr int THREADS = 1024;
constexpr int BINS = 2048;       // the last one's tokens have no weight
constexpr int LIST = 2048;       // tokens that are sorted at once
constexpr int SLICE_LIST = 256;  // tokens of the first bins that a slice lists
constexpr double PER = 64.0;     // bins of a distance of 1
constexpr int UNIT = 30;         // d in units of 2^-30
constexpr int COUNT = 44;        // a bin's word: count above, sum of d below
constexpr unsigned long long LOSSES = (1ull << COUNT) - 1;
constexpr double TOO_FAR = 0x1p49;  // bins from 0: where f64 no longer holds a rest

typedef float f32x4a __attribute__((ext_vector_type(4), aligned(4)));

struct SampleParams {
    const float *logits;
    size_t ld;
    const float *u, *t, *top_p, *min_p;
    const int32_t *top_k;
    int rows, vocab;
    int32_t *token;
    float *prob;
    int *guard;
};

// Order-preserving bits of a logit (of numbers; -0 as 0), and back.
__device__ __forceinline__ uint32_t order_bits(float v) {
    if (v == 0.0f) v = 0.0f;
    const uint32_t b = __float_as_uint(v);
    return (b >> 31) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_bits(uint32_t b) {
    return __uint_as_float((b >> 31) ? b ^ 0x80000000u : ~b);
}
// a token: (order bits, ~index), larger for the one that stands first
__device__ __forceinline__ unsigned long long token_word(float l, int index) {
    return (unsigned long long)order_bits(l) << 32 | (uint32_t)~index;
}

// A logit's place: its bin from the reference on, and the rest as a fraction of a bin in
// units of 2^-32. 2^20 in the sum leaves both in its bits.
struct Place {
    double per = 0.0, ref = 0.0;  // PER / T; the bin of -l / T that is bin 0
    __device__ __forceinline__ Place() {}
    __device__ __forceinline__ Place(float t, float max) {
        per = PER / (double)t;
        refer(max);
    }
    __device__ __forceinline__ void refer(float max) {
        ref = __builtin_floor(-(double)max * per);
        if (__builtin_fma(-(double)max, per, -ref) < 0.0) ref -= 1.0;  // (the product was rounded up to it)
    }
    __device__ __forceinline__ bool too_far(float max) const { return !(fabs((double)max * per) < TOO_FAR); }
    // T so small against the logits that only the largest one's equals can have a weight: a
    // larger T that leaves f64 its rests says the same (the next logit is 2^25 bins away)
    __device__ __forceinline__ void widen(float max) {
        per = TOO_FAR / fabs((double)max);
        refer(max);
    }
    __device__ __forceinline__ int bin(float l, uint32_t *rest) const {
        const double y = __builtin_fma(-(double)l, per, 0x1p20 - ref);  // (+inf for a masked one)
        const unsigned long long b = __builtin_bit_cast(unsigned long long, y);
        *rest = (uint32_t)b;
        return (int)min((uint32_t)(b >> 32) - 0x41300000u, (uint32_t)(BINS - 1));
    }
    // Logits below this one are not in bin b or before it; above it, not in bin b or behind it.
    // (f32: by a part of a bin, and where a bin is narrower than its steps by a few of those)
    __device__ __forceinline__ float below(int b) const {
        const double l = -(ref + (double)b + 1.02) / per;
        return (float)(l - fabs(l) * 0x1p-21);
    }
    __device__ __forceinline__ float above(int b) const {
        const double l = -(ref + (double)b - 0.02) / per;
        return (float)(l + fabs(l) * 0x1p-21);
    }
};
// 1 - exp(-r) of the rest r = f 2^-38 < 2^-6, in units of 2^-30, off by at most one: r itself
// from the bits, the other terms below 2^-13 in f32 (the next of the series is below 2^-36)
__device__ __forceinline__ uint32_t loss(uint32_t f) {
    const float r = (float)f * 0x1p-38f;
    const float q = r * r * __builtin_fmaf(__builtin_fmaf(r, 1.0f / 24, -1.0f / 6), r, 0.5f);
    return (uint32_t)((f >> 8) + (f >> 7 & 1)) - (uint32_t)(int)rintf(q * 0x1p30f);
}
__device__ __forceinline__ void count_token(unsigned long long *hist, const Place &at, float l) {
    uint32_t rest;
    const int b = at.bin(l, &rest);
    if (b < BINS - 1) atomicAdd(&hist[b], (1ull << COUNT) | loss(rest));
}

// 16 of a thread's tokens of the T * 16 from `first` on: 4 times 4 neighbours; those from n on
// are -inf.
template <int T>
struct Tokens {
    f32x4a v[4];
    __device__ __forceinline__ static int index(int k) { return (threadIdx.x + k * T) * 4; }
    __device__ __forceinline__ void load(const float *row, int first, int n) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int i = first + index(k);
            if (i + 3 < n) {
                v[k] = *(const f32x4a *)(row + i);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[k][e] = i + e < n ? row[i + e] : -__builtin_inff();
            }
        }
    }
    template <typename F>
    __device__ __forceinline__ void each(int first, F f) const {
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) f(v[k][e], first + index(k) + e);
    }
};
// Calls f(logit, index) for every token of a row (and, past its end, with -inf). AHEAD: the next
// part is on its way meanwhile, where registers are not short.
template <int T, bool AHEAD, typename F>
__device__ __forceinline__ void each_token(const float *row, int n, F f) {
    Tokens<T> now, next;
    if (AHEAD) next.load(row, 0, n);
    for (int first = 0; first < n; first += T * 16) {
        if (AHEAD) {
            now = next;
            if (first + T * 16 < n) next.load(row, first + T * 16, n);
        } else {
            now.load(row, first, n);
        }
        now.each(first, f);
    }
}

struct Shared {
    unsigned long long hist[BINS];  // counts and losses; what is to be sorted; weights
    double above[BINS];             // the mass before a bin
    uint32_t before[BINS];          // the tokens before a bin
    uint32_t start[BINS];           // where a bin's tokens stand in the list, if they do
    unsigned long long list[LIST];  // tokens, the largest first
    uint32_t slots[LIST];           // of the bins' tokens
    double whole[32], part[64];     // exp(-i), exp(-i / 64)
    double red[16];
    unsigned long long wave64[16];
    unsigned long long best;
    uint32_t n, lo, hi;
    uint32_t wave[16];
};

__device__ __forceinline__ unsigned long long shfl_xor64(unsigned long long v, int o) {
    return (unsigned long long)__shfl_xor((uint32_t)(v >> 32), o, 64) << 32 | (uint32_t)__shfl_xor((uint32_t)v, o, 64);
}
__device__ __forceinline__ unsigned long long wave_most(unsigned long long v) {
#pragma unroll
    for (int o = 32; o; o /= 2) {
        const unsigned long long w = shfl_xor64(v, o);
        v = w > v ? w : v;
    }
    return v;
}
template <typename T>
__device__ __forceinline__ T wave_scan(T v) {  // inclusive
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
        const T w = __shfl_up(v, o, 64);
        if (lane >= o) v = v + w;
    }
    return v;
}

// Block-wide exclusive prefix sums over 2 values a thread; the sum of all.
template <typename T>
__device__ __forceinline__ T block_scan(T a, T b, T *out_a, T *out_b, T *scratch) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const T to = wave_scan<T>(a + b);
    if (lane == 63) scratch[w] = to;
    __syncthreads();
    T base = 0, all = 0;
#pragma unroll
    for (int i = 0; i < THREADS / 64; ++i) {
        if (i == w) base = all;
        all = all + scratch[i];
    }
    const T up = __shfl_up(to, 1, 64);
    *out_a = base + (lane ? up : T(0));
    *out_b = *out_a + a;
    __syncthreads();
    return all;
}

// A row's settings. live: there is something to draw.
struct Settings {
    float u, t, top_p, min_p;
    int top_k;
    bool live;
};
__device__ __forceinline__ Settings settings_of(const SampleParams &p, int r, bool report) {
    Settings c;
    c.u = p.u[r];
    c.t = p.t[r];
    c.top_p = p.top_p ? p.top_p[r] : 1.0f;
    c.min_p = p.min_p ? p.min_p[r] : 0.0f;
    c.top_k = p.top_k ? p.top_k[r] : 0;
    const bool ok = c.u < 1.0f && c.t >= 0.0f && c.t <= 3.40282347e38f && c.top_p == c.top_p &&
                    c.min_p >= 0.0f && c.min_p <= 1.0f;
    c.live = ok && c.u >= 0.0f;
    if (!ok && !(c.u < 0.0f) && report && threadIdx.x == 0) atomicOr(p.guard, 1);
    return c;
}

// What there is to say of a row whose first token is known (WITH_NAN: it has a NaN); true if
// nothing else is.
constexpr unsigned long long WITH_NAN = ~0ull;
__device__ __forceinline__ bool settled(const SampleParams &p, int r, const Settings &c, unsigned long long best) {
    const float max = of_bits((uint32_t)(best >> 32));
    int token = -1;
    float prob;
    if (best == WITH_NAN || max == __builtin_inff())
        prob = __builtin_nanf("");
    else if (max == -__builtin_inff())
        prob = 0.0f;  // the mask leaves no token
    else if (c.t == 0.0f) {
        token = (int)~(uint32_t)best;
        prob = 1.0f;
    } else
        return false;
    if (threadIdx.x == 0) {
        p.token[r] = token;
        if (p.prob) p.prob[r] = prob;
    }
    return true;
}

// What the slices of a row leave for its last kernel.
struct SampleSlices {
    int n;                     // a row's
    unsigned long long *best;  // [rows][n] the first token
    unsigned long long *hist;  // [rows][n][BINS], bins from the slice's largest logit's on
    unsigned long long *list;  // [rows][n][SLICE_LIST] the tokens of the first bins
    int32_t *upto;             // [rows][n][2]: those below this bin, and their number
};

// The n <= LIST tokens in s.list, zeros behind them, the largest first.
__device__ __forceinline__ void sort_list(Shared &s, int n) {
    int pow2 = 64;
    while (pow2 < n) pow2 *= 2;
    __syncthreads();
    for (int k = 2; k <= pow2; k *= 2)
        for (int j = k / 2; j > 0; j /= 2) {
            for (int i = threadIdx.x; i < pow2 / 2; i += THREADS) {
                const int x = i / j * 2 * j + i % j, y = x + j;
                const unsigned long long a = s.list[x], b = s.list[y];
                if (((x & k) == 0) == (a < b)) {
                    s.list[x] = b;
                    s.list[y] = a;
                }
            }
            __syncthreads();
        }
}

// A place in the order: its token's rank in its bin and the bin's weights up to it, in
// units of 2^-30 of the bin's largest.
struct Found {
    uint32_t rank;
    unsigned long long upto;
    uint32_t token, d;
};

// The sums of the losses of the n tokens in s.list up to each, in s.hist.
__device__ __forceinline__ void sum_losses(Shared &s, int n, const Place &at) {
    static_assert(LIST == BINS && LIST == 2 * THREADS, "");
    const int tid = threadIdx.x;
    unsigned long long d[2], e[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int x = tid * 2 + i;
        uint32_t rest;
        d[i] = 0;
        if (x < n) {
            at.bin(of_bits((uint32_t)(s.list[x] >> 32)), &rest);
            d[i] = loss(rest);
        }
    }
    block_scan<unsigned long long>(d[0], d[1], &e[0], &e[1], s.wave64);
#pragma unroll
    for (int i = 0; i < 2; ++i) s.hist[tid * 2 + i] = e[i] + d[i];
    __syncthreads();
}
// The place in the bin of m tokens that stand in s.list from x0 on, as locate finds it.
__device__ __forceinline__ Found place_in(const Shared &s, int x0, int m, bool by_rank, uint32_t rank, double mass,
                                          bool with_equal) {
    const unsigned long long d0 = x0 ? s.hist[x0 - 1] : 0;
    auto upto = [&](int i) { return ((unsigned long long)(i + 1) << UNIT) - (s.hist[x0 + i] - d0); };
    int i = min((int)rank, m - 1);
    if (!by_rank) {
        int z = m - 1;
        for (i = 0; i < z;) {
            const int mid = (i + z) / 2;
            const double w = (double)upto(mid);
            if (with_equal ? w >= mass : w > mass)
                z = mid;
            else
                i = mid + 1;
        }
    }
    Found f;
    f.rank = i;
    f.upto = upto(i);
    f.d = (uint32_t)(s.hist[x0 + i] - (x0 + i ? s.hist[x0 + i - 1] : 0));
    f.token = ~(uint32_t)s.list[x0 + i];
    return f;
}

// The token of rank `rank` in bin `bin` (by_rank), else the first one with weights up to it of
// more than `mass` (or, with_equal, as much). `n`: the bin's tokens.
template <bool AHEAD>
__device__ __forceinline__ Found locate(Shared &s, const float *row, int vocab, const Place &at, int bin, int n,
                                        bool by_rank, uint32_t rank, double mass, bool with_equal) {
    const int tid = threadIdx.x;
    uint32_t lo = 0, hi = 0xffffffffu;  // of the order bits
    const float from = at.below(bin), to = at.above(bin);
    uint32_t rank0 = 0;  // the bin's tokens above them, and their weights
    unsigned long long mass0 = 0;
    auto each_of_bin = [&](auto f) {
        each_token<THREADS, AHEAD>(row, vocab, [&](float l, int i) {
            uint32_t rest;
            const uint32_t key = order_bits(l);
            if (l >= from && l <= to && key >= lo && key <= hi && at.bin(l, &rest) == bin) f(key, rest, i);
        });
    };
    // 1. a bin of too many tokens: ranges of their order bits, the narrowest that hold the place
    while (n > LIST && lo < hi) {
        __syncthreads();
        if (tid == 0) {
            s.lo = 0xffffffffu;
            s.hi = 0;
        }
        for (int i = tid; i < BINS; i += THREADS) s.hist[i] = 0;
        __syncthreads();
        each_of_bin([&](uint32_t key, uint32_t, int) {
            atomicMin(&s.lo, key);
            atomicMax(&s.hi, key);
        });
        __syncthreads();
        lo = s.lo;
        hi = s.hi;
        if (lo == hi) break;
        int shift = 0;
        while ((hi - lo) >> shift >= BINS) ++shift;
        each_of_bin([&](uint32_t key, uint32_t rest, int) {
            atomicAdd(&s.hist[(hi - key) >> shift], (1ull << COUNT) | loss(rest));
        });
        __syncthreads();
        if (tid == 0) {
            uint32_t r = rank0, rl = rank0;
            unsigned long long m = mass0, ml = mass0;
            int last = 0;
            for (int i = 0; i < BINS; ++i) {  // the last range that is not empty where none reaches it
                const uint32_t c = (uint32_t)(s.hist[i] >> COUNT);
                if (c == 0) continue;
                const unsigned long long w = ((unsigned long long)c << UNIT) - (s.hist[i] & LOSSES);
                last = i;
                rl = r;
                ml = m;
                if (by_rank ? r + c > rank : with_equal ? (double)(m + w) >= mass : (double)(m + w) > mass) break;
                r += c;
                m += w;
            }
            s.n = (uint32_t)last;
            s.wave[0] = rl;
            s.best = ml;
        }
        __syncthreads();
        const uint32_t i = s.n, span = hi - lo;
        rank0 = s.wave[0];
        mass0 = s.best;
        n = (int)(s.hist[i] >> COUNT);
        const unsigned long long end = (((unsigned long long)i + 1) << shift) - 1;
        lo = hi - (uint32_t)min(end, (unsigned long long)span);
        hi = hi - (i << shift);
        __syncthreads();
    }
    Found f;
    if (n > LIST) {  // 2. so many equal ones: the place is arithmetic, its index a count
        uint32_t rest;
        at.bin(of_bits(lo), &rest);
        f.d = loss(rest);
        const double w = (double)((1ull << UNIT) - f.d);
        uint32_t k;
        if (by_rank) {
            k = rank - rank0;
        } else {
            const double q = (mass - (double)mass0) / w;  // (weights up to k: k + 1 of them)
            k = q <= 0.0 ? 0 : (uint32_t)fmin(with_equal ? __builtin_ceil(q) - 1.0 : __builtin_floor(q), (double)(n - 1));
        }
        k = min(k, (uint32_t)(n - 1));
        f.rank = rank0 + k;
        f.upto = mass0 + (unsigned long long)(k + 1) * ((1ull << UNIT) - f.d);
        const int seg = (vocab + THREADS - 1) / THREADS, i0 = min(tid * seg, vocab), i1 = min(i0 + seg, vocab);
        uint32_t c = 0, a, b2;
        for (int i = i0; i < i1; ++i) c += order_bits(row[i]) == lo;
        block_scan<uint32_t>(c, 0u, &a, &b2, s.wave);
        if (a <= k && k < a + c) {
            for (int i = i0; i < i1; ++i)
                if (order_bits(row[i]) == lo && a++ == k) s.n = (uint32_t)i;
        }
        __syncthreads();
        f.token = s.n;
        __syncthreads();
        return f;
    }
    // 3. its tokens, gathered and sorted
    __syncthreads();
    if (tid == 0) s.n = 0;
    for (int i = tid; i < LIST; i += THREADS) s.list[i] = 0;
    __syncthreads();
    each_of_bin([&](uint32_t key, uint32_t, int i) {
        s.list[min(atomicAdd(&s.n, 1u), (uint32_t)(LIST - 1))] = (unsigned long long)key << 32 | (uint32_t)~i;
    });
    sort_list(s, n);
    sum_losses(s, n, at);
    f = place_in(s, 0, n, by_rank, rank - rank0, mass - (double)mass0, with_equal);
    f.rank += rank0;
    f.upto += mass0;
    __syncthreads();
    return f;
}

// The smallest logit with exp((l - max) / t) >= min_p in 64 bits: next to where its logarithm puts
// it, the lanes try the f32 around it. (min_p 1: the largest one itself, however many weights beside it are 1 in 64 bits.)
__device__ __forceinline__ float least_of(float max, float t, float min_p) {
    if (min_p == 1.0f) return max;
    const float near = (float)fmax((double)max + (double)t * log((double)min_p), -3.40282347e38);
    const uint32_t key = order_bits(near) + (threadIdx.x & 63) - 32u;
    const float l = of_bits(key);
    const bool in = l <= max && l >= -3.40282347e38f && exp(((double)l - (double)max) / (double)t) >= (double)min_p;
    const unsigned long long keeps = __ballot(in);
    // (next to 0 f32's steps are below what 64 bits tell apart: any of them then)
    if (!keeps) return fminf(max, of_bits(__builtin_amdgcn_readlane(key, 63)));
    return of_bits(__builtin_amdgcn_readlane(key, __builtin_ctzll(keeps)));
}

// The rest, from a row's bins in s.hist, by one workgroup. sl.n 0: no slices. `max`: the largest logit.
template <bool AHEAD>
__device__ __forceinline__ void finish(Shared &s, const SampleParams &p, int r, const Settings &c, float max,
                                       const Place &at, const SampleSlices &sl) {
    const int tid = threadIdx.x, lane = tid & 63, n = p.vocab;
    const float *row = p.logits + r * p.ld;
    if (tid < 32) s.whole[tid] = exp(-(double)tid);
    if (tid >= 64 && tid < 128) s.part[tid - 64] = exp(-(tid - 64) / PER) * (1.0 / (1 << UNIT));
    __syncthreads();
    auto scale = [&](int b) { return s.whole[b >> 6] * s.part[b & 63]; };  // of a bin's units
    uint32_t cnt[2], c0[2];
    double mass[2], m0[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const unsigned long long h = s.hist[tid * 2 + i];
        cnt[i] = (uint32_t)(h >> COUNT);
        mass[i] = scale(tid * 2 + i) * (double)(((unsigned long long)cnt[i] << UNIT) - (h & LOSSES));
    }
    const uint32_t live = block_scan<uint32_t>(cnt[0], cnt[1], &c0[0], &c0[1], s.wave);
    double all = block_scan<double>(mass[0], mass[1], &m0[0], &m0[1], s.red);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        s.before[tid * 2 + i] = c0[i];
        s.above[tid * 2 + i] = m0[i];
    }
    __syncthreads();
    auto tokens = [&](int b) { return (int)((b + 1 < BINS ? s.before[b + 1] : live) - s.before[b]); };
    // The n <= LIST tokens of the bins with a place in s.start, in s.list, the largest first; `each` puts
    // them. Up to 128 go where the number of larger ones says, which as many threads as there are count
    // together (16 reads each at most; 512 would be 256 reads, 8 us more than the following). Of more, a bin of m tokens is cut into m slots, which hold one or two each: a token goes to its slot, and
    // counts the larger ones there. (Of 1000 to 2000 tokens a sort's 55 to 66 steps take 10 to 16 us more; it
    // is left for slots of more than 64, of equal tokens.)
    constexpr uint32_t NONE = ~0u;
    auto sort_bins = [&](int n, auto each) {
        __syncthreads();
        if (tid == 0) s.n = s.hi = 0;
        for (int i = tid; i < LIST; i += THREADS) s.slots[i] = 0;
        __syncthreads();
        each([&](unsigned long long v) { s.hist[min(atomicAdd(&s.n, 1u), (uint32_t)(LIST - 1))] = v; });
        __syncthreads();
        if (n <= 128) {
            int pow2 = 64;
            while (pow2 < n) pow2 *= 2;
            const int x = tid % pow2, part = pow2 * pow2 / THREADS, a = tid / pow2 * part, z = min(a + part, n);
            const unsigned long long v = s.hist[x];
            uint32_t larger = 0;
            for (int i = a; i < z; ++i) larger += s.hist[i] > v;
            if (larger && x < n) atomicAdd(&s.slots[x], larger);
            __syncthreads();
            if (tid < n) s.list[s.slots[tid]] = s.hist[tid];
            __syncthreads();
            return;
        }
        unsigned long long v[2];
        uint32_t slot[2], k[2], c[2], o[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int x = tid + i * THREADS;
            uint32_t rest;
            v[i] = x < n ? s.hist[x] : 0;
            s.list[x] = v[i];
            if (x >= n) continue;
            const int b = at.bin(of_bits((uint32_t)(v[i] >> 32)), &rest);
            slot[i] = s.start[b] + __umulhi(rest, (uint32_t)tokens(b));
            k[i] = atomicAdd(&s.slots[slot[i]], 1u);
            if (k[i] >= 64) s.hi = 1;
        }
        __syncthreads();
        if (s.hi) {
            sort_list(s, n);
            return;
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) c[i] = s.slots[tid * 2 + i];
        block_scan<uint32_t>(c[0], c[1], &o[0], &o[1], s.wave);
#pragma unroll
        for (int i = 0; i < 2; ++i) s.slots[tid * 2 + i] = o[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (tid + i * THREADS < n) s.list[s.slots[slot[i]] + k[i]] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (tid + i * THREADS >= n) continue;
            k[i] = s.slots[slot[i]];
            const int to = slot[i] + 1 < LIST ? (int)s.slots[slot[i] + 1] : n;
            for (int y = (int)k[i]; y < to; ++y) k[i] += s.list[y] > v[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (tid + i * THREADS < n) s.list[k[i]] = v[i];
        __syncthreads();
    };
    // The bin of a rank, and of a mass (the last one that is not empty and starts below it; for a mass of 0 the
    // largest logit's, which is the second one where its rest was rounded up to a whole bin).
    uint32_t first_rest;
    const int first_bin = at.bin(max, &first_rest);
    auto bin_of_rank = [&](uint32_t rank) {
        int b = 0;
        for (int step = BINS / 2; step; step /= 2)
            if (s.before[b + step] <= rank) b += step;
        return b;
    };
    auto bin_of_mass = [&](double m, bool with_equal) {
        int b = 0;
        for (int step = BINS / 2; step; step /= 2)
            if (with_equal ? s.above[b + step] < m : s.above[b + step] <= m) b += step;
        // (the empty ones behind the last token start at the whole mass)
        while (b > 0 && tokens(b) == 0) --b;
        return std::max(b, first_bin);
    };
    uint32_t kept = live;
    const bool by_k = c.top_k > 0 && (uint32_t)c.top_k < live;
    // min_p's place, from the largest logit's bin on (behind all bins: none)
    const double far = c.min_p > 0.0f ? -log((double)c.min_p) * PER + 1.0 : 2.0 * BINS;
    float least = -__builtin_inff();  // the smallest logit that min_p keeps
    if (c.min_p > 0.0f) least = least_of(max, c.t, c.min_p);

    // The bins up to which tokens can be kept: where they hold few, those are sorted
    // together and every question is one of their sums.
    int cut = BINS - 2;
    if (by_k) cut = bin_of_rank((uint32_t)c.top_k - 1);
    if (!(by_k && c.top_p < 1.0f)) {  // (p is of the k's weight)
        if (c.top_p < 1.0f) cut = min(cut, bin_of_mass((double)c.top_p * all, true));
        if (far < cut) cut = (int)far + 1;
    }
    const int few = (int)s.before[cut + 1];
    if (few <= LIST) {
        bool listed = sl.n > 0;
        if (listed) {
            const int32_t *q = sl.upto + (size_t)r * sl.n * 2;
            listed = __all(cut < q[min(lane, sl.n - 1) * 2] && cut < q[min(lane + 64, sl.n - 1) * 2]);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) s.start[tid * 2 + i] = tid * 2 + i <= cut ? c0[i] : NONE;
        sort_bins(few, [&](auto put) {
            if (listed) {
                for (int i = tid / SLICE_LIST; i < sl.n; i += THREADS / SLICE_LIST) {
                    const size_t x = (size_t)r * sl.n + i;
                    const int k = tid % SLICE_LIST;
                    const unsigned long long v = sl.list[x * SLICE_LIST + k];
                    uint32_t rest;
                    if (k < sl.upto[x * 2 + 1] && at.bin(of_bits((uint32_t)(v >> 32)), &rest) <= cut) put(v);
                }
            } else {
                const float from = at.below(cut);
                each_token<THREADS, AHEAD>(row, n, [&](float l, int i) {
                    uint32_t rest;
                    if (l >= from && at.bin(l, &rest) <= cut) put(token_word(l, i));
                });
            }
        });
        double *w = (double *)s.hist;  // weights
        if (tid == 0) s.n = 0;
        __syncthreads();
        for (int x = tid; x < few; x += THREADS) {
            uint32_t rest;
            const float l = of_bits((uint32_t)(s.list[x] >> 32));
            const int b = at.bin(l, &rest);
            w[x] = scale(b) * (double)((1u << UNIT) - loss(rest));
            if (c.min_p > 0.0f && l >= least) atomicAdd(&s.n, 1u);
        }
        __syncthreads();
        if (tid >= 64) return;
        // the first wave: some neighbouring tokens a lane
        const int some = (few + 63) / 64, x0 = min(lane * some, few), x1 = min(x0 + some, few);
        double mine = 0.0;
        for (int x = x0; x < x1; ++x) mine += w[x];
        double base = __shfl_up(wave_scan<double>(mine), 1, 64);  // the weights before the lane's
        if (lane == 0) base = 0.0;
        // the tokens for which f(weights before it, its own) holds, up to some token
        auto upto = [&](auto f) {
            uint32_t k = 0;
            double up = base;
            for (int x = x0; x < x1; ++x) {
                k += f(up, w[x]);
                up += w[x];
            }
            return __shfl(wave_scan<uint32_t>(k), 63, 64);
        };
        auto sum_upto = [&](uint32_t k) {  // of the first k > 0
            double up = base;
            for (int x = x0; x < x1 && x < (int)k; ++x) up += w[x];
            return __shfl(up, (int)(k - 1) / some, 64);
        };
        kept = (uint32_t)few;
        if (by_k && c.top_k <= few) {
            kept = (uint32_t)c.top_k;
            all = sum_upto(kept);
        }
        if (c.top_p < 1.0f) {
            const double goal = (double)c.top_p * all;
            kept = min(kept, std::max(1u, upto([&](double up, double) { return up < goal; })));
        }
        if (c.min_p > 0.0f) kept = min(kept, std::max(1u, s.n));
        all = sum_upto(kept);
        const double goal = (double)c.u * all;
        const uint32_t x = min(upto([&](double up, double v) { return up + v <= goal; }), kept - 1);
        if (lane == 0) {
            p.token[r] = (int)~(uint32_t)s.list[x];
            if (p.prob) p.prob[r] = (float)(w[x] / all);
        }
        return;
    }

    // Else each question ends in one bin, whose tokens decide it. The bins that they can end in are
    // known but for what those tokens change: they are gathered and sorted together, in one
    // reading, and a question that ends in another bin reads the row for itself.
    int from[4], to[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        from[q] = BINS;
        to[q] = -1;
    }
    auto upto_bin = [&](int b) { return b + 1 < BINS ? s.above[b + 1] : all; };
    uint32_t rest;
    const int least_bin = c.min_p > 0.0f ? at.bin(least, &rest) : BINS - 1;
    double a0 = all, a1 = all;  // the kept ones' weights, between
    if (by_k) {
        from[0] = to[0] = bin_of_rank((uint32_t)c.top_k - 1);
        a0 = s.above[from[0]];
        a1 = upto_bin(to[0]);
    }
    if (c.top_p < 1.0f) {
        from[1] = bin_of_mass((double)c.top_p * a0, true);
        to[1] = bin_of_mass((double)c.top_p * a1, true);
        a0 = s.above[from[1]];
        a1 = upto_bin(to[1]);
    }
    if (least_bin < BINS - 1 && s.above[least_bin] < a1) {
        from[2] = to[2] = least_bin;
        a0 = fmin(a0, s.above[least_bin]);
        a1 = fmin(a1, upto_bin(least_bin));
    }
    from[3] = bin_of_mass((double)c.u * a0, false);
    to[3] = bin_of_mass((double)c.u * a1, false);
    uint32_t some[2], start[2];
    bool in[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        in[i] = false;
#pragma unroll
        for (int q = 0; q < 4; ++q) in[i] |= from[q] <= tid * 2 + i && tid * 2 + i <= to[q];
        some[i] = in[i] ? cnt[i] : 0;
    }
    const uint32_t together = block_scan<uint32_t>(some[0], some[1], &start[0], &start[1], s.wave);
    bool listed = together <= LIST;
    if (listed) {
        const int first = std::min(std::min(from[0], from[1]), std::min(from[2], from[3]));
        const int last = std::max(std::max(to[0], to[1]), std::max(to[2], to[3]));
#pragma unroll
        for (int i = 0; i < 2; ++i) s.start[tid * 2 + i] = in[i] ? start[i] : NONE;
        const float least_l = at.below(last), most_l = at.above(first);
        sort_bins((int)together, [&](auto put) {
            each_token<THREADS, AHEAD>(row, n, [&](float l, int i) {
                uint32_t rest;
                if (l >= least_l && l <= most_l && s.start[at.bin(l, &rest)] != NONE) put(token_word(l, i));
            });
        });
        sum_losses(s, (int)together, at);
    }
    for (int question = 0; question < 5; ++question) {
        int b;
        bool by_rank = false, with_equal = false;
        uint32_t rank = 0;
        double goal = 0.0;
        if (question == 0) {  // the k-th
            if (!by_k) continue;
            kept = (uint32_t)c.top_k;
            by_rank = true;
        } else if (question == 1) {  // p of their weight
            if (!(c.top_p < 1.0f)) continue;
            goal = (double)c.top_p * all;
            with_equal = true;
        } else if (question == 2) {  // what min_p keeps
            if (c.min_p == 0.0f) continue;
            if (least_bin == BINS - 1 || s.before[least_bin] >= kept) continue;
            uint32_t k = 0;
            if (listed && s.start[least_bin] != NONE) {
                int i = 0, z = tokens(least_bin);
                const uint32_t key = order_bits(least), x0 = s.start[least_bin];
                while (i < z) {
                    const int mid = (i + z) / 2;
                    if ((uint32_t)(s.list[x0 + mid] >> 32) >= key)
                        i = mid + 1;
                    else
                        z = mid;
                }
                k = s.before[least_bin] + i;
            } else {
                each_token<THREADS, AHEAD>(row, n, [&](float l, int) { k += l >= least; });
                __syncthreads();
                if (tid == 0) s.n = 0;
                __syncthreads();
                atomicAdd(&s.n, k);
                __syncthreads();
                k = s.n;
                __syncthreads();
            }
            k = std::max(1u, k);
            if (k >= kept) continue;
            kept = k;
            by_rank = true;
        } else if (question == 3) {  // the token
            goal = (double)c.u * all;
        } else {  // a rounding put the goal behind the last one
            by_rank = true;
        }
        b = by_rank ? bin_of_rank(kept - 1) : bin_of_mass(goal, with_equal);
        if (by_rank) rank = kept - 1 - s.before[b];
        const double mass = (goal - s.above[b]) / scale(b);
        Found f;
        if (listed && s.start[b] != NONE) {
            f = place_in(s, (int)s.start[b], tokens(b), by_rank, rank, mass, with_equal);
        } else {
            __syncthreads();
            listed = false;  // (the list is written over)
            f = locate<AHEAD>(s, row, n, at, b, tokens(b), by_rank, rank, mass, with_equal);
        }
        const uint32_t upto = s.before[b] + f.rank + 1;
        if (question < 3) {
            if (question == 1 && upto >= kept) continue;
            kept = upto;
            all = s.above[b] + scale(b) * (double)f.upto;
            continue;
        }
        if (question == 3 && upto > kept) continue;
        if (tid == 0) {
            p.token[r] = (int)f.token;
            if (p.prob) p.prob[r] = (float)(scale(b) * (double)((1u << UNIT) - f.d) / all);
        }
        return;
    }
}

// The first token of a row or a slice, by its workgroup.
template <int T>
__device__ __forceinline__ unsigned long long most_of(unsigned long long v, unsigned long long *scratch) {
    v = wave_most(v);
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < T / 64; ++i) v = scratch[i] > v ? scratch[i] : v;
    __syncthreads();
    return v;
}

// The bins of a whole row whose largest logit is known.
__device__ __forceinline__ void count_row(Shared &s, const float *row, int n, const Place &at) {
    for (int i = threadIdx.x; i < BINS; i += THREADS) s.hist[i] = 0;
    __syncthreads();
    each_token<THREADS, false>(row, n, [&](float l, int) { count_token(s.hist, at, l); });
    __syncthreads();
}

// A workgroup a row; two of them on a CU, though 38 vector registers are spilled for that (in the gathers, the scans and the
// decisions; the first reading is free of it): 512 rows of 122753 with mixed settings 115 us, 141 with registers
// enough for one alone. (The last kernel of slices, one a CU, spills 12.)
__global__ __launch_bounds__(THREADS, 8) void sample_row_kernel(SampleParams p) {
    __shared__ Shared s;
    const int r = blockIdx.x, tid = threadIdx.x, n = p.vocab;
    const Settings c = settings_of(p, r, true);
    if (!c.live) return;
    const float *row = p.logits + r * p.ld;
    for (int i = tid; i < BINS; i += THREADS) s.hist[i] = 0;
    unsigned long long best = 0;  // (without the index where T > 0)
    Place at;
    for (int first = 0; first < n; first += THREADS * 16) {
        Tokens<THREADS> now;
        now.load(row, first, n);
        unsigned long long v = 0;
        if (c.t == 0.0f) {
            now.each(first, [&](float l, int i) {
                const unsigned long long t = l == l ? token_word(l, i) : WITH_NAN;
                v = t > v ? t : v;
            });
        } else {
            float m = -__builtin_inff();
            bool nan = false;
            now.each(first, [&](float l, int) {
                nan |= l != l;
                m = fmaxf(m, l);
            });
            v = nan ? WITH_NAN : (unsigned long long)order_bits(m) << 32;
        }
        v = most_of<THREADS>(v, s.wave64);
        if (v == WITH_NAN) {
            best = v;
            break;
        }
        if (v > best) {
            best = v;
            const float max = of_bits((uint32_t)(v >> 32));
            if (c.t > 0.0f && fabsf(max) <= 3.40282347e38f) {
                const Place old = at;
                at = Place(c.t, max);
                // the bins so far move behind by as many as the largest logit came before
                const double d = fmin(old.ref - at.ref, (double)BINS);
                const int by = old.per == 0.0 ? 0 : (int)d;
                if (by > 0) {
                    unsigned long long h[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int x = tid + i * THREADS - by;
                        h[i] = x >= 0 && tid + i * THREADS < BINS - 1 ? s.hist[x] : 0;
                    }
                    __syncthreads();
                    s.hist[tid] = h[0];
                    s.hist[tid + THREADS] = h[1];
                    __syncthreads();
                }
            }
        }
        if (c.t > 0.0f && at.per != 0.0) now.each(first, [&](float l, int) { count_token(s.hist, at, l); });
    }
    if (settled(p, r, c, best)) return;
    const float max = of_bits((uint32_t)(best >> 32));
    __syncthreads();
    // (The last place alone counts. A mask's lowest value may have set one before it that was too far: what
    // was counted there has moved behind all bins since, or that place is within BINS of the last one's, below
    // 2^50, where bins and rests are exact.)
    if (at.too_far(max)) {
        at.widen(max);
        count_row(s, row, n, at);
    }
    finish<false>(s, p, r, c, max, at, SampleSlices{0, nullptr, nullptr, nullptr, nullptr});
}

// Few rows: a workgroup for each slice of them leaves its first token, its bins and the tokens of
// the first ones, then a workgroup a row ends it.
constexpr int SLICE_THREADS = 512, SLICE = SLICE_THREADS * 16;
__global__ __launch_bounds__(SLICE_THREADS) void sample_slice_kernel(SampleParams p, SampleSlices sl) {
    __shared__ unsigned long long hist[BINS], scratch[SLICE_THREADS / 64];
    __shared__ uint32_t wave[SLICE_THREADS / 64], count, last;
    const int r = blockIdx.y, first = blockIdx.x * SLICE, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const float *row = p.logits + r * p.ld;
    Tokens<SLICE_THREADS> now;
    now.load(row, first, p.vocab);
    const Settings c = settings_of(p, r, false);
    if (!c.live) return;
    for (int i = tid; i < BINS; i += SLICE_THREADS) hist[i] = 0;
    if (tid == 0) {
        count = 0;
        last = 0;
    }
    unsigned long long v = 0;
    now.each(first, [&](float l, int i) {
        const unsigned long long t = l == l ? token_word(l, i) : WITH_NAN;
        v = t > v ? t : v;
    });
    v = most_of<SLICE_THREADS>(v, scratch);
    const size_t x = (size_t)r * sl.n + blockIdx.x;
    const float max = of_bits((uint32_t)(v >> 32));
    if (tid == 0) sl.best[x] = v;
    if (v == WITH_NAN || !(fabsf(max) <= 3.40282347e38f) || c.t == 0.0f) {
        // (nothing but its first token is asked of it; a slice without a token has empty bins)
        if (max == -__builtin_inff() && c.t > 0.0f) {
            for (int i = tid; i < BINS; i += SLICE_THREADS) sl.hist[x * BINS + i] = 0;
            if (tid == 0) {
                sl.upto[x * 2] = BINS - 1;
                sl.upto[x * 2 + 1] = 0;
            }
        }
        return;
    }
    const Place at(c.t, max);
    now.each(first, [&](float l, int) { count_token(hist, at, l); });
    __syncthreads();
    // the bins that hold at most SLICE_LIST tokens together
    constexpr int EACH = BINS / SLICE_THREADS;
    uint32_t cnt[EACH], sum = 0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const unsigned long long h = hist[tid * EACH + i];
        sl.hist[x * BINS + tid * EACH + i] = h;
        cnt[i] = (uint32_t)(h >> COUNT);
        sum += cnt[i];
    }
    uint32_t to = wave_scan<uint32_t>(sum);
    if (lane == 63) wave[w] = to;
    __syncthreads();
    to -= sum;
    for (int i = 0; i < w; ++i) to += wave[i];
    int upto = 0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        to += cnt[i];
        if (to <= SLICE_LIST) upto = min(tid * EACH + i + 1, BINS - 1);
    }
    const unsigned long long some = __ballot(upto > 0);
    if (some && lane == 63 - __builtin_clzll(some)) atomicMax(&last, (uint32_t)upto);
    __syncthreads();
    upto = (int)last;
    now.each(first, [&](float l, int i) {
        uint32_t rest;
        if (at.bin(l, &rest) < upto) {
            const uint32_t k = atomicAdd(&count, 1u);
            if (k < SLICE_LIST) sl.list[x * SLICE_LIST + k] = token_word(l, i);
        }
    });
    __syncthreads();
    if (tid == 0) {
        sl.upto[x * 2] = at.too_far(max) ? -1 : upto;
        sl.upto[x * 2 + 1] = (int)count;
    }
}

__global__ __launch_bounds__(THREADS) void sample_finish_kernel(SampleParams p, SampleSlices sl) {
    __shared__ Shared s;
    __shared__ int shift[128];
    const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
    const Settings c = settings_of(p, r, true);
    if (!c.live) return;
    // (a lane two slices at most; by every wave)
    const unsigned long long *bp = sl.best + (size_t)r * sl.n;
    int32_t *up = sl.upto + (size_t)r * sl.n * 2;
    unsigned long long b[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) b[i] = bp[min(lane + 64 * i, sl.n - 1)];
    const unsigned long long best = wave_most(b[0] > b[1] ? b[0] : b[1]);
    if (settled(p, r, c, best)) return;
    const float max = of_bits((uint32_t)(best >> 32));
    Place at(c.t, max);
    if (at.too_far(max)) {
        at.widen(max);
        count_row(s, p.logits + r * p.ld, p.vocab, at);
        finish<true>(s, p, r, c, max, at, SampleSlices{0, nullptr, nullptr, nullptr, nullptr});
        return;
    }
    if (tid < 64) {  // the bins of a slice stand behind the row's by as many as its largest logit's
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float m = of_bits((uint32_t)(b[i] >> 32));
            const int x = lane + 64 * i;
            int by = 0;
            if (m > -__builtin_inff()) by = (int)fmin(Place(c.t, m).ref - at.ref, (double)BINS);
            if (x < sl.n) {
                shift[x] = by;
                up[x * 2] += by;
            }
        }
    }
    __syncthreads();
    unsigned long long h0 = 0, h1 = 0;
    const unsigned long long *h = sl.hist + (size_t)r * sl.n * BINS;
    for (int i = 0; i < sl.n; i += 8) {
        unsigned long long v[8][2];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int x = min(i + k, sl.n - 1), at0 = tid * 2 - shift[x];
            v[k][0] = h[(size_t)x * BINS + std::max(at0, 0)];
            v[k][1] = h[(size_t)x * BINS + std::max(at0 + 1, 0)];
            if (at0 < 0 || i + k >= sl.n) v[k][0] = 0;
            if (at0 + 1 < 0 || i + k >= sl.n) v[k][1] = 0;
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            h0 += v[k][0];
            h1 += v[k][1];
        }
    }
    s.hist[tid * 2] = h0;
    s.hist[tid * 2 + 1] = tid == THREADS - 1 ? 0 : h1;  // (what has no weight)
    __syncthreads();
    finish<true>(s, p, r, c, max, at, sl);
}

// Slices where a row is long and rows do not fill the chip by themselves: two launches and
// the bins' way through memory cost more than a row's own workgroup does from there on. (us with top_k 50 in slices and not:
// a row of 16384 21 and 16, of 30000 21 both, 40000 22 and 26, 122753 25 and 50; 32 of 122753 31 and 52, 64 of 40000 25
// and 27. Beyond: 200 of 30000 33 and 24, but 64 of 122753 38 and 54: the longest rows would still gain.)
int slices_of(int rows, int vocab) {
    const int n = (vocab + SLICE - 1) / SLICE;
    return n >= 4 && (long long)rows * n <= 512 ? n : 0;
}

}  // namespace

size_t sample_work_bytes(int rows, int vocab) {
    const size_t n = slices_of(rows, vocab);
    return rows * n * ((BINS + SLICE_LIST + 1) * 8 + 8);
}

int launch_sample(const SampleArgs &a, hipStream_t st) {
    const SampleParams p{a.logits, a.ld,    a.u,    a.t,     a.top_p, a.min_p,
                         a.top_k,  a.rows, a.vocab, a.token, a.prob,  guard_flag_ptr()};
    SampleSlices sl;
    sl.n = slices_of(a.rows, a.vocab);
    if (sl.n == 0) {
        sample_row_kernel<<<(unsigned)a.rows, THREADS, 0, st>>>(p);
        VMLM_HIP_CHECK(hipGetLastError());
        return VMLM_OK;
    }
    VMLM_GUARD(a.work, "sample: sliced rows need a workspace");
    const size_t x = (size_t)a.rows * sl.n;
    sl.hist = (unsigned long long *)a.work;
    sl.list = sl.hist + x * BINS;
    sl.best = sl.list + x * SLICE_LIST;
    sl.upto = (int32_t *)(sl.best + x);
    sample_slice_kernel<<<dim3((unsigned)sl.n, (unsigned)a.rows), SLICE_THREADS, 0, st>>>(p, sl);
    VMLM_HIP_CHECK(hipGetLastError());
    sample_finish_kernel<<<(unsigned)a.rows, THREADS, 0, st>>>(p, sl);
    VMLM_HIP_CHECK(hipGetLastError());
    return VMLM_OK;
}

}  // namespace vmlm
