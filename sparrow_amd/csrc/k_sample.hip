// k_sample.hip -- one token of each row of logits, drawn with a given random number
// (vmlm_hip_sample).
//
// The tokens stand in the order of their logits, the largest first, of equal ones the
// lowest index; token j has the weight w_j = exp((l_j - l_max) / T). Kept are the first k of
// them, of those the ones before which the weights sum to less than p of the k's, of those
// the ones with w_j >= min_p. The token is the first whose weights up to it sum to more
// than u times the kept ones'.
//
// Nothing is sorted but one bin: the distance x = (l_max - l) / T falls into bins of 1/64,
// and every question (the k-th token, the mass p, the token drawn) is answered by the
// bins' counts and masses down to one bin, whose few tokens are gathered and sorted.
// 2048 bins reach weights of 2^-46; what lies behind has none.
//
// Next to a border between two tokens 32 bits are too few: with 122753 tokens of like weight
// a sum off by 2^-24 takes the neighbour's token once in 50 rows. So x is formed in 64 bits, and a
// token's weight is exp(-bin / 64) (1 - d), d = 1 - exp(-r) < 1/64 of the rest r, held as an
// integer in units of 2^-30: a bin's sum of d and its count are one 64-bit atomic add in
// LDS, whose order changes nothing.
#include "internal.hpp"

namespace vmlm {
namespace {

constexpr int THREADS = 1024;
constexpr int BINS = 2048;      // the last one's tokens have no weight
constexpr int LIST = 2048;      // tokens that are sorted at once
constexpr int SLICE_LIST = 256; // tokens of the first bins that a slice lists
constexpr double PER = 64.0;    // bins of a distance of 1
constexpr int UNIT = 30;        // d in units of 2^-30
constexpr int COUNT = 44;       // a bin's word: count above, sum of d below

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

// Order-preserving bits of a logit (of numbers; -0 as 0).
__device__ __forceinline__ uint32_t order_bits(float v) {
    if (v == 0.0f) v = 0.0f;
    const uint32_t b = __float_as_uint(v);
    return (b >> 31) ? ~b : b | 0x80000000u;
}

// A logit's place: its bin, and the rest of its distance as a fraction of a bin in units of
// 2^-32. 2^20 added to the distance leaves both in the bits of the sum.
struct Place {
    double max, per;  // PER / T
    __device__ __forceinline__ int bin(float l, uint32_t *rest) const {
        const double y = __builtin_fma(max - (double)l, per, 0x1p20);  // (+inf for a masked one)
        const unsigned long long b = __builtin_bit_cast(unsigned long long, y);
        *rest = (uint32_t)b;
        return (int)min((uint32_t)(b >> 32) - 0x41300000u, (uint32_t)(BINS - 1));
    }
    // Logits below this one are not in bin b or before it; above it, not in bin b or behind it.
    // (f32: by a part of a bin, and where a bin is narrower than its steps by a few of those)
    __device__ __forceinline__ float below(int b) const {
        return (float)(max - ((double)b + 1.02) / per - fabs(max) * 0x1p-21);
    }
    __device__ __forceinline__ float above(int b) const {
        return (float)(max - ((double)b - 0.02) / per + fabs(max) * 0x1p-21);
    }
};
// 1 - exp(-r) of the rest r = f 2^-38 < 2^-6, in units of 2^-30, off by at most one: r itself
// from the bits, the other terms below 2^-13 in f32 (the next of the series is below 2^-36)
__device__ __forceinline__ uint32_t loss(uint32_t f) {
    const float r = (float)f * 0x1p-38f;
    const float q = r * r * __builtin_fmaf(__builtin_fmaf(r, 1.0f / 24, -1.0f / 6), r, 0.5f);
    return (uint32_t)((f >> 8) + (f >> 7 & 1)) - (uint32_t)(int)rintf(q * 0x1p30f);
}

// Calls f(logit, index) for the tokens [0, n) at `row`: 16 of a thread at a time, loaded
// before the first is used. T: threads.
template <int T, typename F>
__device__ __forceinline__ void each_token(const float *row, int n, F f) {
    int i = threadIdx.x * 4;
    for (; i + 3 + 3 * T * 4 < n; i += 4 * T * 4) {
        f32x4a v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = *(const f32x4a *)(row + i + k * T * 4);
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) f(v[k][e], i + k * T * 4 + e);
    }
    for (; i + 3 < n; i += T * 4) {
        const f32x4a v = *(const f32x4a *)(row + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) f(v[e], i + e);
    }
    for (; i < n; ++i) f(row[i], i);
}

struct Shared {
    unsigned long long hist[BINS];  // counts and losses; then, in a bin, of key ranges, and up to a token
    double above[BINS];             // the mass before a bin
    uint32_t before[BINS];          // the tokens before a bin
    unsigned long long list[LIST];  // (order bits, ~index), the largest first
    uint32_t rank[512];
    double red[16];
    unsigned long long wave64[16];
    unsigned long long best;
    uint32_t n, lo, hi;
    uint32_t wave[16];
};

// Block-wide exclusive prefix sums over 2 values a thread.
template <typename T>
__device__ T block_scan(T a, T b, T *out_a, T *out_b, T *scratch) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    T to = a + b;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
        const T v = __shfl_up(to, o, 64);
        if (lane >= o) to = to + v;
    }
    if (lane == 63) scratch[w] = to;
    __syncthreads();
    T base = 0, all = 0;
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

// The n <= LIST tokens that `each` puts, (order bits, ~index), in s.list: the largest first. Up
// to 512 by the number of larger ones, which as many threads as there are count together
// (256 tokens: 64 reads each, where a sort of them has 36 steps); more by a bitonic sort.
template <typename F>
__device__ void gather(Shared &s, int n, F each) {
    const int tid = threadIdx.x;
    const bool count = n <= 512;
    unsigned long long *raw = count ? s.hist : s.list;
    __syncthreads();
    if (tid == 0) s.n = 0;
    int pow2 = 64;
    while (pow2 < n) pow2 *= 2;
    for (int i = tid; i < pow2; i += THREADS) raw[i] = 0;
    if (count && tid < 512) s.rank[tid] = 0;
    __syncthreads();
    each([&](unsigned long long v) {
        const uint32_t k = atomicAdd(&s.n, 1u);
        if (k < LIST) raw[k] = v;
    });
    __syncthreads();
    if (count) {
        const int parts = THREADS / pow2, x = tid % pow2, each_part = pow2 / parts, a = tid / pow2 * each_part;
        const unsigned long long v = raw[x];
        uint32_t larger = 0;
        for (int i = a; i < a + each_part; ++i) larger += raw[i] > v;
        if (larger) atomicAdd(&s.rank[x], larger);
        __syncthreads();
        if (tid < n) s.list[s.rank[tid]] = raw[tid];
        __syncthreads();
        return;
    }
    for (int k = 2; k <= pow2; k *= 2)
        for (int j = k / 2; j > 0; j /= 2) {
            for (int i = tid; i < pow2 / 2; i += THREADS) {
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

// The token of rank `rank` in bin `bin` (by_rank), else the first one with weights up to it of
// more than `mass` (or, with_equal, as much). `n`: the bin's tokens.
__device__ Found locate(Shared &s, const float *row, int vocab, const Place &at, int bin, int n,
                        bool by_rank, uint32_t rank, double mass, bool with_equal) {
    const int tid = threadIdx.x;
    uint32_t lo = 0, hi = 0xffffffffu;  // of the order bits
    const float from = at.below(bin), to = at.above(bin);
    uint32_t rank0 = 0;                 // the bin's tokens above them, and their weights
    unsigned long long mass0 = 0;
    // 1. a bin of too many tokens: ranges of their order bits, the narrowest that hold the place
    while (n > LIST && lo < hi) {
        __syncthreads();
        if (tid == 0) {
            s.lo = 0xffffffffu;
            s.hi = 0;
        }
        for (int i = tid; i < BINS; i += THREADS) s.hist[i] = 0;
        __syncthreads();
        each_token<THREADS>(row, vocab, [&](float l, int) {
            uint32_t rest;
            const uint32_t key = order_bits(l);
            if (l >= from && l <= to && at.bin(l, &rest) == bin && key >= lo && key <= hi) {
                atomicMin(&s.lo, key);
                atomicMax(&s.hi, key);
            }
        });
        __syncthreads();
        lo = s.lo;
        hi = s.hi;
        if (lo == hi) break;
        int shift = 0;
        while ((hi - lo) >> shift >= BINS) ++shift;
        each_token<THREADS>(row, vocab, [&](float l, int) {
            uint32_t rest;
            const uint32_t key = order_bits(l);
            if (l >= from && l <= to && at.bin(l, &rest) == bin && key >= lo && key <= hi)
                atomicAdd(&s.hist[(hi - key) >> shift], (1ull << COUNT) | loss(rest));
        });
        __syncthreads();
        if (tid == 0) {
            uint32_t r = rank0;
            unsigned long long m = mass0;
            int i = 0, last = 0;
            uint32_t rl = r;
            unsigned long long ml = m;
            for (; i < BINS; ++i) {  // the last range that is not empty where none reaches it
                const uint32_t c = (uint32_t)(s.hist[i] >> COUNT);
                if (c == 0) continue;
                const unsigned long long w =
                    ((unsigned long long)c << UNIT) - (s.hist[i] & ((1ull << COUNT) - 1));
                last = i;
                rl = r;
                ml = m;
                if (by_rank ? r + c > rank
                            : with_equal ? (double)(m + w) >= mass : (double)(m + w) > mass)
                    break;
                r += c;
                m += w;
            }
            s.n = (uint32_t)last;
            s.wave[0] = rl;
            s.best = ml;
        }
        __syncthreads();
        const int i = (int)s.n;
        rank0 = s.wave[0];
        mass0 = s.best;
        n = (int)(s.hist[i] >> COUNT);
        const uint32_t top = hi - ((uint32_t)i << shift);
        const uint32_t bottom = hi - (uint32_t)min((((unsigned long long)i + 1) << shift) - 1, (unsigned long long)(hi - lo));
        hi = top;
        lo = bottom;
        __syncthreads();
    }
    Found f;
    if (n > LIST) {  // 2. so many equal ones: the place is arithmetic, its index a count
        __syncthreads();
        if (tid == 0) s.n = 0;
        __syncthreads();
        each_token<THREADS>(row, vocab, [&](float l, int) {
            uint32_t rest;
            if (order_bits(l) == lo) {
                at.bin(l, &rest);
                s.n = loss(rest);
            }
        });
        __syncthreads();
        f.d = s.n;
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
    gather(s, n, [&](auto put) {
        each_token<THREADS>(row, vocab, [&](float l, int i) {
            uint32_t rest;
            const uint32_t key = order_bits(l);
            if (l >= from && l <= to && key >= lo && key <= hi && at.bin(l, &rest) == bin) put((unsigned long long)key << 32 | (uint32_t)~i);
        });
    });
    static_assert(LIST == BINS && LIST == 2 * THREADS, "");
    unsigned long long *sum = s.hist, d[2], e[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int x = tid * 2 + i;
        uint32_t rest;
        d[i] = 0;
        if (x < n) {
            at.bin(row[~(uint32_t)s.list[x]], &rest);
            d[i] = loss(rest);
        }
    }
    block_scan<unsigned long long>(d[0], d[1], &e[0], &e[1], s.wave64);
    if (tid == 0) s.lo = n - 1;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int x = tid * 2 + i;
        if (x >= n) continue;
        sum[x] = e[i] + d[i];
        const unsigned long long w = mass0 + ((unsigned long long)(x + 1) << UNIT) - (e[i] + d[i]);
        const bool hit = by_rank ? rank0 + x == rank
                                 : with_equal ? (double)w >= mass : (double)w > mass;
        if (hit) atomicMin(&s.lo, (uint32_t)x);
    }
    __syncthreads();
    const uint32_t x = s.lo;
    f.rank = rank0 + x;
    f.upto = mass0 + ((unsigned long long)(x + 1) << UNIT) - sum[x];
    f.d = (uint32_t)(sum[x] - (x ? sum[x - 1] : 0));
    f.token = ~(uint32_t)s.list[x];
    __syncthreads();
    return f;
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

__device__ __forceinline__ unsigned long long wave_most(unsigned long long v) {
#pragma unroll
    for (int o = 32; o; o /= 2) {
        const unsigned long long w = (unsigned long long)__shfl_xor((uint32_t)(v >> 32), o, 64) << 32 |
                                     (uint32_t)__shfl_xor((uint32_t)v, o, 64);
        v = w > v ? w : v;
    }
    return v;
}

// The largest of some tokens, the first of equal ones: (order bits, ~index); a NaN above all.
constexpr unsigned long long WITH_NAN = ~0ull;
template <int T>
__device__ unsigned long long largest(const float *row, int n, int first, unsigned long long *scratch) {
    uint32_t best = 0, index = 0;
    bool nan = false;
    each_token<T>(row, n, [&](float l, int i) {
        nan |= l != l;
        const uint32_t key = order_bits(l);
        if (key > best) {
            best = key;
            index = i;
        }
    });
    unsigned long long v = nan ? WITH_NAN : (unsigned long long)best << 32 | (uint32_t)~(first + index);
    v = wave_most(v);
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < T / 64; ++i) v = scratch[i] > v ? scratch[i] : v;
    __syncthreads();
    return v;
}
// the logit that the order bits came from
__device__ __forceinline__ float of_bits(uint32_t b) { return __uint_as_float((b >> 31) ? b ^ 0x80000000u : ~b); }

// Counts and losses of some tokens into the bins.
template <int T>
__device__ __forceinline__ void count_bins(unsigned long long *hist, const float *row, int n, const Place &at) {
    each_token<T>(row, n, [&](float l, int) {
        uint32_t rest;
        const int b = at.bin(l, &rest);
        if (b < BINS - 1) atomicAdd(&hist[b], (1ull << COUNT) | loss(rest));
    });
}

// What the slices of a row leave for its last kernel.
struct SampleSlices {
    int n, each;                     // their number and tokens
    unsigned long long *best;        // [rows][n] the largest token
    unsigned long long *hist;        // [rows][n][BINS]
    unsigned long long *list;        // [rows][n][SLICE_LIST] the tokens of the first bins
    int32_t *upto;                   // [rows][n][2]: those below this bin, and their number
};

// 3. The rest, from a row's bins in s.hist: by one workgroup.
__device__ void finish(Shared &s, const SampleParams &p, int r, const Settings &c, float first,
                       const SampleSlices &sl) {
    const int tid = threadIdx.x, n = p.vocab;
    const float *row = p.logits + r * p.ld;
    const float u = c.u, t = c.t;
    auto answer = [&](int token, float prob) {
        if (tid == 0) {
            p.token[r] = token;
            if (p.prob) p.prob[r] = prob;
        }
    };
    const Place at{(double)first, PER / (double)t};
    uint32_t cnt[2], c0[2];
    double mass[2], m0[2];
    const double unit = 1.0 / (1 << UNIT);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const unsigned long long h = s.hist[tid * 2 + i];
        cnt[i] = (uint32_t)(h >> COUNT);
        mass[i] = exp(-(tid * 2 + i) / PER) * unit *
                  (double)(((unsigned long long)cnt[i] << UNIT) - (h & ((1ull << COUNT) - 1)));
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
    auto scale = [&](int b) { return exp(-b / PER) * unit; };
    // the bin of a rank, and of a mass (the last one that is not empty and starts below it)
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
        return b;
    };
    uint32_t kept = live;
    const bool by_k = c.top_k > 0 && (uint32_t)c.top_k < live;
    const double far = -log((double)c.min_p) * PER;  // min_p's place (+inf: none)

    // The bins up to which tokens can be kept: where they hold few, those are sorted
    // together and every question is one of their sums.
    int cut = BINS - 2;
    if (by_k) cut = bin_of_rank((uint32_t)c.top_k - 1);
    if (!(by_k && c.top_p < 1.0f)) {  // (p is of the k's weight)
        if (c.top_p < 1.0f) cut = bin_of_mass((double)c.top_p * all, true);
        if (far < cut) cut = (int)far + 1;
    }
    const int few = (int)s.before[cut + 1];
    if (few <= LIST) {
        bool listed = sl.n > 0;
        if (listed) {
            const int lane = tid & 63;
            const int32_t *q = sl.upto + (size_t)r * sl.n * 2;
            listed = __all(cut < q[min(lane, sl.n - 1) * 2] && cut < q[min(lane + 64, sl.n - 1) * 2]);
        }
        gather(s, few, [&](auto put) {
            if (listed) {
                for (int i = tid / SLICE_LIST; i < sl.n; i += THREADS / SLICE_LIST) {
                    const size_t x = (size_t)r * sl.n + i;
                    const int k = tid % SLICE_LIST;
                    if (k >= sl.upto[x * 2 + 1]) continue;
                    const unsigned long long v = sl.list[x * SLICE_LIST + k];
                    uint32_t rest;
                    if (at.bin(of_bits((uint32_t)(v >> 32)), &rest) <= cut) put(v);
                }
            } else {
                const float from = at.below(cut);
                each_token<THREADS>(row, n, [&](float l, int i) {
                    uint32_t rest;
                    if (l >= from && at.bin(l, &rest) <= cut) put((unsigned long long)order_bits(l) << 32 | (uint32_t)~i);
                });
            }
        });
        double w[2], up[2];
        bool over[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int x = tid * 2 + i;
            w[i] = 0.0;
            over[i] = false;
            if (x < few) {
                uint32_t rest;
                const float l = of_bits((uint32_t)(s.list[x] >> 32));
                const int b = at.bin(l, &rest);
                w[i] = scale(b) * (double)((1u << UNIT) - loss(rest));
                over[i] = c.min_p == 0.0f || exp(((double)l - at.max) / (double)t) >= (double)c.min_p;
            }
        }
        block_scan<double>(w[0], w[1], &up[0], &up[1], s.red);  // weights before a token
        // counts of a condition that holds up to some token
        auto upto = [&](bool a, bool b) {
            uint32_t x, y;
            return block_scan<uint32_t>(a, b, &x, &y, s.wave);
        };
        auto sum_upto = [&](uint32_t k) {  // of the first k > 0
            if (tid == (int)(k - 1) / 2) s.red[0] = (k - 1) % 2 ? up[1] + w[1] : up[0] + w[0];
            __syncthreads();
            const double v = s.red[0];
            __syncthreads();
            return v;
        };
        kept = (uint32_t)few;
        if (by_k && c.top_k <= few) {
            kept = (uint32_t)c.top_k;
            all = sum_upto(kept);
        }
        if (c.top_p < 1.0f) {
            const double goal = (double)c.top_p * all;
            kept = min(kept, max(1u, upto(tid * 2 < few && up[0] < goal, tid * 2 + 1 < few && up[1] < goal)));
        }
        if (c.min_p > 0.0f) kept = min(kept, max(1u, upto(over[0], over[1])));
        all = sum_upto(kept);
        const double goal = (double)u * all;
        const uint32_t x = min(upto(tid * 2 < few && up[0] + w[0] <= goal, tid * 2 + 1 < few && up[1] + w[1] <= goal),
                               kept - 1);
        if (tid == (int)x / 2) {
            p.token[r] = (int)~(uint32_t)s.list[x];
            if (p.prob) p.prob[r] = (float)((x % 2 ? w[1] : w[0]) / all);
        }
        return;
    }

    // Else each question by its bin.
    if (by_k) {
        kept = (uint32_t)c.top_k;
        const int b = bin_of_rank(kept - 1);
        const Found f = locate(s, row, n, at, b, tokens(b), true, kept - 1 - s.before[b], 0.0, false);
        all = s.above[b] + scale(b) * (double)f.upto;
    }
    if (c.top_p < 1.0f) {
        const double goal = (double)c.top_p * all;
        const int b = bin_of_mass(goal, true);
        const Found f = locate(s, row, n, at, b, tokens(b), false, 0, (goal - s.above[b]) / scale(b), true);
        const uint32_t k = s.before[b] + f.rank + 1;
        if (k < kept) {
            kept = k;
            all = s.above[b] + scale(b) * (double)f.upto;
        }
    }
    if (c.min_p > 0.0f) {
        // (weights next to the border in 64 bits, the others by their bin)
        uint32_t k = 0;
        each_token<THREADS>(row, n, [&](float l, int) {
            uint32_t rest;
            const int b = at.bin(l, &rest);
            if (b == BINS - 1) return;
            if (fabs((double)b - far) > 2.0)
                k += (double)b < far;
            else
                k += exp(((double)l - at.max) / (double)t) >= (double)c.min_p;
        });
        if (tid == 0) s.n = 0;
        __syncthreads();
        atomicAdd(&s.n, k);
        __syncthreads();
        k = s.n;
        __syncthreads();
        if (k < kept) {
            kept = k;
            const int b = bin_of_rank(kept - 1);
            const Found f = locate(s, row, n, at, b, tokens(b), true, kept - 1 - s.before[b], 0.0, false);
            all = s.above[b] + scale(b) * (double)f.upto;
        }
    }
    const double goal = (double)u * all;
    int b = bin_of_mass(goal, false);
    Found f = locate(s, row, n, at, b, tokens(b), false, 0, (goal - s.above[b]) / scale(b), false);
    if (s.before[b] + f.rank >= kept) {  // (a rounding put the goal behind the last one)
        b = bin_of_rank(kept - 1);
        f = locate(s, row, n, at, b, tokens(b), true, kept - 1 - s.before[b], 0.0, false);
    }
    answer((int)f.token, (float)(scale(b) * (double)((1u << UNIT) - f.d) / all));
}

// What there is to say of a row whose largest token is known; true if nothing else is.
__device__ __forceinline__ bool settled(const SampleParams &p, int r, const Settings &c, unsigned long long best,
                                        bool write) {
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
    if (write && threadIdx.x == 0) {
        p.token[r] = token;
        if (p.prob) p.prob[r] = prob;
    }
    return true;
}

// A workgroup a row.
__global__ __launch_bounds__(THREADS) void sample_row_kernel(SampleParams p) {
    __shared__ Shared s;
    const int r = blockIdx.x;
    const Settings c = settings_of(p, r, true);
    if (!c.live) return;
    const float *row = p.logits + r * p.ld;
    for (int i = threadIdx.x; i < BINS; i += THREADS) s.hist[i] = 0;
    const unsigned long long best = largest<THREADS>(row, p.vocab, 0, s.wave64);
    if (settled(p, r, c, best, true)) return;
    const float max = of_bits((uint32_t)(best >> 32));
    count_bins<THREADS>(s.hist, row, p.vocab, Place{(double)max, PER / (double)c.t});
    __syncthreads();
    finish(s, p, r, c, max, SampleSlices{0, 0, nullptr, nullptr, nullptr, nullptr});
}

// Few rows: a workgroup for each slice of them finds its largest token, then its bins and the
// tokens of the first ones, then a workgroup a row ends it.
constexpr int SLICE = 8192, SLICE_THREADS = 512;
__global__ __launch_bounds__(SLICE_THREADS) void sample_best_kernel(SampleParams p, SampleSlices sl) {
    __shared__ unsigned long long scratch[SLICE_THREADS / 64];
    const int r = blockIdx.y, first = blockIdx.x * sl.each;
    if (!settings_of(p, r, false).live) return;
    const unsigned long long v = largest<SLICE_THREADS>(p.logits + r * p.ld + first, min(sl.each, p.vocab - first),
                                                        first, scratch);
    if (threadIdx.x == 0) sl.best[(size_t)r * sl.n + blockIdx.x] = v;
}

__device__ __forceinline__ unsigned long long best_of(const SampleSlices &sl, int r) {
    // (a lane two of them at most; by whole waves)
    const int lane = threadIdx.x & 63;
    const unsigned long long *p = sl.best + (size_t)r * sl.n;
    const unsigned long long a = p[min(lane, sl.n - 1)], b = p[min(lane + 64, sl.n - 1)];
    return wave_most(a > b ? a : b);
}

__global__ __launch_bounds__(SLICE_THREADS) void sample_bins_kernel(SampleParams p, SampleSlices sl) {
    __shared__ unsigned long long hist[BINS];
    __shared__ uint32_t wave[SLICE_THREADS / 64], n, last;
    const int r = blockIdx.y, first = blockIdx.x * sl.each, tid = threadIdx.x, len = min(sl.each, p.vocab - first);
    const Settings c = settings_of(p, r, false);
    if (!c.live) return;
    for (int i = tid; i < BINS; i += SLICE_THREADS) hist[i] = 0;
    const unsigned long long best = best_of(sl, r);
    if (settled(p, r, c, best, false)) return;
    const Place at{(double)of_bits((uint32_t)(best >> 32)), PER / (double)c.t};
    const float *row = p.logits + r * p.ld + first;
    if (tid == 0) {
        n = 0;
        last = 0;
    }
    __syncthreads();
    count_bins<SLICE_THREADS>(hist, row, len, at);
    __syncthreads();
    // the bins that hold at most SLICE_LIST tokens together
    constexpr int EACH = BINS / SLICE_THREADS;
    const size_t x = (size_t)r * sl.n + blockIdx.x;
    uint32_t cnt[EACH], sum = 0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const unsigned long long h = hist[tid * EACH + i];
        sl.hist[x * BINS + tid * EACH + i] = h;
        cnt[i] = (uint32_t)(h >> COUNT);
        sum += cnt[i];
    }
    uint32_t to = sum;
    const int lane = tid & 63, w = tid >> 6;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
        const uint32_t v = __shfl_up(to, o, 64);
        if (lane >= o) to += v;
    }
    if (lane == 63) wave[w] = to;
    __syncthreads();
    to -= sum;
    for (int i = 0; i < w; ++i) to += wave[i];
#pragma unroll
    for (int i = 0; i < EACH; ++i) {  // bin tid EACH + i is listed where the count up to it fits
        to += cnt[i];
        if (to <= SLICE_LIST) atomicMax(&last, (uint32_t)min(tid * EACH + i + 1, BINS - 1));
    }
    __syncthreads();
    const int upto = (int)last;
    const float from = at.below(upto - 1);
    each_token<SLICE_THREADS>(row, len, [&](float l, int i) {
        uint32_t rest;
        if (l >= from && at.bin(l, &rest) < upto) {
            const uint32_t k = atomicAdd(&n, 1u);
            if (k < SLICE_LIST)
                sl.list[x * SLICE_LIST + k] = (unsigned long long)order_bits(l) << 32 | (uint32_t)~(first + i);
        }
    });
    __syncthreads();
    if (tid == 0) {
        sl.upto[x * 2] = upto;
        sl.upto[x * 2 + 1] = (int)n;
    }
}

__global__ __launch_bounds__(THREADS) void sample_finish_kernel(SampleParams p, SampleSlices sl) {
    __shared__ Shared s;
    const int r = blockIdx.x, tid = threadIdx.x;
    const Settings c = settings_of(p, r, true);
    if (!c.live) return;
    const unsigned long long best = best_of(sl, r);
    if (settled(p, r, c, best, true)) return;
    unsigned long long a = 0, b = 0;
    const unsigned long long *h = sl.hist + (size_t)r * sl.n * BINS + tid * 2;
    for (int i = 0; i < sl.n; i += 8) {
        ulonglong2 v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = *(const ulonglong2 *)(h + (size_t)min(i + k, sl.n - 1) * BINS);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            a += i + k < sl.n ? v[k].x : 0;
            b += i + k < sl.n ? v[k].y : 0;
        }
    }
    s.hist[tid * 2] = a;
    s.hist[tid * 2 + 1] = b;
    __syncthreads();
    finish(s, p, r, c, of_bits((uint32_t)(best >> 32)), sl);
}

// SampleSlices where a row is long and they do not fill the chip by themselves: their three launches
// and the bins' way through memory cost more than a row's own workgroup does from there on.
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
    sl.each = SLICE;
    sl.hist = (unsigned long long *)a.work;
    sl.list = sl.hist + x * BINS;
    sl.best = sl.list + x * SLICE_LIST;
    sl.upto = (int32_t *)(sl.best + x);
    const dim3 grid((unsigned)sl.n, (unsigned)a.rows);
    sample_best_kernel<<<grid, SLICE_THREADS, 0, st>>>(p, sl);
    VMLM_HIP_CHECK(hipGetLastError());
    sample_bins_kernel<<<grid, SLICE_THREADS, 0, st>>>(p, sl);
    VMLM_HIP_CHECK(hipGetLastError());
    sample_finish_kernel<<<(unsigned)a.rows, THREADS, 0, st>>>(p, sl);
    VMLM_HIP_CHECK(hipGetLastError());
    return VMLM_OK;
}

}  // namespace vmlm
