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
constexpr int LIST = 2048;      // tokens of a bin that are sorted
constexpr double PER = 64.0;    // bins of 1
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

// A logit's place: its bin, and the rest of its distance in [0, 1) of a bin.
struct Place {
    double max, per;  // PER / T
    __device__ __forceinline__ int bin(float l, double *rest) const {
        const double x = (max - (double)l) * per;  // (+inf for a masked one)
        if (!(x < BINS - 1)) return BINS - 1;
        const double f = __builtin_floor(x);
        *rest = x - f;
        return (int)f;
    }
};
// 1 - exp(-r / 64), in units of 2^-30 (the next term of the series is below 2^-36)
__device__ __forceinline__ uint32_t loss(double rest) {
    const double r = rest * (1.0 / PER);
    const double d = r * (1.0 - r * (0.5 - r * (1.0 / 6 - r * (1.0 / 24))));
    return (uint32_t)(int)__builtin_rint(d * (double)(1 << UNIT));
}

// Calls f(logit, index) for every token of the row.
template <typename F>
__device__ __forceinline__ void each_token(const float *row, int n, F f) {
    const int step = THREADS * 4;
    int i = threadIdx.x * 4;
    for (; i + 3 < n; i += step) {
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
        each_token(row, vocab, [&](float l, int) {
            double rest;
            const uint32_t key = order_bits(l);
            if (at.bin(l, &rest) == bin && key >= lo && key <= hi) {
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
        each_token(row, vocab, [&](float l, int) {
            double rest;
            const uint32_t key = order_bits(l);
            if (at.bin(l, &rest) == bin && key >= lo && key <= hi)
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
        each_token(row, vocab, [&](float l, int) {
            double rest;
            if (order_bits(l) == lo && at.bin(l, &rest) == bin) s.n = loss(rest);
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
    __syncthreads();
    if (tid == 0) s.n = 0;
    int pow2 = 64;
    while (pow2 < n) pow2 *= 2;
    for (int i = tid; i < pow2; i += THREADS) s.list[i] = 0;
    __syncthreads();
    each_token(row, vocab, [&](float l, int i) {
        double rest;
        const uint32_t key = order_bits(l);
        if (key >= lo && key <= hi && at.bin(l, &rest) == bin)
            s.list[atomicAdd(&s.n, 1u)] = (unsigned long long)key << 32 | (uint32_t)~i;
    });
    __syncthreads();
    for (int k = 2; k <= pow2; k *= 2)
        for (int j = k / 2; j > 0; j /= 2) {
            for (int i = tid; i < pow2 / 2; i += THREADS) {
                const int x = i / j * 2 * j + i % j, y = x + j;
                const unsigned long long a = s.list[x], b = s.list[y];
                if (((x & k) == 0) == (a < b)) {  // the largest first
                    s.list[x] = b;
                    s.list[y] = a;
                }
            }
            __syncthreads();
        }
    static_assert(LIST == BINS && LIST == 2 * THREADS, "");
    unsigned long long *sum = s.hist, d[2], e[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int x = tid * 2 + i;
        double rest;
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

__global__ __launch_bounds__(THREADS) void sample_kernel(SampleParams p) {
    __shared__ Shared s;
    const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const float u = p.u[r], t = p.t[r], top_p = p.top_p ? p.top_p[r] : 1.0f,
                min_p = p.min_p ? p.min_p[r] : 0.0f;
    const int top_k = p.top_k ? p.top_k[r] : 0, n = p.vocab;
    if (u < 0.0f) return;  // an idle row
    if (!(u < 1.0f) || !(t >= 0.0f && t <= 3.40282347e38f) || !(top_p == top_p) ||
        !(min_p >= 0.0f && min_p <= 1.0f)) {
        if (tid == 0) atomicOr(p.guard, 1);
        return;
    }
    const float *row = p.logits + r * p.ld;
    auto answer = [&](int token, float prob) {
        if (tid == 0) {
            p.token[r] = token;
            if (p.prob) p.prob[r] = prob;
        }
    };
    // 1. the largest, the first of equal ones; NaN anywhere
    uint32_t best = 0, index = 0xffffffffu;
    bool nan = false;
    each_token(row, n, [&](float l, int i) {
        nan |= l != l;
        const uint32_t key = order_bits(l);
        if (key > best) {
            best = key;
            index = i;
        }
    });
    if (tid == 0) {
        s.best = 0;
        s.n = 0;
    }
    for (int i = tid; i < BINS; i += THREADS) s.hist[i] = 0;
    __syncthreads();
    if (nan) s.n = 1;
    atomicMax(&s.best, (unsigned long long)best << 32 | (uint32_t)~index);
    __syncthreads();
    index = ~(uint32_t)s.best;
    const bool any_nan = s.n != 0;
    __syncthreads();
    const float max = row[index < (uint32_t)n ? index : 0];
    if (any_nan || max == __builtin_inff()) return answer(-1, __builtin_nanf(""));
    if (max == -__builtin_inff()) return answer(-1, 0.0f);  // the mask leaves no token
    if (t == 0.0f) return answer((int)index, 1.0f);

    // 2. the bins
    const Place at{(double)max, PER / (double)t};
    each_token(row, n, [&](float l, int) {
        double rest;
        const int b = at.bin(l, &rest);
        if (b < BINS - 1) atomicAdd(&s.hist[b], (1ull << COUNT) | loss(rest));
    });
    __syncthreads();
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
    // 3. what is kept: the first `kept` of the order, of weight `all`
    uint32_t kept = live;
    if (top_k > 0 && (uint32_t)top_k < kept) {
        kept = (uint32_t)top_k;
        const int b = bin_of_rank(kept - 1);
        const Found f = locate(s, row, n, at, b, tokens(b), true, kept - 1 - s.before[b], 0.0, false);
        all = s.above[b] + scale(b) * (double)f.upto;
    }
    if (top_p < 1.0f) {
        const double goal = (double)top_p * all;
        const int b = bin_of_mass(goal, true);
        const Found f = locate(s, row, n, at, b, tokens(b), false, 0, (goal - s.above[b]) / scale(b), true);
        const uint32_t k = s.before[b] + f.rank + 1;
        if (k < kept) {
            kept = k;
            all = s.above[b] + scale(b) * (double)f.upto;
        }
    }
    if (min_p > 0.0f) {
        // (weights next to the border in 64 bits, the others by their bin)
        const double x = -log((double)min_p) * PER;
        uint32_t k = 0;
        each_token(row, n, [&](float l, int) {
            double rest;
            const int b = at.bin(l, &rest);
            if (b == BINS - 1) return;
            if (fabs((double)b - x) > 2.0)
                k += (double)b < x;
            else
                k += exp(((double)l - at.max) / (double)t) >= (double)min_p;
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
    // 4. the token
    const double goal = (double)u * all;
    int b = bin_of_mass(goal, false);
    Found f = locate(s, row, n, at, b, tokens(b), false, 0, (goal - s.above[b]) / scale(b), false);
    if (s.before[b] + f.rank >= kept) {  // (a rounding put the goal behind the last one)
        b = bin_of_rank(kept - 1);
        f = locate(s, row, n, at, b, tokens(b), true, kept - 1 - s.before[b], 0.0, false);
    }
    answer((int)f.token, (float)(scale(b) * (double)((1u << UNIT) - f.d) / all));
}

}  // namespace

size_t sample_work_bytes(int rows, int vocab) { return 0; }

int launch_sample(const SampleArgs &a, hipStream_t st) {
    const SampleParams p{a.logits, a.ld,    a.u,    a.t,     a.top_p, a.min_p,
                         a.top_k,  a.rows, a.vocab, a.token, a.prob,  guard_flag_ptr()};
    sample_kernel<<<(unsigned)a.rows, THREADS, 0, st>>>(p);
    VMLM_HIP_CHECK(hipGetLastError());
    return VMLM_OK;
}

}  // namespace vmlm
