// k_kv4.hip -- rows into the 4-bit KV cache and out of it
// (vmlm_hip_kv4_append, vmlm_hip_kv4_read); the format is in kv4.hpp.
#include <algorithm>

#include "kv4.hpp"

namespace vmlm {
namespace {

typedef float f32x4a __attribute__((ext_vector_type(4), aligned(4)));

struct Kv4Params {
    Kv4View c;
    const float *k, *v;  // append: rows [B][S][ld]
    float *ko, *vo;      // read
    size_t ldk, ldv;
    const int32_t *pos0, *count;
    int S;
    int *guard;
};

// The rows [t0, t1) of sequence b that fall into block `blk` of those that its
// rows touch, and the position of row 0; false if there are none.
__device__ __forceinline__ bool kv4_rows(const Kv4Params &p, int b, int blk, int *first, int *pos,
                                         int *t0, int *t1) {
    const int pos0 = p.pos0[b];
    if (pos0 < 0) return false;  // idle
    int n = p.count ? min(max(p.count[b], 0), p.S) : p.S;
    const int room = p.c.cap - pos0;
    if (n > max(room, 0) && blk == 0 && blockIdx.y == 0 && threadIdx.x == 0) atomicOr(p.guard, 1);
    n = min(n, room);
    if (n <= 0) return false;
    *first = (pos0 / KV4_BLOCK + blk) * KV4_BLOCK;
    *pos = pos0;
    *t0 = max(0, *first - pos0);
    *t1 = min(n, *first + KV4_BLOCK - pos0);
    return *t0 < *t1;
}

// One workgroup per (32-position block, head, K or V, sequence). Eight lanes quantise 32
// channels of a position; V's codes cross LDS to be packed along positions, and a
// block's bytes that hold other positions keep their nibbles. Bound by the f32 rows;
// all of a thread's loads are issued before the first is used. 16 prompts of up to 128
// rows, 36 heads of 64, 31 MB of rows and codes: 11 us, 2.8 TB/s; the two dozen operations a
// value and V's way through LDS are what a copy does not have. (K and V in one workgroup: 7.0 us
// instead of 6.1 then for 3 x 333 rows of 8 heads of 128.)
template <int HD>
__global__ __launch_bounds__(256) void kv4_append_kernel(Kv4Params p) {
    constexpr int NG = HD / 32, LD = HD + 4;  // bytes of a position in LDS
    __shared__ __align__(4) uint8_t codes[KV4_BLOCK * LD];
    const int b = blockIdx.z, h = blockIdx.y >> 1, isv = blockIdx.y & 1, tid = threadIdx.x;
    int first, pos0, t0, t1;
    if (!kv4_rows(p, b, blockIdx.x, &first, &pos0, &t0, &t1)) return;
    const size_t head = (size_t)b * p.c.Hkv + h;
    const float *src = isv ? p.v : p.k;
    const size_t ld = isv ? p.ldv : p.ldk;
    uint32_t *meta = isv ? p.c.vm : p.c.km;
    const int l = tid & 7;
    f32x4a row[NG];
#pragma unroll
    for (int i = 0; i < NG; ++i) {
        const int task = (tid >> 3) + i * 32, o = task / NG, g = task % NG;
        const int t = min(max(first + o - pos0, t0), t1 - 1);
        row[i] = *(const f32x4a *)(src + ((size_t)b * p.S + t) * ld + (size_t)h * HD + g * 32 + 4 * l);
    }
#pragma unroll
    for (int i = 0; i < NG; ++i) {
        const int task = (tid >> 3) + i * 32, o = task / NG, g = task % NG;
        const int t = first + o - pos0, ch = g * 32 + 4 * l;
        if (t < t0 || t >= t1) continue;  // the same for the eight lanes
        const size_t pos = head * p.c.cap + first + o;
        const float x[4] = {row[i][0], row[i][1], row[i][2], row[i][3]};
        const uint32_t m = kv4_meta8(x);
        uint32_t c[4];
        kv4_codes(x, m, c);
        if (isv)
            *(uint32_t *)(codes + o * LD + ch) = kv4_bytes(c);
        else
            *(uint16_t *)(p.c.k + pos * (HD / 2) + ch / 2) = kv4_nibbles(c);
        if (l == 0) meta[pos * NG + g] = m;
    }
    if (!isv) return;
    __syncthreads();
    const int o0 = pos0 + t0 - first, o1 = pos0 + t1 - first;  // offsets that are new
    uint32_t *vb = (uint32_t *)(p.c.v + (head * (p.c.cap / KV4_BLOCK) + first / KV4_BLOCK) *
                                            (size_t)(HD * 16));
    if (tid >= HD) return;
    // four channels, eight positions: byte e of a dword holds 2e and 2e + 1
    const int ch = tid / 4 * 4, base = (tid & 3) * 8;
    uint32_t w[4], out[4], mask = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint8_t *a = codes + (base + 2 * e) * LD + ch;
        // (positions without a new row hold anything)
        w[e] = (*(const uint32_t *)a & 0x0f0f0f0fu) |
               (*(const uint32_t *)(a + LD) << 4 & 0xf0f0f0f0u);
    }
    transpose_bytes(w, out);
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (base + e >= o0 && base + e < o1) mask |= 15u << (4 * e);
    if (mask == 0) return;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        uint32_t *at = vb + (ch + k) * 4 + (tid & 3);
        *at = mask == 0xffffffffu ? out[k] : (out[k] & mask) | (*at & ~mask);
    }
}

// Neighbouring heads of a workgroup that reads: 128 channels, fewer workgroups to start
// (for 16 prompts of up to 128 rows, 36 heads of 64, 7.8 us instead of 8.3; appending takes
// 11 us either way).
constexpr int read_heads(int hd) { return hd < 128 ? 128 / hd : 1; }

// The block's codes and meta through LDS, then four channels of a position a thread:
// whole 16-byte stores of a row. Bound by the f32 rows that it writes: 16 prompts of up to
// 128 rows, 36 heads of 64, 31 MB in 7.8 us, 4.0 TB/s.
template <int HD>
__global__ __launch_bounds__(256) void kv4_read_kernel(Kv4Params p) {
    constexpr int NH = read_heads(HD), NG = HD / 32, LV = 20;  // LDS bytes of a V channel
    constexpr int CODES = HD * 4, METAS = KV4_BLOCK * NG;      // dwords of a head's block
    __shared__ __align__(4) uint8_t codes[NH * HD * LV];
    __shared__ uint32_t meta[NH * METAS];
    const int b = blockIdx.z, h0 = (blockIdx.y >> 1) * NH, isv = blockIdx.y & 1, tid = threadIdx.x;
    const int nh = min(NH, p.c.Hkv - h0);
    int first, pos0, t0, t1;
    if (!kv4_rows(p, b, blockIdx.x, &first, &pos0, &t0, &t1)) return;
    const size_t pos = ((size_t)b * p.c.Hkv + h0) * p.c.cap + first;
    // a V block is as long as its positions' K rows; a head's is cap positions on
    const uint32_t *cb = (const uint32_t *)((isv ? p.c.v : p.c.k) + pos * (HD / 2));
    const uint32_t *mb = (isv ? p.c.vm : p.c.km) + pos * NG;
    uint32_t c[NH * CODES / 256];
#pragma unroll
    for (int i = 0; i < NH * CODES / 256; ++i) {
        const int x = tid + i * 256, h = min(x / CODES, nh - 1);
        c[i] = cb[(size_t)h * p.c.cap * (HD / 8) + x % CODES];
    }
    const int mh = min(tid / METAS, nh - 1);
    const uint32_t m0 = mb[(size_t)mh * p.c.cap * NG + tid % METAS];
#pragma unroll
    for (int i = 0; i < NH * CODES / 256; ++i) {
        const int x = tid + i * 256;
        *(uint32_t *)(codes + (isv ? x / 4 * LV + x % 4 * 4 : x * 4)) = c[i];
    }
    if (tid < NH * METAS) meta[tid] = m0;
    __syncthreads();
    float *dst = isv ? p.vo : p.ko;
    const size_t ld = isv ? p.ldv : p.ldk;
#pragma unroll
    for (int i = 0; i < NH * NG; ++i) {
        constexpr int RD = NH * HD / 4;  // threads of a position
        const int x = tid + i * 256, o = x / RD, all = x % RD * 4, t = first + o - pos0;
        const int h = all / HD, ch = all % HD;
        if (t < t0 || t >= t1 || h >= nh) continue;
        const uint32_t m = meta[h * METAS + o * NG + ch / 32];
        uint32_t c;
        if (isv) {
            c = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                c |= ((uint32_t)codes[(all + e) * LV + o / 2] >> (4 * (o & 1)) & 15u) << (4 * e);
        } else {
            c = ((const uint16_t *)codes)[(h * KV4_BLOCK + o) * (HD / 4) + ch / 4];
        }
        f32x4a y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = kv4_value(c >> (4 * e), kv4_min(m), kv4_scale(m));
        *(f32x4a *)(dst + ((size_t)b * p.S + t) * ld + (size_t)(h0 + h) * HD + ch) = y;
    }
}

template <int HD>
void launch_hd(const Kv4Params &p, dim3 grid, hipStream_t st) {
    if (p.k)
        kv4_append_kernel<HD><<<grid, 256, 0, st>>>(p);
    else
        kv4_read_kernel<HD><<<grid, 256, 0, st>>>(p);
}

dim3 kv4_grid(const Kv4View &c, int S, int heads) {
    // the blocks that S rows can touch, from any position of the first
    const size_t blocks = std::min((size_t)c.cap / KV4_BLOCK, ((size_t)S + 30) / KV4_BLOCK + 1);
    return dim3((unsigned)blocks, 2 * cdiv((size_t)c.Hkv, heads), (unsigned)c.B);
}

int launch_kv4(const Kv4Params &p, hipStream_t st) {
    const dim3 grid = kv4_grid(p.c, p.S, p.k ? 1 : read_heads(p.c.hd));
    switch (p.c.hd) {
    case 32: launch_hd<32>(p, grid, st); break;
    case 64: launch_hd<64>(p, grid, st); break;
    case 128: launch_hd<128>(p, grid, st); break;
    default: launch_hd<256>(p, grid, st); break;
    }
    VMLM_HIP_CHECK(hipGetLastError());
    return VMLM_OK;
}

}  // namespace

int launch_kv4_append(const Kv4View &c, const float *k, size_t ldk, const float *v, size_t ldv,
                      const int32_t *pos0, const int32_t *count, int S, hipStream_t st) {
    return launch_kv4(Kv4Params{c, k, v, nullptr, nullptr, ldk, ldv, pos0, count, S,
                                guard_flag_ptr()}, st);
}

int launch_kv4_read(const Kv4View &c, float *k, size_t ldk, float *v, size_t ldv,
                    const int32_t *pos0, const int32_t *count, int S, hipStream_t st) {
    return launch_kv4(Kv4Params{c, nullptr, nullptr, k, v, ldk, ldv, pos0, count, S,
                                guard_flag_ptr()}, st);
}

}  // namespace vmlm
