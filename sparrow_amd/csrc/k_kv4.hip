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
    if (n > room) {
        if (blk == 0 && blockIdx.y == 0 && threadIdx.x == 0) atomicOr(p.guard, 1);
        if (room <= 0) return false;
        n = room;
    }
    *first = (pos0 / KV4_BLOCK + blk) * KV4_BLOCK;
    *pos = pos0;
    *t0 = max(0, *first - pos0);
    *t1 = min(n, *first + KV4_BLOCK - pos0);
    return *t0 < *t1;
}

// One workgroup per (32-position block, head, sequence). Eight lanes quantise 32
// channels of a position; V's codes cross LDS to be packed along positions, and a
// block's bytes that hold other positions keep their nibbles.
__global__ __launch_bounds__(256) void kv4_append_kernel(Kv4Params p) {
    __shared__ uint8_t codes[KV4_BLOCK * KV4_MAX_HD];
    const int b = blockIdx.z, h = blockIdx.y, tid = threadIdx.x, hd = p.c.hd, ng = hd / 32;
    int first, pos0, t0, t1;
    if (!kv4_rows(p, b, blockIdx.x, &first, &pos0, &t0, &t1)) return;
    const size_t head = (size_t)b * p.c.Hkv + h;
    const int l = tid & 7;
    for (int task = tid >> 3; task < KV4_BLOCK * ng; task += 32) {
        const int o = task / ng, g = task - o * ng, t = first + o - pos0;
        if (t < t0 || t >= t1) continue;  // the same for the eight lanes
        const size_t row = (size_t)b * p.S + t, pos = head * p.c.cap + first + o;
        const int ch = g * 32 + 4 * l;
        float x[4];
        f32x4a r = *(const f32x4a *)(p.k + row * p.ldk + (size_t)h * hd + ch);
        for (int e = 0; e < 4; ++e) x[e] = r[e];
        uint32_t m = kv4_meta8(x);
        float mn = kv4_min(m), sc = kv4_scale(m);
        uint32_t c[4];
        for (int e = 0; e < 4; ++e) c[e] = kv4_code(x[e], mn, sc);
        *(uint16_t *)(p.c.k + pos * (hd / 2) + ch / 2) =
            (uint16_t)(c[0] | c[1] << 4 | c[2] << 8 | c[3] << 12);
        if (l == 0) p.c.km[pos * ng + g] = m;
        r = *(const f32x4a *)(p.v + row * p.ldv + (size_t)h * hd + ch);
        for (int e = 0; e < 4; ++e) x[e] = r[e];
        m = kv4_meta8(x);
        mn = kv4_min(m);
        sc = kv4_scale(m);
        for (int e = 0; e < 4; ++e) c[e] = kv4_code(x[e], mn, sc);
        *(uint32_t *)(codes + o * hd + ch) = c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24;
        if (l == 0) p.c.vm[pos * ng + g] = m;
    }
    __syncthreads();
    const int o0 = pos0 + t0 - first, o1 = pos0 + t1 - first;  // offsets that are new
    uint32_t *vb = (uint32_t *)(p.c.v + (head * (p.c.cap / KV4_BLOCK) + first / KV4_BLOCK) *
                                            (size_t)(hd * 16));
    for (int i = tid; i < hd * 4; i += 256) {  // dword: channel i / 4, offsets 8 (i % 4) ..
        const int ch = i >> 2, base = (i & 3) * 8;
        uint32_t w = 0, mask = 0;
        for (int e = 0; e < 8; ++e) {
            const int o = base + e;
            if (o >= o0 && o < o1) {
                w |= (uint32_t)codes[o * hd + ch] << (4 * e);
                mask |= 15u << (4 * e);
            }
        }
        if (mask == 0) continue;
        if (mask != 0xffffffffu) w |= vb[i] & ~mask;
        vb[i] = w;
    }
}

__global__ __launch_bounds__(256) void kv4_read_kernel(Kv4Params p) {
    const int b = blockIdx.z, h = blockIdx.y, tid = threadIdx.x, hd = p.c.hd, ng = hd / 32;
    int first, pos0, t0, t1;
    if (!kv4_rows(p, b, blockIdx.x, &first, &pos0, &t0, &t1)) return;
    const size_t head = (size_t)b * p.c.Hkv + h;
    const uint8_t *vb = p.c.v + (head * (p.c.cap / KV4_BLOCK) + first / KV4_BLOCK) *
                                    (size_t)(hd * 16);
    for (int i = tid; i < KV4_BLOCK * hd / 4; i += 256) {
        const int o = i / (hd / 4), ch = (i - o * (hd / 4)) * 4, t = first + o - pos0;
        if (t < t0 || t >= t1) continue;
        const size_t row = (size_t)b * p.S + t, pos = head * p.c.cap + first + o;
        const uint32_t km = p.c.km[pos * ng + ch / 32], vm = p.c.vm[pos * ng + ch / 32];
        const uint32_t kc = *(const uint16_t *)(p.c.k + pos * (hd / 2) + ch / 2);
        f32x4a k, v;
        for (int e = 0; e < 4; ++e) {
            k[e] = kv4_value(kc >> (4 * e), kv4_min(km), kv4_scale(km));
            v[e] = kv4_value((uint32_t)vb[(ch + e) * 16 + o / 2] >> (4 * (o & 1)), kv4_min(vm),
                             kv4_scale(vm));
        }
        *(f32x4a *)(p.ko + row * p.ldk + (size_t)h * hd + ch) = k;
        *(f32x4a *)(p.vo + row * p.ldv + (size_t)h * hd + ch) = v;
    }
}

dim3 kv4_grid(const Kv4View &c, int S) {
    // the blocks that S rows can touch, from any position of the first
    const size_t blocks = std::min((size_t)c.cap / KV4_BLOCK, ((size_t)S + 30) / KV4_BLOCK + 1);
    return dim3((unsigned)blocks, (unsigned)c.Hkv, (unsigned)c.B);
}

}  // namespace

int launch_kv4_append(const Kv4View &c, const float *k, size_t ldk, const float *v, size_t ldv,
                      const int32_t *pos0, const int32_t *count, int S, hipStream_t st) {
    Kv4Params p{c, k, v, nullptr, nullptr, ldk, ldv, pos0, count, S, guard_flag_ptr()};
    kv4_append_kernel<<<kv4_grid(c, S), 256, 0, st>>>(p);
    VMLM_HIP_CHECK(hipGetLastError());
    return VMLM_OK;
}

int launch_kv4_read(const Kv4View &c, float *k, size_t ldk, float *v, size_t ldv,
                    const int32_t *pos0, const int32_t *count, int S, hipStream_t st) {
    Kv4Params p{c, nullptr, nullptr, k, v, ldk, ldv, pos0, count, S, guard_flag_ptr()};
    kv4_read_kernel<<<kv4_grid(c, S), 256, 0, st>>>(p);
    VMLM_HIP_CHECK(hipGetLastError());
    return VMLM_OK;
}

}  // namespace vmlm
