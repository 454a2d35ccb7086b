// kv4.hpp -- the KV cache in 4 bits, as its kernels see it (vmlm_kv4_cache).
//
// 32 channels of one position's head share (min, scale), two bf16 in one dword
// (scale in the low half): min is their lowest value rounded down, scale a
// fifteenth of the way to their highest rounded up, so that the 16 steps reach
// both. A value is held as u = rint((x - min) / scale) in 0..15 and stands for
// min + scale * u; the nibble is u ^ 8, the two's complement of u - 8, which an
// int8 matrix product reads with one mask. The difference and both quotients are
// f32, correctly rounded. 5 bits a value.
//
// K codes lie by position ([hd/2] bytes: channels 2i and 2i + 1 in byte i): the
// scores' products run over channels. V codes lie in blocks of 32 positions
// ([hd][16] bytes: positions 2i and 2i + 1 of a channel): the output's run over
// positions, and a lane's 16-byte load is 32 positions of one channel.
#pragma once

#include "internal.hpp"

namespace vmlm {

constexpr int KV4_BLOCK = 32;

// The meta of 32 values with lowest lo and highest hi (NaN among them gives both
// NaN); NaN twice where one of them is not finite or their range leaves f32. (Judged
// before the bits are rounded outward, where a NaN's may wrap to zero.)
__device__ __forceinline__ uint32_t kv4_meta(float lo, float hi) {
    const uint32_t b = __float_as_uint(lo);
    const uint32_t mn = ((b >> 31) ? b + 0xffffu : b) & 0xffff0000u;
    const float q = (hi - __uint_as_float(mn)) / 15.0f;
    const uint32_t sc = (__float_as_uint(q) + 0xffffu) & 0xffff0000u;
    const bool ok = fabsf(lo) <= 3.40282347e38f && fabsf(q) <= 3.40282347e38f &&
                    (mn & 0x7f800000u) != 0x7f800000u && (sc & 0x7f800000u) != 0x7f800000u;
    return ok ? mn | (sc >> 16) : 0x7fc07fc0u;
}
__device__ __forceinline__ float kv4_scale(uint32_t meta) { return __uint_as_float(meta << 16); }
__device__ __forceinline__ float kv4_min(uint32_t meta) {
    return __uint_as_float(meta & 0xffff0000u);
}
// the code of x, by the definition's quotient
__device__ __forceinline__ uint32_t kv4_code(float x, float mn, float sc) {
    const float u = sc > 0.0f ? fminf(fmaxf(rintf((x - mn) / sc), 0.0f), 15.0f) : 0.0f;
    return (uint32_t)u;
}
// Four codes as 16 bits of nibbles, and as a byte each with the nibble in its low half.
__device__ __forceinline__ uint16_t kv4_nibbles(const uint32_t (&c)[4]) {
    return (uint16_t)((c[0] | c[1] << 4 | c[2] << 8 | c[3] << 12) ^ 0x8888u);
}
__device__ __forceinline__ uint32_t kv4_bytes(const uint32_t (&c)[4]) {
    const uint32_t a = __builtin_amdgcn_perm(c[1], c[0], 0x0c0c0400u);
    const uint32_t b = __builtin_amdgcn_perm(c[3], c[2], 0x04000c0cu);
    return (a | b) ^ 0x08080808u;
}
// The codes u = nibble ^ 8 of four values, each in the low 16 bits of its dword. A
// product with 1 / scale is within 2^-22 of the quotient relative to it, 2^-18 in all, so
// it decides every code whose quotient is not nearer than 2^-16 to a half; the wave takes
// the quotients themselves where one is, or where the scale is so small or large that its
// reciprocal is not normal. (Clamped first: 0 and 15 are no halves. 1.5 * 2^23 added
// rounds to an integer and leaves it in the low bits.)
__device__ __forceinline__ void kv4_codes(const float (&x)[4], uint32_t meta, uint32_t (&c)[4]) {
    const float mn = kv4_min(meta), sc = kv4_scale(meta), r = __builtin_amdgcn_rcpf(sc);
    float off[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float q = __builtin_amdgcn_fmed3f((x[e] - mn) * r, 0.0f, 15.0f);
        const float t = q + 0x1.8p23f;
        off[e] = fabsf(q - (t - 0x1.8p23f));
        c[e] = __float_as_uint(t);
    }
    const float most = fmaxf(fmaxf(off[0], off[1]), fmaxf(off[2], off[3]));
    if (__builtin_expect(__any(!(sc > 1e-36f && sc < 1e36f && most < 0.5f - 0x1p-16f)), 0)) {
#pragma unroll
        for (int e = 0; e < 4; ++e) c[e] = kv4_code(x[e], mn, sc);
    }
}
// the value of a nibble (in the low four bits)
__device__ __forceinline__ float kv4_value(uint32_t nib, float mn, float sc) {
    return sc * (float)((nib & 15u) ^ 8u) + mn;
}

// The meta of 32 values held by 8 neighbouring lanes, four each; the same in all
// eight. (Minimum and maximum that keep a NaN; lanes swapped within a quad, then the
// half row mirrored. All eight take part: no lane's own value is kept for an absent one.)
template <int CTRL>
__device__ __forceinline__ float kv4_swap(float v) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xF, 0xF, true));
}
__device__ __forceinline__ uint32_t kv4_meta8(const float (&x)[4]) {
    float lo = __builtin_elementwise_minimum(__builtin_elementwise_minimum(x[0], x[1]),
                                             __builtin_elementwise_minimum(x[2], x[3]));
    float hi = __builtin_elementwise_maximum(__builtin_elementwise_maximum(x[0], x[1]),
                                             __builtin_elementwise_maximum(x[2], x[3]));
    lo = __builtin_elementwise_minimum(lo, kv4_swap<0xB1>(lo));
    hi = __builtin_elementwise_maximum(hi, kv4_swap<0xB1>(hi));
    lo = __builtin_elementwise_minimum(lo, kv4_swap<0x4E>(lo));
    hi = __builtin_elementwise_maximum(hi, kv4_swap<0x4E>(hi));
    lo = __builtin_elementwise_minimum(lo, kv4_swap<0x141>(lo));
    hi = __builtin_elementwise_maximum(hi, kv4_swap<0x141>(hi));
    return kv4_meta(lo, hi);
}

}  // namespace vmlm
