// k_attn4.hip -- decode attention over the 4-bit KV cache
// (vmlm_hip_attention_decode_kv4); the format is in kv4.hpp.
#include "kv4.hpp"

namespace vmlm {
namespace {

// One workgroup per (query head, sequence): 256 positions at a time, a running
// maximum and sum.
__global__ __launch_bounds__(256) void attn4_simple(Kv4View c, const float *q, size_t ldq,
                                                    const int32_t *posp, float *out, size_t ldo,
                                                    int H, float scale, int *guard) {
    __shared__ float qs[KV4_MAX_HD], ps[256], red[4], os[256];
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, hd = c.hd, ng = hd / 32;
    const int pos = posp[b], kvh = h / (H / c.Hkv);
    if (pos < 0) return;
    if (pos >= c.cap) {
        if (h == 0 && tid == 0) atomicOr(guard, 1);
        return;
    }
    const size_t head = (size_t)b * c.Hkv + kvh;
    if (tid < hd) qs[tid] = q[b * ldq + (size_t)h * hd + tid] * scale;
    __syncthreads();
    float m = -__builtin_inff(), L = 0.0f, o = 0.0f;
    const int parts = 256 / hd, ch = tid % hd, part = tid / hd;
    for (int p0 = 0; p0 <= pos; p0 += 256) {
        const int p = p0 + tid;
        float s = -__builtin_inff();
        if (p <= pos) {
            s = 0.0f;
            const uint8_t *kr = c.k + (head * c.cap + p) * (size_t)(hd / 2);
            for (int g = 0; g < ng; ++g) {
                const uint32_t mt = c.km[(head * c.cap + p) * ng + g];
                for (int i = 0; i < 32; ++i)
                    s = __builtin_fmaf(qs[g * 32 + i],
                                       kv4_value(kr[(g * 32 + i) / 2] >> (4 * (i & 1)),
                                                 kv4_min(mt), kv4_scale(mt)), s);
            }
        }
        float mx = wave_max(s);
        if ((tid & 63) == 0) red[tid >> 6] = mx;
        __syncthreads();
        mx = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
        const float mn = fmaxf(m, mx), corr = __expf(m - mn);
        const float pr = p <= pos ? expf(s - mn) : 0.0f;
        ps[tid] = pr;
        __syncthreads();
        o *= corr;
        L *= corr;
        m = mn;
        const int n = min(256, pos + 1 - p0);
        for (int i = 0; i < n; ++i) L += ps[i];
        for (int i = part; i < n; i += parts) {
            const size_t at = p0 + i;
            const uint32_t mt = c.vm[(head * c.cap + at) * ng + ch / 32];
            const uint8_t vb = c.v[((head * (c.cap / 32) + at / 32) * hd + ch) * 16 + at % 32 / 2];
            o = __builtin_fmaf(ps[i], kv4_value(vb >> (4 * (at & 1)), kv4_min(mt), kv4_scale(mt)),
                               o);
        }
        __syncthreads();
    }
    os[tid] = o;
    __syncthreads();
    if (tid < hd) {
        for (int i = 1; i < parts; ++i) o += os[tid + i * hd];
        out[b * ldo + (size_t)h * hd + tid] = o / L;
    }
}

}  // namespace

size_t attn4_work_floats(const Kv4View &c, int H) { return 0; }

int launch_attn4(const Attn4Args &a, hipStream_t st) {
    if (a.k_new) {
        int rc = launch_kv4_append(a.c, a.k_new, a.ldkv, a.v_new, a.ldkv, a.pos, nullptr, 1, st);
        if (rc) return rc;
    }
    attn4_simple<<<dim3((unsigned)a.H, (unsigned)a.c.B), 256, 0, st>>>(
        a.c, a.q, a.ldq, a.pos, a.out, a.ldo, a.H, a.scale, guard_flag_ptr());
    VMLM_HIP_CHECK(hipGetLastError());
    return VMLM_OK;
}

}  // namespace vmlm
