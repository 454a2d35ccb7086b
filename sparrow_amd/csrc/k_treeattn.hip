// k_treeattn.hip -- attention of several tokens a sequence over the 4-bit KV cache
// (vmlm_hip_attention_tree_kv4); the format is in kv4.hpp.
//
// Token t of a sequence stands at position pos0 + t, its row already in the cache. It sees
// the positions before pos0, and of the tokens itself and its ancestors (a tree) or those
// before it (a chain): s_p = scale * q . k_p over the positions seen, o = sum_p exp(s_p - m) v_p /
// sum_p exp(s_p - m).
#include "kv4.hpp"
#include "tree.hpp"

namespace vmlm {
namespace {

struct TreeAttnParams {
    Kv4View c;
    const float *q;
    size_t ldq, ldo;
    const int32_t *pos0, *count, *parent;
    int S, H, G;
    float *out;
    float scale;
    int *guard;
};

// A wave for one query head of one token.
__global__ __launch_bounds__(64) void tree_attn_kernel(TreeAttnParams p) {
    __shared__ float qs[KV4_MAX_HD], w[64];
    const int h = blockIdx.x, t = blockIdx.y, b = blockIdx.z, lane = threadIdx.x, hd = p.c.hd;
    const TreeRows r = tree_rows(p.pos0, p.count, p.parent, p.S, p.c.cap, b, p.guard, h == 0 && t == 0);
    if (t >= r.n) return;
    const unsigned long long seen = p.parent ? tree_ancestors(r.parent, t) : ~0ull;
    const int ng = hd / 32, last = r.pos0 + t;
    const size_t head = (size_t)b * p.c.Hkv + h / p.G;
    const float *q = p.q + ((size_t)b * p.S + t) * p.ldq + (size_t)h * hd;
    int bad = 0;
    for (int c = lane; c < hd; c += 64) {
        qs[c] = q[c];
        bad |= !(fabsf(q[c]) <= 3.40282347e38f);
    }
    bad = __any(bad);
    __syncthreads();
    float m = -3.40282347e38f, l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int p0 = 0; p0 <= last; p0 += 64) {
        const int pos = p0 + lane, own = pos - r.pos0;
        const bool in = pos <= last && (own < 0 || !p.parent || (seen >> own & 1));
        float s = -__builtin_inff();
        if (in) {
            const size_t row = head * p.c.cap + pos;
            float acc = 0.0f;
            for (int g = 0; g < ng; ++g) {
                const uint32_t meta = p.c.km[row * ng + g];
                for (int i = 0; i < 16; ++i) {
                    const uint32_t byte = p.c.k[row * (hd / 2) + g * 16 + i];
                    acc = __builtin_fmaf(qs[g * 32 + 2 * i], kv4_value(byte, kv4_min(meta), kv4_scale(meta)), acc);
                    acc = __builtin_fmaf(qs[g * 32 + 2 * i + 1], kv4_value(byte >> 4, kv4_min(meta), kv4_scale(meta)), acc);
                }
            }
            s = acc * p.scale;
        }
        const float mx = fmaxf(m, wave_max(s));
        const float corr = expf(m - mx), e = in ? expf(s - mx) : 0.0f;
        l = l * corr + wave_sum(e);
        m = mx;
        __syncthreads();
        w[lane] = e;
        __syncthreads();
        const unsigned long long live = __ballot(in);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int c = lane + i * 64;
            if (c >= hd) break;
            o[i] *= corr;
            for (int x = 0; x < 64; ++x) {
                if (!(live >> x & 1)) continue;
                const int at = p0 + x;
                const uint32_t byte = p.c.v[((head * (p.c.cap / 32) + at / 32) * hd + c) * 16 + at % 32 / 2];
                const uint32_t meta = p.c.vm[(head * p.c.cap + at) * ng + c / 32];
                o[i] = __builtin_fmaf(w[x], kv4_value(byte >> (4 * (at & 1)), kv4_min(meta), kv4_scale(meta)), o[i]);
            }
        }
    }
    float *out = p.out + ((size_t)b * p.S + t) * p.ldo + (size_t)h * hd;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (lane + i * 64 < hd) out[lane + i * 64] = bad ? __builtin_nanf("") : o[i] / l;
}

}  // namespace

size_t tree_attn_work_floats(const Kv4View &c, int H, int S) { return 0; }

int launch_tree_attn(const TreeAttnArgs &a, hipStream_t st) {
    const TreeAttnParams p{a.c, a.q,   a.ldq, a.ldo, a.pos0, a.count, a.parent,
                           a.S, a.H,   a.H / a.c.Hkv, a.out, a.scale, guard_flag_ptr()};
    tree_attn_kernel<<<dim3((unsigned)a.H, (unsigned)a.S, (unsigned)a.c.B), 64, 0, st>>>(p);
    VMLM_HIP_CHECK(hipGetLastError());
    return VMLM_OK;
}

}  // namespace vmlm
