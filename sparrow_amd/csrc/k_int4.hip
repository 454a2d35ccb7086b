// k_int4.hip -- C[m][j] = sum over groups g of scale[j][g] * (A[m] . Q[j]) over
// the group's k, Q in 4 bits (vmlm_hip_gemm_nt_int4).
//
// Q is [N][K/2] bytes, byte i of a row holding k = 2i (low nibble) and 2i + 1,
// two's complement. K is a multiple of 32; the last group may be short.
#include "internal.hpp"

namespace vmlm {
namespace {

// One wave per output element, lanes over the row's 32-k runs.
__global__ __launch_bounds__(256) void gemm_int4_simple(const float *__restrict__ A,
                                                        const uint8_t *__restrict__ Q,
                                                        const float *__restrict__ scale,
                                                        float *__restrict__ C, int M, int N, int K,
                                                        int G, int ng) {
    const int j = blockIdx.x * 4 + (threadIdx.x >> 6), m = blockIdx.y, lane = threadIdx.x & 63;
    if (j >= N) return;
    const float *a = A + (size_t)m * K;
    const uint8_t *q = Q + (size_t)j * (K / 2);
    float acc = 0.0f;
    for (int k = lane * 32; k < K; k += 64 * 32) {
        float s = 0.0f;
        for (int i = 0; i < 16; ++i) {
            const int b = q[k / 2 + i];
            s = __builtin_fmaf(a[k + 2 * i], (float)((int8_t)(b << 4) >> 4), s);
            s = __builtin_fmaf(a[k + 2 * i + 1], (float)((int8_t)b >> 4), s);
        }
        acc = __builtin_fmaf(s, scale[(size_t)j * ng + k / G], acc);
    }
    acc = wave_sum(acc);
    if (lane == 0) C[(size_t)m * N + j] = acc;
}

}  // namespace

int launch_gemm_int4(const Int4Args &a, hipStream_t st) {
    gemm_int4_simple<<<dim3(cdiv((size_t)a.N, 4), (unsigned)a.M), 256, 0, st>>>(
        a.A, a.Q, a.scale, a.C, a.M, a.N, a.K, a.G, (a.K + a.G - 1) / a.G);
    VMLM_HIP_CHECK(hipGetLastError());
    return VMLM_OK;
}

}  // namespace vmlm
